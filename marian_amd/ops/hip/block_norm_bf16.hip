// Block-join kernels for bf16 rows.
#include "block_norm.h"

template int mamd::join_fwd_launch<mamd::bf16_t>(const mamd::NormPlan&, unsigned,
                                              hipStream_t);
template int mamd::join_bwd_launch<mamd::bf16_t>(const mamd::NormPlan&, unsigned,
                                              hipStream_t);
