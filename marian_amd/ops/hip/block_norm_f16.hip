// Block-join kernels for f16 rows.
#include "block_norm.h"

template int mamd::join_fwd_launch<mamd::f16_t>(const mamd::NormPlan&, unsigned,
                                              hipStream_t);
template int mamd::join_bwd_launch<mamd::f16_t>(const mamd::NormPlan&, unsigned,
                                              hipStream_t);
