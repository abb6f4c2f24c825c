// Block-join kernels for f32 rows.
#include "block_norm.h"

template int mamd::join_fwd_launch<float>(const mamd::NormPlan&, unsigned,
                                              hipStream_t);
template int mamd::join_bwd_launch<float>(const mamd::NormPlan&, unsigned,
                                              hipStream_t);
