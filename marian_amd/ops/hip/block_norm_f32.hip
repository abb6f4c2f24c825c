// Block-join kernels for f32 rows.
#include "block_norm.h"

template void mamd::join_fwd_launch<float>(const mamd::NormPlan&, unsigned,
                                               hipStream_t);
template void mamd::join_bwd_launch<float>(const mamd::NormPlan&, unsigned,
                                               hipStream_t);
