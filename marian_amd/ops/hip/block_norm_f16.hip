// Block-join kernels for f16 rows.
#include "block_norm.h"

template void mamd::join_fwd_launch<mamd::f16_t>(const mamd::NormPlan&, unsigned,
                                               hipStream_t);
template void mamd::join_bwd_launch<mamd::f16_t>(const mamd::NormPlan&, unsigned,
                                               hipStream_t);
