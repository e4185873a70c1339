// The kernels around a residual block for one element type (residual_norm_kernels.h).
#include "residual_norm_kernels.h"

template void rn::launch_fwd<DT_F32>(const ResidualNormParams& p, hipStream_t s);
template void rn::launch_bwd<DT_F32>(const ResidualNormParams& p, hipStream_t s);
