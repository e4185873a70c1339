// Entry points of the seam between two residual blocks: checks and the choice of the element type
// (kernels: residual_norm_kernels.h).
#include <algorithm>
#include <stdexcept>

#include "residual_norm_kernels.h"

extern template void rn::launch_fwd<DT_BF16>(const ResidualNormParams& p, hipStream_t s);
extern template void rn::launch_fwd<DT_F16>(const ResidualNormParams& p, hipStream_t s);
extern template void rn::launch_fwd<DT_F32>(const ResidualNormParams& p, hipStream_t s);
extern template void rn::launch_bwd<DT_BF16>(const ResidualNormParams& p, hipStream_t s);
extern template void rn::launch_bwd<DT_F16>(const ResidualNormParams& p, hipStream_t s);
extern template void rn::launch_bwd<DT_F32>(const ResidualNormParams& p, hipStream_t s);

namespace {

void check(const ResidualNormParams& p) {
  if (p.C < 1 || p.C > RESIDUAL_NORM_MAX_C) throw std::invalid_argument("residual_norm: 1 to 8192 channels");
  if (p.P < 0 || p.P > 0x7ff00000) throw std::invalid_argument("residual_norm: too many rows");
  if (!(p.eps > 0.f)) throw std::invalid_argument("residual_norm: eps has to be positive");   // rows of zeros
  if (p.gate_mode == GATE_GROUP && (p.group_rows < 1 || p.P % p.group_rows))
    throw std::invalid_argument("residual_norm: the rows of a gate's groups have to divide the rows");
  if ((p.post_gamma || p.gate_mode != GATE_NONE) && !p.y)
    throw std::invalid_argument("residual_norm: a gate or post_gamma without y");
  if ((p.post_beta && !p.post_gamma) || (p.pre_beta && !p.pre_gamma) || (!p.layer && (p.post_beta || p.pre_beta)))
    throw std::invalid_argument("residual_norm: a beta goes with its gamma and with norm='layer'");
}

}  // namespace

size_t residual_norm_workspace_floats(const ResidualNormParams& p) {
  if (p.P <= 0 || p.C < 1 || (p.gate_mode == GATE_GROUP && p.group_rows < 1)) return 0;
  // enough for either kind of kernel: the caller need not know which one its call takes
  return (size_t)5 * std::max(rn::plan_bwd(p, true).blocks, rn::plan_bwd(p, false).blocks) * p.C;
}

void launch_residual_norm_fwd(const ResidualNormParams& p, hipStream_t s) {
  check(p);
  if (p.P == 0) return;
  DTF_DT_SWITCH(p.dt, rn::launch_fwd<DT>(p, s));
}

void launch_residual_norm_bwd(const ResidualNormParams& p, hipStream_t s) {
  check(p);
  if (p.P == 0) return;         // the caller clears the vectors' gradients
  if ((p.dz != nullptr) != (p.pre_gamma != nullptr))
    throw std::invalid_argument("residual_norm_grad: dz goes with pre_gamma");
  if (!p.dz && !p.dh) throw std::invalid_argument("residual_norm_grad: neither dh nor dz");
  DTF_DT_SWITCH(p.dt, rn::launch_bwd<DT>(p, s));
}
