// The seam between two residual blocks (residual_norm.hip): arguments and launchers.
#pragma once
#include "common.h"

enum ResidualGate { GATE_NONE = 0, GATE_GROUP = 1, GATE_ELEMENT = 2 };

struct ResidualNormParams {
  // forward: x, y (or null), gate -> h, z.   backward: dh (or null), dz, h, y, gate -> dx, dy, dgate and the
  // gradients of the four vectors.  Rows of `C` channels; ld*: elements from one row to the next.
  const void *x = nullptr, *y = nullptr, *gate = nullptr, *dh = nullptr, *dz = nullptr;
  void *h = nullptr, *z = nullptr, *dx = nullptr, *dy = nullptr, *dgate = nullptr;
  const float *post_gamma = nullptr, *post_beta = nullptr, *pre_gamma = nullptr, *pre_beta = nullptr;
  float *dpost_gamma = nullptr, *dpost_beta = nullptr, *dpre_gamma = nullptr, *dpre_beta = nullptr;
  float* ws = nullptr;          // backward: residual_norm_workspace_floats() of them
  int64_t ldx = 0, ldy = 0, ldgate = 0, lddh = 0, lddz = 0;
  int P = 0, C = 0;
  int group_rows = 0;           // GATE_GROUP: rows that share a gate row
  int gate_mode = GATE_NONE, sigmoid = 0, layer = 0, dt = DT_BF16;
  float scale = 1.f, eps = 1e-6f;
};

constexpr int RESIDUAL_NORM_MAX_C = 8192;
size_t residual_norm_workspace_floats(const ResidualNormParams& p);
void launch_residual_norm_fwd(const ResidualNormParams& p, hipStream_t s);
void launch_residual_norm_bwd(const ResidualNormParams& p, hipStream_t s);
