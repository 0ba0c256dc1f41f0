// Products of float matrices with what stands around them in a layer: a gated pair of projections, a projection with bias,
// activation and residual, and their backward passes.
#pragma once

#include "tesm_hip_internal.h"

namespace tesm {

enum Act : int { kActNone = 0, kActSilu = 1, kActGelu = 2 };

// h = act(x w^T) * (x w2^T) (w2 given), or y = act(x w^T + bias) + residual.  z, z2: what stands before the activation, kept for the
// backward pass.
struct DenseArgs {
  int dt = 0, act = kActNone;
  int64_t M = 0, K = 0, N = 0;
  const void* x = nullptr;  // (M, ld_x)
  int64_t ld_x = 0;
  const void* w = nullptr;  // (N, ld_w)
  int64_t ld_w = 0;
  const void* w2 = nullptr;
  int64_t ld_w2 = 0;
  const void* bias = nullptr;      // optional (N)
  const void* residual = nullptr;  // optional (M, ld_r)
  int64_t ld_r = 0;
  void* y = nullptr;  // (M, ld_y)
  int64_t ld_y = 0;
  void* z = nullptr;  // optional (M, N): float32, or 24 bits (dense_mfma.h)
  void* z2 = nullptr;
};

struct DenseBwdArgs {
  DenseArgs in;                // bias, residual, y not used; z (and z2) those kept
  const void* grad = nullptr;  // (M, ld_g)
  int64_t ld_g = 0;
  void* dx = nullptr;   // optional (M, K)
  void* dw = nullptr;   // optional (N, K)
  void* dw2 = nullptr;
  void* dbias = nullptr;  // optional (N)
};

int64_t dense_ws_bytes(const DenseArgs& a);
int64_t dense_bwd_ws_bytes(const DenseBwdArgs& a);
int launch_dense(const DenseArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);
int launch_dense_bwd(const DenseBwdArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);

}  // namespace tesm
