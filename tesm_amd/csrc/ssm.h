// Selective state space layer pieces: arguments shared by the kernels (conv.hip, ssm.hip) and the C-ABI layer.
#pragma once

#include "tesm_hip_internal.h"

namespace tesm {

constexpr int64_t kConvMaxW = 8;
constexpr int64_t kSsmMaxN = 256;

struct ConvArgs {
  int dt = 0, w_dt = 0;
  int64_t B = 0, L = 0, C = 0, W = 0, S = 0;  // S sequences (B of L rows, or packed into L rows by seq_starts)
  int silu = 1;
  const void* x = nullptr;       // row r at x[r * ld_x], B * L rows
  int64_t ld_x = 0;
  const void* weight = nullptr;  // (C, W) w_dt
  const void* bias = nullptr;    // optional (C) w_dt
  const int32_t* seq_starts = nullptr;  // optional (S + 1): sequence s is rows [seq_starts[s], seq_starts[s + 1])
  const void* state = nullptr;   // optional (S, W - 1, C) dt: the rows before each sequence, oldest first
  void* y = nullptr;
  int64_t ld_y = 0;
  void* state_out = nullptr;     // optional (S, W - 1, C) dt: each sequence's last W - 1 rows
};
int launch_causal_conv(const ConvArgs& a, hipStream_t st);

struct SsmArgs {
  int dt = 0;
  int64_t B = 0, L = 0, H = 0, P = 0, G = 0, N = 0, S = 0;
  int softplus = 1;
  const void* x = nullptr;   // (row, h, p) at x[row * ld_x + h * P + p]
  int64_t ld_x = 0;
  const void* dts = nullptr; // (row, h) at dts[row * ld_dt + h]
  int64_t ld_dt = 0;
  const float* A = nullptr;  // (H)
  const void* Bm = nullptr;  // (row, g, n) at Bm[row * ld_b + g * N + n]
  int64_t ld_b = 0;
  const void* Cm = nullptr;
  int64_t ld_c = 0;
  const float* D = nullptr;        // optional (H)
  const void* z = nullptr;         // optional, as x
  int64_t ld_z = 0;
  const float* dt_bias = nullptr;  // optional (H)
  const int32_t* seq_starts = nullptr;
  const float* h0 = nullptr;       // optional (S, H, P, N)
  void* y = nullptr;               // as x
  int64_t ld_y = 0;
  float* h_out = nullptr;          // optional (S, H, P, N)
};
int64_t selective_scan_ws_bytes(const SsmArgs& a);
int launch_selective_scan(const SsmArgs& a, void* ws, int64_t ws_bytes, hipStream_t st);

struct SsmStepArgs {
  int dt = 0, w_dt = 0;
  int64_t B = 0, H = 0, P = 0, G = 0, N = 0, W = 0;
  int softplus = 1, silu = 1;
  const void* row = nullptr;         // (B, H * P + 2 * G * N): x, B, C of the token, before the convolution
  int64_t ld_row = 0;
  const void* conv_weight = nullptr; // optional (C, W) w_dt; without it the row is used as it is
  const void* conv_bias = nullptr;   // optional (C) w_dt
  const void* conv_state = nullptr;  // (B, W - 1, C) dt
  void* conv_state_out = nullptr;    // (B, W - 1, C) dt, another buffer
  const void* dts = nullptr;         // (B, H)
  int64_t ld_dt = 0;
  const float* A = nullptr;
  const float* D = nullptr;
  const void* z = nullptr;           // optional (B, H * P)
  int64_t ld_z = 0;
  const float* dt_bias = nullptr;
  float* state = nullptr;            // (B, H, P, N), updated in place
  void* y = nullptr;                 // (B, H * P)
  int64_t ld_y = 0;
};
int launch_selective_scan_step(const SsmStepArgs& a, hipStream_t st);

__device__ __forceinline__ float siluf_(float v) { return v * __builtin_amdgcn_rcpf(1.0f + fast_exp(-v)); }

// The real rows [a, b) of packed sequence s, whatever the array holds: inside [0, M), b >= a.
__device__ __forceinline__ void seq_rows(const int32_t* starts, int64_t s, int64_t M, int64_t& a, int64_t& b) {
  const int64_t lo = starts[s], hi = starts[s + 1];
  a = lo < 0 ? 0 : (lo > M ? M : lo);
  b = hi < a ? a : (hi > M ? M : hi);
}

}  // namespace tesm
