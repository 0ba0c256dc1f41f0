// Selective state space scan of a multi-head layer.  Per head h with its group's B and C, per row t:
//   d_t = softplus(dt_t + dt_bias)        a_t = exp(d_t A)
//   h_t = a_t h_{t-1} + d_t x_t B_t^T     (P x N, float32)
//   y_t = h_t C_t + D x_t                 times silu(z_t) where there is a gate
#include "ssm.h"

namespace tesm {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float softplusf_(float v) { return v > 20.0f ? v : log1pf(expf(v)); }
__device__ __forceinline__ float siluf_(float v) { return v * sigmoidf_(v); }

// One wave per (sequence, head, p): lanes over the N states, row after row.
template <int DT>
__global__ __launch_bounds__(256) void ssm_rows_kernel(SsmArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (u >= a.S * a.H * a.P) return;
  const int64_t s = u / (a.H * a.P), h = u / a.P % a.H, p = u % a.P, g = h / (a.H / a.G);
  int64_t first, end;
  if (a.seq_starts) {
    seq_rows(a.seq_starts, s, a.B * a.L, first, end);
  } else {
    first = s * a.L;
    end = first + a.L;
  }
  float st4[4];
  for (int i = 0; i < 4; ++i) {
    const int64_t n = lane + 64 * i;
    st4[i] = a.h0 && n < a.N ? a.h0[u * a.N + n] : 0.0f;
  }
  for (int64_t r = first; r < end; ++r) {
    const float raw = ld<DT>(a.dts, r * a.ld_dt + h) + (a.dt_bias ? a.dt_bias[h] : 0.0f);
    const float d = a.softplus ? softplusf_(raw) : raw;
    const float decay = fast_exp(d * a.A[h]);
    const float x = ld<DT>(a.x, r * a.ld_x + h * a.P + p);
    float acc = 0.0f;
    for (int i = 0; i < 4; ++i) {
      const int64_t n = lane + 64 * i;
      if (n >= a.N) continue;
      st4[i] = decay * st4[i] + d * x * ld<DT>(a.Bm, r * a.ld_b + g * a.N + n);
      acc += st4[i] * ld<DT>(a.Cm, r * a.ld_c + g * a.N + n);
    }
    float y = wave_sum_f<64>(acc);
    if (a.D) y += a.D[h] * x;
    if (a.z) y *= siluf_(ld<DT>(a.z, r * a.ld_z + h * a.P + p));
    if (lane == 0) st<DT>(a.y, r * a.ld_y + h * a.P + p, y);
  }
  if (a.h_out)
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.N) a.h_out[u * a.N + lane + 64 * i] = st4[i];
}

// Convolved value of channel c of the token; the state moves on where `keep`.
template <int DT>
__device__ __forceinline__ float step_channel(const SsmStepArgs& a, int64_t b, int64_t c, int64_t C, bool keep) {
  const float now = ld<DT>(a.row, b * a.ld_row + c);
  if (!a.conv_weight) return now;
  const int W = static_cast<int>(a.W);
  float acc = a.conv_bias ? (a.w_dt == kBF16 ? ld<kBF16>(a.conv_bias, c) : ld<kF32>(a.conv_bias, c)) : 0.0f;
  for (int j = 0; j < W; ++j) {
    const float v = j < W - 1 ? ld<DT>(a.conv_state, (b * (W - 1) + j) * C + c) : now;
    const float w = a.w_dt == kBF16 ? ld<kBF16>(a.conv_weight, c * W + j) : ld<kF32>(a.conv_weight, c * W + j);
    acc = __builtin_fmaf(v, w, acc);
    if (keep && j > 0) st<DT>(a.conv_state_out, (b * (W - 1) + j - 1) * C + c, v);
  }
  return a.silu ? siluf_(acc) : acc;
}

// One workgroup per (sequence, head).
template <int DT>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStepArgs a) {
  __shared__ float bs[kSsmMaxN], cs[kSsmMaxN];
  const int64_t b = blockIdx.y, h = blockIdx.x, hg = a.H / a.G, g = h / hg;
  const int64_t HP = a.H * a.P, C = HP + 2 * a.G * a.N;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t n = threadIdx.x; n < a.N; n += 256) {
    bs[n] = step_channel<DT>(a, b, HP + g * a.N + n, C, h % hg == 0);
    cs[n] = step_channel<DT>(a, b, HP + (a.G + g) * a.N + n, C, h % hg == 0);
  }
  const float raw = ld<DT>(a.dts, b * a.ld_dt + h) + (a.dt_bias ? a.dt_bias[h] : 0.0f);
  const float d = a.softplus ? softplusf_(raw) : raw;
  const float decay = fast_exp(d * a.A[h]);
  __syncthreads();
  for (int64_t p = wave; p < a.P; p += 4) {
    const float x = step_channel<DT>(a, b, h * a.P + p, C, lane == 0);
    float* row = a.state + ((b * a.H + h) * a.P + p) * a.N;
    float acc = 0.0f;
    for (int64_t n = lane; n < a.N; n += 64) {
      const float v = decay * row[n] + d * x * bs[n];
      row[n] = v;
      acc += v * cs[n];
    }
    float y = wave_sum_f<64>(acc);
    if (a.D) y += a.D[h] * x;
    if (a.z) y *= siluf_(ld<DT>(a.z, b * a.ld_z + h * a.P + p));
    if (lane == 0) st<DT>(a.y, b * a.ld_y + h * a.P + p, y);
  }
}

}  // namespace

int64_t selective_scan_ws_bytes(const SsmArgs&) { return 0; }

int launch_selective_scan(const SsmArgs& a, void*, int64_t, hipStream_t st) {
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, "selective scan: dtype must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.L >= 0 && a.S >= 0 && a.H >= 1 && a.P >= 1 && a.G >= 1 && a.N >= 1 && a.H % a.G == 0 &&
                   a.B < (1LL << 31) && a.L < (1LL << 31) && a.B * a.L < (1LL << 31) && a.S < (1LL << 24) &&
                   a.H < (1LL << 20) && a.P < (1LL << 20) && a.H * a.P < (1LL << 24),
               kErrInvalidArg, "selective scan: bad sizes (n_groups must divide the heads)");
  TESM_REQUIRE(a.N <= kSsmMaxN, kErrUnsupported, "selective scan: need at most 256 states");
  TESM_REQUIRE(a.seq_starts ? a.B == 1 : a.S == a.B, kErrInvalidArg,
               "selective scan: packed sequences lie in one row axis (B = 1), others have S = B");
  TESM_REQUIRE(a.A && (a.B * a.L == 0 || (a.x && a.dts && a.Bm && a.Cm && a.y)), kErrInvalidArg,
               "selective scan: need x, dt, A, B, C and y");
  TESM_REQUIRE(a.ld_x >= a.H * a.P && a.ld_y >= a.H * a.P && a.ld_dt >= a.H && a.ld_b >= a.G * a.N &&
                   a.ld_c >= a.G * a.N && (!a.z || a.ld_z >= a.H * a.P),
               kErrInvalidArg, "selective scan: a row pitch is shorter than its row");
  TESM_REQUIRE(!a.h_out || a.h_out != a.h0, kErrInvalidArg, "selective scan: the states out need a buffer of their own");
  TESM_REQUIRE(a.S * a.H * a.P < (1LL << 32), kErrUnsupported, "selective scan: too many states");
  if (a.S == 0) return kOk;
  const unsigned grid = static_cast<unsigned>((a.S * a.H * a.P + 3) / 4);
  if (a.dt == kBF16)
    ssm_rows_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, ssm_rows_kernel<kBF16>)>>>(a);
  else
    ssm_rows_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, ssm_rows_kernel<kF32>)>>>(a);
  return check_launch("selective scan");
}

int launch_selective_scan_step(const SsmStepArgs& a, hipStream_t st) {
  TESM_REQUIRE((a.dt == kF32 || a.dt == kBF16) && (a.w_dt == kF32 || a.w_dt == kBF16), kErrInvalidArg,
               "selective scan step: dtypes must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.H >= 1 && a.P >= 1 && a.G >= 1 && a.N >= 1 && a.H % a.G == 0 && a.B < 65536 &&
                   a.H < (1LL << 20) && a.P < (1LL << 20) && a.H * a.P < (1LL << 24),
               kErrInvalidArg, "selective scan step: bad sizes (n_groups must divide the heads)");
  TESM_REQUIRE(a.N <= kSsmMaxN, kErrUnsupported, "selective scan step: need at most 256 states");
  const int64_t C = a.H * a.P + 2 * a.G * a.N;
  TESM_REQUIRE(a.B == 0 || (a.row && a.dts && a.A && a.state && a.y), kErrInvalidArg,
               "selective scan step: need row, dt, A, state and y");
  TESM_REQUIRE(a.ld_row >= C && a.ld_dt >= a.H && a.ld_y >= a.H * a.P && (!a.z || a.ld_z >= a.H * a.P), kErrInvalidArg,
               "selective scan step: a row pitch is shorter than its row");
  if (a.conv_weight) {
    TESM_REQUIRE(a.W >= 2 && a.W <= kConvMaxW, kErrUnsupported, "selective scan step: need 2 <= W <= 8");
    TESM_REQUIRE(a.B == 0 || (a.conv_state && a.conv_state_out && a.conv_state != a.conv_state_out), kErrInvalidArg,
                 "selective scan step: the convolution needs its state, and another buffer for the state after");
  }
  if (a.B == 0) return kOk;
  const dim3 grid(static_cast<unsigned>(a.H), static_cast<unsigned>(a.B));
  if (a.dt == kBF16)
    ssm_step_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, ssm_step_kernel<kBF16>)>>>(a);
  else
    ssm_step_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, ssm_step_kernel<kF32>)>>>(a);
  return check_launch("selective scan step");
}

}  // namespace tesm
