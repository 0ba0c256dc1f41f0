// Short causal convolution over time, one filter per channel:
//   y[t, c] = act(bias[c] + sum_{j < W} weight[c, j] x[t - W + 1 + j, c]),  act = silu or the identity,
// over B sequences of L rows, or over sequences packed one behind the other (seq_starts).  Rows before a sequence
// come from its state (W - 1 rows, oldest first) and are zero without one; the state out is the last W - 1 rows of
// state and sequence together.  Sums in float32, one rounding to the layer type.
#include "ssm.h"

namespace tesm {

namespace {

constexpr int kConvRows = 8;  // rows per thread

// Sequence of packed row r: the last s with seq_starts[s] <= r (S - 1 at most, 0 at least).
__device__ __forceinline__ int64_t conv_seq_of(const int32_t* starts, int64_t S, int64_t r) {
  int64_t lo = 0, hi = S;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (starts[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <int DT>
__global__ __launch_bounds__(256) void causal_conv_kernel(ConvArgs a) {
  const int64_t c = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x;
  if (c >= a.C) return;
  const int64_t M = a.B * a.L;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kConvRows, r1 = r0 + kConvRows < M ? r0 + kConvRows : M;
  const int W = static_cast<int>(a.W);
  for (int64_t r = r0; r < r1; ++r) {
    int64_t s, first, end;
    if (a.seq_starts) {
      s = conv_seq_of(a.seq_starts, a.S, r);
      seq_rows(a.seq_starts, s, M, first, end);
      if (r < first || r >= end) continue;
    } else {
      s = r / a.L;
      first = s * a.L;
    }
    float acc = a.bias ? (a.w_dt == kBF16 ? ld<kBF16>(a.bias, c) : ld<kF32>(a.bias, c)) : 0.0f;
    for (int j = 0; j < W; ++j) {
      const int64_t src = r - (W - 1) + j;
      float v = 0.0f;
      if (src >= first)
        v = ld<DT>(a.x, src * a.ld_x + c);
      else if (a.state)
        v = ld<DT>(a.state, (s * (W - 1) + (W - 1) + (src - first)) * a.C + c);
      const float w = a.w_dt == kBF16 ? ld<kBF16>(a.weight, c * W + j) : ld<kF32>(a.weight, c * W + j);
      acc = __builtin_fmaf(v, w, acc);
    }
    if (a.silu) acc = acc * sigmoidf_(acc);
    st<DT>(a.y, r * a.ld_y + c, acc);
  }
}

template <int DT>
__global__ __launch_bounds__(256) void conv_state_kernel(ConvArgs a) {
  const int64_t c = static_cast<int64_t>(blockIdx.y) * 256 + threadIdx.x;
  if (c >= a.C) return;
  const int64_t W1 = a.W - 1, s = blockIdx.x / W1, j = blockIdx.x % W1;
  int64_t first, end;
  if (a.seq_starts) {
    seq_rows(a.seq_starts, s, a.B * a.L, first, end);
  } else {
    first = s * a.L;
    end = first + a.L;
  }
  const int64_t src = end - W1 + j;
  float v = 0.0f;
  if (src >= first)
    v = ld<DT>(a.x, src * a.ld_x + c);
  else if (a.state)
    v = ld<DT>(a.state, (s * W1 + W1 + (src - first)) * a.C + c);
  st<DT>(a.state_out, (s * W1 + j) * a.C + c, v);
}

}  // namespace

int launch_causal_conv(const ConvArgs& a, hipStream_t st) {
  TESM_REQUIRE((a.dt == kF32 || a.dt == kBF16) && (a.w_dt == kF32 || a.w_dt == kBF16), kErrInvalidArg,
               "causal conv: dtypes must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.L >= 0 && a.C >= 1 && a.S >= 0 && a.B < (1LL << 31) && a.L < (1LL << 31) &&
                   a.C < (1LL << 23) && a.B * a.L < (1LL << 31) && a.S < (1LL << 24),
               kErrInvalidArg, "causal conv: bad sizes");
  TESM_REQUIRE(a.W >= 2 && a.W <= kConvMaxW, kErrUnsupported, "causal conv: need 2 <= W <= 8");
  TESM_REQUIRE(a.seq_starts ? a.B == 1 : a.S == a.B, kErrInvalidArg,
               "causal conv: packed sequences lie in one row axis (B = 1), others have S = B");
  TESM_REQUIRE(a.weight && (a.B * a.L == 0 || (a.x && a.y)) && a.ld_x >= a.C && a.ld_y >= a.C, kErrInvalidArg,
               "causal conv: need weight, x (ld_x >= C) and y (ld_y >= C)");
  TESM_REQUIRE(!a.state_out || a.state_out != a.state, kErrInvalidArg,
               "causal conv: the state out needs a buffer of its own");
  const unsigned gy = static_cast<unsigned>((a.C + 255) / 256);
  const int64_t M = a.B * a.L;
  if (M > 0 && a.S > 0) {
    const dim3 grid(static_cast<unsigned>((M + kConvRows - 1) / kConvRows), gy);
    if (a.dt == kBF16)
      causal_conv_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, causal_conv_kernel<kBF16>)>>>(a);
    else
      causal_conv_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, causal_conv_kernel<kF32>)>>>(a);
  }
  if (a.state_out && a.S > 0) {
    const dim3 grid(static_cast<unsigned>(a.S * (a.W - 1)), gy);
    if (a.dt == kBF16)
      conv_state_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, conv_state_kernel<kBF16>)>>>(a);
    else
      conv_state_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, conv_state_kernel<kF32>)>>>(a);
  }
  return check_launch("causal conv");
}

}  // namespace tesm
