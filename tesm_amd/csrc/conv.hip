// Short causal convolution over time, one filter per channel:
//   y[t, c] = act(bias[c] + sum_{j < W} weight[c, j] x[t - W + 1 + j, c]),  act = silu or the identity,
// over B sequences of L rows, or over sequences packed one behind the other (seq_starts).  Rows before a sequence
// come from its state (W - 1 rows, oldest first) and are zero without one; the state out is the last W - 1 rows of
// state and sequence together.  Sums in float32, one rounding to the layer type.
//
// Bound by HBM up to 4 taps, with float32 rows up to 8: each row is read once and written once.  A thread owns 16 bytes of
// channels, at any alignment, and walks kConvRows rows with its filter and the last W - 1 rows in registers, as float32: for
// 8 bfloat16 channels and 5 to 8 taps these do not fit the 128 registers that four waves per SIMD leave, and 22 to 220 of them
// spill.  The W - 1 rows before a thread's own are read again, from the cache.  Measured, 8192 rows of 1792 channels with 4, 5,
// 6, 7 and 8 taps: bfloat16 15, 21, 39, 72 and 101 us (a copy of the same 29 MB 11.3), float32 22, 24, 25, 26 and 27.  The last thread of a row ends with the row, so it may form some of its neighbour's channels too (the same
// values).  The states out are written by threads behind those of the rows, in the same launch.
#include "ssm.h"

namespace tesm {

namespace {

constexpr int kConvRows = 8;  // rows per thread

// Sequence of packed row r: the last s with seq_starts[s] <= r (S - 1 at most, 0 at least).
__device__ __forceinline__ int conv_seq_of(const int32_t* starts, int64_t S, int r) {
  int lo = 0, hi = static_cast<int>(S);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// 16 bytes at any address of an element.
typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ uint4 load16(const void* p) { return __builtin_bit_cast(uint4, *static_cast<const any16*>(p)); }
// (non-temporal: y is written once and read by another kernel, and the cache is left to the rows that two threads read;
// 29 MB of bfloat16 rows 15.3 us against 16.6, 51 MB of float32 ones 27 against 33)
__device__ __forceinline__ void store16(void* p, const uint4& v) {
  __builtin_nontemporal_store(__builtin_bit_cast(any16, v), static_cast<any16*>(p));
}

// V elements of a row.
template <int DT, int V>
struct ConvVec;
template <int DT>
struct ConvVec<DT, 1> {
  using R = uint32_t;  // raw bits
  static __device__ __forceinline__ R load(const void* p, int64_t i) { return ld_bits<DT>(p, i); }
  static __device__ __forceinline__ R zero() { return 0; }
  static __device__ __forceinline__ void get(R r, float (&v)[1]) { v[0] = from_bits<DT>(r); }
  static __device__ __forceinline__ void put(void* p, int64_t i, const float (&v)[1]) { st<DT>(p, i, v[0]); }
  static __device__ __forceinline__ void raw(void* p, int64_t i, R r) {
    if constexpr (DT == kBF16)
      static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(r);
    else
      static_cast<uint32_t*>(p)[i] = r;
  }
};
template <>
struct ConvVec<kBF16, 8> {
  using R = uint4;
  static __device__ __forceinline__ R load(const void* p, int64_t i) {
    return load16(static_cast<const uint16_t*>(p) + i);
  }
  static __device__ __forceinline__ R zero() { return make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ void get(const R& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void put(void* p, int64_t i, const float (&v)[8]) {
    store16(static_cast<uint16_t*>(p) + i,
            make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
  }
  static __device__ __forceinline__ void raw(void* p, int64_t i, const R& r) {
    store16(static_cast<uint16_t*>(p) + i, r);
  }
};
template <>
struct ConvVec<kF32, 4> {
  using R = uint4;
  static __device__ __forceinline__ R load(const void* p, int64_t i) {
    return load16(static_cast<const float*>(p) + i);
  }
  static __device__ __forceinline__ R zero() { return make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ void get(const R& r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ void put(void* p, int64_t i, const float (&v)[4]) {
    store16(static_cast<float*>(p) + i, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
  }
  static __device__ __forceinline__ void raw(void* p, int64_t i, const R& r) {
    store16(static_cast<float*>(p) + i, r);
  }
};

// silu of a bfloat16 result: the exponent's rounding (2^-24 |v| log2 e) is far below the result's.
template <int DT>
__device__ __forceinline__ float conv_silu(float v) {
  if constexpr (DT == kF32) return siluf_(v);
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}

// Row `back` rows before row `first` of sequence s (1 is the last one before it).
template <int DT, int V>
__device__ __forceinline__ typename ConvVec<DT, V>::R conv_before(const ConvArgs& a, int s, int back, int c) {
  const int W1 = static_cast<int>(a.W) - 1;
  if (!a.state || back > W1) return ConvVec<DT, V>::zero();
  return ConvVec<DT, V>::load(a.state, (static_cast<int64_t>(s) * W1 + W1 - back) * a.C + c);
}

// The filters of V channels from c on: their n = V * W values lie one behind the other.
template <int WDT, int W, int V>
__device__ __forceinline__ void conv_filter(const void* weight, const void* bias, int c, float (&w)[W][V], float (&b)[V]) {
  constexpr int EV = WDT == kBF16 ? 8 : 4, N = V * W / EV;
  if constexpr (V * W % EV != 0) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][i] = ld<WDT>(weight, static_cast<int64_t>(c + i) * W + j);
  } else {
    uint4 u[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
      u[k] = load16(static_cast<const char*>(weight) + static_cast<int64_t>(c) * W * (16 / EV) + 16 * k);
    float f[V * W];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float v[EV];
      ConvVec<WDT, EV>::get(u[k], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) f[k * EV + e] = v[e];
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) w[j][i] = f[i * W + j];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = bias ? ld<WDT>(bias, c + i) : 0.0f;
}

// Threads below runs * cv: kConvRows rows of V channels each; behind them one per state row out.
template <int DT, int WDT, int W, int V>
__global__ __launch_bounds__(256, 4) void causal_conv_kernel(ConvArgs a, int runs, int cv, int64_t total) {
  using CV = ConvVec<DT, V>;
  using R = typename CV::R;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (u >= total) return;
  const int run = static_cast<int>(u / cv), c = min(static_cast<int>(u - static_cast<int64_t>(run) * cv) * V, static_cast<int>(a.C) - V);
  const int M = static_cast<int>(a.B * a.L), L = static_cast<int>(a.L);
  if (run >= runs) {  // state out: row j of sequence s
    const int e = run - runs, s = e / (W - 1), j = e - s * (W - 1);
    int64_t first = static_cast<int64_t>(s) * L, end = first + L;
    if (a.seq_starts) seq_rows(a.seq_starts, s, M, first, end);
    const int64_t src = end - (W - 1) + j;
    const R v = src >= first ? CV::load(a.x, src * a.ld_x + c) : conv_before<DT, V>(a, s, static_cast<int>(first - src), c);
    CV::raw(a.state_out, static_cast<int64_t>(e) * a.C + c, v);
    return;
  }
  float w[W][V], bias[V];
  conv_filter<WDT, W, V>(a.weight, a.bias, c, w, bias);
  const int r0 = run * kConvRows, r1 = min(r0 + kConvRows, M);
  // the sequence of the first row
  int s;
  int64_t first, end;
  if (a.seq_starts) {
    s = conv_seq_of(a.seq_starts, a.S, r0);
    seq_rows(a.seq_starts, s, M, first, end);
  } else {
    s = r0 / L;
    first = static_cast<int64_t>(s) * L;
    end = first + L;
  }
  float past[W - 1][V];  // the rows before the current one, oldest first
  auto fill = [&](int r) {
#pragma unroll
    for (int j = 0; j < W - 1; ++j) {
      const int64_t src = r - (W - 1) + j;
      CV::get(src >= first ? CV::load(a.x, src * a.ld_x + c) : conv_before<DT, V>(a, s, static_cast<int>(first - src), c), past[j]);
    }
  };
  auto emit = [&](int r, const R& raw) {
    float x[V], y[V];
    CV::get(raw, x);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float acc = bias[i];
#pragma unroll
      for (int j = 0; j < W - 1; ++j) acc = __builtin_fmaf(past[j][i], w[j][i], acc);
      acc = __builtin_fmaf(x[i], w[W - 1][i], acc);
      y[i] = a.silu ? conv_silu<DT>(acc) : acc;
    }
    CV::put(a.y, r * a.ld_y + c, y);
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int j = 0; j + 1 < W - 1; ++j) past[j][i] = past[j + 1][i];
      past[W - 2][i] = x[i];
    }
  };
  if (r0 >= first && r1 <= end && r1 == r0 + kConvRows) {  // whole run inside one sequence: every load ahead
    R raw[kConvRows];
#pragma unroll
    for (int k = 0; k < kConvRows; ++k) raw[k] = CV::load(a.x, (r0 + k) * a.ld_x + c);
    fill(r0);
#pragma unroll
    for (int k = 0; k < kConvRows; ++k) emit(r0 + k, raw[k]);
    return;
  }
  bool filled = false;
  for (int r = r0; r < r1; ++r) {
    if (r < first) continue;  // in front of the first sequence
    while (r >= end && s + 1 < a.S) {
      ++s;
      filled = false;
      if (a.seq_starts) {
        seq_rows(a.seq_starts, s, M, first, end);
      } else {
        first = static_cast<int64_t>(s) * L;
        end = first + L;
      }
    }
    if (r < first || r >= end) continue;
    if (!filled) fill(r);
    filled = true;
    emit(r, CV::load(a.x, r * a.ld_x + c));
  }
}

template <int DT, int WDT, int W, int V>
int run_conv(const ConvArgs& a, hipStream_t st) {
  const int64_t M = a.S > 0 ? a.B * a.L : 0;
  const int64_t runs = (M + kConvRows - 1) / kConvRows, states = a.state_out ? a.S * (W - 1) : 0;
  const int cv = static_cast<int>((a.C + V - 1) / V);
  const int64_t total = (runs + states) * cv, blocks = (total + 255) / 256;
  if (total == 0) return kOk;
  TESM_REQUIRE(blocks < (1LL << 31), kErrUnsupported, "causal conv: too many rows and channels for one call");
  causal_conv_kernel<DT, WDT, W, V><<<static_cast<unsigned>(blocks), 256, 0, TESM_LOGGED(st, causal_conv_kernel<DT, WDT, W, V>)>>>(
      a, static_cast<int>(runs), cv, total);
  return check_launch("causal conv");
}

template <int DT, int WDT, int V>
int run_conv_w(const ConvArgs& a, hipStream_t st) {
  switch (a.W) {
    case 2: return run_conv<DT, WDT, 2, V>(a, st);
    case 3: return run_conv<DT, WDT, 3, V>(a, st);
    case 4: return run_conv<DT, WDT, 4, V>(a, st);
    case 5: return run_conv<DT, WDT, 5, V>(a, st);
    case 6: return run_conv<DT, WDT, 6, V>(a, st);
    case 7: return run_conv<DT, WDT, 7, V>(a, st);
    default: return run_conv<DT, WDT, 8, V>(a, st);
  }
}

template <int DT, int WDT>
int run_conv_v(const ConvArgs& a, hipStream_t st) {
  constexpr int V = DT == kBF16 ? 8 : 4;
  return a.C >= V ? run_conv_w<DT, WDT, V>(a, st) : run_conv_w<DT, WDT, 1>(a, st);
}

}  // namespace

int launch_causal_conv(const ConvArgs& a, hipStream_t st) {
  TESM_REQUIRE((a.dt == kF32 || a.dt == kBF16) && (a.w_dt == kF32 || a.w_dt == kBF16), kErrInvalidArg,
               "causal conv: dtypes must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.L >= 0 && a.C >= 1 && a.S >= 0 && a.B < (1LL << 31) && a.L < (1LL << 31) &&
                   a.C < (1LL << 23) && a.B * a.L < (1LL << 31) - 65536 && a.S < (1LL << 24),
               kErrInvalidArg, "causal conv: bad sizes");
  TESM_REQUIRE(a.W >= 2 && a.W <= kConvMaxW, kErrUnsupported, "causal conv: need 2 <= W <= 8");
  TESM_REQUIRE(a.seq_starts ? a.B == 1 : a.S == a.B, kErrInvalidArg,
               "causal conv: packed sequences lie in one row axis (B = 1), others have S = B");
  TESM_REQUIRE(a.weight && (a.B * a.L == 0 || (a.x && a.y)) && a.ld_x >= a.C && a.ld_y >= a.C, kErrInvalidArg,
               "causal conv: need weight, x (ld_x >= C) and y (ld_y >= C)");
  TESM_REQUIRE(!a.state_out || a.state_out != a.state, kErrInvalidArg,
               "causal conv: the state out needs a buffer of its own");
  if (a.dt == kBF16)
    return a.w_dt == kBF16 ? run_conv_v<kBF16, kBF16>(a, st) : run_conv_v<kBF16, kF32>(a, st);
  return a.w_dt == kBF16 ? run_conv_v<kF32, kBF16>(a, st) : run_conv_v<kF32, kF32>(a, st);
}

}  // namespace tesm
