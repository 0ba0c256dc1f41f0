// Rows of logits x: with lse = logsumexp(x) and p = exp(x - lse),
//   log probability of a given token t: x_t - lse,   entropy: H = -sum p (x - lse),
// and the n largest logits' log probabilities; backward, with gradients g of the log probability and e of the entropy,
//   dx_v = g [v = t] - p_v (g + e ((x_v - lse) + H)).
//
// One pass over a row (row_pass.h): terms 2^(x L - ref), their sum S and the sum Q of the terms times their exponents, so that
// lse = ref ln 2 + log S and H = log S - Q ln 2 / S.  Parts of a row are joined in 64 bits.
//
// The backward pass forms p again as 2^((x - m) L - d), m near the row's largest logit and d in two floats: the high one goes into
// the exponent's fused operation, the low one into the row's two coefficients, so that an element costs one exponential and five
// more operations.
//
// Bound by HBM: 8192 x 151936 bfloat16 forward 459 us, backward 939 (5.4 TB/s); one row with its 20 best by latency, 10 us and 5 to join
// its parts.
#include "logp.h"
#include "row_pass.h"

namespace tesm {

namespace {

__device__ unsigned g_logp_status;

constexpr int kLogpWaves = 4;
constexpr double kLn2 = 0.69314718055994530942;

// exp(x - ref) summed, and (x - ref) exp(x - ref) summed.
struct LogpSum {
  double ref, sum, dot;
};
// The sums of groups of WIDTH lanes, on every lane of a group.  (Equal references may be infinite; a part of -infinities alone has an
// infinite distance and nothing to add; a NaN sum stays one.)
template <int WIDTH>
__device__ __forceinline__ LogpSum join_lanes(const LogpSum& a) {
  double ref = a.ref;
#pragma unroll
  for (int d = 1; d < WIDTH; d <<= 1) ref = fmax(ref, __shfl_xor(ref, d));
  const double far = a.ref == ref ? 0.0 : a.ref - ref, f = exp(far);
  double sum = f * a.sum, dot = f == 0.0 ? 0.0 * a.sum : f * (a.dot + far * a.sum);
#pragma unroll
  for (int d = 1; d < WIDTH; d <<= 1) {
    sum += __shfl_xor(sum, d);
    dot += __shfl_xor(dot, d);
  }
  return {ref, sum, dot};
}

// What a row's sums and list say, by one wave.
__device__ __forceinline__ void finish_row(const LogpArgs& a, int64_t r, const LogpSum& s, uint64_t list, int DT) {
  const int lane = threadIdx.x & 63;
  const double log_sum = log(s.sum), entropy = log_sum - s.dot / s.sum;
  if (lane < a.top) {
    a.top_logp[r * a.top + lane] = static_cast<float>((static_cast<double>(key_value(list)) - s.ref) - log_sum);
    a.top_tokens[r * a.top + lane] = key_index(list);
  }
  if (lane != 0) return;
  const int64_t t = a.targets[r];
  float lp = 0.0f;
  if (t != a.ignore) {
    if (t >= 0 && t < a.V) {
      const int64_t i = r * a.ld + t;
      const float x = DT == kBF16 ? ld<kBF16>(a.logits, i) : ld<kF32>(a.logits, i);
      lp = static_cast<float>((static_cast<double>(x) - s.ref) - log_sum);
    } else {
      lp = __builtin_nanf("");
      __hip_atomic_fetch_or(&g_logp_status, 4u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  a.logp[r] = lp;
  a.entropy[r] = static_cast<float>(entropy);
  if (a.kept) {
    // exp(x - lse) = 2^((x - m) log2 e - d) with m near the largest logit: neither term leaves float32 in any row
    const float m = static_cast<float>(s.ref);
    const double d = ((s.ref - static_cast<double>(m)) + log_sum) * 1.4426950408889634074;
    const float hi = static_cast<float>(d);
    float* k = a.kept + 4 * r;
    k[0] = m;
    k[1] = hi;
    k[2] = static_cast<float>(d - static_cast<double>(hi));
    k[3] = static_cast<float>(entropy);
  }
}

// Part blockIdx.x % parts of row blockIdx.x / parts, a quarter of it per wave.
template <int DT, bool LIST>
__global__ __launch_bounds__(64 * kLogpWaves) void logp_row_kernel(LogpArgs a, int m, int parts, int part, uint64_t* keys, LogpSum* sums) {
  __shared__ uint64_t buffer[kLogpWaves][LIST ? 64 + 64 * (DT == kBF16 ? 8 : 4) : 1];
  __shared__ LogpSum ps[kLogpWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x / parts;
  const int at = static_cast<int>(blockIdx.x % parts);
  const char* row = static_cast<const char*>(a.logits) + r * a.ld * (DT == kBF16 ? 2 : 4);
  const int each = part / kLogpWaves, V = static_cast<int>(a.V);
  const int64_t from = static_cast<int64_t>(at) * part + wave * each;
  const int lo = from < V ? static_cast<int>(from) : V, hi = V - lo < each ? V : lo + each;
  RowPart p = row_pass<DT, false, LIST, true>(row, lo, hi, m, buffer[wave]);
  float mx = wave_max<64>(p.max);
  const bool again = __any(sum_is_off(p, mx));
  if (again) {
    p = row_pass<DT, true, LIST, true>(row, lo, hi, m, buffer[wave]);
    mx = wave_max<64>(p.max);
  }
  const float top = fmaxf(mx, again ? -FLT_MAX : -kFar), own = fmaxf(p.max, again ? -FLT_MAX : -kFar);
  const float far = p.max == mx ? 0.0f : again ? (own - top) * kLog2e : own * kLog2e - top * kLog2e;
  const float scale = __builtin_amdgcn_exp2f(far);
  const float s = wave_sum_f<64>(p.sum * scale), q = wave_sum_f<64>(scale * __builtin_fmaf(fmaxf(far, -1.0e5f), p.sum, p.dot));
  // (the reference as in beam search: the rounding of the largest logit's product taken off again, in 64 bits)
  const double t = top, over = t * static_cast<double>(kLog2e) - static_cast<double>(top * kLog2e);
  const double ref = again || mx == -__builtin_inff() ? static_cast<double>(mx) : t - kLn2 * over;
  if (lane == 0) ps[wave] = {ref, s, kLn2 * q};
  if constexpr (LIST) buffer[wave][lane] = p.list;
  __syncthreads();
  if (wave) return;
  if constexpr (LIST)
    for (int w = 1; w < kLogpWaves; ++w) p.list = merge_lists(p.list, buffer[w][lane]);
  const LogpSum o = join_lanes<kLogpWaves>(ps[lane % kLogpWaves]);
  if (parts == 1) return finish_row(a, r, o, p.list, DT);
  if constexpr (LIST)
    if (lane < m) keys[static_cast<int64_t>(blockIdx.x) * m + lane] = p.list;
  if (lane == 0) sums[blockIdx.x] = o;
}

// A workgroup per row joins its parts: a lane each for their sums, and, with lists, a wave each for runs of 64 keys, then merged in
// pairs.
template <int DT, bool LIST>
__global__ __launch_bounds__(64 * (LIST ? 8 : 1)) void logp_join_kernel(LogpArgs a, int m, int parts, const uint64_t* keys, const LogpSum* sums) {
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const LogpSum* sr = sums + r * parts;
  LogpSum s = {-__builtin_inf(), 0.0, 0.0};
  if (wave == 0 && lane < parts) s = sr[lane];
  uint64_t list = 0;
  if constexpr (LIST) {
    __shared__ uint64_t lists[8][64];
    const uint64_t* kr = keys + r * parts * m;
    const int count = parts * m;
#pragma unroll 1
    for (int c = wave * 64; c < count; c += 512) list = merge64(list, c + lane < count ? kr[c + lane] : 0);
    const int waves = count < 512 ? (count + 63) / 64 : 8;
#pragma unroll 1
    for (int d = 1; d < waves; d <<= 1) {
      lists[wave][lane] = list;
      __syncthreads();
      if (wave % (2 * d) == 0 && wave + d < waves) list = merge_lists(list, lists[wave + d][lane]);
      __syncthreads();
    }
    if (wave) return;
  }
  s = join_lanes<64>(s);
  for (int c = 64; c < parts; c += 64) {  // (more than 64 parts: joined 64 at a time)
    const LogpSum more = join_lanes<64>(c + lane < parts ? sr[c + lane] : LogpSum{-__builtin_inf(), 0.0, 0.0});
    s = join_lanes<2>(lane & 1 ? more : s);
  }
  finish_row(a, r, s, list, DT);
}

// Elements [part blockIdx.x % parts) of row blockIdx.x / parts, 16 bytes per lane and load, four loads under way.
template <int DT, bool ENT>
__global__ __launch_bounds__(256) void logp_bwd_kernel(LogpBwdArgs a, int parts, int64_t part) {
  constexpr int EV = DT == kBF16 ? 8 : 4, ES = 16 / EV, U = 4;
  const int64_t r = blockIdx.x / parts, at = blockIdx.x % parts;
  const float* k = a.kept + 4 * r;
  const int64_t t = a.targets[r];
  float g = a.grad_logp ? a.grad_logp[r] : 0.0f;
  const float e = ENT ? a.grad_entropy[r] : 0.0f;
  if (t == a.ignore)
    g = 0.0f;
  else if (t < 0 || t >= a.V)
    g = __builtin_nanf("");
  const float mx = k[0], c = k[1], low = k[2], scale = __builtin_amdgcn_exp2f(-low), ln2 = 0.69314718055994530942f;
  const float A = -scale * (ENT ? __builtin_fmaf(e, __builtin_fmaf(-low, ln2, k[3]), g) : g), B = ENT ? -scale * e * ln2 : 0.0f;
  const int64_t lo = at * part, hi = a.V - lo < part ? a.V : lo + part;
  const int hot = t >= lo && t < hi && t != a.ignore ? static_cast<int>(t - lo) : -1;
  const char* src = static_cast<const char*>(a.logits) + (r * a.ld + lo) * ES;
  char* dst = static_cast<char*>(a.grad_logits) + (r * a.ld_g + lo) * ES;
  const int n = static_cast<int>(hi - lo);
  auto value = [&](float x) {
    float y = __builtin_fmaf(x - mx, kLog2e, -c);
    if constexpr (ENT) {
      y = y < -150.0f ? -150.0f : y;  // (keeps a NaN)
      return __builtin_amdgcn_exp2f(y) * __builtin_fmaf(B, y, A);
    }
    return __builtin_amdgcn_exp2f(y) * A;
  };
  for (int i0 = threadIdx.x * EV; i0 < n; i0 += 256 * EV * U) {
    any16 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 256 * EV;
      if (i + EV <= n) raw[u] = *reinterpret_cast<const any16*>(src + static_cast<int64_t>(i) * ES);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 256 * EV;
      if (i >= n) break;
      if (i + EV <= n) {
        float v[EV];
        unpack_logits<DT>(raw[u], v);
#pragma unroll
        for (int q = 0; q < EV; ++q) v[q] = value(v[q]);
        if (static_cast<unsigned>(hot - i) < static_cast<unsigned>(EV)) {
#pragma unroll
          for (int q = 0; q < EV; ++q)
            if (hot - i == q) v[q] += g;
        }
        any16 o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = DT == kBF16 ? pack_bf16x2(v[2 * q % EV], v[(2 * q + 1) % EV]) : __float_as_uint(v[q % EV]);
        *reinterpret_cast<any16*>(dst + static_cast<int64_t>(i) * ES) = o;
      } else {
        for (int q = i; q < n; ++q) {
          float v = value(ld<DT>(src, q));
          if (q == hot) v += g;
          st<DT>(dst, q, v);
        }
      }
    }
  }
}

int64_t up256(int64_t v) { return round_up(std::max<int64_t>(v, 1), 256); }

// Logits per workgroup: rows are divided until about 4 workgroups per CU run, into at least one step per wave.
int64_t logp_part(const LogpArgs& a) {
  const int64_t step = 64 * kRowVecs * (a.dt == kBF16 ? 8 : 4) * kLogpWaves;
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, a.rows));
  return std::max<int64_t>(1, ((a.V + want - 1) / want + step - 1) / step) * step;
}
int64_t logp_parts(const LogpArgs& a) {
  const int64_t part = logp_part(a);
  return (a.V + part - 1) / part;
}

int logp_check(int dt, int64_t rows, int64_t V, const char* who) {
  const std::string w = std::string(who) + ": ";
  TESM_REQUIRE(dt == kF32 || dt == kBF16, kErrInvalidArg, w + "dtype must be 0 or 1");
  TESM_REQUIRE(rows >= 0 && V >= 1 && rows < (1LL << 31) && V < (1LL << 30), kErrInvalidArg, w + "bad sizes");
  return kOk;
}

}  // namespace

int64_t logp_ws_bytes(const LogpArgs& a) {
  if (logp_check(a.dt, a.rows, a.V, "token log probs") != kOk || a.top < 0 || a.top > kLogpMaxTop) return -1;
  const int64_t parts = logp_parts(a);
  if (parts == 1) return 0;
  const int64_t all = a.rows * parts;
  return up256(all * std::min(a.top, a.V) * 8) + up256(all * static_cast<int64_t>(sizeof(LogpSum)));
}

int launch_token_logp(const LogpArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (int rc = logp_check(a.dt, a.rows, a.V, "token log probs")) return rc;
  TESM_REQUIRE(a.top >= 0 && a.top <= kLogpMaxTop && a.top <= a.V, kErrUnsupported,
               "token log probs: at most 64 alternatives, and no more than there are tokens");
  TESM_REQUIRE(a.ld >= a.V, kErrInvalidArg, "token log probs: ld < V");
  if (a.rows == 0) return kOk;
  TESM_REQUIRE(a.logits && a.targets && a.logp && a.entropy && (a.top == 0 || (a.top_logp && a.top_tokens)), kErrInvalidArg,
               "token log probs: need logits, targets and the outputs");
  const int64_t need = logp_ws_bytes(a);
  TESM_REQUIRE(need == 0 || (ws && ws_bytes >= need && aligned(ws, 8)), kErrWorkspace,
               "token log probs: workspace too small or not 8-byte aligned");
  const int parts = static_cast<int>(logp_parts(a)), part = static_cast<int>(logp_part(a)), m = static_cast<int>(a.top);
  TESM_REQUIRE(fits_grid(a.rows * parts, 64 * kLogpWaves), kErrUnsupported, "token log probs: too many rows for one call");
  uint64_t* keys = static_cast<uint64_t*>(ws);
  LogpSum* sums = reinterpret_cast<LogpSum*>(static_cast<char*>(ws) + up256(a.rows * parts * m * 8));
  const unsigned blocks = static_cast<unsigned>(a.rows * parts);
  constexpr int T = 64 * kLogpWaves;
#define TESM_LOGP(DT, LIST)                                                                                                     \
  do {                                                                                                                          \
    logp_row_kernel<DT, LIST><<<blocks, T, 0, TESM_LOGGED(st, logp_row_kernel<DT, LIST>)>>>(a, m, parts, part, keys, sums);     \
    if (parts > 1)                                                                                                              \
      logp_join_kernel<DT, LIST><<<static_cast<unsigned>(a.rows), LIST ? 512 : 64, 0, TESM_LOGGED(st, logp_join_kernel<DT, LIST>)>>>(        \
          a, m, parts, keys, sums);                                                                                             \
  } while (0)
  if (a.dt == kBF16) {
    if (m)
      TESM_LOGP(kBF16, true);
    else
      TESM_LOGP(kBF16, false);
  } else {
    if (m)
      TESM_LOGP(kF32, true);
    else
      TESM_LOGP(kF32, false);
  }
#undef TESM_LOGP
  return check_launch("token log probs");
}

int launch_token_logp_bwd(const LogpBwdArgs& a, hipStream_t st) {
  if (int rc = logp_check(a.dt, a.rows, a.V, "token log probs backward")) return rc;
  TESM_REQUIRE(a.ld >= a.V && a.ld_g >= a.V, kErrInvalidArg, "token log probs backward: ld < V");
  if (a.rows == 0) return kOk;
  TESM_REQUIRE(a.logits && a.targets && a.kept && a.grad_logits, kErrInvalidArg,
               "token log probs backward: need logits, targets, what the forward call kept and the output");
  const int64_t unit = 256 * 4 * (a.dt == kBF16 ? 8 : 4), many = (a.V + 4 * unit - 1) / (4 * unit);
  const int64_t part = round_up((a.V + many - 1) / many, unit), parts = (a.V + part - 1) / part;
  TESM_REQUIRE(fits_grid(a.rows * parts, 256), kErrUnsupported, "token log probs backward: too many rows for one call");
  const unsigned blocks = static_cast<unsigned>(a.rows * parts);
  const int p = static_cast<int>(parts);
#define TESM_LOGP_BWD(DT, ENT) logp_bwd_kernel<DT, ENT><<<blocks, 256, 0, TESM_LOGGED(st, logp_bwd_kernel<DT, ENT>)>>>(a, p, part)
  if (a.dt == kBF16) {
    if (a.grad_entropy)
      TESM_LOGP_BWD(kBF16, true);
    else
      TESM_LOGP_BWD(kBF16, false);
  } else {
    if (a.grad_entropy)
      TESM_LOGP_BWD(kF32, true);
    else
      TESM_LOGP_BWD(kF32, false);
  }
#undef TESM_LOGP_BWD
  return check_launch("token log probs backward");
}

int logp_status(unsigned* out, int clear) {
  unsigned v = 0;
  hipError_t e = hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_logp_status), sizeof(v), 0, hipMemcpyDeviceToHost);
  if (e == hipSuccess && clear && v != 0) {
    const unsigned zero = 0;
    e = hipMemcpyToSymbol(HIP_SYMBOL(g_logp_status), &zero, sizeof(zero), 0, hipMemcpyHostToDevice);
  }
  if (e != hipSuccess) return fail(kErrLaunch, std::string("device status: ") + hipGetErrorString(e));
  *out = v;
  return kOk;
}

}  // namespace tesm
