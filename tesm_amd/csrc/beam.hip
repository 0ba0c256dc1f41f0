// Beam search.  A beam k of a request with score s_k and logits l_k offers every token v at
//   s_k + l_k[v] - logsumexp(l_k),
// and the n best of all beams' offers are chosen, equal ones in the order of k * V + v.  Offers that are not a number
// (a NaN logit, a row with an infinite one) and all offers of a beam without a finite score count as -infinity; a
// finished beam offers its padding token alone, at its own score.
//
// Inside a beam the order of the offers is the order of the logits, so each row is reduced to its n largest logits and
// its logsumexp in one pass (beam_row_kernel), and requests then merge their beams' lists, the offers compared in 64
// bits (beam_merge_kernel).  The floor is reading the logits once.  A wave issues 14 vector and 7 scalar instructions per
// logit (unpacking for the maximum, the sum and the test; the exponential, at a quarter of the rate; the list's upkeep);
// counters over 512 rows: the vector unit issues in 43 % of the cycles, a wave waits for memory or LDS in 47 % of its time and
// for an issue slot in 17 %, so that no one unit is the bound.  Measured, bfloat16, a quarter of the beams finished: 512 rows
// of 151936 logits (117 MB read) 46 us + 11 for the merge, 2.5 TB/s, whatever part of a row is masked; float32 (none finished,
// 311 MB) 72 us in all; 4 rows 8.5 + 6.3 us.
#include <float.h>

#include <type_traits>

#include "beam.h"

namespace tesm {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// A logit and its index as one number: the larger is the better, equal logits by the lower index.  0 is below all.
__device__ __forceinline__ uint64_t top_key(float v, int i) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 is 0)
  return static_cast<uint64_t>(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t b = static_cast<uint32_t>(k >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int key_index(uint64_t k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

// The value of the lane D away (D a power of 2), by the vector unit alone: a step of a sorting network waits for it, and by
// way of LDS it takes several times as long (4 rows of 151936 logits: 10.0 us against 8.5).
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  constexpr int kRowRor8 = 0x128, kQuadReverse = 0x1B;
  const int i = static_cast<int>(v);
  if constexpr (D == 1) return dpp_mov<kDppXor1>(i);
  if constexpr (D == 2) return dpp_mov<kDppXor2>(i);
  if constexpr (D == 4) return dpp_mov<kQuadReverse>(dpp_mov<kDppHalfMirror>(i));  // 7 away, then 3
  if constexpr (D == 8) return dpp_mov<kRowRor8>(i);
  if constexpr (D == 16) {  // (rows 0, 0, 2, 2 and 1, 1, 3, 3)
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  }
  if constexpr (D == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
// f(D) for D = FROM, FROM / 2 .. 1
template <int FROM, typename F>
__device__ __forceinline__ void each_distance(F&& f) {
  f(std::integral_constant<int, FROM>{});
  if constexpr (FROM > 1) each_distance<FROM / 2>(f);
}
// Steps of a bitonic network over the lanes: the larger of a lane and the one D away goes to the lower lane where `down`.
template <int FROM>
__device__ __forceinline__ uint64_t bitonic(uint64_t v, bool down) {
  each_distance<FROM>([&](auto d) __attribute__((always_inline)) {
    constexpr int D = decltype(d)::value;
    const uint64_t o = static_cast<uint64_t>(lane_xor<D>(static_cast<uint32_t>(v >> 32))) << 32 | lane_xor<D>(static_cast<uint32_t>(v));
    const bool low = (threadIdx.x & D) == 0;
    v = (v > o) == (low == down) ? v : o;
  });
  return v;
}
// The 64 best of a falling list (one per lane) and 64 more keys in any order, as a falling list.
__device__ __forceinline__ uint64_t merge64(uint64_t list, uint64_t more) {
  const int lane = threadIdx.x & 63;
  more = bitonic<1>(more, (lane & 2) != 0);  // `more` rising
  more = bitonic<2>(more, (lane & 4) != 0);
  more = bitonic<4>(more, (lane & 8) != 0);
  more = bitonic<8>(more, (lane & 16) != 0);
  more = bitonic<16>(more, (lane & 32) != 0);
  more = bitonic<32>(more, false);
  return bitonic<32>(list > more ? list : more, true);
}
// The same for two falling lists.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, uint64_t b) {
  const int r = 63 - (threadIdx.x & 63);
  const uint32_t lo = __shfl(static_cast<int>(b), r), hi = __shfl(static_cast<int>(b >> 32), r);
  const uint64_t o = static_cast<uint64_t>(hi) << 32 | lo;
  return bitonic<32>(a > o ? a : o, true);
}
// The values in falling order.
__device__ __forceinline__ float sorted(float v) {
  const int lane = threadIdx.x & 63;
  auto steps = [&](auto from, bool down) __attribute__((always_inline)) {
    each_distance<decltype(from)::value>([&](auto d) __attribute__((always_inline)) {
      constexpr int D = decltype(d)::value;
      const float o = __uint_as_float(lane_xor<D>(__float_as_uint(v)));
      v = ((lane & D) == 0) == down ? fmaxf(v, o) : fminf(v, o);
    });
  };
  steps(std::integral_constant<int, 1>{}, (lane & 2) == 0);
  steps(std::integral_constant<int, 2>{}, (lane & 4) == 0);
  steps(std::integral_constant<int, 4>{}, (lane & 8) == 0);
  steps(std::integral_constant<int, 8>{}, (lane & 16) == 0);
  steps(std::integral_constant<int, 16>{}, (lane & 32) == 0);
  steps(std::integral_constant<int, 32>{}, true);
  return v;
}
__device__ __forceinline__ uint64_t readlane_u64(uint64_t v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(2)));

template <int DT>
__device__ __forceinline__ void unpack_logits(const any16& u, float (&v)[DT == kBF16 ? 8 : 4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == kBF16) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    } else {
      v[i] = __uint_as_float(u[i]);
    }
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// What a wave knows of its part of a row.
struct RowPart {
  uint64_t list;   // falling, one key per lane
  float max, sum;  // per lane: the largest logit, and the sum of exp(logit - max)
};
struct PartSum {
  double ref, sum;  // the sum of exp(logit) is sum * exp(ref)
};
__device__ __forceinline__ PartSum add(const PartSum& a, const PartSum& b) {
  const double ref = fmax(a.ref, b.ref);  // (equal references may be infinite)
  return {ref, (a.ref == ref ? a.sum : a.sum * exp(a.ref - ref)) + (b.ref == ref ? b.sum : b.sum * exp(b.ref - ref))};
}

constexpr int kBeamWaves = 4, kBeamVecs = 4;  // waves per workgroup, 16-byte vectors per lane and step
constexpr float kFar = 1.0e6f;

// One pass over logits [lo, hi) of a row by one wave.  A lane keeps its running maximum and sum.  A logit that may belong
// to the n best (not below the last of the list) is put into a buffer in LDS; from 64 on it is sorted and merged into the
// list.  The n-th largest of the lanes' own maxima is not above the n-th largest logit so far: taken as the bound after
// the first step and whenever the steps have doubled, it lets few logits through.
// The sum's terms are 2^(logit L - ref) with L = log2 e and ref = L times the maximum, rounded: one fused operation and the
// exponential.  The largest logit's own term is then 2^d, d the rounding of ref: within a sixteenth of 0 for maxima up to
// kFar either way, but up to 64 at 1e9.  A lane whose maximum is below -kFar takes ref from -kFar, and its terms may all be
// 0; sum_is_off tells where that matters.  There, and where a logit is NaN or the maximum above kFar, the pass is made again
// with CLEAN: terms 2^((logit - max) L), a NaN counts as -infinity.
template <int DT, bool CLEAN>
__device__ __forceinline__ RowPart row_pass(const void* row, int lo, int hi, int n, uint64_t* buffer) {
  constexpr int EV = DT == kBF16 ? 8 : 4, ES = 16 / EV, STEP = 64 * EV * kBeamVecs;
  const int lane = threadIdx.x & 63;
  const float inf = __builtin_inff();
  RowPart p{0, -inf, 0.0f};
  float bound = -inf;          // a logit below is not among the n best
  int bound_index = INT32_MAX;  // one equal to it is, up to this index
  int held = 0, step = 0;
  auto flush = [&]() {
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int c = 0; c < held; c += 64) p.list = merge64(p.list, c + lane < held ? buffer[c + lane] : 0);
    __builtin_amdgcn_wave_barrier();
    held = 0;
    const uint64_t last = readlane_u64(p.list, n - 1);
    if (last) {
      bound = key_value(last);
      bound_index = key_index(last);
    }
  };
  any16 raw[kBeamVecs], ahead[kBeamVecs];
  auto load = [&](int at, any16 (&to)[kBeamVecs]) {
    const bool whole = at + STEP <= hi;
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) {
      const int i = at + (u * 64 + lane) * EV;
      const char* q = static_cast<const char*>(row) + static_cast<int64_t>(i) * ES;
      if (whole || i + EV <= hi) {
        to[u] = *reinterpret_cast<const any16*>(q);
      } else {  // the last ones: -infinity behind the end, which no test below takes for a logit
        to[u] = DT == kBF16 ? any16{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}
                            : any16{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
#pragma unroll
        for (int e = 0; e < EV; ++e)
          if (i + e < hi) {
            if constexpr (DT == kBF16) {
              const uint32_t b = reinterpret_cast<const uint16_t*>(q)[e];
              to[u][e / 2] = e % 2 ? (to[u][e / 2] & 0xffffu) | b << 16 : (to[u][e / 2] & 0xffff0000u) | b;
            } else {
              to[u][e] = reinterpret_cast<const uint32_t*>(q)[e];
            }
          }
      }
    }
  };
  if (lo < hi) load(lo, ahead);
  for (int at = lo; at < hi; at += STEP) {
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) raw[u] = ahead[u];
    if (at + STEP < hi) load(at + STEP, ahead);  // under this step's arithmetic
    float vmax[kBeamVecs], top = -inf;
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) {
      float v[EV];
      unpack_logits<DT>(raw[u], v);
      if constexpr (CLEAN) {
        vmax[u] = -inf;
#pragma unroll
        for (int e = 0; e < EV; ++e) vmax[u] = fmaxf(vmax[u], v[e]);
        top = fmaxf(top, vmax[u]);
      } else {  // (the library's fmaxf first quiets each operand; a NaN voids this pass anyway)
        vmax[u] = max3(v[0], v[1], max3(v[2], v[3], v[3]));
        if constexpr (EV == 8) vmax[u] = max3(vmax[u], v[4], max3(v[5], v[6], v[7]));
        top = max3(top, vmax[u], vmax[u]);
      }
    }
    const float mx = fmaxf(p.max, top);
    float ref, scale;
    if constexpr (CLEAN) {
      ref = fmaxf(mx, -FLT_MAX);
      scale = p.max == mx ? 1.0f : __builtin_amdgcn_exp2f((fmaxf(p.max, -FLT_MAX) - ref) * kLog2e);
    } else {
      ref = fmaxf(mx, -kFar) * kLog2e;
      scale = __builtin_amdgcn_exp2f(fmaxf(p.max, -kFar) * kLog2e - ref);
    }
    float sum = p.sum * scale;
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) {
      float v[EV];
      unpack_logits<DT>(raw[u], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        if constexpr (CLEAN) {
          const float x = __builtin_amdgcn_exp2f((v[e] - ref) * kLog2e);
          sum += x == x ? x : v[e] == v[e] ? 1.0f : 0.0f;  // (infinity - infinity; a NaN logit)
        } else {
          sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], kLog2e, -ref));
        }
      }
    }
    p.max = mx;
    p.sum = sum;
    if ((step & (step + 1)) == 0) {  // after 1, 2, 4, 8 .. steps
      float s = sorted(mx == mx ? mx : -inf);
      s = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s), n - 1));
      if (s > bound) {
        bound = s;
        bound_index = INT32_MAX;
      }
    }
    ++step;
#pragma unroll
    for (int u = 0; u < kBeamVecs; ++u) {
      if (!__any(vmax[u] >= bound)) continue;
      float v[EV];
      unpack_logits<DT>(raw[u], v);
      const int i = at + (u * 64 + lane) * EV;
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        float x = v[e];
        if (CLEAN && !(x == x)) x = -inf;
        const bool take = x >= bound && (x > bound || i + e <= bound_index) && i + e < hi;
        const uint64_t who = __ballot(take);
        const int place = held + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(who >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(who), 0));
        if (take) buffer[place] = top_key(x, i + e);  // (below 64 + 64 EV)
        held += __popcll(who);
      }
      if (held >= 64) flush();
    }
  }
  if (held) flush();
  return p;
}

// Whether a lane's sum of the first form does not hold its largest terms, and the part's sum (`top`: its largest logit) needs
// them: terms 200 below the largest are lost in it anyway (a lane that met masked logits alone).
__device__ __forceinline__ bool sum_is_off(const RowPart& p, float top) {
  if (p.max > kFar || !(p.sum == p.sum)) return true;
  return p.sum < 0.5f && p.max > -__builtin_inff() && p.max >= top - 200.0f;
}

// Part blockIdx.x of row blockIdx.y, a quarter of it per wave: its m best keys and its sum.
template <int DT>
__global__ __launch_bounds__(64 * kBeamWaves) void beam_row_kernel(BeamArgs a, int m, int part, uint64_t* keys, PartSum* sums) {
  __shared__ uint64_t buffer[kBeamWaves][64 + 64 * (DT == kBF16 ? 8 : 4)];
  __shared__ PartSum ps[kBeamWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.y;
  // (offers that do not depend on the logits)
  if ((a.finished && a.finished[r]) || !(fabsf(a.scores[r]) < __builtin_inff())) return;
  const char* row = static_cast<const char*>(a.logits) + r * a.ld * (DT == kBF16 ? 2 : 4);
  const int each = part / kBeamWaves, V = static_cast<int>(a.V);
  const int lo = min(static_cast<int>(blockIdx.x) * part + wave * each, V), hi = min(lo + each, V);
  RowPart p = row_pass<DT, false>(row, lo, hi, m, buffer[wave]);
  float mx = wave_max<64>(p.max);
  const bool again = __any(sum_is_off(p, mx));
  if (again) {
    p = row_pass<DT, true>(row, lo, hi, m, buffer[wave]);
    mx = wave_max<64>(p.max);
  }
  // over the lanes, then the waves
  const float top = fmaxf(mx, again ? -FLT_MAX : -kFar), own = fmaxf(p.max, again ? -FLT_MAX : -kFar);
  const float scale = p.max == mx ? 1.0f : __builtin_amdgcn_exp2f(again ? (own - top) * kLog2e : own * kLog2e - top * kLog2e);
  const float s = wave_sum_f<64>(p.sum * scale);
  // The first form's terms are exp(logit - top) times 2^(top L - r) in the float L, r the rounded product: in 64 bits the
  // product of two floats is exact, and what the sum has too much is taken off its reference (r ln 2 would be off by 1.3e-8
  // top, L's own error).  A part of -infinities alone keeps such a reference.
  const double t = top, over = t * static_cast<double>(kLog2e) - static_cast<double>(top * kLog2e);
  const double ref = again || mx == -__builtin_inff() ? static_cast<double>(mx) : t - 0.69314718055994530942 * over;
  if (lane == 0) ps[wave] = {ref, s};
  buffer[wave][lane] = p.list;
  __syncthreads();
  if (wave) return;
  for (int w = 1; w < kBeamWaves; ++w) p.list = merge_lists(p.list, buffer[w][lane]);
  const int64_t at = r * gridDim.x + blockIdx.x;
  if (lane < m) keys[at * m + lane] = p.list;
  if (lane == 0) {
    PartSum o = ps[0];
    for (int w = 1; w < kBeamWaves; ++w) o = add(o, ps[w]);
    sums[at] = o;
  }
}

// Larger first, equal ones by index.
__device__ __forceinline__ bool before(double v, int64_t i, double w, int64_t j) { return v > w || (v == w && i < j); }

struct Offer {
  double value;
  int64_t flat;  // k * V + v
};

// One workgroup per request: a wave per beam merges its parts' lists into the beam's m best offers; the offers' ranks
// among all beams' are then counted.  Bound by latency: the chains of sorting steps and of the 64-bit exponentials and
// logarithm, 6 to 12 us; all that a beam needs is read at once (4 beams 6.2 us against 6.8).  The ranking compares all offers
// with all: 64 beams and 64 candidates take 2.9 ms.
__global__ __launch_bounds__(512) void beam_merge_kernel(BeamArgs a, int m, int parts, const uint64_t* keys, const PartSum* sums) {
  extern __shared__ __attribute__((aligned(16))) char lds_beam[];
  Offer* const offers = reinterpret_cast<Offer*>(lds_beam);
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int K = static_cast<int>(a.K), n = static_cast<int>(a.n), count = K * m;
  const double inf = __builtin_inf();
  for (int k = wave; k < K; k += 8) {
    const int64_t r = b * K + k;
    const uint64_t* const kr = keys + r * parts * m;
    const PartSum* const sr = sums + r * parts;
    // (under way together, also where they turn out not to be wanted)
    const float score = a.scores[r];
    const uint8_t fin = a.finished ? a.finished[r] : 0;
    const uint64_t first = lane < parts * m ? kr[lane] : 0, second = lane + 64 < parts * m ? kr[lane + 64] : 0;
    const PartSum own = lane < parts ? sr[lane] : PartSum{-inf, 0.0};
    const bool live = fabsf(score) < __builtin_inff(), done = fin != 0;
    double value = -inf;
    int64_t token = lane;
    if (live && done) {
      token = lane == 0 ? a.pad : (lane <= a.pad ? lane - 1 : lane);
      if (lane == 0) value = score;
    } else if (live) {
      uint64_t list = 0, next = first;
#pragma unroll 1
      for (int c = 0; c < parts * m; c += 64) {
        list = merge64(list, next);
        next = c == 0 ? second : c + 64 + lane < parts * m ? kr[c + 64 + lane] : 0;
      }
      double ref = own.ref, s = 0.0;
      for (int c = lane + 64; c < parts; c += 64) ref = fmax(ref, sr[c].ref);
      for (int d = 32; d > 0; d >>= 1) ref = fmax(ref, __shfl_xor(ref, d));
      if (lane < parts) s = own.ref == ref ? own.sum : own.sum * exp(own.ref - ref);
      for (int c = lane + 64; c < parts; c += 64) s += sr[c].ref == ref ? sr[c].sum : sr[c].sum * exp(sr[c].ref - ref);
      s = wave_sum_d<64>(s);
      const double lse = ref + log(s);
      if (fabs(lse) < inf) {
        value = static_cast<double>(score) + (static_cast<double>(key_value(list)) - lse);
        token = key_index(list);
      }
    }
    if (lane < m) offers[k * m + lane] = {value, k * a.V + token};
  }
  __syncthreads();
  for (int c = tid; c < count; c += 512) {
    const Offer o = offers[c];
    int rank = 0;
    if (c % m >= n) continue;
#pragma unroll 8
    for (int j = 0; j < count; ++j) {
      const Offer q = offers[j];
      rank += before(q.value, q.flat, o.value, o.flat);
    }
    if (rank >= n) continue;
    const int64_t k = c / m, token = o.flat - k * a.V;
    a.out_scores[b * n + rank] = static_cast<float>(o.value);
    a.parents[b * n + rank] = k;
    a.tokens[b * n + rank] = token;
    if (a.finished_out)
      a.finished_out[b * n + rank] = (a.finished && a.finished[b * K + k]) || (a.eos >= 0 && token == a.eos);
  }
}

// ---------------------------------------------------------------------------
// Reordering: row b * K + k of every tensor becomes the old row b * K + parents[b][k], in place.
// ---------------------------------------------------------------------------
__device__ unsigned g_reorder_status;

struct ReorderTable {
  int count;
  struct Entry {
    char* p;
    int64_t pitch, bytes;
    int unit;         // bytes moved at once: 16, 4 or 1
    unsigned block0;  // first workgroup
  } t[kReorderTensors];
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A thread moves one unit of all K rows of a request: every load before the first store, so a row may be the parent
// of several others and be overwritten itself.  Rows that stay are neither read nor written: in their place one that is
// read anyway is read again (a branch per row around the loads would keep them from being under way together).  Bound by
// HBM where the rows are long: 16 requests of 8 beams, 655 MB if all rows moved, 104 us; a layer stack's small caches 4.3 us.
template <typename U, int KM>
__device__ __forceinline__ void reorder_unit(char* at, int64_t pitch, const int (&from)[KM], uint64_t moves) {
  U v[KM];
#pragma clang loop unroll(full)
  for (int k = 0; k < KM; ++k) v[k] = *reinterpret_cast<const U*>(at + from[k] * pitch);
#pragma clang loop unroll(full)
  for (int k = 0; k < KM; ++k)
    if (moves >> k & 1) *reinterpret_cast<U*>(at + k * pitch) = v[k];
}

template <int KM>
__global__ __launch_bounds__(256) void reorder_rows_kernel(ReorderTable tab, const int64_t* __restrict__ parents, int K) {
  const int64_t b = blockIdx.y;
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].block0 <= blockIdx.x)
      lo = mid;
    else
      hi = mid;
  }
  const ReorderTable::Entry& e = tab.t[lo];
  // the rows' sources, uniform over the workgroup
  int from[KM], any = 0;
  uint64_t moves = 0;
  bool bad = false;
#pragma clang loop unroll(full)
  for (int k = 0; k < KM; ++k) {
    from[k] = k;
    if (k < K) {
      const int64_t p = parents[b * K + k];
      if (p < 0 || p >= K)
        bad = true;
      else
        from[k] = __builtin_amdgcn_readfirstlane(static_cast<int>(p));
    }
    if (from[k] != k) moves |= 1ull << k, any = from[k];
  }
  if (bad && blockIdx.x == 0 && threadIdx.x == 0)
    __hip_atomic_fetch_or(&g_reorder_status, 2u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const int64_t off = (static_cast<int64_t>(blockIdx.x - e.block0) * 256 + threadIdx.x) * e.unit;
  if (moves == 0 || off >= e.bytes) return;
#pragma clang loop unroll(full)
  for (int k = 0; k < KM; ++k)
    if (!(moves >> k & 1)) from[k] = any;
  char* at = e.p + b * K * e.pitch + off;
  if (e.unit == 16)
    reorder_unit<u32x4, KM>(at, e.pitch, from, moves);
  else if (e.unit == 4)
    reorder_unit<uint32_t, KM>(at, e.pitch, from, moves);
  else
    reorder_unit<uint8_t, KM>(at, e.pitch, from, moves);
}

int64_t round256(int64_t v) { return round_up(std::max<int64_t>(v, 1), 256); }

// Logits per workgroup: rows are divided until about 4 workgroups per CU run, into at least one step per wave.  More of
// them sort and merge more often, fewer leave loads uncovered: 512 rows of 151936 logits in 512, 1024, 2048 and 4096
// workgroups 51, 46, 50 and 54 us.
int64_t beam_part(const BeamArgs& a) {
  const int64_t step = 64 * kBeamVecs * (a.dt == kBF16 ? 8 : 4) * kBeamWaves;
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, a.B * a.K));
  return std::max<int64_t>(1, ((a.V + want - 1) / want + step - 1) / step) * step;
}
int64_t beam_parts(const BeamArgs& a) {
  const int64_t part = beam_part(a);
  return (a.V + part - 1) / part;
}

int beam_check(const BeamArgs& a) {
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, "beam select: dtype must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.K >= 1 && a.V >= 1 && a.n >= 1 && a.B < (1LL << 24) && a.V < (1LL << 30),
               kErrInvalidArg, "beam select: bad sizes");
  TESM_REQUIRE(a.K <= kBeamMaxN && a.n <= kBeamMaxN, kErrUnsupported,
               "beam select: at most 64 beams and 64 chosen candidates");
  TESM_REQUIRE(a.n <= a.K * a.V, kErrInvalidArg, "beam select: more candidates asked for than there are");
  return kOk;
}

}  // namespace

int64_t beam_select_ws_bytes(const BeamArgs& a) {
  if (beam_check(a) != kOk) return -1;
  const int64_t all = a.B * a.K * beam_parts(a), m = std::min(a.n, a.V);
  return round256(all * m * 8) + round256(all * static_cast<int64_t>(sizeof(PartSum)));
}

int launch_beam_select(const BeamArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (int rc = beam_check(a)) return rc;
  TESM_REQUIRE(a.ld >= a.V, kErrInvalidArg, "beam select: ld < V");
  TESM_REQUIRE(!a.finished || (a.pad >= 0 && a.pad < a.V), kErrInvalidArg, "beam select: pad outside the vocabulary");
  TESM_REQUIRE(a.eos < a.V, kErrInvalidArg, "beam select: eos outside the vocabulary");
  if (a.B == 0) return kOk;
  TESM_REQUIRE(a.logits && a.scores && a.out_scores && a.parents && a.tokens, kErrInvalidArg,
               "beam select: need logits, scores and the three outputs");
  TESM_REQUIRE(a.B * a.K < 65536, kErrUnsupported, "beam select: too many beams for one call");
  TESM_REQUIRE(ws && ws_bytes >= beam_select_ws_bytes(a) && aligned(ws, 8), kErrWorkspace,
               "beam select: workspace too small or not 8-byte aligned");
  const int m = static_cast<int>(std::min(a.n, a.V)), parts = static_cast<int>(beam_parts(a));
  const int part = static_cast<int>(beam_part(a));
  const int64_t rows = a.B * a.K;
  uint64_t* keys = static_cast<uint64_t*>(ws);
  PartSum* sums = reinterpret_cast<PartSum*>(static_cast<char*>(ws) + round256(rows * parts * m * 8));
  const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(rows));
  constexpr int T = 64 * kBeamWaves;
  if (a.dt == kBF16)
    beam_row_kernel<kBF16><<<grid, T, 0, TESM_LOGGED(st, beam_row_kernel<kBF16>)>>>(a, m, part, keys, sums);
  else
    beam_row_kernel<kF32><<<grid, T, 0, TESM_LOGGED(st, beam_row_kernel<kF32>)>>>(a, m, part, keys, sums);
  const unsigned lds = static_cast<unsigned>(a.K * m * static_cast<int64_t>(sizeof(Offer)));
  beam_merge_kernel<<<static_cast<unsigned>(a.B), 512, lds, TESM_LOGGED(st, beam_merge_kernel)>>>(a, m, parts, keys, sums);
  return check_launch("beam select");
}

int launch_reorder_rows(const ReorderRows* t, int64_t count, const int64_t* parents, int64_t B, int64_t K,
                        hipStream_t st) {
  TESM_REQUIRE(count >= 0 && B >= 0 && K >= 1 && B < 65536, kErrInvalidArg, "reorder rows: bad sizes");
  TESM_REQUIRE(K <= kBeamMaxN, kErrUnsupported, "reorder rows: at most 64 beams");
  TESM_REQUIRE(count == 0 || B == 0 || (t && parents), kErrInvalidArg, "reorder rows: need the tensors and parents");
  for (int64_t i = 0; i < count; ++i)
    TESM_REQUIRE(t[i].bytes >= 0 && t[i].bytes < (1LL << 36) && (B * K <= 1 || t[i].pitch >= t[i].bytes) &&
                     (t[i].p || t[i].bytes == 0),
                 kErrInvalidArg, "reorder rows: a tensor has no memory or a pitch shorter than its row");
  if (B == 0) return kOk;
  for (int64_t i0 = 0; i0 < count; i0 += kReorderTensors) {
    ReorderTable tab;
    tab.count = 0;
    int64_t blocks = 0;
    for (int64_t i = i0; i < std::min<int64_t>(count, i0 + kReorderTensors); ++i) {
      if (t[i].bytes == 0) continue;
      ReorderTable::Entry& e = tab.t[tab.count++];
      e.p = static_cast<char*>(t[i].p);
      e.pitch = t[i].pitch;
      e.bytes = t[i].bytes;
      e.unit = 1;
      for (int u : {4, 16})
        if (aligned(e.p, u) && e.pitch % u == 0 && e.bytes % u == 0) e.unit = u;
      e.block0 = static_cast<unsigned>(blocks);
      blocks += (e.bytes + 256 * e.unit - 1) / (256 * e.unit);
      TESM_REQUIRE(blocks < (1LL << 31), kErrUnsupported, "reorder rows: rows too long");
    }
    if (tab.count == 0) continue;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(B));
    const int k = static_cast<int>(K);
#define TESM_REORDER(KM) \
  reorder_rows_kernel<KM><<<grid, 256, 0, TESM_LOGGED(st, reorder_rows_kernel<KM>)>>>(tab, parents, k)
    if (K <= 4)
      TESM_REORDER(4);
    else if (K <= 8)
      TESM_REORDER(8);
    else if (K <= 16)
      TESM_REORDER(16);
    else if (K <= 32)
      TESM_REORDER(32);
    else
      TESM_REORDER(64);
#undef TESM_REORDER
  }
  return check_launch("reorder rows");
}

int reorder_status(unsigned* out, int clear) {
  unsigned v = 0;
  hipError_t e = hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_reorder_status), sizeof(v), 0, hipMemcpyDeviceToHost);
  if (e == hipSuccess && clear && v != 0) {
    const unsigned zero = 0;
    e = hipMemcpyToSymbol(HIP_SYMBOL(g_reorder_status), &zero, sizeof(zero), 0, hipMemcpyHostToDevice);
  }
  if (e != hipSuccess) return fail(kErrLaunch, std::string("device status: ") + hipGetErrorString(e));
  *out = v;
  return kOk;
}

}  // namespace tesm
