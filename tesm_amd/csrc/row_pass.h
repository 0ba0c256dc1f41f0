// Device helpers of the operators over rows of logits: the largest logits in order, and one pass over a part of a row.
#pragma once

#include <float.h>

#include <type_traits>

#include "tesm_hip_internal.h"

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
  float dot;       // (ENT) that sum's terms times their logarithms to base 2
};
constexpr int kRowVecs = 4;  // 16-byte vectors per lane and step
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
// With ENT it also forms the sum of the terms times their exponents (exponents below -150 belong to terms that are 0; a NaN or
// +infinite logit makes the sums NaN, here as in the first form).  Without LIST it keeps no list.
template <int DT, bool CLEAN, bool LIST = true, bool ENT = false>
__device__ __forceinline__ RowPart row_pass(const void* row, int lo, int hi, int n, uint64_t* buffer) {
  constexpr int EV = DT == kBF16 ? 8 : 4, ES = 16 / EV, STEP = 64 * EV * kRowVecs;
  const int lane = threadIdx.x & 63;
  const float inf = __builtin_inff();
  RowPart p{0, -inf, 0.0f, 0.0f};
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
  any16 raw[kRowVecs], ahead[kRowVecs];
  auto load = [&](int at, any16 (&to)[kRowVecs]) {
    const bool whole = at + STEP <= hi;
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
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
    for (int u = 0; u < kRowVecs; ++u) raw[u] = ahead[u];
    if (at + STEP < hi) load(at + STEP, ahead);  // under this step's arithmetic
    float vmax[kRowVecs], top = -inf;
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
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
    float ref, scale, dot = 0.0f;
    if constexpr (CLEAN) {
      ref = fmaxf(mx, -FLT_MAX);
      if constexpr (ENT) dot = (fmaxf(p.max, -FLT_MAX) - ref) * kLog2e;
      scale = p.max == mx ? 1.0f : __builtin_amdgcn_exp2f((fmaxf(p.max, -FLT_MAX) - ref) * kLog2e);
    } else {
      ref = fmaxf(mx, -kFar) * kLog2e;
      scale = __builtin_amdgcn_exp2f(fmaxf(p.max, -kFar) * kLog2e - ref);
      if constexpr (ENT) dot = fmaxf(p.max, -kFar) * kLog2e - ref;
    }
    float sum = p.sum * scale;
    if constexpr (ENT) dot = scale * __builtin_fmaf(fmaxf(dot, -1.0e5f), p.sum, p.dot);  // the earlier terms' exponents move too
#pragma unroll
    for (int u = 0; u < kRowVecs; ++u) {
      float v[EV];
      unpack_logits<DT>(raw[u], v);
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        if constexpr (ENT) {
          float t;
          if constexpr (CLEAN)
            t = (v[e] - ref) * kLog2e;
          else
            t = __builtin_fmaf(v[e], kLog2e, -ref);
          const float x = __builtin_amdgcn_exp2f(t);
          sum += x;
          dot = __builtin_fmaf(x, fmaxf(t, -150.0f), dot);
        } else if constexpr (CLEAN) {
          const float x = __builtin_amdgcn_exp2f((v[e] - ref) * kLog2e);
          sum += x == x ? x : v[e] == v[e] ? 1.0f : 0.0f;  // (infinity - infinity; a NaN logit)
        } else {
          sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], kLog2e, -ref));
        }
      }
    }
    p.max = mx;
    p.sum = sum;
    if constexpr (ENT) p.dot = dot;
    if constexpr (LIST) {
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
      for (int u = 0; u < kRowVecs; ++u) {
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
  }
  if constexpr (LIST) {
    if (held) flush();
  }
  return p;
}

// Whether a lane's sum of the first form does not hold its largest terms, and the part's sum (`top`: its largest logit) needs
// them: terms 200 below the largest are lost in it anyway (a lane that met masked logits alone).
__device__ __forceinline__ bool sum_is_off(const RowPart& p, float top) {
  if (p.max > kFar || !(p.sum == p.sum)) return true;
  return p.sum < 0.5f && p.max > -__builtin_inff() && p.max >= top - 200.0f;
}

}  // namespace

}  // namespace tesm
