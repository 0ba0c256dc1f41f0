// Gated linear recurrence over rows t, per channel:
//   a_t = sigmoid(decay_t + bias),  u_t = sigmoid(write_t) tanh(value_t),  h_t = a_t h_{t-1} + u_t
// and its backward pass, with g_t the gradient of h_t by every way and c_t = a_t g_t what it hands to the row before:
//   g_t = dh_t + c_{t+1}  (the last row: + the final state's gradient),
//   d decay_t = g_t h_{t-1} a_t (1 - a_t), d write_t = g_t u_t (1 - sigmoid(write_t)),
//   d value_t = g_t sigmoid(write_t) (1 - tanh^2), d h_0 = c_1.
// Both are first-order recurrences x <- A x + U, and runs of them compose: (A, U) then (A', U') is (A' A, A' U + U').
//
// One pass over the data.  A tile is 128 rows of one sequence by 64 or 128 channels; each of 8 waves takes 16 rows, a lane one or
// two channels; inputs are read once and stay in registers as gates.  Waves scan their rows from zero, their (A, U) meet in
// LDS, and tiles of one sequence and channel group hand on their state in a chain: a tile publishes its (A, U); from these
// and the state in front of its group of 16 tiles every tile forms its own carry, always in the same order, so results
// repeat bit for bit; the last tile of a group publishes the state behind it.  Tiles are taken by ticket, predecessors first, so that
// whatever a tile waits for is already running.  The forward pass can keep every tile's carry (1/128 of a float32 copy of the
// states); the backward pass then forms the states again in registers and walks the chain from the end.
//
// Published values and flags go by agent-scope atomic accesses (coherent over the XCDs' caches); a wave waits for its
// value stores before it sets its flag.  A poll gives up after kSpinLimit rounds: the states are then NaN and bit 0 of the
// status word is set.
#include "recur.h"

namespace tesm {

namespace {

constexpr int kWaves = 8, kRows = 16, kTile = kWaves * kRows, kGroup = 16;
static_assert(kTile == kRecurRows && kGroup == 2 * kWaves, "a wave composes two earlier tiles");
constexpr int kSpinLimit = 1 << 20;
constexpr float kLog2e = 1.44269504088896340736f;

__device__ unsigned g_recur_status;
int g_spin_limit = kSpinLimit;

// ---------------------------------------------------------------------------
// gates
// ---------------------------------------------------------------------------
// The exponent's rounding moves a sigmoid by at most 0.23 * 2^-24, so it needs no second part.  Infinite arguments give the limits,
// NaN stays NaN.
struct Sig {
  float p, q;  // sigmoid(x), sigmoid(-x), each to a few ulp of itself
};
__device__ __forceinline__ float sig(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -kLog2e)); }
__device__ __forceinline__ Sig sig2(float x) {
  const float e = __builtin_amdgcn_exp2f(x * -kLog2e), p = __builtin_amdgcn_rcpf(1.0f + e);
  return {p, p < 0.5f ? 1.0f - p : e * p};
}
struct Tanh {
  float t, d;  // tanh(x), 1 - tanh^2(x)
};
// With r = 1 / (e^{2|x|} + 1) in (0, 1/2]: tanh = 1 - 2 r, derivative 4 r (1 - r).  The difference loses the bits of small
// values, which take the odd series instead: below 1/4 to x^9 for float32 (2^-27 off), below 1/32 to x^3 where the
// operands are bfloat16 (relative 2^-17 from the difference, 2^-22 from the series).
template <int DT>
__device__ __forceinline__ Tanh tanh2(float x) {
  const float r = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(fabsf(x) * (2.0f * kLog2e)) + 1.0f);
  const float big = __builtin_copysignf(__builtin_fmaf(r, -2.0f, 1.0f), x);
  const float x2 = x * x;
  float p;
  if constexpr (DT == kF32) {
    p = __builtin_fmaf(x2, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = __builtin_fmaf(x2, p, 2.0f / 15.0f);
    p = __builtin_fmaf(x2, p, -1.0f / 3.0f);
  } else {
    p = -1.0f / 3.0f;
  }
  const float small = __builtin_fmaf(x * x2, p, x);
  return {fabsf(x) < (DT == kF32 ? 0.25f : 0.03125f) ? small : big, 4.0f * r * (1.0f - r)};
}

// ---------------------------------------------------------------------------
// a lane's channels of a row
// ---------------------------------------------------------------------------
template <int DT, int CPT>
struct Row {
  uint32_t w;  // one float32, one bfloat16 or two
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (CPT == 2)
      w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p) + i);
    else
      w = ld_bits<DT>(p, i);
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (CPT == 2) return __uint_as_float(j ? w & 0xffff0000u : w << 16);
    return from_bits<DT>(w);
  }
  static __device__ __forceinline__ void store(void* p, int64_t i, const float (&v)[CPT]) {
    if constexpr (CPT == 2)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p) + i) = pack_bf16x2(v[0], v[1]);
    else
      st<DT>(p, i, v[0]);
  }
};

// ---------------------------------------------------------------------------
// the chain of a sequence's tiles
// ---------------------------------------------------------------------------
struct Chain {
  int* flags = nullptr;     // (G, slots)
  unsigned* tickets = nullptr;  // a 256-byte line per channel group
  unsigned long long* values = nullptr;  // (G, slots, 64 CPT): (A, U) of a tile, or the state behind a group's last one
  const int32_t* starts = nullptr;   // packed: S + 1 starts, inside the rows and not decreasing
  int64_t slots = 0;
  int G = 0, tiles = 0;  // channel groups; tiles per sequence of a dense batch
  int spin_limit = 0;
};
constexpr int kTicketStride = 64;

struct Place {
  int64_t row0, len, seq, slot0;  // the sequence's first row and length, its number and first slot
  int tile, tiles;
  bool any;
};

// The tile of slot `at` in walking order; `back`: from the end.
__device__ __forceinline__ Place place_of(const RecurArgs& a, const Chain& c, int64_t at, bool back) {
  Place p;
  if (!c.starts) {
    p.seq = at % a.B;
    const int pos = static_cast<int>(at / a.B);
    p.tile = back ? c.tiles - 1 - pos : pos;
    p.tiles = c.tiles;
    p.row0 = p.seq * a.L;
    p.len = a.L;
    p.slot0 = p.seq * c.tiles;
    p.any = true;
    return p;
  }
  const int64_t slot = back ? c.slots - 1 - at : at;
  // sequence s has the slots from start / kTile + s on, at least one
  int64_t lo = 0, hi = a.S;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (c.starts[mid] / kTile + mid <= slot)
      lo = mid;
    else
      hi = mid;
  }
  p.seq = lo;
  p.row0 = c.starts[lo];
  p.len = c.starts[lo + 1] - p.row0;
  p.slot0 = p.row0 / kTile + lo;
  p.tile = static_cast<int>(slot - p.slot0);
  p.tiles = static_cast<int>((p.len + kTile - 1) / kTile);
  if (p.tiles < 1) p.tiles = 1;  // (an empty sequence hands its state through)
  p.any = p.tile >= 0 && p.tile < p.tiles;
  return p;
}

__device__ __forceinline__ unsigned long long pack2(float a, float u) {
  return static_cast<unsigned long long>(__float_as_uint(u)) << 32 | __float_as_uint(a);
}
__device__ __forceinline__ float2 unpack2(unsigned long long v) {
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

template <int CPT>
struct ChainTile {
  float2 part[kWaves][64 * CPT];   // the waves' rows
  float2 before[kWaves][64 * CPT];  // the tiles in front, two per wave
  float base[64 * CPT];             // the state in front of the group
  int bad;
  unsigned ticket;
};

// Publishes a wave's values for slot `s`: the values first, then the flag.
template <int CPT>
__device__ __forceinline__ void publish(const Chain& c, int64_t s, int lane, const float2 (&v)[CPT]) {
#pragma unroll
  for (int j = 0; j < CPT; ++j)
    __hip_atomic_store(c.values + (s * 64 + lane) * CPT + j, pack2(v[j].x, v[j].y), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (lane == 0) __hip_atomic_store(c.flags + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Waits for the flags of slots s and (with `two`) s2; whether they came.
__device__ __forceinline__ bool await(const Chain& c, int64_t s, int64_t s2, bool two) {
  bool ok = false;
  for (int i = 0; i <= c.spin_limit && !ok; ++i) {
    int f = __hip_atomic_load(c.flags + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (two) f &= __hip_atomic_load(c.flags + s2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    ok = __builtin_amdgcn_readfirstlane(f) != 0;
    if (!ok) __builtin_amdgcn_s_sleep(1);
  }
  asm volatile("" ::: "memory");
  return ok;
}

// The state entering the wave's rows.  part: the wave's (A, U).  In walking order: pos of the tile, order of the wave; slot(p):
// the slot of position p; first: the sequence's own first state.  `entry` returns the tile's carry, `leave` the state behind the
// tile (of use to the last wave in order).
template <int CPT, typename Slot, typename First>
__device__ __forceinline__ void chain_carry(const Chain& c, ChainTile<CPT>& sh, int lane, int order, int pos, int count,
                                            const float2 (&part)[CPT], Slot&& slot, First&& first, float (&carry)[CPT],
                                            float (&entry)[CPT], float (&leave)[CPT]) {
#pragma unroll
  for (int j = 0; j < CPT; ++j) sh.part[order][lane * CPT + j] = part[j];
  if (order == 0 && lane == 0) sh.bad = 0;
  __syncthreads();
  const int g0 = pos & ~(kGroup - 1);
  const bool last_of_group = (pos & (kGroup - 1)) == kGroup - 1, more = pos + 1 < count;
  float2 all[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    all[j] = make_float2(1.0f, 0.0f);
    for (int w = 0; w < kWaves; ++w) {
      const float2 q = sh.part[w][lane * CPT + j];
      all[j] = make_float2(q.x * all[j].x, __builtin_fmaf(q.x, all[j].y, q.y));
    }
  }
  if (order == 0 && more && !last_of_group) publish<CPT>(c, slot(pos), lane, all);
  // two tiles in front of this one, in order
  const int p0 = g0 + 2 * order;
  bool ok = true;
  float2 b[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) b[j] = make_float2(1.0f, 0.0f);
  if (p0 < pos) {
    const bool two = p0 + 1 < pos;
    const int64_t s0 = slot(p0), s1 = slot(two ? p0 + 1 : p0);
    ok = await(c, s0, s1, two);
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const float2 x = unpack2(__hip_atomic_load(c.values + (s0 * 64 + lane) * CPT + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      const float2 y = unpack2(__hip_atomic_load(c.values + (s1 * 64 + lane) * CPT + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      b[j] = two ? make_float2(y.x * x.x, __builtin_fmaf(y.x, x.y, y.y)) : x;
    }
  }
#pragma unroll
  for (int j = 0; j < CPT; ++j) sh.before[order][lane * CPT + j] = b[j];
  if (order == kWaves - 1) {  // (it has the fewest tiles to wait for)
    if (g0 == 0) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) sh.base[lane * CPT + j] = first(j);
    } else {
      const int64_t s = slot(g0 - 1);
      ok = await(c, s, s, false) && ok;
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        sh.base[lane * CPT + j] =
            unpack2(__hip_atomic_load(c.values + (s * 64 + lane) * CPT + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)).y;
    }
  }
  if (!ok && lane == 0) sh.bad = 1;
  __syncthreads();
  const bool bad = sh.bad != 0;
  if (bad && order == 0 && lane == 0) __hip_atomic_fetch_or(&g_recur_status, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    float x = sh.base[lane * CPT + j];
    if (pos != g0)
      for (int w = 0; w < kWaves; ++w) {
        const float2 q = sh.before[w][lane * CPT + j];
        x = __builtin_fmaf(q.x, x, q.y);
      }
    if (bad) x = __builtin_nanf("");
    entry[j] = x;
    leave[j] = __builtin_fmaf(all[j].x, x, all[j].y);
    for (int w = 0; w < order; ++w) {
      const float2 q = sh.part[w][lane * CPT + j];
      x = __builtin_fmaf(q.x, x, q.y);
    }
    carry[j] = x;
  }
  if (order == 0 && more && last_of_group) {
    float2 v[CPT];
#pragma unroll
    for (int j = 0; j < CPT; ++j) v[j] = make_float2(0.0f, leave[j]);
    publish<CPT>(c, slot(pos), lane, v);
  }
}

// The workgroup's tile in walking order: by ticket where tiles wait for each other, else by its index.
template <int CPT>
__device__ __forceinline__ int64_t take_ticket(const Chain& c, ChainTile<CPT>& sh, int g) {
  if (!c.tickets) return blockIdx.x / c.G;
  if (threadIdx.x == 0)
    sh.ticket = __hip_atomic_fetch_add(c.tickets + static_cast<int64_t>(g) * kTicketStride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return sh.ticket;
}

template <int DT, int CPT>
__global__ __launch_bounds__(64 * kWaves) void recur_fwd_kernel(RecurArgs a, Chain c) {
  __shared__ ChainTile<CPT> sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % c.G;
  const Place p = place_of(a, c, take_ticket(c, sh, g), false);
  if (!p.any) return;
  const int64_t mine = static_cast<int64_t>(g) * 64 * CPT + lane * CPT;
  const bool on = mine < a.C;
  const int64_t ch = on ? mine : a.C - CPT;
  const int64_t t0 = static_cast<int64_t>(p.tile) * kTile + wave * kRows;
  const int n = static_cast<int>(p.len - t0 < 0 ? 0 : p.len - t0 < kRows ? p.len - t0 : kRows);
  float bias[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) bias[j] = a.bias ? a.bias[ch + j] : 0.0f;
  float A[kRows][CPT], U[kRows][CPT];
  float2 part[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) part[j] = make_float2(1.0f, 0.0f);
  if (n > 0) {
    Row<DT, CPT> v[kRows], w[kRows], d[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {  // (rows behind the end read the last one again)
      const int64_t r = p.row0 + t0 + (i < n ? i : n - 1);
      d[i].load(a.decay, r * a.ld_d + ch);
      w[i].load(a.write, r * a.ld_w + ch);
      v[i].load(a.value, r * a.ld_v + ch);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        A[i][j] = sig(d[i].get(j) + bias[j]);
        U[i][j] = sig(w[i].get(j)) * tanh2<DT>(v[i].get(j)).t;
        if (i < n) part[j] = make_float2(A[i][j] * part[j].x, __builtin_fmaf(A[i][j], part[j].y, U[i][j]));
      }
  }
  float h[CPT], entry[CPT], leave[CPT];
  auto first = [&](int j) { return a.h0 ? a.h0[p.seq * a.C + ch + j] : 0.0f; };
  auto slot = [&](int q) { return g * c.slots + p.slot0 + q; };
  chain_carry<CPT>(c, sh, lane, wave, p.tile, p.tiles, part, slot, first, h, entry, leave);
  if (!on) return;
  if (wave == kWaves - 1) {
    if (a.carries) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) a.carries[(p.slot0 + p.tile) * a.C + ch + j] = entry[j];
    }
    if (p.tile == p.tiles - 1) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) a.h_out[p.seq * a.C + ch + j] = leave[j];
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (i < n) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) h[j] = __builtin_fmaf(A[i][j], h[j], U[i][j]);
      Row<DT, CPT>::store(a.h, (p.row0 + t0 + i) * a.ld_h + ch, h);
    }
}

template <int DT, int CPT>
__global__ __launch_bounds__(64 * kWaves) void recur_bwd_kernel(RecurBwdArgs b, Chain c, float* sums) {
  __shared__ ChainTile<CPT> sh;
  __shared__ float2 fwd[kWaves][64 * CPT];
  const RecurArgs& a = b.in;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % c.G;
  const Place p = place_of(a, c, take_ticket(c, sh, g), true);
  if (!p.any) return;
  const int64_t mine = static_cast<int64_t>(g) * 64 * CPT + lane * CPT;
  const bool on = mine < a.C;
  const int64_t ch = on ? mine : a.C - CPT;
  const int64_t t0 = static_cast<int64_t>(p.tile) * kTile + wave * kRows;
  const int n = static_cast<int>(p.len - t0 < 0 ? 0 : p.len - t0 < kRows ? p.len - t0 : kRows);
  float bias[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) bias[j] = a.bias ? a.bias[ch + j] : 0.0f;
  Row<DT, CPT> v[kRows], w[kRows], d[kRows], dh[kRows];
  float A[kRows][CPT], U[kRows][CPT];
  float2 part[CPT], from[CPT];  // the rows backwards and forwards
#pragma unroll
  for (int j = 0; j < CPT; ++j) part[j] = from[j] = make_float2(1.0f, 0.0f);
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = p.row0 + t0 + (i < n ? i : n - 1);
      d[i].load(a.decay, r * a.ld_d + ch);
      w[i].load(a.write, r * a.ld_w + ch);
      v[i].load(a.value, r * a.ld_v + ch);
      dh[i].load(b.grad, r * b.ld_g + ch);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        A[i][j] = sig(d[i].get(j) + bias[j]);
        U[i][j] = sig(w[i].get(j)) * tanh2<DT>(v[i].get(j)).t;
        if (i < n) from[j] = make_float2(A[i][j] * from[j].x, __builtin_fmaf(A[i][j], from[j].y, U[i][j]));
      }
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        if (i < n) part[j] = make_float2(A[i][j] * part[j].x, A[i][j] * (part[j].y + dh[i].get(j)));
  }
#pragma unroll
  for (int j = 0; j < CPT; ++j) fwd[wave][lane * CPT + j] = from[j];
  // The chain's state is c; in front of it (behind the last row) stands the final state's gradient.
  float back[CPT], entry[CPT], leave[CPT];
  const int pos = p.tiles - 1 - p.tile;
  auto first = [&](int j) { return b.grad_state ? b.grad_state[p.seq * a.C + ch + j] : 0.0f; };
  auto slot = [&](int q) { return g * c.slots + p.slot0 + (p.tiles - 1 - q); };
  chain_carry<CPT>(c, sh, lane, kWaves - 1 - wave, pos, p.tiles, part, slot, first, back, entry, leave);
  // the states again, from the tile's kept carry
  float h[kRows][CPT];  // in front of each row
  float db[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    float x = a.carries[(p.slot0 + p.tile) * a.C + ch + j];
    for (int q = 0; q < wave; ++q) {
      const float2 f = fwd[q][lane * CPT + j];
      x = __builtin_fmaf(f.x, x, f.y);
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      h[i][j] = x;
      if (n > 0) x = __builtin_fmaf(A[i][j], x, U[i][j]);
    }
    db[j] = 0.0f;
  }
  if (n > 0) {
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i)
      if (i < n) {
        float ov[CPT], ow[CPT], od[CPT];
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          const Sig s = sig2(w[i].get(j));
          const Tanh t = tanh2<DT>(v[i].get(j));
          const float q = sig2(d[i].get(j) + bias[j]).q;
          const float grad = back[j] + dh[i].get(j);
          ov[j] = grad * s.p * t.d;
          ow[j] = grad * U[i][j] * s.q;
          od[j] = grad * h[i][j] * A[i][j] * q;
          db[j] += od[j];
          back[j] = A[i][j] * grad;
        }
        if (on) {
          const int64_t r = p.row0 + t0 + i;
          Row<DT, CPT>::store(b.d_value, r * b.ld_dv + ch, ov);
          Row<DT, CPT>::store(b.d_write, r * b.ld_dw + ch, ow);
          Row<DT, CPT>::store(b.d_decay, r * b.ld_dd + ch, od);
        }
      }
  }
  if (on && wave == 0 && p.tile == 0 && b.d_h0) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) b.d_h0[p.seq * a.C + ch + j] = leave[j];
  }
  if (sums) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) sh.before[wave][lane * CPT + j].x = db[j];
    __syncthreads();
    if (wave == 0 && on) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        float x = 0.0f;
        for (int q = 0; q < kWaves; ++q) x += sh.before[q][lane * CPT + j].x;
        sums[(p.slot0 + p.tile) * a.C + ch + j] = x;
      }
    }
  }
}

// The bias gradient: tiles' sums (slots without rows hold zeros), 16 runs of slots per workgroup of 64 channels, joined in order.
__global__ __launch_bounds__(1024) void recur_bias_kernel(const float* sums, int64_t slots, int64_t C, float* out) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  float x = 0.0f;
  if (ch < C) {
    const int64_t each = (slots + 15) / 16, lo = run * each, hi = lo + each < slots ? lo + each : slots;
#pragma unroll 8
    for (int64_t s = lo; s < hi; ++s) x += sums[s * C + ch];
  }
  part[run][lane] = x;
  __syncthreads();
  if (run == 0 && ch < C) {
    for (int q = 1; q < 16; ++q) x += part[q][lane];
    out[ch] = x;
  }
}

// Workgroup 0 of a packed call brings the starts inside the rows and in order (a running maximum); the others clear words.
__global__ __launch_bounds__(256) void recur_reset_kernel(uint32_t* words, int64_t n, const int32_t* starts, int64_t count, int64_t rows,
                                                          int32_t* ordered) {
  if (starts && blockIdx.x == gridDim.x - 1) {
    __shared__ int32_t top[256];
    int32_t run = 0;
    for (int64_t i0 = 0; i0 < count; i0 += 256) {
      const int64_t i = i0 + threadIdx.x;
      int64_t v = i < count ? starts[i] : 0;
      v = v < 0 ? 0 : v > rows ? rows : v;
      top[threadIdx.x] = static_cast<int32_t>(v);
      __syncthreads();
      for (int d = 1; d < 256; d <<= 1) {
        const int32_t o = threadIdx.x >= d ? top[threadIdx.x - d] : 0;
        __syncthreads();
        if (o > top[threadIdx.x]) top[threadIdx.x] = o;
        __syncthreads();
      }
      const int32_t m = top[threadIdx.x] > run ? top[threadIdx.x] : run, last = top[255];
      if (i < count) ordered[i] = m;
      run = last > run ? last : run;
      __syncthreads();
    }
    return;
  }
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) words[i] = 0;
}

template <int DT>
__global__ __launch_bounds__(256) void recur_step_kernel(RecurStepArgs a) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, b = blockIdx.y;
  if (c >= a.C) return;
  const float d = ld<DT>(a.decay, b * a.ld_d + c), w = ld<DT>(a.write, b * a.ld_w + c), v = ld<DT>(a.value, b * a.ld_v + c);
  const float h = __builtin_fmaf(sig(d + (a.bias ? a.bias[c] : 0.0f)), a.state[b * a.C + c], sig(w) * tanh2<DT>(v).t);
  a.state[b * a.C + c] = h;
  st<DT>(a.h, b * a.ld_h + c, h);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int recur_check(const RecurArgs& a) {
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, "gated scan: dtype must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.L >= 0 && a.C >= 0 && a.S >= 0 && a.B < (1LL << 31) && a.L < (1LL << 31) && a.C < (1LL << 24) &&
                   a.S < (1LL << 24) && a.B * a.L < (1LL << 31),
               kErrInvalidArg, "gated scan: bad sizes");
  TESM_REQUIRE(a.seq_starts ? a.B == 1 : a.S == a.B, kErrInvalidArg,
               "gated scan: one sequence per batch row, or with starts one row axis");
  return kOk;
}

// Two bfloat16 channels per lane where every row begins on four bytes.
bool in_pairs(int dt, int64_t C, std::initializer_list<std::pair<const void*, int64_t>> rows) {
  if (dt != kBF16 || C % 2) return false;
  for (const auto& r : rows)
    if (r.first && (!aligned(r.first, 4) || r.second % 2)) return false;
  return true;
}

struct Plan {
  int64_t slots = 0, words = 0;  // words to clear, at most: tickets, flags
  int64_t at_values = 0, at_starts = 0, at_sums = 0, total = 0;
  bool chained = false;
};
int64_t up256(int64_t v) { return round_up(v, 256); }
Plan plan_of(const RecurArgs& a, bool sums) {
  Plan p;
  const int64_t G = 2 * ((a.C + 127) / 128);  // (64 channels each, or half as many of 128)
  const int64_t tiles = (a.L + kTile - 1) / kTile;
  p.slots = a.seq_starts ? a.B * a.L / kTile + a.S : a.B * std::max<int64_t>(tiles, 1);
  p.chained = a.seq_starts || tiles > 1;
  if (p.chained) p.words = G * kTicketStride + G * p.slots;
  p.at_values = up256(4 * p.words);
  p.at_starts = p.at_values + (p.chained ? up256(G * p.slots * 64 * 8) : 0);
  p.at_sums = p.at_starts + (a.seq_starts ? up256(4 * (a.S + 1)) : 0);
  p.total = p.at_sums + (sums ? up256(4 * p.slots * a.C) : 0);
  return p;
}

Chain chain_of(const RecurArgs& a, const Plan& p, void* ws, int cpt) {
  Chain c;
  char* base = static_cast<char*>(ws);
  c.slots = p.slots;
  c.G = static_cast<int>((a.C + 64 * cpt - 1) / (64 * cpt));
  c.tiles = static_cast<int>(std::max<int64_t>(1, (a.L + kTile - 1) / kTile));
  c.spin_limit = g_spin_limit;
  if (p.chained) {
    c.tickets = reinterpret_cast<unsigned*>(base);
    c.flags = reinterpret_cast<int*>(base) + static_cast<int64_t>(c.G) * kTicketStride;
    c.values = reinterpret_cast<unsigned long long*>(base + p.at_values);
  }
  if (a.seq_starts) c.starts = reinterpret_cast<int32_t*>(base + p.at_starts);
  return c;
}

int reset(const RecurArgs& a, const Plan& p, const Chain& c, void* ws, bool sums, hipStream_t st) {
  if (!p.chained) return kOk;
  // (sums lie behind the rest and are cleared with packed rows only: every slot of a dense batch is a tile)
  const int64_t words = static_cast<int64_t>(c.G) * (kTicketStride + p.slots);
  const unsigned blocks = static_cast<unsigned>((words + 255) / 256 + (a.seq_starts ? 1 : 0));
  recur_reset_kernel<<<blocks, 256, 0, TESM_LOGGED(st, recur_reset_kernel)>>>(
      static_cast<uint32_t*>(ws), words, a.seq_starts, a.S + 1, a.B * a.L, const_cast<int32_t*>(c.starts));
  if (sums && a.seq_starts) {
    const int64_t n = p.slots * a.C;
    recur_reset_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, TESM_LOGGED(st, recur_reset_kernel)>>>(
        reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + p.at_sums), n, nullptr, 0, 0, nullptr);
  }
  return kOk;
}

}  // namespace

int64_t recur_slots(const RecurArgs& a) { return recur_check(a) == kOk ? plan_of(a, false).slots : -1; }
int64_t recur_ws_bytes(const RecurArgs& a) { return recur_check(a) == kOk ? plan_of(a, false).total : -1; }
int64_t recur_bwd_ws_bytes(const RecurArgs& a, bool bias) { return recur_check(a) == kOk ? plan_of(a, bias).total : -1; }

int launch_gated_scan(const RecurArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (int rc = recur_check(a)) return rc;
  if (a.C == 0 || a.S == 0) return kOk;
  const bool rows = a.B * a.L > 0;
  TESM_REQUIRE(a.h_out && (!rows || (a.value && a.write && a.decay && a.h)), kErrInvalidArg, "gated scan: need the gates, h and h_out");
  TESM_REQUIRE(!rows || (a.ld_v >= a.C && a.ld_w >= a.C && a.ld_d >= a.C && a.ld_h >= a.C), kErrInvalidArg,
               "gated scan: a row pitch below the channels");
  const Plan p = plan_of(a, false);
  TESM_REQUIRE(p.total == 0 || (ws && ws_bytes >= p.total && aligned(ws, 8)), kErrWorkspace,
               "gated scan: workspace too small or not 8-byte aligned");
  const bool pairs = in_pairs(a.dt, a.C, {{a.value, a.ld_v}, {a.write, a.ld_w}, {a.decay, a.ld_d}, {a.h, a.ld_h}});
  const Chain c = chain_of(a, p, ws, pairs ? 2 : 1);
  const int64_t blocks = p.slots * c.G;
  TESM_REQUIRE(blocks < (1LL << 31), kErrUnsupported, "gated scan: too many tiles for one call");
  if (int rc = reset(a, p, c, ws, false, st)) return rc;
  constexpr int T = 64 * kWaves;
  const unsigned n = static_cast<unsigned>(blocks);
  if (a.dt == kF32)
    recur_fwd_kernel<kF32, 1><<<n, T, 0, TESM_LOGGED(st, recur_fwd_kernel<kF32, 1>)>>>(a, c);
  else if (pairs)
    recur_fwd_kernel<kBF16, 2><<<n, T, 0, TESM_LOGGED(st, recur_fwd_kernel<kBF16, 2>)>>>(a, c);
  else
    recur_fwd_kernel<kBF16, 1><<<n, T, 0, TESM_LOGGED(st, recur_fwd_kernel<kBF16, 1>)>>>(a, c);
  return check_launch("gated scan");
}

int launch_gated_scan_bwd(const RecurBwdArgs& b, void* ws, int64_t ws_bytes, hipStream_t st) {
  const RecurArgs& a = b.in;
  if (int rc = recur_check(a)) return rc;
  if (a.C == 0) return kOk;
  const bool rows = a.B * a.L > 0;
  TESM_REQUIRE(a.S == 0 || (a.carries && (!rows || (a.value && a.write && a.decay && b.grad && b.d_value && b.d_write && b.d_decay))),
               kErrInvalidArg, "gated scan backward: need the gates, the kept carries, the gradient and its outputs");
  TESM_REQUIRE(!rows || (a.ld_v >= a.C && a.ld_w >= a.C && a.ld_d >= a.C && b.ld_g >= a.C && b.ld_dv >= a.C && b.ld_dw >= a.C &&
                         b.ld_dd >= a.C),
               kErrInvalidArg, "gated scan backward: a row pitch below the channels");
  const Plan p = plan_of(a, b.d_bias != nullptr);
  TESM_REQUIRE(p.total == 0 || (ws && ws_bytes >= p.total && aligned(ws, 8)), kErrWorkspace,
               "gated scan backward: workspace too small or not 8-byte aligned");
  const bool pairs = in_pairs(a.dt, a.C, {{a.value, a.ld_v}, {a.write, a.ld_w}, {a.decay, a.ld_d}, {b.grad, b.ld_g},
                                          {b.d_value, b.ld_dv}, {b.d_write, b.ld_dw}, {b.d_decay, b.ld_dd}});
  const Chain c = chain_of(a, p, ws, pairs ? 2 : 1);
  const int64_t blocks = a.S ? p.slots * c.G : 0;
  TESM_REQUIRE(blocks < (1LL << 31), kErrUnsupported, "gated scan backward: too many tiles for one call");
  float* sums = b.d_bias ? reinterpret_cast<float*>(static_cast<char*>(ws) + p.at_sums) : nullptr;
  if (blocks > 0) {
    if (int rc = reset(a, p, c, ws, sums != nullptr, st)) return rc;
    constexpr int T = 64 * kWaves;
    const unsigned n = static_cast<unsigned>(blocks);
    if (a.dt == kF32)
      recur_bwd_kernel<kF32, 1><<<n, T, 0, TESM_LOGGED(st, recur_bwd_kernel<kF32, 1>)>>>(b, c, sums);
    else if (pairs)
      recur_bwd_kernel<kBF16, 2><<<n, T, 0, TESM_LOGGED(st, recur_bwd_kernel<kBF16, 2>)>>>(b, c, sums);
    else
      recur_bwd_kernel<kBF16, 1><<<n, T, 0, TESM_LOGGED(st, recur_bwd_kernel<kBF16, 1>)>>>(b, c, sums);
  }
  if (b.d_bias) {
    const unsigned n = static_cast<unsigned>((a.C + 63) / 64);
    recur_bias_kernel<<<n, 1024, 0, TESM_LOGGED(st, recur_bias_kernel)>>>(sums, a.S ? p.slots : 0, a.C, b.d_bias);
  }
  return check_launch("gated scan backward");
}

int launch_gated_scan_step(const RecurStepArgs& a, hipStream_t st) {
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, "gated scan step: dtype must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.C >= 0 && a.B < 65536 && a.C < (1LL << 24), kErrInvalidArg, "gated scan step: bad sizes");
  if (a.B == 0 || a.C == 0) return kOk;
  TESM_REQUIRE(a.value && a.write && a.decay && a.state && a.h, kErrInvalidArg, "gated scan step: need the gates, the state and h");
  TESM_REQUIRE(a.ld_v >= a.C && a.ld_w >= a.C && a.ld_d >= a.C && a.ld_h >= a.C, kErrInvalidArg,
               "gated scan step: a row pitch below the channels");
  const dim3 grid(static_cast<unsigned>((a.C + 255) / 256), static_cast<unsigned>(a.B));
  if (a.dt == kF32)
    recur_step_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, recur_step_kernel<kF32>)>>>(a);
  else
    recur_step_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, recur_step_kernel<kBF16>)>>>(a);
  return check_launch("gated scan step");
}

int recur_status(unsigned* out, int clear) {
  unsigned v = 0;
  hipError_t e = hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_recur_status), sizeof(v), 0, hipMemcpyDeviceToHost);
  if (e == hipSuccess && clear && v != 0) {
    const unsigned zero = 0;
    e = hipMemcpyToSymbol(HIP_SYMBOL(g_recur_status), &zero, sizeof(zero), 0, hipMemcpyHostToDevice);
  }
  if (e != hipSuccess) return fail(kErrLaunch, std::string("device status: ") + hipGetErrorString(e));
  *out = v;
  return kOk;
}

void recur_set_spin_limit(int limit) { g_spin_limit = limit < 0 ? -1 : limit; }

}  // namespace tesm
