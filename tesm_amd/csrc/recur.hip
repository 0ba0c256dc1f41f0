// Gated linear recurrence over rows t, per channel:
//   a_t = sigmoid(decay_t + bias),  u_t = sigmoid(write_t) tanh(value_t),  h_t = a_t h_{t-1} + u_t
// and its backward pass, with g_t the gradient of h_t by every way and c_t = a_t g_t what it hands to the row before:
//   g_t = dh_t + c_{t+1}  (the last row: + the final state's gradient),
//   d decay_t = g_t h_{t-1} a_t (1 - a_t), d write_t = g_t u_t (1 - sigmoid(write_t)),
//   d value_t = g_t sigmoid(write_t) (1 - tanh^2), d h_0 = c_1.
// Both are first-order recurrences x <- A x + U, and runs of them compose: (A, U) then (A', U') is (A' A, A' U + U').
//
// One pass over the data.  A tile is 64 rows of one sequence (forward, where long sequences are more than the caches hold, 128 bfloat16 rows) by
// 64 or 128 channels; each of 8 waves takes 8 (16) rows, a lane one or two channels; inputs are read once and stay in registers as gates.  Waves scan their rows from zero, their (A, U) meet in
// LDS, and tiles of one sequence and channel group hand on their state in a chain: a tile publishes its (A, U); from these
// and the state in front of its group of 16 tiles every tile forms its own carry, always in the same order, so results
// repeat bit for bit; the last tile of a group publishes the state behind it.  Tiles are taken by ticket, predecessors first, so that
// whatever a tile waits for is already running.  The forward pass can keep the state in front of every 64 rows (1/64 of a
// float32 copy of the states; a tile of 128 rows keeps two); the backward pass, whose tiles have 64 rows, then forms the states again in
// registers and walks the chain from the end.
//
// Published values go by agent-scope atomic accesses of 8 bytes (coherent over the XCDs' caches).  A value says by itself that it is
// there, its bits are those of no number before: a flag beside it would cost the chain three more trips through memory (one for the
// values to arrive before the flag, two for the reader).  A poll gives up after kSpinLimit rounds: the states are then NaN and bit 0 of
// the status word is set.
//
// Bound by HBM where there is much of it: 32768 x 8192 bfloat16 forward 498 us (4.3 TB/s; a copy's 5.9 would take 364), backward 844 (637; accesses past the caches take as long);
// 16384 x 4096 float32 231 us (182) and 353 (318).  The vector unit is busy for 58 to 63 % of the bfloat16 passes, the chain costs 7 %, the
// tickets 5 %; workgroups that stay and load their next tile ahead took 610 and 1103 us.  Short calls by latency: 4 x 2048 x 384 12 and
// 16 us.
#include <type_traits>
#include <utility>

#include "linear_dev.h"
#include "recur.h"

namespace tesm {

namespace {

constexpr int kWaves = 8, kGroup = 16;
static_assert(kGroup == 2 * kWaves, "a wave looks after two earlier tiles");
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
// (where e overflows, p is 0; every use of q has p as a factor)
__device__ __forceinline__ Sig sig_of(float e) {
  const float p = __builtin_amdgcn_rcpf(1.0f + e);
  return {p, fminf(e, 3.4e38f) * p};
}
// The decay, of x + b: added first, since b log2 e and x log2 e, rounded apart, lose what is left where the two nearly cancel (biases of
// 300: a decay 1e-5 of itself off).  A state that is kept for n rows holds n times what a decay is off to one side, so this
// reciprocal takes a Newton step, 1 - p (1 + e) = (1 - p) - p e being exact where p is near 1 (decays that keep 400 rows: the bias's
// gradient is 1.6e-6 of itself off without it, 3.3e-7 with it; both passes of 32768 x 8192 take 1362 us instead of 1357).
__device__ __forceinline__ Sig decay_of(float x, float b) {
  const float e = __builtin_amdgcn_exp2f((x + b) * -kLog2e);
  const float r = __builtin_amdgcn_rcpf(1.0f + e), most = fminf(e, 3.4e38f);
  const float p = __builtin_fmaf(r, __builtin_fmaf(-most, r, 1.0f - r), r);
  return {p, most * p};
}
__device__ __forceinline__ Sig sig2(float x) { return sig_of(__builtin_amdgcn_exp2f(x * -kLog2e)); }
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
  const float small = x * __builtin_fmaf(x2, p, 1.0f);
  return {fabsf(x) < (DT == kF32 ? 0.25f : 0.03125f) ? small : big, 4.0f * r * (1.0f - r)};
}

// ---------------------------------------------------------------------------
// a lane's channels of a row
// ---------------------------------------------------------------------------
template <int DT, int CPT>
struct Row {
  uint32_t w;  // one float32, one bfloat16 or two
  // (row: the same for all lanes; off: the lane's bytes in it)
  __device__ __forceinline__ void load(const char* row, uint32_t off) {
    if constexpr (DT == kBF16 && CPT == 1)
      w = *reinterpret_cast<const uint16_t*>(row + off);
    else
      w = *reinterpret_cast<const uint32_t*>(row + off);
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (CPT == 2) return __uint_as_float(j ? w & 0xffff0000u : w << 16);
    return from_bits<DT>(w);
  }
  static __device__ __forceinline__ void store(char* row, uint32_t off, const float (&v)[CPT]) {
    if constexpr (CPT == 2)
      *reinterpret_cast<uint32_t*>(row + off) = pack_bf16x2(v[0], v[1]);
    else if constexpr (DT == kBF16)
      *reinterpret_cast<uint16_t*>(row + off) = f32_to_bf16(v[0]);
    else
      *reinterpret_cast<float*>(row + off) = v[0];
  }
};
// The wave's first row of an array, and its rows' distance in bytes.
struct RowsOf {
  char* p;
  int64_t step;
};
template <int DT>
__device__ __forceinline__ RowsOf rows_of(const void* p, int64_t ld, int64_t row) {
  constexpr int ES = DT == kBF16 ? 2 : 4;
  return {const_cast<char*>(static_cast<const char*>(p)) + row * ld * ES, ld * ES};
}

// ---------------------------------------------------------------------------
// the chain of a sequence's tiles
// ---------------------------------------------------------------------------
struct Chain {
  unsigned* tickets = nullptr;  // a 256-byte line per channel group
  unsigned long long* values = nullptr;  // (G, slots, 64 CPT): (A, U) of a tile, or the state behind a group's last one; kUnset before
  const int32_t* starts = nullptr;   // packed: S + 1 starts, inside the rows and not decreasing
  int slots = 0;
  int G = 0, tiles = 0;  // channel groups; tiles per sequence of a dense batch
  int kept = 0;          // kept carries per sequence of a dense batch
  int spin_limit = 0;
};
constexpr int kTicketStride = 64;
constexpr uint32_t kUnset = 0xffffffffu;  // as U: no value yet (a NaN is published with other bits)

struct Place {  // (rows, sequences and slots are below 2^31)
  int row0, len, seq, slot0;  // the sequence's first row and length, its number and first slot
  int tile, tiles;            // tiles < 0: none
};

// The tile of slot `at` in walking order; `back`: from the end.
template <int ROWS>
__device__ __forceinline__ Place place_of(const RecurArgs& a, const Chain& c, int at, bool back) {
  Place p;
  if (!c.starts) {
    const unsigned B = static_cast<unsigned>(a.B), pos = static_cast<unsigned>(at) / B;
    p.seq = static_cast<int>(static_cast<unsigned>(at) - pos * B);
    p.tiles = c.tiles;
    p.tile = back ? c.tiles - 1 - static_cast<int>(pos) : static_cast<int>(pos);
    p.len = static_cast<int>(a.L);
    p.row0 = p.seq * p.len;
    p.slot0 = p.seq * c.tiles;
    return p;
  }
  const int slot = back ? c.slots - 1 - at : at;
  // sequence s has the slots from start / ROWS + s on, at least one
  int lo = 0, hi = static_cast<int>(a.S);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__builtin_amdgcn_readfirstlane(c.starts[mid]) / ROWS + mid <= slot)
      lo = mid;
    else
      hi = mid;
  }
  p.seq = lo;
  p.row0 = __builtin_amdgcn_readfirstlane(c.starts[lo]);
  p.len = __builtin_amdgcn_readfirstlane(c.starts[lo + 1]) - p.row0;
  p.slot0 = p.row0 / ROWS + lo;
  p.tile = slot - p.slot0;
  p.tiles = p.len > 0 ? (p.len + ROWS - 1) / ROWS : 1;  // (an empty sequence hands its state through)
  if (p.tile < 0 || p.tile >= p.tiles) p.tiles = -1;
  return p;
}

__device__ __forceinline__ float2 unpack2(unsigned long long v) {
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}
__device__ __forceinline__ void publish(const Chain& c, int64_t at, float a, float u) {
  const uint32_t bits = u == u ? __float_as_uint(u) : 0x7fc00000u;
  __hip_atomic_store(c.values + at, static_cast<unsigned long long>(bits) << 32 | __float_as_uint(a), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long published(const Chain& c, int64_t at) {
  return __hip_atomic_load(c.values + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool is_set(unsigned long long v) { return static_cast<uint32_t>(v >> 32) != kUnset; }

template <int CPT>
struct ChainTile {
  float2 part[kWaves][64 * CPT];    // the waves' rows
  float2 before[kWaves][64 * CPT];  // the tiles in front, two per wave
  float base[64 * CPT];             // the state in front of the group
  int bad;
  unsigned ticket;
};

// The state entering the wave's rows.  part: the wave's (A, U).  In walking order: pos of the tile, order of the wave; at(p): where
// position p publishes this lane's values; first: the sequence's own first state.  `leave` returns, to the first wave in order, the
// state behind the tile.
template <int CPT, typename At, typename First>
__device__ __forceinline__ void chain_carry(const Chain& c, ChainTile<CPT>& sh, int lane, int order, int pos, int count,
                                            const float2 (&part)[CPT], At&& at, First&& first, float (&carry)[CPT],
                                            float (&leave)[CPT]) {
#pragma unroll
  for (int j = 0; j < CPT; ++j) sh.part[order][lane * CPT + j] = part[j];
  if (order == 0 && lane == 0) sh.bad = 0;
  __syncthreads();
  const int g0 = pos & ~(kGroup - 1), front = pos - g0;
  const bool last_of_group = front == kGroup - 1, more = pos + 1 < count;
  float2 all[CPT];
  if (order == 0) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      all[j] = sh.part[0][lane * CPT + j];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        const float2 q = sh.part[w][lane * CPT + j];
        all[j] = make_float2(q.x * all[j].x, __builtin_fmaf(q.x, all[j].y, q.y));
      }
      if (more && !last_of_group) publish(c, at(pos) + j, all[j].x, all[j].y);
    }
  }
  // two tiles in front of this one, in order; the last wave has one, and the state in front of the group
  const int p0 = g0 + 2 * order;
  const bool one = p0 < pos, two = p0 + 1 < pos, base = order == kWaves - 1 && g0 > 0;
  if (one || base) {
    const int64_t at0 = at(one ? p0 : g0 - 1), at1 = at(two ? p0 + 1 : base ? g0 - 1 : p0);
    unsigned long long x[CPT] = {}, y[CPT] = {};
    bool ok = false;
    // (polled by the first lane's value alone: all lanes' would be more traffic than the rows)
    const int64_t look0 = at0 - lane * CPT, look1 = at1 - lane * CPT;
    for (int i = 0; i <= c.spin_limit && !ok; ++i) {
      bool set = true;
      if (lane == 0) set = is_set(published(c, look0)) && is_set(published(c, look1));
      if (!__all(set)) {
        __builtin_amdgcn_s_sleep(2);
        continue;
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        x[j] = published(c, at0 + j);
        y[j] = published(c, at1 + j);
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j) set = set && is_set(x[j]) && is_set(y[j]);
      ok = __all(set);
    }
    if (!ok && lane == 0) sh.bad = 1;
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      const float2 u = unpack2(x[j]), v = unpack2(y[j]);
      if (one) sh.before[order][lane * CPT + j] = two ? make_float2(v.x * u.x, __builtin_fmaf(v.x, u.y, v.y)) : u;
      if (base) sh.base[lane * CPT + j] = v.y;
    }
  }
  if (order == kWaves - 1 && g0 == 0) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) sh.base[lane * CPT + j] = first(j);
  }
  __syncthreads();
  const bool bad = sh.bad != 0;
  if (bad && order == 0 && lane == 0) __hip_atomic_fetch_or(&g_recur_status, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    float x = sh.base[lane * CPT + j];
    for (int w = 0; w < (front + 1) / 2; ++w) {
      const float2 q = sh.before[w][lane * CPT + j];
      x = __builtin_fmaf(q.x, x, q.y);
    }
    if (bad) x = __builtin_nanf("");
    if (order == 0) {
      leave[j] = __builtin_fmaf(all[j].x, x, all[j].y);
      if (more && last_of_group) publish(c, at(pos) + j, 0.0f, leave[j]);
    }
    for (int w = 0; w < order; ++w) {
      const float2 q = sh.part[w][lane * CPT + j];
      x = __builtin_fmaf(q.x, x, q.y);
    }
    carry[j] = x;
  }
}

// The workgroup's tile in walking order: by ticket where tiles wait for each other, else by its index.  (Uniform: what follows
// from it costs no vector operations.)
template <int CPT>
__device__ __forceinline__ int take_ticket(const Chain& c, ChainTile<CPT>& sh, int g) {
  if (!c.tickets) return static_cast<int>(blockIdx.x / static_cast<unsigned>(c.G));
  if (threadIdx.x == 0)
    sh.ticket = __hip_atomic_fetch_add(c.tickets + static_cast<int64_t>(g) * kTicketStride, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(static_cast<int>(sh.ticket));
}

// A wave's rows of a tile: the first one in the array, and how many there are.
struct Part {
  int row, n;
};
template <int T>
__device__ __forceinline__ Part part_of(const Place& p, int wave) {
  const int t0 = (p.tile * kWaves + wave) * T, left = p.tiles > 0 ? p.len - t0 : 0;
  return {p.row0 + t0, left < 0 ? 0 : left < T ? left : T};
}
// Its inputs, rows behind the end read as the last one.
template <int DT, int CPT, int T, bool WHOLE, int ARRAYS>
__device__ __forceinline__ void load_rows(const Part& q, const void* const (&&p)[ARRAYS], const int64_t (&&ld)[ARRAYS], uint32_t off,
                                          Row<DT, CPT> (&to)[ARRAYS][T]) {
  RowsOf r[ARRAYS];
#pragma unroll
  for (int k = 0; k < ARRAYS; ++k) r[k] = rows_of<DT>(p[k], ld[k], q.row);
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int k = 0; k < ARRAYS; ++k) {
      to[k][i].load(r[k].p, off);
      if (WHOLE || i + 1 < q.n) r[k].p += r[k].step;
    }
}

template <int DT, int CPT, int T>
__global__ __launch_bounds__(64 * kWaves) void recur_fwd_kernel(RecurArgs a, Chain c) {
  __shared__ ChainTile<CPT> sh;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.x % c.G;
  const Place p = place_of<kWaves * T>(a, c, take_ticket(c, sh, g), false);
  if (p.tiles < 0) return;
  const int64_t mine = static_cast<int64_t>(g) * 64 * CPT + lane * CPT;
  const bool on = mine < a.C;
  const int64_t ch = on ? mine : a.C - CPT;
  constexpr int ES = DT == kBF16 ? 2 : 4;
  const uint32_t off = static_cast<uint32_t>(ch * ES);
  const Part q = part_of<T>(p, wave);
  float A[T][CPT], U[T][CPT];
  float2 part[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) part[j] = make_float2(1.0f, 0.0f);
  // (whole parts apart: without a branch per row their rows are worked on side by side)
  auto gates = [&](auto whole) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole)::value;
    Row<DT, CPT> raw[3][T];
    load_rows<DT, CPT, T, WHOLE, 3>(q, {a.decay, a.write, a.value}, {a.ld_d, a.ld_w, a.ld_v}, off, raw);
    float bias[CPT];
#pragma unroll
    for (int j = 0; j < CPT; ++j) bias[j] = a.bias ? a.bias[ch + j] : 0.0f;
#pragma unroll
    for (int i = 0; i < T; ++i)
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        A[i][j] = decay_of(raw[0][i].get(j), bias[j]).p;
        U[i][j] = sig(raw[1][i].get(j)) * tanh2<DT>(raw[2][i].get(j)).t;
        if (WHOLE || i < q.n) part[j] = make_float2(A[i][j] * part[j].x, __builtin_fmaf(A[i][j], part[j].y, U[i][j]));
      }
  };
  if (q.n == T)
    gates(std::true_type{});
  else if (q.n > 0)
    gates(std::false_type{});
  float h[CPT], leave[CPT];
  auto first = [&](int j) { return a.h0 ? a.h0[p.seq * a.C + ch + j] : 0.0f; };
  auto at = [&](int k) { return ((static_cast<int64_t>(g) * c.slots + (p.slot0 + k)) * 64 + lane) * CPT; };
  chain_carry<CPT>(c, sh, lane, wave, p.tile, p.tiles, part, at, first, h, leave);
  if (!on) return;
  if (wave == 0 && p.tile == p.tiles - 1) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) a.h_out[p.seq * a.C + ch + j] = leave[j];
  }
  // the state in front of every kRecurRows rows (an empty sequence has one such place)
  const int t0 = (p.tile * kWaves + wave) * T;
  if (a.carries && t0 % kRecurRows == 0 && (t0 < p.len || t0 == 0)) {
    const int64_t slot0 = c.starts ? p.row0 / kRecurRows + p.seq : static_cast<int64_t>(p.seq) * c.kept;
#pragma unroll
    for (int j = 0; j < CPT; ++j) a.carries[(slot0 + t0 / kRecurRows) * a.C + ch + j] = h[j];
  }
  auto states = [&](auto whole) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole)::value;
    RowsOf rh = rows_of<DT>(a.h, a.ld_h, q.row);
#pragma unroll
    for (int i = 0; i < T; ++i) {
      if (!WHOLE && i >= q.n) break;
#pragma unroll
      for (int j = 0; j < CPT; ++j) h[j] = __builtin_fmaf(A[i][j], h[j], U[i][j]);
      Row<DT, CPT>::store(rh.p, off, h);
      rh.p += rh.step;
    }
  };
  if (q.n == T)
    states(std::true_type{});
  else
    states(std::false_type{});
}

template <int DT, int CPT>
__global__ __launch_bounds__(64 * kWaves, 4) void recur_bwd_kernel(RecurBwdArgs b, Chain c, float* sums) {
  constexpr int T = kRecurRows / kWaves;
  __shared__ ChainTile<CPT> sh;
  __shared__ float2 fwd[kWaves][64 * CPT];
  const RecurArgs& a = b.in;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int order = kWaves - 1 - wave;  // in walking order, from the end
  const int g = blockIdx.x % c.G;
  const Place p = place_of<kRecurRows>(a, c, take_ticket(c, sh, g), true);
  const int64_t mine = static_cast<int64_t>(g) * 64 * CPT + lane * CPT;
  const bool on = mine < a.C;
  const int64_t ch = on ? mine : a.C - CPT;
  if (p.tiles < 0) {  // (a slot without a tile: nothing to add to the bias's sums)
    if (sums && wave == 0 && on) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) sums[static_cast<int64_t>(p.slot0 + p.tile) * a.C + ch + j] = 0.0f;
    }
    return;
  }
  constexpr int ES = DT == kBF16 ? 2 : 4;
  const uint32_t off = static_cast<uint32_t>(ch * ES);
  const Part q = part_of<T>(p, wave);
  float kept[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) kept[j] = a.carries[static_cast<int64_t>(p.slot0 + p.tile) * a.C + ch + j];
  // Per row: a, and what the gradient is multiplied with for value, write and decay; U: u.
  Row<DT, CPT> dh[T];
  float A[T][CPT], U[T][CPT], fv[T][CPT], fw[T][CPT], fd[T][CPT];
  float2 part[CPT], from[CPT];  // the rows backwards and forwards
#pragma unroll
  for (int j = 0; j < CPT; ++j) part[j] = from[j] = make_float2(1.0f, 0.0f);
  auto gates = [&](auto whole) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole)::value;
    Row<DT, CPT> raw[4][T];
    load_rows<DT, CPT, T, WHOLE, 4>(q, {a.decay, a.write, a.value, b.grad}, {a.ld_d, a.ld_w, a.ld_v, b.ld_g}, off, raw);
    float bias[CPT];
#pragma unroll
    for (int j = 0; j < CPT; ++j) bias[j] = a.bias ? a.bias[ch + j] : 0.0f;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      dh[i] = raw[3][i];
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const Sig f = decay_of(raw[0][i].get(j), bias[j]), s = sig2(raw[1][i].get(j));
        const Tanh t = tanh2<DT>(raw[2][i].get(j));
        A[i][j] = f.p;
        fd[i][j] = f.p * f.q;
        U[i][j] = s.p * t.t;
        fv[i][j] = s.p * t.d;
        fw[i][j] = U[i][j] * s.q;
        if (WHOLE || i < q.n) from[j] = make_float2(A[i][j] * from[j].x, __builtin_fmaf(A[i][j], from[j].y, U[i][j]));
      }
    }
#pragma unroll
    for (int i = T - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < CPT; ++j)
        if (WHOLE || i < q.n) part[j].y = A[i][j] * (part[j].y + dh[i].get(j));
#pragma unroll
    for (int j = 0; j < CPT; ++j) part[j].x = from[j].x;
  };
  if (q.n == T)
    gates(std::true_type{});
  else if (q.n > 0)
    gates(std::false_type{});
#pragma unroll
  for (int j = 0; j < CPT; ++j) fwd[wave][lane * CPT + j] = from[j];
  // The chain's state is c; in front of it (behind the last row) stands the final state's gradient.
  float back[CPT], leave[CPT];
  auto first = [&](int j) { return b.grad_state ? b.grad_state[p.seq * a.C + ch + j] : 0.0f; };
  auto at = [&](int k) { return ((static_cast<int64_t>(g) * c.slots + (p.slot0 + (p.tiles - 1 - k))) * 64 + lane) * CPT; };
  chain_carry<CPT>(c, sh, lane, order, p.tiles - 1 - p.tile, p.tiles, part, at, first, back, leave);
  // the states again, from the tile's kept carry
  float db[CPT];
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    db[j] = 0.0f;
    if (q.n > 0) {
      float x = kept[j];
      for (int w = 0; w < wave; ++w) {
        const float2 f = fwd[w][lane * CPT + j];
        x = __builtin_fmaf(f.x, x, f.y);
      }
#pragma unroll
      for (int i = 0; i < T; ++i) {
        fd[i][j] *= x;
        x = __builtin_fmaf(A[i][j], x, U[i][j]);
      }
    }
  }
  auto grads = [&](auto whole) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int64_t row = static_cast<int64_t>(q.row) + (WHOLE ? T : q.n) - 1;
    RowsOf rv = rows_of<DT>(b.d_value, b.ld_dv, row), rw = rows_of<DT>(b.d_write, b.ld_dw, row), rd = rows_of<DT>(b.d_decay, b.ld_dd, row);
#pragma unroll
    for (int i = T - 1; i >= 0; --i) {
      if (!WHOLE && i >= q.n) continue;
      float ov[CPT], ow[CPT], od[CPT];
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const float grad = back[j] + dh[i].get(j);
        ov[j] = grad * fv[i][j];
        ow[j] = grad * fw[i][j];
        od[j] = grad * fd[i][j];
        db[j] += od[j];
        back[j] = A[i][j] * grad;
      }
      Row<DT, CPT>::store(rv.p, off, ov);
      Row<DT, CPT>::store(rw.p, off, ow);
      Row<DT, CPT>::store(rd.p, off, od);
      rv.p -= rv.step, rw.p -= rw.step, rd.p -= rd.step;
    }
  };
  if (on) {
    if (q.n == T)
      grads(std::true_type{});
    else
      grads(std::false_type{});
  }
  if (on && order == 0 && p.tile == 0 && b.d_h0) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) b.d_h0[p.seq * a.C + ch + j] = leave[j];
  }
  if (sums) {  // (the waves are past the carry's barrier: nobody reads `before` any more but this)
    __syncthreads();
#pragma unroll
    for (int j = 0; j < CPT; ++j) sh.before[wave][lane * CPT + j].x = db[j];
    __syncthreads();
    if (wave == 0 && on) {
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        float x = 0.0f;
        for (int w = 0; w < kWaves; ++w) x += sh.before[w][lane * CPT + j].x;
        sums[static_cast<int64_t>(p.slot0 + p.tile) * a.C + ch + j] = x;
      }
    }
  }
}

// The bias gradient: tiles' sums (zeros where a slot has no tile), in 64 bits: 16 runs of slots per workgroup of 64
// channels, joined in order.
__global__ __launch_bounds__(1024) void recur_bias_kernel(const float* sums, int64_t slots, int64_t C, float* out) {
  __shared__ double part[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int64_t ch = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  double x = 0.0;
  if (ch < C) {
    const int64_t each = (slots + 15) / 16, lo = run * each, hi = lo + each < slots ? lo + each : slots;
#pragma unroll 8
    for (int64_t s = lo; s < hi; ++s) x += sums[s * C + ch];
  }
  part[run][lane] = x;
  __syncthreads();
  if (run == 0 && ch < C) {
    for (int q = 1; q < 16; ++q) x += part[q][lane];
    out[ch] = static_cast<float>(x);
  }
}

// Clears the tickets and marks the values unset.  The last workgroup of a packed call brings the starts inside the rows and in
// order (a running maximum).
__global__ __launch_bounds__(256) void recur_reset_kernel(uint4* tickets, int64_t n_tickets, uint4* values, int64_t n_values, const int32_t* starts,
                                                          int64_t count, int64_t rows, int32_t* ordered) {
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
  if (i < n_tickets)
    tickets[i] = make_uint4(0, 0, 0, 0);
  else if (i < n_tickets + n_values)
    values[i - n_tickets] = make_uint4(kUnset, kUnset, kUnset, kUnset);
}
// The rows of no sequence set to zero in up to three arrays, a row per workgroup (starts in order).
struct RestArgs {
  void* p[3];
  int64_t ld[3];
  int64_t C, rows, S;
  const int32_t* starts;
};
template <int DT>
__global__ __launch_bounds__(256) void recur_rest_kernel(RestArgs a) {
  const int64_t lo = a.starts[0], hi = a.starts[a.S];
  for (int64_t i = blockIdx.x; i < lo + (a.rows - hi); i += gridDim.x) {
    const int64_t r = i < lo ? i : hi + (i - lo);
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (a.p[k])
        for (int64_t c = threadIdx.x; c < a.C; c += 256) st<DT>(a.p[k], r * a.ld[k] + c, 0.0f);
  }
}

// One token: a channel per thread (64 x 8192 bfloat16 3.4 us, 2.5 TB/s).
template <int DT>
__global__ __launch_bounds__(256) void recur_step_kernel(RecurStepArgs a) {
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, b = blockIdx.y;
  if (c >= a.C) return;
  const float d = ld<DT>(a.decay, b * a.ld_d + c), w = ld<DT>(a.write, b * a.ld_w + c), v = ld<DT>(a.value, b * a.ld_v + c);
  const float h = __builtin_fmaf(decay_of(d, a.bias ? a.bias[c] : 0.0f).p, a.state[b * a.C + c], sig(w) * tanh2<DT>(v).t);
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
  int64_t slots = 0;
  int64_t at_values = 0, at_starts = 0, at_sums = 0, total = 0;  // tickets first
  bool chained = false;
};
int64_t up256(int64_t v) { return round_up(v, 256); }
Plan plan_of(const RecurArgs& a, bool sums, int rows = kRecurRows) {
  Plan p;
  const int64_t G = 2 * ((a.C + 127) / 128);  // (64 channels each, or half as many of 128)
  const int64_t tiles = (a.L + rows - 1) / rows;
  p.slots = a.seq_starts ? a.B * a.L / rows + a.S : a.B * std::max<int64_t>(tiles, 1);
  p.chained = a.seq_starts || tiles > 1;
  p.at_values = p.chained ? up256(4 * G * kTicketStride) : 0;
  p.at_starts = p.at_values + (p.chained ? up256(G * p.slots * 64 * 8) : 0);
  p.at_sums = p.at_starts + (a.seq_starts ? up256(4 * (a.S + 1)) : 0);
  p.total = p.at_sums + (sums ? up256(4 * p.slots * a.C) : 0);
  return p;
}

Chain chain_of(const RecurArgs& a, const Plan& p, void* ws, int cpt, int rows = kRecurRows) {
  Chain c;
  char* base = static_cast<char*>(ws);
  c.slots = static_cast<int>(p.slots);
  c.G = static_cast<int>((a.C + 64 * cpt - 1) / (64 * cpt));
  c.tiles = static_cast<int>(std::max<int64_t>(1, (a.L + rows - 1) / rows));
  c.kept = static_cast<int>(std::max<int64_t>(1, (a.L + kRecurRows - 1) / kRecurRows));
  c.spin_limit = g_spin_limit;
  if (p.chained) {
    c.tickets = reinterpret_cast<unsigned*>(base);
    c.values = reinterpret_cast<unsigned long long*>(base + p.at_values);
  }
  if (a.seq_starts) c.starts = reinterpret_cast<int32_t*>(base + p.at_starts);
  return c;
}

int reset(const RecurArgs& a, const Plan& p, const Chain& c, int cpt, RestArgs rest, hipStream_t st) {
  if (!p.chained) return kOk;
  const int64_t n_tickets = static_cast<int64_t>(c.G) * kTicketStride / 4, n_values = c.G * p.slots * 64 * cpt / 2;
  const unsigned blocks = static_cast<unsigned>((n_tickets + n_values + 255) / 256 + (a.seq_starts ? 1 : 0));
  recur_reset_kernel<<<blocks, 256, 0, TESM_LOGGED(st, recur_reset_kernel)>>>(
      reinterpret_cast<uint4*>(c.tickets), n_tickets, reinterpret_cast<uint4*>(c.values), n_values, a.seq_starts, a.S + 1, a.B * a.L,
      const_cast<int32_t*>(c.starts));
  if (a.seq_starts && a.zero_rest && a.B * a.L > 0) {
    rest.C = a.C, rest.rows = a.B * a.L, rest.S = a.S;
    rest.starts = c.starts;
    const unsigned n = static_cast<unsigned>(std::min<int64_t>(a.B * a.L, 4096));
    if (a.dt == kBF16)
      recur_rest_kernel<kBF16><<<n, 256, 0, TESM_LOGGED(st, recur_rest_kernel<kBF16>)>>>(rest);
    else
      recur_rest_kernel<kF32><<<n, 256, 0, TESM_LOGGED(st, recur_rest_kernel<kF32>)>>>(rest);
  }
  return kOk;
}

// Two channels per lane once the tiles of 128 channels are four per CU; before that twice as many of 64 hide more of their
// waits (4 x 2048 rows of 384 channels forward 11.0 us and 14.4, backward 15.7 and 18.7).
bool many_tiles(const RecurArgs& a) {
  return plan_of(a, false).slots * ((a.C + 127) / 128) >= 4 * static_cast<int64_t>(std::max(device_limits().cus, 1));
}

}  // namespace

int64_t recur_slots(const RecurArgs& a) { return recur_check(a) == kOk ? plan_of(a, false).slots : -1; }
int64_t recur_ws_bytes(const RecurArgs& a) { return recur_check(a) == kOk ? plan_of(a, false).total : -1; }
int64_t recur_bwd_ws_bytes(const RecurArgs& a, bool bias) { return recur_check(a) == kOk ? plan_of(a, bias).total : -1; }

int launch_gated_scan(const RecurArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (int rc = recur_check(a)) return rc;
  if (a.C == 0) return kOk;
  if (a.S == 0) {  // (no sequence: every row is of none)
    TESM_REQUIRE(!a.zero_rest || a.B * a.L == 0, kErrUnsupported, "gated scan: zero_rest needs a sequence");
    return kOk;
  }
  const bool rows = a.B * a.L > 0;
  TESM_REQUIRE(a.h_out && (!rows || (a.value && a.write && a.decay && a.h)), kErrInvalidArg, "gated scan: need the gates, h and h_out");
  TESM_REQUIRE(!rows || (a.ld_v >= a.C && a.ld_w >= a.C && a.ld_d >= a.C && a.ld_h >= a.C), kErrInvalidArg,
               "gated scan: a row pitch below the channels");
  const Plan small = plan_of(a, false);
  TESM_REQUIRE(small.total == 0 || (ws && ws_bytes >= small.total && aligned(ws, 16)), kErrWorkspace,
               "gated scan: workspace too small or not 16-byte aligned");
  const bool pairs = many_tiles(a) && in_pairs(a.dt, a.C, {{a.value, a.ld_v}, {a.write, a.ld_w}, {a.decay, a.ld_d}, {a.h, a.ld_h}});
  // Tiles of 128 rows where the call's four arrays are more than the last cache holds and sequences are long: half as many hand-overs, and
  // twice the loads under way (us with 64 rows and with 128: 1 x 32768 x 8192 525 and 492, of 8190 channels 577 and 551; smaller arrays
  // 4 x 2048 x 2048 37.1 and 37.5; short sequences, where half a tile may stay empty, 64 x 192 x 8192 185 and 208).
  const int64_t all_rows = a.B * a.L;
  const bool tall = pairs && all_rows * a.C * 2 * 4 > (256LL << 20) && all_rows >= 1024 * a.S;
  const int tile = tall ? 2 * kRecurRows : kRecurRows;
  const Plan p = plan_of(a, false, tile);
  const Chain c = chain_of(a, p, ws, pairs ? 2 : 1, tile);
  const int64_t blocks = p.slots * c.G;
  TESM_REQUIRE(fits_grid(blocks, 64 * kWaves), kErrUnsupported, "gated scan: too many tiles for one call");
  if (int rc = reset(a, p, c, pairs ? 2 : 1, RestArgs{{a.h}, {a.ld_h}}, st)) return rc;
  const unsigned n = static_cast<unsigned>(blocks);
#define TESM_RECUR(DT, CPT, T) recur_fwd_kernel<DT, CPT, T><<<n, 64 * kWaves, 0, TESM_LOGGED(st, recur_fwd_kernel<DT, CPT, T>)>>>(a, c)
  if (a.dt == kF32)
    TESM_RECUR(kF32, 1, 8);
  else if (tall)
    TESM_RECUR(kBF16, 2, 16);
  else if (pairs)
    TESM_RECUR(kBF16, 2, 8);
  else
    TESM_RECUR(kBF16, 1, 8);
#undef TESM_RECUR
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
  TESM_REQUIRE(p.total == 0 || (ws && ws_bytes >= p.total && aligned(ws, 16)), kErrWorkspace,
               "gated scan backward: workspace too small or not 16-byte aligned");
  const bool pairs = many_tiles(a) && in_pairs(a.dt, a.C, {{a.value, a.ld_v}, {a.write, a.ld_w}, {a.decay, a.ld_d}, {b.grad, b.ld_g},
                                          {b.d_value, b.ld_dv}, {b.d_write, b.ld_dw}, {b.d_decay, b.ld_dd}});
  const Chain c = chain_of(a, p, ws, pairs ? 2 : 1);
  const int64_t blocks = a.S ? p.slots * c.G : 0;
  TESM_REQUIRE(fits_grid(blocks, 64 * kWaves), kErrUnsupported, "gated scan backward: too many tiles for one call");
  float* sums = b.d_bias ? reinterpret_cast<float*>(static_cast<char*>(ws) + p.at_sums) : nullptr;
  if (blocks > 0) {
    if (int rc = reset(a, p, c, pairs ? 2 : 1, RestArgs{{b.d_value, b.d_write, b.d_decay}, {b.ld_dv, b.ld_dw, b.ld_dd}}, st)) return rc;
    const unsigned n = static_cast<unsigned>(blocks);
#define TESM_RECUR(DT, CPT) recur_bwd_kernel<DT, CPT><<<n, 64 * kWaves, 0, TESM_LOGGED(st, recur_bwd_kernel<DT, CPT>)>>>(b, c, sums)
    if (a.dt == kF32)
      TESM_RECUR(kF32, 1);
    else if (pairs)
      TESM_RECUR(kBF16, 2);
    else
      TESM_RECUR(kBF16, 1);
#undef TESM_RECUR
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
