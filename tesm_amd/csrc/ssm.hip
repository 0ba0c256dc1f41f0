// Selective state space scan of a multi-head layer.  Per head h with its group's B and C, per row t:
//   d_t = softplus(dt_t + dt_bias)        a_t = exp(d_t A)
//   h_t = a_t h_{t-1} + d_t x_t B_t^T     (P x N, float32)
//   y_t = h_t C_t + D x_t                 times silu(z_t) where there is a gate
#include <type_traits>

#include "ssm.h"
#include "ssm_chunk.h"

namespace tesm {

namespace {

// log(1 + e^v) = max(v, 0) + log(1 + u), u = e^-|v|, and with s = u / (2 + u) <= 1/3 the logarithm is 2 artanh(s) =
// 2 s (1 + s^2 / 3 + s^4 / 5 + ..), cut after s^12 (what is left is below 2e-8 of it).  NaN stays NaN.
__device__ __forceinline__ float softplusf_(float v) {
  const float u = fast_exp(-fabsf(v));
  const float s = u * __builtin_amdgcn_rcpf(2.0f + u), s2 = s * s;
  float p = 1.0f / 13.0f;
  p = __builtin_fmaf(p, s2, 1.0f / 11.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 9.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 7.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 5.0f);
  p = __builtin_fmaf(p, s2, 1.0f / 3.0f);
  p = __builtin_fmaf(p, s2, 1.0f);
  return (v < 0.0f ? 0.0f : v) + (v == -__builtin_inff() || v == __builtin_inff() ? 0.0f : 2.0f * s * p);
}
// silu for a bfloat16 result: the exponent's rounding (2^-24 |v| log2 e) is far below the result's, so it is taken as it is.
template <int DT>
__device__ __forceinline__ float gatef_(float v) {
  if constexpr (DT == kF32) return siluf_(v);
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// The scan in chunks of 32 rows.  With c_i the sum of d A over the chunk's rows up to i, and h the state on entry:
//   Y = W X + exp(c) C h,   W_ij = (C_i . B_j) exp(c_i - c_j) d_j for j <= i, else 0
//   h' = exp(c_Q) h + sum_j exp(c_Q - c_j) d_j x_j B_j^T
// so that all of it is matrix products.  A workgroup of 4 waves walks a segment of one sequence for 128 columns of one
// group (4 slices of 32 columns, each inside one head, one per wave); a wave keeps its slice's state in its
// accumulators.  The products are formed transposed, with the state's layout in mind:
//   scores  S^T = B C^T   (shared by the heads of the workgroup), scaled to W and kept in LDS, a matrix per head
//   Y^T     = h C^T, scaled by exp(c_i) per column, + X^T W^T
//   h       = exp(c_Q) h + B^T (w x)
// where a result's lane holds 4 consecutive rows of one column.  Rows of a 32-wide block are taken in the order
// row m of tile T  <->  8 (m / 4) + 4 T + m % 4: two tiles of the state are then the 8 consecutive states per lane that
// the next product's operand needs, with no exchange, and two tiles of Y are 8 consecutive columns of one row, one
// 16-byte store.
//
// A chunk's x, B and C come through registers, read one chunk ahead, into LDS (two chunks' worth for bfloat16, so that
// one barrier separates a chunk's writes from its reads; float32 rows fill it with one).  Three of the waves form the
// scores; the fourth meanwhile forms d and the sums c of the next chunk (in 64 bits: c is a difference's operand, and is
// kept as a high and a low float).  With bfloat16 operands W and the h that C reads go into their products as two bfloat16
// parts each, which leaves y the error of its own rounding; the state takes its addends in three parts, unrounded.  (One
// rounded part each: y's error 1.9e-3 of it instead of 1.7e-3, with narrow states 2.3e-3, single values up to 30 times what
// the formula in float32 leaves, for 72 us instead of 78 and 800 instead of 880.)
//
// Bound by the vector unit first: with 128 bfloat16 states a wave issues some 800 of its instructions per chunk, 91
// matrix ones among them and the exponentials and reciprocals at a quarter of the rate.  Counters over 32768 rows: the
// vector unit issues in 63 % of the cycles, the matrix unit works in 27 %, LDS conflicts take 10 %; a wave waits for an issue
// slot in 29 % of its time and for memory, LDS or one of the two barriers per chunk in 22 %, which the two waves per SIMD that
// the state's and the next operands' registers leave do not cover for each other.  Chunks of 64 rows
// (one staged, with the work inside a chunk doubled) took 628 us where these took 520.  Measured, bfloat16 with 128
// states: 4 x 2048 rows of 1536 columns 50 us + 31 for the states of the segments, 32768 rows of 8192 columns (1.76 GB)
// 676 + 271 us, 1.9 TB/s.
// ---------------------------------------------------------------------------
constexpr int kCols = 128;  // columns per workgroup

template <int DT>
struct Tile;
template <>
struct Tile<kBF16> {
  using E = uint16_t;
  static constexpr int EV = 8, PAD = 8, NB = 2;  // elements per 16 bytes, padding, chunks staged at once
  // Rows of U 16-byte units (4, 8, 16 or 32) lie one behind the other without padding; unit u of row r is kept at
  // u ^ swz(r).  Then the 8 rows of one unit that a row operand reads at once, and the 4 rows x 4 units of a column
  // operand, fall on different banks (64 of 4 bytes).
  template <int U>
  static __device__ __forceinline__ int swz(int r) {
    const int block = U >= 16 ? r & 3 : U == 8 ? (r >> 1) & 1 : 0;
    return block << 2 | ((r >> 2) & 3);
  }
  template <int U>
  static constexpr int pitch() { return U * EV; }
  template <int U>
  static __device__ __forceinline__ int unit(int r, int u) { return r * U * EV + (u ^ swz<U>(r)) * EV; }
  using Frag = uint4;  // 8 consecutive k of one row: lane l holds row l & 15, k = 8 (l >> 4) ..
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ Frag row(const E* p) { return *reinterpret_cast<const uint4*>(p); }
  // Rows r0 + m (r0 a multiple of 16), columns 32 s + 8 g .. + 7
  template <int U>
  static __device__ __forceinline__ Frag rows(const E* p, int r0, int m, int g, int s) {
    return row(p + r0 * U * EV + unit<U>(m, 4 * s + g));
  }
  // Rows r0 + 8 g .. + 7 (r0 a multiple of 16), one column per lane: 32 s + 8 (m / 4) + 4 T + m % 4
  template <int U>
  static __device__ __forceinline__ Frag column(const E* p, int r0, int m, int g, int s, int T) {
    const int r = 8 * g + (m >> 2);  // the lane's place: 4 columns of row m / 4, then of the row 4 below
    const uint2 a = tr(p + r0 * U * EV + unit<U>(r, 4 * s + (m & 3)) + 4 * T);
    const uint2 b = tr(p + r0 * U * EV + unit<U>(r + 4, 4 * s + (m & 3)) + 4 * T);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  static __device__ __forceinline__ uint2 tr(const E* p) {
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
    return __builtin_bit_cast(uint2, v);
  }
  static __device__ __forceinline__ Frag pack(const f32x4& lo, const f32x4& hi) {
    return make_uint4(pack_bf16x2(lo[0], lo[1]), pack_bf16x2(lo[2], lo[3]), pack_bf16x2(hi[0], hi[1]),
                      pack_bf16x2(hi[2], hi[3]));
  }
  static __device__ __forceinline__ void unpack(const Frag& f, float (&v)[8]) {
    const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  // Float32 values as two bfloat16 parts: the first cut off, the second what that leaves, rounded (2^-15 of the value off).
  static constexpr int PARTS = 2;
  static __device__ __forceinline__ uint2 cut(const f32x4& v, f32x4& rest) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[i] = __float_as_uint(v[i]);
      rest[i] = v[i] - __uint_as_float(b[i] & 0xffff0000u);
    }
    return make_uint2(__builtin_amdgcn_perm(b[1], b[0], 0x07060302), __builtin_amdgcn_perm(b[3], b[2], 0x07060302));
  }
  static __device__ __forceinline__ void parts(const f32x4& lo, const f32x4& hi, Frag (&f)[PARTS]) {
    f32x4 a, b;
    const uint2 u = cut(lo, a), v = cut(hi, b);
    f[0] = make_uint4(u.x, u.y, v.x, v.y);
    f[1] = pack(a, b);
  }
  static __device__ __forceinline__ void store4(E* p, int part_pitch, const f32x4& v) {
    f32x4 rest;
    *reinterpret_cast<uint2*>(p) = cut(v, rest);
    *reinterpret_cast<uint2*>(p + part_pitch) = make_uint2(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]));
  }
};
template <>
struct Tile<kF32> {
  using E = float;
  static constexpr int EV = 4, PAD = 4, NB = 1;
  template <int U>
  static constexpr int pitch() { return U * EV + PAD; }
  template <int U>
  static __device__ __forceinline__ int unit(int r, int u) { return r * pitch<U>() + u * EV; }
  struct Frag {
    float v[8];
  };
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag row(const E* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    return Frag{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
  }
  template <int U>
  static __device__ __forceinline__ Frag rows(const E* p, int r0, int m, int g, int s) {
    return row(p + (r0 + m) * pitch<U>() + 32 * s + 8 * g);
  }
  template <int U>
  static __device__ __forceinline__ Frag column(const E* p, int r0, int m, int g, int s, int T) {
    const E* q = p + (r0 + 8 * g) * pitch<U>() + 32 * s + 8 * (m >> 2) + 4 * T + (m & 3);
    Frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = q[e * pitch<U>()];
    return f;
  }
  static __device__ __forceinline__ Frag pack(const f32x4& lo, const f32x4& hi) {
    return Frag{{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
  }
  static __device__ __forceinline__ void unpack(const Frag& f, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f.v[i];
  }
  static constexpr int PARTS = 1;
  static __device__ __forceinline__ void parts(const f32x4& lo, const f32x4& hi, Frag (&f)[PARTS]) { f[0] = pack(lo, hi); }
  static __device__ __forceinline__ void store4(E* p, int, const f32x4& v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
};

// The compiler is to form what depends on h, and what is read from memory, anew from here on (kept values would have
// to be spilled).
template <int NS>
__device__ __forceinline__ void anew(f32x4 (&h)[NS][2][2]) {
#pragma unroll
  for (int s = 0; s < NS; ++s) asm volatile("" : "+v"(h[s][0][0]), "+v"(h[s][0][1]), "+v"(h[s][1][0]), "+v"(h[s][1][1])::"memory");
}

typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any address of an element
__device__ __forceinline__ uint4 load16(const void* p) { return __builtin_bit_cast(uint4, *static_cast<const any16*>(p)); }
__device__ __forceinline__ void store16(void* p, const uint4& v) { *static_cast<any16*>(p) = __builtin_bit_cast(any16, v); }

// How the launch divides the work.
struct SsmGrid {
  int64_t seg = 0;      // rows per segment, a multiple of 64
  int64_t slots = 0;    // segments of all sequences (packed: at most)
  int ps = 0, sg = 0;   // slices per head, per group
  int wpg = 0;          // workgroups per group
  int nh = 0;           // heads per workgroup, at most
  float* carry = nullptr;  // (slots, G * wpg, kCols * 32 NS): a segment's end state, in accumulator order
  float* decay = nullptr;  // (slots, H): the product of its decays
};

struct Segment {  // uniform over the workgroup, in scalar registers
  int seq, k, r0, r1;  // sequence, its k-th segment, rows
  bool last, valid;
};

__device__ __forceinline__ int64_t segments_of(int64_t len, int64_t seg) { return len <= seg ? 1 : (len + seg - 1) / seg; }

// Segment `slot`, counted through the sequences; every sequence has one at least.
__device__ __forceinline__ Segment find_segment(const SsmArgs& a, const SsmGrid& gr, int slot) {
  Segment s;
  int64_t first, end;
  int seq = 0, k = 0;
  bool valid = true;
  if (!a.seq_starts) {
    const int n = static_cast<int>(segments_of(a.L, gr.seg));
    seq = slot / n;
    k = slot - seq * n;
    first = seq * a.L;
    end = first + a.L;
  } else {
    const int lane = threadIdx.x & 63;
    const int64_t M = a.B * a.L;
    int before = 0;
    valid = false;
    for (int base = 0; base < static_cast<int>(a.S) && !valid; base += 64) {
      int n = 0;
      if (base + lane < a.S) {
        seq_rows(a.seq_starts, base + lane, M, first, end);
        n = static_cast<int>(segments_of(end - first, gr.seg));
      }
      int upto = n;
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
      const uint64_t past = __ballot(before + upto > slot);
      if (past) {
        const int l = __ffsll(static_cast<long long>(past)) - 1;
        seq = base + l;
        k = slot - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
        valid = true;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (valid)
      seq_rows(a.seq_starts, seq, M, first, end);
    else
      first = end = 0;
  }
  s.valid = valid;
  s.seq = __builtin_amdgcn_readfirstlane(seq);
  s.k = __builtin_amdgcn_readfirstlane(k);
  const int64_t r0 = first + k * gr.seg, r1 = r0 + gr.seg < end ? r0 + gr.seg : end;
  s.r0 = __builtin_amdgcn_readfirstlane(static_cast<int>(r0));
  s.r1 = __builtin_amdgcn_readfirstlane(static_cast<int>(r1));
  s.last = s.r1 >= __builtin_amdgcn_readfirstlane(static_cast<int>(end));
  return s;
}

// EV elements of a row from column `col` of `count`, zeros past its end.
template <int DT>
__device__ __forceinline__ uint4 load_unit(const void* p, int64_t at, int col, int count) {
  using TT = Tile<DT>;
  using E = typename TT::E;
  const E* q = static_cast<const E*>(p) + at + col;
  if (col + TT::EV <= count) return load16(q);
  E v[TT::EV];
#pragma unroll
  for (int i = 0; i < TT::EV; ++i) v[i] = col + i < count ? q[i] : E(0);
  uint4 o;
  __builtin_memcpy(&o, v, 16);
  return o;
}

__device__ __forceinline__ double readlane_d(double v, int l) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(b), l);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), l);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Inclusive sums over each half of the wave: shifts inside rows of 16 lanes, then the total of the row before.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double half_scan_d(double v) {
  v = dpp_add<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = dpp_add<0x112, 0xF>(v);
  v = dpp_add<0x114, 0xF>(v);
  v = dpp_add<0x118, 0xF>(v);
  return dpp_add<0x142, 0xA>(v);  // lane 15 of the row before, to rows 1 and 3
}

template <int DT, int NS, bool FULL>
struct SsmLds {
  using TT = Tile<DT>;
  static constexpr int UX = kCols / TT::EV, UB = 32 * NS / TT::EV;  // 16-byte units per row
  static constexpr int XP = TT::template pitch<UX>(), NP = TT::template pitch<UB>(), WP = kQ + TT::PAD;
  static constexpr int kStage = kQ * (XP + (FULL ? 2 : 1) * NP);  // x, B and C of a chunk
  static constexpr int kSmall = 6 * kQ;  // per head: c high, c low, d, exp(c_Q - c) d, exp(c), and exp(c_Q) at 5 kQ
  static constexpr int64_t bytes(int nh) {
    const int64_t e = sizeof(typename TT::E);
    return TT::NB * kStage * e + (FULL ? TT::PARTS * nh * kQ * WP * e : 0) + 2 * nh * kSmall * 4;
  }
};

// FULL: y and the final state of a segment from its carried-in state; otherwise the segment's end state from zero.
// VEC: whole 32-column slices and 32-state steps, and 32-bit offsets inside a chunk.
// (Two waves per SIMD also where float32 operands with 128 states then spill 37 registers, 40 with edges: 14 sequences of 600
// rows and 24 heads 179 us, with one wave and no spill 186; 256 states need the registers of one and spill 4 to 10 with float32
// operands.  The states' pass with float32 operands and 128 states spills 1 register, 15 with edges.)
template <int DT, int NS, bool FULL, bool VEC>
__global__ __launch_bounds__(256, NS == 8 ? 1 : FULL ? 2 : 3) void ssm_chunk_kernel(SsmArgs a, SsmGrid gr) {
  using TT = Tile<DT>;
  using E = typename TT::E;
  using Frag = typename TT::Frag;
  using Lds = SsmLds<DT, NS, FULL>;
  constexpr int EV = TT::EV, NB = TT::NB, WP = Lds::WP, UX = Lds::UX, UB = Lds::UB;
  using XU = ChunkUnits<UX>;
  using BU = ChunkUnits<UB>;
  constexpr int XR = XU::kEach, BR = BU::kEach;  // units per thread
  extern __shared__ __attribute__((aligned(16))) char lds_s[];
  E* const stages = reinterpret_cast<E*>(lds_s);
  E* const Ws = stages + NB * Lds::kStage;
  constexpr int PARTS = TT::PARTS;
  const int wpart = gr.nh * kQ * WP;  // from W's first parts to its second
  float* const smalls = reinterpret_cast<float*>(Ws + (FULL ? PARTS * wpart : 0));

  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Segment sg = find_segment(a, gr, blockIdx.y);
  if (!sg.valid || (!FULL && sg.last)) return;
  const int grp = blockIdx.x / gr.wpg, wgi = blockIdx.x % gr.wpg;
  const int hg = static_cast<int>(a.H / a.G);
  const int N = static_cast<int>(a.N), P = static_cast<int>(a.P);
  // this wave's slice, and the heads of the workgroup
  const int sl = wgi * 4 + wave, head0 = wgi * 4 / gr.ps;  // within the group
  const bool active = sl < gr.sg;
  const int last_sl = min(wgi * 4 + 3, gr.sg - 1), nh = last_sl / gr.ps - head0 + 1;
  const int hh = active ? sl / gr.ps - head0 : 0, head = grp * hg + head0 + hh, p0 = (sl % gr.ps) * 32;
  // this thread's column of x and of B and C
  const int xc = (tid % UX) * EV, xsl = wgi * 4 + xc / 32, xhead = xsl / gr.ps, xp = (xsl % gr.ps) * 32 + xc % 32;
  const bool xok = xsl < gr.sg;
  const int bc = (tid % UB) * EV;

  // state: tile (s, T2) of rows n = 32 s + 8 (m / 4) + 4 T2 + m % 4, tile T of columns p0 + 8 (m / 4) + 4 T + m % 4;
  // this lane: states 32 s + 8 g + 4 T2 .. + 3 of column p0 + 8 (m / 4) + 4 T + m % 4
  f32x4 h[NS][2][2];
  const int64_t frags = static_cast<int64_t>(NS) * 4 * 64;  // vectors of 4 per wave
  const int64_t wg_all = static_cast<int64_t>(gr.wpg) * a.G;
  const f32x4* carry_in = nullptr;
  if (FULL && sg.k > 0)
    carry_in = reinterpret_cast<const f32x4*>(gr.carry) + (((blockIdx.y - 1) * wg_all + blockIdx.x) * 4 + wave) * frags;
#pragma unroll
  for (int s = 0; s < NS; ++s)
#pragma unroll
    for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        h[s][t2][T] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!FULL || !active) continue;
        if (carry_in) {
          h[s][t2][T] = carry_in[((s * 2 + t2) * 2 + T) * 64 + lane];
        } else if (a.h0) {
          const int p = p0 + 8 * (m >> 2) + 4 * T + (m & 3), n = 32 * s + 8 * g + 4 * t2;
          const float* src = a.h0 + (static_cast<int64_t>(sg.seq) * a.H + head) * P * N + p * N + n;
          if (VEC || (p < P && n + 4 <= N)) {
            h[s][t2][T] = __builtin_bit_cast(f32x4, load16(src));
          } else {
#pragma unroll
            for (int r = 0; r < 3; ++r)
              if (p < P && n + r < N) h[s][t2][T][r] = src[r];
          }
        }
      }

  // A chunk's units, one chunk ahead of their use: uniform bases and 32-bit offsets.  Rows past the end read the last one
  // and are cleared when staged.
  uint4 xr[XR], br[BR], cr[FULL ? BR : 1], zr[2][8 / EV];
  const int64_t es = sizeof(E), gn = static_cast<int64_t>(grp) * N, hp = static_cast<int64_t>(head) * P;
  const bool xin = VEC ? xok : xok && xp < P, bin = VEC || bc < N;
  // at: the uniform address of the chunk's first row and the operand's first column here, moved on chunk by chunk
  const char* xat = static_cast<const char*>(a.x) + (sg.r0 * a.ld_x + static_cast<int64_t>(grp * hg + head0) * P) * es;
  const char* bat = static_cast<const char*>(a.Bm) + (sg.r0 * a.ld_b + gn) * es;
  const char* cat = static_cast<const char*>(a.Cm) + (sg.r0 * a.ld_c + gn) * es;
  const char* zat = static_cast<const char*>(a.z) + (sg.r0 * a.ld_z + hp + p0) * es;
  char* yat = static_cast<char*>(a.y) + (sg.r0 * a.ld_y + hp + p0) * es;
  const uint32_t px = static_cast<uint32_t>(a.ld_x * es), pb = static_cast<uint32_t>(a.ld_b * es), pc = static_cast<uint32_t>(a.ld_c * es);
  const uint32_t pz = static_cast<uint32_t>(a.ld_z * es), py = static_cast<uint32_t>(a.ld_y * es);
  auto load_rows = [&](const char* at, uint32_t pitch, int last, auto whole, int r, int col, int count, bool in) __attribute__((always_inline)) {
    const uint32_t off = static_cast<uint32_t>(chunk_source(whole.value, r, last)) * pitch;
    if constexpr (VEC) return load16(at + (off + static_cast<uint32_t>(col * sizeof(E))));
    return in ? load_unit<DT>(at + off, 0, col, count) : make_uint4(0, 0, 0, 0);
  };
  const int xcol = xok ? (xhead - head0) * P + xp : 0;
  auto load_as = [&](int row0, auto whole) __attribute__((always_inline)) {
    const int last = sg.r1 - 1 - row0;
#pragma unroll
    for (int i = 0; i < XR; ++i)
      xr[i] = load_rows(xat, px, last, whole, XU::row(tid, i), xcol, xcol - xp + P, xin);
#pragma unroll
    for (int i = 0; i < BR; ++i) {
      br[i] = load_rows(bat, pb, last, whole, BU::row(tid, i), bc, N, bin);
      if constexpr (FULL) cr[i] = load_rows(cat, pc, last, whole, BU::row(tid, i), bc, N, bin);
    }
    if (FULL && a.z && active) {  // the gate of this lane's outputs
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int k = 0; k < 8 / EV; ++k)
          zr[q][k] = load_rows(zat, pz, last, whole, 16 * q + m, 8 * g + k * EV, P - p0, p0 + 8 * g + k * EV < P);
    }
    xat += kQ * static_cast<int64_t>(px);
    bat += kQ * static_cast<int64_t>(pb);
    if constexpr (FULL) {
      cat += kQ * static_cast<int64_t>(pc);
      zat += kQ * static_cast<int64_t>(pz);
    }
  };
  auto load_chunk = [&](int row0) __attribute__((always_inline)) {
    if (row0 + kQ <= sg.r1)
      load_as(row0, std::true_type{});
    else
      load_as(row0, std::false_type{});
  };

  // d and the sums c of a chunk, formed by one wave for two heads at a time, 32 lanes each, while the others work on the
  // chunk before; dt is read two chunks ahead.
  uint32_t dtr[2] = {0, 0};
  float Ar[2] = {0.0f, 0.0f}, biasr[2] = {0.0f, 0.0f};
  const int dh = lane >> 5;
  auto load_dt = [&](int row0) __attribute__((always_inline)) {
    const int r = min(row0 + (lane & 31), sg.r1 - 1);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (2 * k + dh < nh) dtr[k] = ld_bits<DT>(a.dts, r * a.ld_dt + grp * hg + head0 + 2 * k + dh);
  };
  auto sums = [&](int row0, float* to) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (2 * k >= nh) break;
      const float raw = from_bits<DT>(dtr[k]) + biasr[k];
      const float d = row0 + (lane & 31) < sg.r1 ? (a.softplus ? softplusf_(raw) : raw) : 0.0f;
      // in units of log 2, 64 bits split into two floats.  A row below -2^16 clears the state like one of -2^16 (no growth that
      // float32 holds makes up for either), which leaves the sums' last bits to the rows around it.
      double each = static_cast<double>(d) * static_cast<double>(Ar[k]) * 1.4426950408889634074;
      if (each < -0x1p16) each = -0x1p16;
      const double c = half_scan_d(each);
      const double all = dh ? readlane_d(c, 63) : readlane_d(c, 31);
      if (2 * k + dh < nh) {
        float* sm = to + (2 * k + dh) * Lds::kSmall + (lane & 31);
        const float hi = static_cast<float>(c), lo = static_cast<float>(c - static_cast<double>(hi));
        sm[0] = hi;
        sm[kQ] = lo;
        sm[2 * kQ] = d;
        sm[3 * kQ] = __builtin_amdgcn_exp2f(static_cast<float>(all - c)) * d;
        sm[4 * kQ] = __builtin_amdgcn_exp2f(hi);
        if ((lane & 31) == 0) sm[5 * kQ] = __builtin_amdgcn_exp2f(static_cast<float>(all));
      }
    }
  };

  float decay = 1.0f;  // of the segment so far (this wave's head)
  float scale = 1.0f;  // of h
  const float skip = FULL && a.D && active ? a.D[head] : 0.0f;
  if (sg.r0 < sg.r1) {
    load_chunk(sg.r0);
    if (wave == 3) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (2 * k + dh < nh) {
          Ar[k] = a.A[grp * hg + head0 + 2 * k + dh];
          if (a.dt_bias) biasr[k] = a.dt_bias[grp * hg + head0 + 2 * k + dh];
        }
      load_dt(sg.r0);
      sums(sg.r0, smalls);
      load_dt(sg.r0 + kQ);
    }
    if constexpr (FULL) {  // the block of W above the diagonal that a 32-wide step reads: zero throughout
      for (int e = tid; e < PARTS * gr.nh * 256; e += 256) Ws[((e >> 8) * kQ + ((e >> 4) & 15)) * WP + 16 + (e & 15)] = E(0);
    }
  }
  int buf = 0;
  for (int row0 = sg.r0; row0 < sg.r1; row0 += kQ, buf ^= 1) {
    const int left = sg.r1 - row0;
    E* const X = stages + (NB == 2 ? buf * Lds::kStage : 0);
    E* const Bs = X + kQ * Lds::XP;
    E* const Cs = Bs + kQ * Lds::NP;
    const float* const sw = smalls + buf * gr.nh * Lds::kSmall;
    float* const next = smalls + (buf ^ 1) * gr.nh * Lds::kSmall;
    if (left < kQ) {
#pragma unroll
      for (int i = 0; i < XR; ++i)
        if (XU::row(tid, i) >= left) xr[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < BR; ++i)
        if (BU::row(tid, i) >= left) {
          br[i] = make_uint4(0, 0, 0, 0);
          if constexpr (FULL) cr[i] = make_uint4(0, 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < XR; ++i) *reinterpret_cast<uint4*>(X + TT::template unit<UX>(XU::row(tid, i), tid % UX)) = xr[i];
#pragma unroll
    for (int i = 0; i < BR; ++i) {
      if (!BU::stages(tid)) break;
      const int at = TT::template unit<UB>(BU::row(tid, i), tid % UB);
      *reinterpret_cast<uint4*>(Bs + at) = br[i];
      if constexpr (FULL) *reinterpret_cast<uint4*>(Cs + at) = cr[i];
    }
    uint4 zc[2][8 / EV];
    if constexpr (FULL) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int k = 0; k < 8 / EV; ++k) zc[q][k] = zr[q][k];
    }
    lds_barrier();
    if (left > kQ) load_chunk(row0 + kQ);
    const float* const sm = sw + hh * Lds::kSmall;
    if (wave == 3) {
      if (left > kQ) {
        sums(row0 + kQ, next);
        if (left > 2 * kQ) load_dt(row0 + 2 * kQ);
      }
    } else if (FULL) {
      // scores: one 16 x 16 tile (it, jt) of the lower triangle per wave, then W of every head of the workgroup
      const int it = wave ? 1 : 0, jt = wave == 2 ? 1 : 0;
      f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NS; ++k)
        sc = TT::mma(TT::template rows<UB>(Bs, 16 * jt, m, g, k), TT::template rows<UB>(Cs, 16 * it, m, g, k), sc);
      const int i = 16 * it + m, j0 = 16 * jt + 4 * g;
      for (int w = 0; w < nh; ++w) {
        const float* const s = sw + w * Lds::kSmall;
        // the low halves of the sums matter where the sums are large against the result's own rounding
        const bool low = DT == kF32 || !(__builtin_amdgcn_readfirstlane(__float_as_int(fabsf(s[kQ - 1]))) < __float_as_int(512.0f));
        const float hi = s[i];
        const f32x4 hj = *reinterpret_cast<const f32x4*>(s + j0), dj = *reinterpret_cast<const f32x4*>(s + 2 * kQ + j0);
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = hi - hj[r];
        if (low) {
          const float lo = s[kQ + i];
          const f32x4 lj = *reinterpret_cast<const f32x4*>(s + kQ + j0);
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] += lo - lj[r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = sc[r] * __builtin_amdgcn_exp2f(v[r]) * dj[r];
        if (it == jt) {  // on the diagonal
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (j0 + r > i) v[r] = 0.0f;
        }
        TT::store4(Ws + (w * kQ + i) * WP + j0, wpart, v);
      }
    }
    Frag xf[2];  // x of this wave's columns, 8 rows of a column per lane
    if (active) {
#pragma unroll
      for (int T = 0; T < 2; ++T) xf[T] = TT::template column<UX>(X, 0, m, g, wave, T);
    }
    if constexpr (FULL) {
      f32x4 y[2][2];
      // exp(c_i) C_i . h
      auto across = [&]() __attribute__((always_inline)) {
        anew(h);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int T = 0; T < 2; ++T) y[q][T] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          Frag h0[PARTS], h1[PARTS];
          TT::parts(h[s][0][0], h[s][1][0], h0);
          TT::parts(h[s][0][1], h[s][1][1], h1);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const Frag c = TT::template rows<UB>(Cs, 16 * q, m, g, s);
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
              y[q][0] = TT::mma(h0[part], c, y[q][0]);
              y[q][1] = TT::mma(h1[part], c, y[q][1]);
            }
          }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float e = sm[4 * kQ + 16 * q + m] * scale;
          y[q][0] *= e;
          y[q][1] *= e;
        }
      };
      if (active) across();
      lds_barrier();
      if (active) {
        // + W x over the rows up to each
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            const Frag w = TT::row(Ws + part * wpart + (hh * kQ + 16 * q + m) * WP + 8 * g);
            y[q][0] = TT::mma(xf[0], w, y[q][0]);
            y[q][1] = TT::mma(xf[1], w, y[q][1]);
          }
        // An infinite or NaN x must not reach the rows before it through a weight 0.  Rows with one near have sums
        // that are not finite: they are formed again without such values, which are then added from their row on.
        bool odd = false;
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int T = 0; T < 2; ++T)
            odd |= !(fabsf(y[q][T][0]) + fabsf(y[q][T][1]) + fabsf(y[q][T][2]) + fabsf(y[q][T][3]) < __builtin_inff());
        if (__any(odd)) {
          across();
#pragma unroll
          for (int T = 0; T < 2; ++T) {
            float v[8];
            TT::unpack(TT::template column<UX>(X, 0, m, g, wave, T), v);
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = fabsf(v[r]) < __builtin_inff() ? v[r] : 0.0f;
            const Frag f = TT::pack(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]});
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int part = 0; part < PARTS; ++part)
                y[q][T] = TT::mma(f, TT::row(Ws + part * wpart + (hh * kQ + 16 * q + m) * WP + 8 * g), y[q][T]);
          }
#pragma unroll 1
          for (int j = 0; j < kQ; ++j)
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              const float x = ld<DT>(X, TT::template unit<UX>(j, (32 * wave + 8 * g + c) / EV) + c % EV);
              if (fabsf(x) < __builtin_inff()) continue;
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int i = 16 * q + m;
                const float add = j <= i ? ld<DT>(Ws, (hh * kQ + i) * WP + j) * x : 0.0f;
#pragma unroll
                for (int r = 0; r < 8; ++r)
                  if (r == c) y[q][r >> 2][r & 3] += add;
              }
            }
        }
        const int pcol = p0 + 8 * g;  // this lane's outputs: columns pcol .. + 7 of rows 16 q + m
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int i = 16 * q + m;
          if (i >= left || pcol >= P) continue;
          float v[8], x[8];
          TT::unpack(TT::template rows<UX>(X, 16 * q, m, g, wave), x);
#pragma unroll
          for (int r = 0; r < 8; ++r) v[r] = y[q][r >> 2][r & 3];
          if (a.D) {
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = __builtin_fmaf(skip, x[r], v[r]);
          }
          if (a.z) {
            float z[8];
            TT::unpack(__builtin_bit_cast(Frag, zc[q]), z);
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] *= gatef_<DT>(z[r]);
          }
          uint32_t at = static_cast<uint32_t>(i) * py + 8 * g * static_cast<uint32_t>(es);
          asm volatile("" : "+v"(at));  // formed here, not kept over the loop
          const Frag o = TT::pack(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]});
          if (VEC || pcol + 8 <= P) {
            const __attribute__((ext_vector_type(4))) uint32_t* u = reinterpret_cast<const __attribute__((ext_vector_type(4))) uint32_t*>(&o);
#pragma unroll
            for (int k = 0; k < 8 / EV; ++k) *reinterpret_cast<any16*>(yat + at + 16 * k) = u[k];
          } else {
#pragma unroll
            for (int r = 0; r < 7; ++r)
              if (pcol + r < P) st<DT>(yat + at, r, v[r]);
          }
        }
      }
    }
    if constexpr (FULL) yat += kQ * static_cast<int64_t>(py);
    if (active) {  // the state
      const float tot = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(sm[5 * kQ])));
      decay *= tot;
      // The state is kept as h * scale: the chunk's decay goes to the scale, and what is added is divided by it; only
      // where the scale has left 2^-8 .. 2^8 is h itself multiplied (so that neither runs out of its range early).
      scale *= tot;
      if (scale < 0x1p-8f || scale > 0x1p8f) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int T = 0; T < 2; ++T) h[s][t2][T] *= scale;
        scale = 1.0f;
      }
      const float per = __builtin_amdgcn_rcpf(scale);
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(sm + 3 * kQ + 8 * g) * per;
      const f32x4 w1 = *reinterpret_cast<const f32x4*>(sm + 3 * kQ + 8 * g + 4) * per;
      // w x: float32, or as three bfloat16 parts that hold all its 24 bits, each a product of its own
      constexpr int ADDENDS = DT == kBF16 ? 3 : 1;
      Frag wx[ADDENDS][2];
#pragma unroll
      for (int T = 0; T < 2; ++T) {
        float v[8];
        TT::unpack(xf[T], v);
        f32x4 v0, v1;
#pragma unroll
        for (int r = 0; r < 4; ++r) v0[r] = v[r] * w0[r], v1[r] = v[4 + r] * w1[r];
#pragma unroll
        for (int part = 0; part < ADDENDS; ++part) {
          wx[part][T] = TT::pack(v0, v1);
          if (part + 1 == ADDENDS) break;
          TT::unpack(wx[part][T], v);
#pragma unroll
          for (int r = 0; r < 4; ++r) v0[r] -= v[r], v1[r] -= v[4 + r];  // (an infinity's states become NaN)
        }
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        Frag b[2];
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) b[t2] = TT::template column<UB>(Bs, 0, m, g, s, t2);
#pragma unroll
        for (int part = 0; part < ADDENDS; ++part)
#pragma unroll
          for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
            for (int T = 0; T < 2; ++T) h[s][t2][T] = TT::mma(b[t2], wx[part][T], h[s][t2][T]);
      }
    }
    if (NB == 1) lds_barrier();
  }

  if (!active) return;
  if constexpr (!FULL) {
    f32x4* out = reinterpret_cast<f32x4*>(gr.carry) + ((blockIdx.y * wg_all + blockIdx.x) * 4 + wave) * frags;
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int T = 0; T < 2; ++T) out[((s * 2 + t2) * 2 + T) * 64 + lane] = h[s][t2][T] * scale;
    if (lane == 0) gr.decay[blockIdx.y * a.H + head] = decay;  // (slices of one head write the same value)
  } else if (sg.last && a.h_out) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2)
#pragma unroll
        for (int T = 0; T < 2; ++T) {
          const int p = p0 + 8 * (m >> 2) + 4 * T + (m & 3), n = 32 * s + 8 * g + 4 * t2;
          float* dst = a.h_out + (static_cast<int64_t>(sg.seq) * a.H + head) * P * N + p * N + n;
          const f32x4 v = h[s][t2][T] * scale;
          if (VEC || (p < P && n + 4 <= N)) {
            store16(dst, __builtin_bit_cast(uint4, v));
          } else {
#pragma unroll
            for (int r = 0; r < 3; ++r)
              if (p < P && n + r < N) dst[r] = v[r];
          }
        }
  }
}

// The segments' end states from zero become the states at their ends: a sequence's are folded in order, one vector of
// 4 states per thread, the reads of eight segments under way together.  Bound by the bytes: 8 segments of 4 MB, 63 MB
// read and written, in 12 us.
template <int NS>
__global__ __launch_bounds__(256) void ssm_carry_kernel(SsmArgs a, SsmGrid gr) {
  constexpr int VW = NS * 4 * 64;  // vectors per wave
  const int64_t wg_all = static_cast<int64_t>(gr.wpg) * a.G;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;  // vector of a slot
  const int64_t wg = u / (4 * VW);
  const int wave = static_cast<int>(u / VW % 4), v = static_cast<int>(u % VW);
  const int grp = static_cast<int>(wg / gr.wpg), sl = static_cast<int>(wg % gr.wpg) * 4 + wave;
  int64_t slot = 0, nseg;
  if (!a.seq_starts) {
    nseg = segments_of(a.L, gr.seg);
    slot = blockIdx.y * nseg;
  } else {
    int64_t first, end;
    for (int64_t s = threadIdx.x & 63; s < static_cast<int64_t>(blockIdx.y); s += 64) {
      seq_rows(a.seq_starts, s, a.B * a.L, first, end);
      slot += segments_of(end - first, gr.seg);
    }
    for (int d = 32; d > 0; d >>= 1) slot += __shfl_xor(static_cast<long long>(slot), d);
    seq_rows(a.seq_starts, blockIdx.y, a.B * a.L, first, end);
    nseg = segments_of(end - first, gr.seg);
  }
  if (sl >= gr.sg || nseg < 2 || slot + nseg > gr.slots) return;  // (more segments than rows allow: starts that decrease)
  const int hg = static_cast<int>(a.H / a.G), head = grp * hg + sl / gr.ps;
  const int lane = v & 63, m = lane & 15, g = lane >> 4, T = (v >> 6) & 1, t2 = (v >> 7) & 1, s = v >> 8;
  f32x4 h = {0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t p = (sl % gr.ps) * 32 + 8 * (m >> 2) + 4 * T + (m & 3), n = 32 * s + 8 * g + 4 * t2;
  if (a.h0 && p < a.P) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < a.N) h[r] = a.h0[((blockIdx.y * a.H + head) * a.P + p) * a.N + n + r];
  }
  f32x4* c = reinterpret_cast<f32x4*>(gr.carry) + (slot * wg_all + wg) * 4 * VW + wave * VW + v;
  const float* dec = gr.decay + slot * a.H + head;
  for (int64_t k0 = 0; k0 + 1 < nseg; k0 += 8) {  // eight segments' loads at once
    f32x4 own[8];
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i + 1 < nseg) {
        own[i] = c[(k0 + i) * wg_all * 4 * VW];
        d[i] = dec[(k0 + i) * a.H];
      }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i + 1 < nseg) {
        h = h * d[i] + own[i];
        c[(k0 + i) * wg_all * 4 * VW] = h;
      }
  }
}

// ---------------------------------------------------------------------------
// One token.  A workgroup owns one head of one sequence: its state, read and written once, is what the call costs.  Rows of
// N states are held 4 per lane by LPR lanes, 256 / LPR rows at a time; the state's loads are issued first, and the
// convolution of the head's x and its group's B and C (in float32, to LDS) runs while they are on their way.  Every head
// forms its group's B and C again; the first head of a group writes their convolution state.  The states go past the
// caches both ways: 16 to 512 MB of them are never slower for it, used again at once or not (256 MB 96 us against 96 and
// 108, 512 MB 189 against 206).  Measured: 64 sequences of 128 heads of 64 x 128 states, 537 MB read and written, 98 us, 5.5 TB/s.
// ---------------------------------------------------------------------------
// A channel's inputs, as raw bits: the rows before the token and the token's, its filter and bias.
struct StepChannel {
  uint32_t past[kConvMaxW], w[kConvMaxW], bias;
};
template <int DT, int WDT>
__device__ __forceinline__ void step_load(const SsmStepArgs& a, int64_t b, int c, int64_t C, StepChannel& s) {
  const int W = a.conv_weight ? static_cast<int>(a.W) : 1;
#pragma unroll
  for (int j = 0; j < kConvMaxW; ++j)
    if (j < W - 1) {
      s.past[j] = ld_bits<DT>(a.conv_state, (b * (W - 1) + j) * C + c);
      s.w[j] = ld_bits<WDT>(a.conv_weight, static_cast<int64_t>(c) * W + j);
    }
  s.past[kConvMaxW - 1] = ld_bits<DT>(a.row, b * a.ld_row + c);
  if (a.conv_weight) s.w[kConvMaxW - 1] = ld_bits<WDT>(a.conv_weight, static_cast<int64_t>(c) * W + W - 1);
  s.bias = 0;
  if (a.conv_bias) s.bias = ld_bits<WDT>(a.conv_bias, c);
}
// Its convolved value; the state moves on where `keep`.
template <int DT, int WDT>
__device__ __forceinline__ float step_value(const SsmStepArgs& a, int64_t b, int c, int64_t C, const StepChannel& s, bool keep) {
  if (!a.conv_weight) return from_bits<DT>(s.past[kConvMaxW - 1]);
  const int W = static_cast<int>(a.W);
  auto put = [&](int j, uint32_t v) {
    if constexpr (DT == kBF16)
      static_cast<uint16_t*>(a.conv_state_out)[(b * (W - 1) + j) * C + c] = static_cast<uint16_t>(v);
    else
      static_cast<uint32_t*>(a.conv_state_out)[(b * (W - 1) + j) * C + c] = v;
  };
  float acc = from_bits<WDT>(s.bias);
#pragma unroll
  for (int j = 0; j < kConvMaxW; ++j)
    if (j < W - 1) {
      acc = __builtin_fmaf(from_bits<DT>(s.past[j]), from_bits<WDT>(s.w[j]), acc);
      if (keep && j > 0) put(j - 1, s.past[j]);
    }
  acc = __builtin_fmaf(from_bits<DT>(s.past[kConvMaxW - 1]), from_bits<WDT>(s.w[kConvMaxW - 1]), acc);
  if (keep) put(W - 2, s.past[kConvMaxW - 1]);
  return a.silu ? siluf_(acc) : acc;
}

// Sum over groups of LPR lanes, in every lane.
template <int LPR>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LPR >= 2) v += __int_as_float(dpp_mov<kDppXor1>(__float_as_int(v)));
  if constexpr (LPR >= 4) v += __int_as_float(dpp_mov<kDppXor2>(__float_as_int(v)));
  if constexpr (LPR >= 8) v += __int_as_float(dpp_mov<kDppHalfMirror>(__float_as_int(v)));
  if constexpr (LPR >= 16) v += __int_as_float(dpp_mov<kDppMirror>(__float_as_int(v)));
  if constexpr (LPR >= 32) v += __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), kSwzXor16));
  if constexpr (LPR >= 64) v += __shfl_xor(v, 32);
  return v;
}

// N4: rows are whole vectors of 4 states.
template <int DT, int WDT, int LPR, bool N4>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStepArgs a) {
  constexpr int RP = 256 / LPR, K = 8;  // rows at a time, and how many times ahead
  extern __shared__ __attribute__((aligned(16))) float lds_step[];
  const int N = static_cast<int>(a.N), P = static_cast<int>(a.P), n4 = (N + 3) & ~3;
  float* const bs = lds_step;  // B, C: n4 each; x: P; y: P
  float* const cs = bs + n4;
  float* const xs = cs + n4;
  float* const ys = xs + P;
  const int64_t b = blockIdx.y;
  const int h = blockIdx.x, hg = static_cast<int>(a.H / a.G), grp = h / hg;
  const int HP = static_cast<int>(a.H) * P;
  const int64_t C = HP + 2 * a.G * a.N;
  const int tid = threadIdx.x, n = (tid % LPR) * 4, p0 = tid / LPR;
  float* const state = a.state + (b * a.H + h) * P * static_cast<int64_t>(N);
  any16 raw[K];
  auto load = [&](int p, any16& v) {
    v = any16{0, 0, 0, 0};
    if (p >= P || n >= N) return;
    const float* q = state + static_cast<int64_t>(p) * N + n;
    if (N4 || n + 4 <= N) {
      v = __builtin_nontemporal_load(reinterpret_cast<const any16*>(q));
    } else {
#pragma unroll
      for (int r = 0; r < 3; ++r)
        if (n + r < N) v[r] = __float_as_uint(q[r]);
    }
  };
#pragma unroll
  for (int k = 0; k < K; ++k) load(p0 + k * RP, raw[k]);
  const uint32_t in = ld_bits<DT>(a.dts, b * a.ld_dt + h);
  const float bias = a.dt_bias ? a.dt_bias[h] : 0.0f, rate = a.A[h], skip = a.D ? a.D[h] : 0.0f;
  const int64_t zat = b * a.ld_z + static_cast<int64_t>(h) * P;
  const uint32_t z0 = a.z && tid < P ? ld_bits<DT>(a.z, zat + tid) : 0;
  // two channels of B, C and x at a time: both are on their way before either is used
  const int count = 2 * n4 + P;
  auto channel = [&](int e) {  // -1: padding
    if (e >= 2 * n4) return h * P + e - 2 * n4;
    const int c = e >= n4, i = e - c * n4;
    return i < N ? HP + (c * static_cast<int>(a.G) + grp) * N + i : -1;
  };
  for (int e = tid; e < count; e += 512) {
    StepChannel s[2];
    int c[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c[k] = e + 256 * k < count ? channel(e + 256 * k) : -1;
      if (c[k] >= 0) step_load<DT, WDT>(a, b, c[k], C, s[k]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (e + 256 * k < count)
        lds_step[e + 256 * k] = c[k] < 0 ? 0.0f : step_value<DT, WDT>(a, b, c[k], C, s[k], c[k] < HP || h % hg == 0);
  }
  const float sum_in = from_bits<DT>(in) + bias;
  const float d = a.softplus ? softplusf_(sum_in) : sum_in;
  const float decay = fast_exp(d * rate);
  __syncthreads();
  f32x4 bv = {0.0f, 0.0f, 0.0f, 0.0f}, cv = bv;
  if (n < N) {
    bv = *reinterpret_cast<const f32x4*>(bs + n) * d;
    cv = *reinterpret_cast<const f32x4*>(cs + n);
  }
  for (int pb = p0; pb < P; pb += K * RP) {
    float sum[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int p = pb + k * RP;
      const float x = p < P ? xs[p] : 0.0f;
      const f32x4 v = __builtin_bit_cast(f32x4, raw[k]) * decay + bv * x;
      sum[k] = (v[0] * cv[0] + v[1] * cv[1]) + (v[2] * cv[2] + v[3] * cv[3]);
      if (p < P && n < N) {
        float* q = state + static_cast<int64_t>(p) * N + n;
        if (N4 || n + 4 <= N) {
          __builtin_nontemporal_store(__builtin_bit_cast(any16, v), reinterpret_cast<any16*>(q));
        } else {
#pragma unroll
          for (int r = 0; r < 3; ++r)
            if (n + r < N) q[r] = v[r];
        }
      }
    }
    if (pb + K * RP - p0 < P) {
#pragma unroll
      for (int k = 0; k < K; ++k) load(pb + (K + k) * RP, raw[k]);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      sum[k] = lanes_sum<LPR>(sum[k]);
      if (tid % LPR == 0 && pb + k * RP < P) ys[pb + k * RP] = sum[k];
    }
  }
  __syncthreads();
  for (int p = tid; p < P; p += 256) {
    float y = ys[p];
    if (a.D) y += skip * xs[p];
    if (a.z) y *= siluf_(from_bits<DT>(p < 256 ? z0 : ld_bits<DT>(a.z, zat + p)));
    st<DT>(a.y, b * a.ld_y + static_cast<int64_t>(h) * P + p, y);
  }
}

}  // namespace

namespace {

int states32(const SsmArgs& a) {  // 32-state steps, rounded up to an instantiation
  const int n = static_cast<int>((a.N + 31) / 32);
  return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8;
}

// Segments: a divided sequence costs a second pass over its x, B and dt, a state per segment written, read, written and
// read again, and two launches, so that three of them at least are made, of 64 rows at least: as many as give each CU a
// workgroup, and where they keep 128 rows then, two (as many as fit).  Bfloat16 with 24 heads of 64 channels and 128
// states, divided against in one pass: 2048 rows 4 x 72 us against 172, 8 x 101 against 172, 16 x (two segments) 204
// against 175; 512 rows 25 us against 44 in segments of 256; 160 rows 19.3 against 19.5; 128 rows (two) 20 against 17.
SsmGrid ssm_grid(const SsmArgs& a) {
  SsmGrid g;
  const int64_t hg = a.H / a.G;
  g.ps = static_cast<int>((a.P + 31) / 32);
  g.sg = static_cast<int>(hg * g.ps);
  g.wpg = (g.sg + 3) / 4;
  g.nh = 4 % g.ps == 0 ? 4 / g.ps : g.ps % 4 == 0 ? 1 : 2;
  const int64_t wgs = a.G * g.wpg, rows = a.seq_starts ? a.B * a.L : a.L;
  const int64_t each = a.seq_starts ? 1 : std::max<int64_t>(a.S, 1);
  auto rows_for = [&](int64_t all) {
    const int64_t n = std::max<int64_t>(1, all / std::max<int64_t>(1, wgs * each));
    return round_up((rows + n - 1) / n, 64);
  };
  g.seg = std::max<int64_t>(64, std::min(rows_for(256), std::max<int64_t>(128, rows_for(512))));
  if (!a.seq_starts && a.L <= 2 * g.seg) g.seg = round_up(std::max<int64_t>(a.L, 1), 64);
  if (a.seq_starts)
    g.slots = rows / g.seg + a.S;
  else
    g.slots = a.S * std::max<int64_t>(1, (a.L + g.seg - 1) / g.seg);
  return g;
}

bool ssm_split(const SsmArgs& a, const SsmGrid& g) { return (a.seq_starts ? a.B * a.L : a.L) > g.seg; }

template <int DT, int NS, bool VEC>
int run_ssm(const SsmArgs& a, const SsmGrid& g, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.G * g.wpg), static_cast<unsigned>(g.slots));
  if (ssm_split(a, g)) {
    const unsigned part = static_cast<unsigned>(SsmLds<DT, NS, false>::bytes(g.nh));
    ssm_chunk_kernel<DT, NS, false, VEC><<<grid, 256, part, TESM_LOGGED(st, ssm_chunk_kernel<DT, NS, false, VEC>)>>>(a, g);
    const dim3 cg(static_cast<unsigned>(a.G * g.wpg * NS * 4), static_cast<unsigned>(a.S));
    ssm_carry_kernel<NS><<<cg, 256, 0, TESM_LOGGED(st, ssm_carry_kernel<NS>)>>>(a, g);
  }
  const unsigned full = static_cast<unsigned>(SsmLds<DT, NS, true>::bytes(g.nh));
  ssm_chunk_kernel<DT, NS, true, VEC><<<grid, 256, full, TESM_LOGGED(st, ssm_chunk_kernel<DT, NS, true, VEC>)>>>(a, g);
  return check_launch("selective scan");
}

template <int DT, bool VEC>
int run_ssm_dt(const SsmArgs& a, const SsmGrid& g, hipStream_t st) {
  switch (states32(a)) {
    case 1: return run_ssm<DT, 1, VEC>(a, g, st);
    case 2: return run_ssm<DT, 2, VEC>(a, g, st);
    case 4: return run_ssm<DT, 4, VEC>(a, g, st);
    default: return run_ssm<DT, 8, VEC>(a, g, st);
  }
}

int ssm_check(const SsmArgs& a) {
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, "selective scan: dtype must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.L >= 0 && a.S >= 0 && a.H >= 1 && a.P >= 1 && a.G >= 1 && a.N >= 1 && a.H % a.G == 0 &&
                   a.B < (1LL << 31) && a.L < (1LL << 31) && a.B * a.L < (1LL << 31) && a.S < (1LL << 24) &&
                   a.H < (1LL << 20) && a.P < (1LL << 20) && a.H * a.P < (1LL << 24),
               kErrInvalidArg, "selective scan: bad sizes (n_groups must divide the heads)");
  TESM_REQUIRE(a.N <= kSsmMaxN, kErrUnsupported, "selective scan: need at most 256 states");
  TESM_REQUIRE(a.seq_starts ? a.B == 1 : a.S == a.B, kErrInvalidArg,
               "selective scan: packed sequences lie in one row axis (B = 1), others have S = B");
  return kOk;
}

}  // namespace

int64_t selective_scan_ws_bytes(const SsmArgs& a) {
  if (ssm_check(a) != kOk) return -1;
  const SsmGrid g = ssm_grid(a);
  if (!ssm_split(a, g)) return 0;
  return round_up(g.slots * a.G * g.wpg * kCols * 32 * states32(a) * 4, 256) + round_up(g.slots * a.H * 4, 256);
}

int launch_selective_scan(const SsmArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  if (int rc = ssm_check(a)) return rc;
  TESM_REQUIRE(a.A && (a.B * a.L == 0 || (a.x && a.dts && a.Bm && a.Cm && a.y)), kErrInvalidArg,
               "selective scan: need x, dt, A, B, C and y");
  TESM_REQUIRE(a.ld_x >= a.H * a.P && a.ld_y >= a.H * a.P && a.ld_dt >= a.H && a.ld_b >= a.G * a.N &&
                   a.ld_c >= a.G * a.N && (!a.z || a.ld_z >= a.H * a.P),
               kErrInvalidArg, "selective scan: a row pitch is shorter than its row");
  TESM_REQUIRE(!a.h_out || a.h_out != a.h0, kErrInvalidArg, "selective scan: the states out need a buffer of their own");
  if (a.S == 0) return kOk;
  SsmGrid g = ssm_grid(a);
  TESM_REQUIRE(g.slots < 65536, kErrUnsupported, "selective scan: too many sequences");
  if (ssm_split(a, g)) {
    TESM_REQUIRE(ws && ws_bytes >= selective_scan_ws_bytes(a) && aligned(ws, 16), kErrWorkspace,
                 "selective scan: workspace too small or not 16-byte aligned");
    g.carry = static_cast<float*>(ws);
    g.decay = g.carry + round_up(g.slots * a.G * g.wpg * kCols * 32 * states32(a) * 4, 256) / 4;
  }
  // 32-bit offsets inside a chunk: 32 rows of pitch ld, 4 bytes at most
  const int64_t ld = std::max({a.ld_x, a.ld_b, a.ld_c, a.z ? a.ld_z : 0, a.ld_y});
  TESM_REQUIRE(ld < (1LL << 24), kErrUnsupported, "selective scan: row pitches must be below 2^24 elements");
  const bool v = a.P % 32 == 0 && a.N == 32 * states32(a);
  if (a.dt == kBF16) return v ? run_ssm_dt<kBF16, true>(a, g, st) : run_ssm_dt<kBF16, false>(a, g, st);
  return v ? run_ssm_dt<kF32, true>(a, g, st) : run_ssm_dt<kF32, false>(a, g, st);
}

namespace {

template <int DT, int WDT, int LPR>
int run_step(const SsmStepArgs& a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.H), static_cast<unsigned>(a.B));
  const unsigned lds = static_cast<unsigned>((2 * round_up(a.N, 4) + 2 * a.P) * 4);
  if (a.N % 4 == 0)
    ssm_step_kernel<DT, WDT, LPR, true><<<grid, 256, lds, TESM_LOGGED(st, ssm_step_kernel<DT, WDT, LPR, true>)>>>(a);
  else
    ssm_step_kernel<DT, WDT, LPR, false><<<grid, 256, lds, TESM_LOGGED(st, ssm_step_kernel<DT, WDT, LPR, false>)>>>(a);
  return check_launch("selective scan step");
}

template <int DT, int WDT>
int run_step_dt(const SsmStepArgs& a, hipStream_t st) {
  if (a.N <= 16) return run_step<DT, WDT, 4>(a, st);
  if (a.N <= 32) return run_step<DT, WDT, 8>(a, st);
  if (a.N <= 64) return run_step<DT, WDT, 16>(a, st);
  return a.N <= 128 ? run_step<DT, WDT, 32>(a, st) : run_step<DT, WDT, 64>(a, st);
}

}  // namespace

int launch_selective_scan_step(const SsmStepArgs& a, hipStream_t st) {
  TESM_REQUIRE((a.dt == kF32 || a.dt == kBF16) && (a.w_dt == kF32 || a.w_dt == kBF16), kErrInvalidArg,
               "selective scan step: dtypes must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.H >= 1 && a.P >= 1 && a.G >= 1 && a.N >= 1 && a.H % a.G == 0 && a.B < 65536 &&
                   a.H < (1LL << 20) && a.P <= 4096 && a.H * a.P < (1LL << 24),
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
  if (a.dt == kBF16) return a.w_dt == kBF16 ? run_step_dt<kBF16, kBF16>(a, st) : run_step_dt<kBF16, kF32>(a, st);
  return a.w_dt == kBF16 ? run_step_dt<kF32, kBF16>(a, st) : run_step_dt<kF32, kF32>(a, st);
}

}  // namespace tesm
