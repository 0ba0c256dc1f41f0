// Products of bfloat16 matrices for the dense operators.
//
// A workgroup owns BM x BN results: WM x WN waves of TM x TN tiles of 32 x 32, with a gated pair two accumulators per tile and
// two weight tiles.  Weights are the MFMA's first operand, so that a lane holds 4 consecutive columns of one row.  Operand tiles of
// BK values of k go straight from memory to LDS in NS stages.  A fragment's LDS reads are issued one k-step ahead of its MFMAs, one
// after each MFMA, and so are the loads of a later tile in a tile's last k-step: issued together behind the barrier, they held
// up all waves at once (8192 x 16384 x 4096 1097 us, one after each MFMA 1040).  One barrier per tile, before its last k-step, where the
// next tile has landed.
//
// A tile with k along its rows has rows of BK values, 16-byte chunk q of row r at q ^ (r / (16 / CPR)) % CPR (CPR chunks per
// row): 16 rows' reads of one chunk fall on 256 different bytes.  A tile with k down its rows has BK rows of BM (BN) values; its
// fragments come through the transposing read of 4 x 16 values (lane i of 16 gives the address of 4 columns of row i / 4 and
// gets column i of the 4 rows), with the 64-byte blocks of row k turned by k so that 4 rows fall on different banks.
// What lies behind the end of the contraction is read as zeros (an offset beyond the buffer's range), what lies behind the last
// row or column repeats the last one and is never stored.
//
// Bound by the matrix unit and the power it draws: counters over 8192 x 16384 x 4096 showed it busy in 60 % of the cycles of the first form,
// LDS in 25 %, without bank conflicts, at clocks between 1.6 (all along) and 2.1 GHz.
#include <type_traits>

#include "dense_mfma.h"

namespace tesm {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kRange = 0x80000000u;  // bytes from a tile's first value that a load can reach; offsets from here on give zeros

typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 buffer_at(uint64_t p) {
  return i32x4{static_cast<int>(p), static_cast<int>(p >> 32) & 0xffff, static_cast<int>(kRange), 0x00027000};
}
// 64 lanes x 16 bytes from the buffer's first value + `off` (each lane's own) to LDS in lane order.  In assembly, since the compiler
// lets every transposing LDS read wait for all such loads, which would leave none of them ahead; the instruction writes no
// register, and what waits for it is wait_vmcnt.  (Nothing else in this file uses m0, which the compiler sets anew where it does.)
__device__ __forceinline__ void to_lds(i32x4 buf, char* dst, uint32_t off) {
  const uint32_t at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(dst)));
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(buf));
}

// The products of parts that count, smallest first; the last one has sums of its own, which the others' join at the end.
constexpr int kOrder[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};

template <int KIND, int PARTS_, int WM_, int WN_, int TM_, int TN_, int BK_, int NS_>
struct Shape {
  static constexpr int PARTS = PARTS_, ORDERS = PARTS == 1 ? 1 : 6, SETS = PARTS == 1 ? 1 : 2;
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, BK = BK_, NS = NS_;
  static constexpr int NP = KIND == kProdGated ? 2 : 1;  // products
  static constexpr int NW = WM * WN, NT = NW * 64, BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE = PARTS * (A_BYTES + NP * B_BYTES);
  static constexpr int NA = A_BYTES / 1024, NB = B_BYTES / 1024, BLOCKS = PARTS * (NA + NP * NB);  // 1 KB per load instruction
  static constexpr int D = BLOCKS / NW;
  static_assert(BLOCKS % NW == 0 && PARTS * NA % NW == 0 && PARTS * NB % NW == 0, "every wave loads as many blocks of each operand");
  static constexpr int STEPS = BK / 16;
  static constexpr int PITCH = TN * 32 * 4 + 16, SLAB = NP * 32 * PITCH;
  static constexpr int SMEM = NS * STAGE > NW * SLAB ? NS * STAGE : NW * SLAB;
  static_assert(NS >= 2 && STEPS >= 2 && SMEM <= 160 * 1024, "stages");
  // With two stages a tile's own stage is refilled before its last k-step, whose fragments are in registers by then; with more of
  // them the previous tile's, so that no wave has to wait for its LDS reads in front of the barrier.
  static constexpr bool OWN = NS == 2;
  static constexpr int AHEAD = OWN ? 2 : NS - 1;  // tiles between the one in work and the one asked for
};

// How far the 64-byte blocks of row k of a tile that lies down are turned: 4 rows' blocks then fall on different banks (of 256
// bytes: rows of 128 are two to that).
template <int BX>
__device__ __forceinline__ int turn_of(int k) {
  static_assert(BX >= 64, "rows of two blocks at least");
  return BX == 64 ? (k >> 1) & 1 : k & 3;
}

// Where lane `lane` of a 1 KB block reads: the offset from the tile's first value, and the value of k (within the tile).
template <int BK, int BX, bool DOWN>
__device__ __forceinline__ void load_place(int block, int lane, int64_t ld, int64_t extent, uint32_t& off, int& k) {
  if constexpr (!DOWN) {
    constexpr int CPR = BK / 8, RPB = 64 / CPR, TURN = 16 / CPR;
    const int row = block * RPB + lane / CPR, q = (lane % CPR) ^ ((row / TURN) % CPR);
    const int64_t r = row < extent ? row : extent - 1;
    off = static_cast<uint32_t>(r * ld * 2) + q * 16;
    k = q * 8;
  } else {
    constexpr int UPR = BX / 8, RPB = 64 / UPR;
    k = block * RPB + lane / UPR;
    const int u = (lane % UPR) ^ (turn_of<BX>(k) << 2);
    const int64_t x = u * 8 < extent ? u * 8 : extent - 8;
    off = static_cast<uint32_t>(k * ld * 2 + x * 2);
  }
}

// A lane's fragment addresses: tile i (32 rows or columns from x0 + 32 i), k-step 0.
template <int BK, int BX, bool DOWN, int T>
struct Frag {
  int at[T];
  int turn;
  __device__ __forceinline__ void init(int x0, int lane) {
    if constexpr (!DOWN) {
#pragma unroll
      for (int i = 0; i < T; ++i) at[i] = (x0 + 32 * i + (lane & 31)) * BK * 2;
      turn = (((lane & 31) / (16 / (BK / 8))) % (BK / 8)) ^ (lane >> 5);  // (x0 is a multiple of 32)
    } else {
      const int i16 = lane & 15, kk = i16 >> 2, low = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
      const int row = 8 * (lane >> 5) + kk;
#pragma unroll
      for (int i = 0; i < T; ++i)
        at[i] = row * BX * 2 + ((((x0 >> 5) + i) ^ turn_of<BX>(kk)) * 4 + low) * 16 + 8 * (i16 & 1);
      turn = 0;
    }
  }
  // What a read gives: put together where it is used, since a copy behind the read would wait for it.
  struct Down {
    s16x4 lo, hi;
  };
  using Value = std::conditional_t<DOWN, Down, b16x8>;
  __device__ __forceinline__ Value read(const char* tile, int i, int s) const {
    if constexpr (!DOWN) {
      return *reinterpret_cast<const b16x8*>(tile + at[i] + ((turn ^ (2 * s)) * 16));
    } else {
      const char* p = tile + at[i] + s * 16 * BX * 2;
      return {__builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * BX * 2))};
    }
  }
  static __device__ __forceinline__ b16x8 value(const Value& v) {
    if constexpr (!DOWN)
      return v;
    else
      return __builtin_bit_cast(b16x8, __builtin_shufflevector(v.lo, v.hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};

// 8 consecutive columns of one row from the float32 slab to their places, 16 bytes of bfloat16 or 2 x 16 of float32 at once.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (DT == kBF16) {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      v[2 * q] = __uint_as_float(u[q] << 16);
      v[2 * q + 1] = __uint_as_float(u[q] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i)[q];
      v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
    }
  }
}
template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (DT == kBF16) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}
template <int DT>
__device__ __forceinline__ void keep_eight(void* z, int64_t all, int64_t i, const float (&v)[8]) {
  if constexpr (DT == kBF16) {
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = to_24(v[e]);
    uint4 hi;
    hi.x = __builtin_amdgcn_perm(b[1], b[0], 0x07060302), hi.y = __builtin_amdgcn_perm(b[3], b[2], 0x07060302);
    hi.z = __builtin_amdgcn_perm(b[5], b[4], 0x07060302), hi.w = __builtin_amdgcn_perm(b[7], b[6], 0x07060302);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(z) + i) = hi;
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] >>= 8;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(z) + 2 * all + i) =
        make_uint2(pack_low_bytes(b[0], b[1], b[2], b[3]), pack_low_bytes(b[4], b[5], b[6], b[7]));
  } else {
    store8<DT>(z, i, v);
  }
}
template <int KIND, int DT>
__device__ __forceinline__ void store_eight(const ProductArgs& a, void* out, int64_t m, int64_t n, float (&v)[8], float (&v2)[8]) {
  if constexpr (KIND == kProdGated) {
    if (a.z) {
      keep_eight<DT>(a.z, a.M * a.N, m * a.N + n, v);
      keep_eight<DT>(a.z2, a.M * a.N, m * a.N + n, v2);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = act_value(v[e], a.act) * v2[e];
  } else if constexpr (KIND == kProdLinear) {
    if (a.bias) {
      float b[8];
      load8<DT>(a.bias, n, b);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += b[e];
    }
    if (a.z) keep_eight<DT>(a.z, a.M * a.N, m * a.N + n, v);
    if (a.act != kActNone) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = act_value(v[e], a.act);
    }
    if (a.residual) {
      float r[8];
      load8<DT>(a.residual, m * a.ld_r + n, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += r[e];
    }
  }
  store8<DT>(out, m * a.ldo + n, v);
}

template <int KIND, int DT, int PARTS, bool ADOWN, bool BDOWN, int WM, int WN, int TM, int TN, int BK, int NS>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(ProductArgs a) {
  using S = Shape<KIND, PARTS, WM, WN, TM, TN, BK, NS>;
  __shared__ __attribute__((aligned(1024))) char smem[S::SMEM];
  constexpr int NP = S::NP;
  const int t = threadIdx.x;
  __builtin_assume(t < S::NT);
  const int lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int64_t ntm = (a.M + S::BM - 1) / S::BM, ntn = (a.N + S::BN - 1) / S::BN;
  int64_t tm, tn;
  xcd_tile_of<4>(blockIdx.x, ntm, ntn, tm, tn);
  const int64_t m0 = tm * S::BM, n0 = tn * S::BN;

  // this wave's loads: block b of an operand is block b % NA of its part b / NA
  constexpr int DA = PARTS * S::NA / S::NW, DB = PARTS * S::NB / S::NW;
  uint32_t off_a[DA], off_b[DB];
  int k_a[DA], k_b[DB];
#pragma unroll
  for (int i = 0; i < DA; ++i)
    load_place<BK, S::BM, ADOWN>((wave + i * S::NW) % S::NA, lane, a.lda, (ADOWN ? a.ext_a : a.M) - m0, off_a[i], k_a[i]);
#pragma unroll
  for (int i = 0; i < DB; ++i)
    load_place<BK, S::BN, BDOWN>((wave + i * S::NW) % S::NB, lane, a.ldb, (BDOWN ? a.ext_b : a.N) - n0, off_b[i], k_b[i]);
  auto part_of = [&](int block, int per, int64_t stride) __attribute__((always_inline)) {
    return PARTS == 1 ? 0 : static_cast<uint64_t>(block / per) * static_cast<uint64_t>(stride) * 2;
  };
  const int64_t a_first = ADOWN ? m0 : m0 * a.lda, b_first = BDOWN ? n0 : n0 * a.ldb;
  const int64_t a_step = ADOWN ? BK * a.lda : BK, b_step = BDOWN ? BK * a.ldb : BK;
  const int nk = static_cast<int>((a.K + BK - 1) / BK);
  const int all = nk * a.pairs;
  int first = 0, steps = all;  // this split's run
  if (KIND == kProdPartial) {
    first = static_cast<int>(static_cast<int64_t>(all) * blockIdx.y / a.splits);
    steps = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.y + 1) / a.splits) - first;
  }
  // The next tile to ask for: its values' addresses, kept in scalar registers.  A new pair's addresses are waited for where they
  // are read: left to the loop, that wait would hold up every tile's LDS reads (they share a counter).
  int pair = first / nk, kt = first % nk;
  uint64_t at_a, at_b, at_b2 = 0;
  auto begin = [&]() {
    at_a = reinterpret_cast<uint64_t>(a.A[pair] + a_first + kt * a_step);
    at_b = reinterpret_cast<uint64_t>(a.B[pair] + b_first + kt * b_step);
    if constexpr (NP == 2) at_b2 = reinterpret_cast<uint64_t>(a.B2[pair] + b_first + kt * b_step);
    asm volatile("" : "+s"(at_a), "+s"(at_b), "+s"(at_b2));
  };
  begin();
  // Load number i of the D that the wave asks for per tile; the last one moves on to the next tile.
  auto issue = [&](char* stage, bool live, int i) __attribute__((always_inline)) {
    const int end = live ? static_cast<int>(a.K - static_cast<int64_t>(kt) * BK) : 0;  // values of k from here on are zeros
    if (i < DA) {
      to_lds(buffer_at(at_a + part_of(wave + i * S::NW, S::NA, a.part_a)), stage + (wave + i * S::NW) * 1024, k_a[i] < end ? off_a[i] : kRange);
    } else {
      const int p = (i - DA) / DB, j = (i - DA) % DB;
      to_lds(buffer_at((p ? at_b2 : at_b) + part_of(wave + j * S::NW, S::NB, a.part_b)),
             stage + PARTS * (S::A_BYTES + p * S::B_BYTES) + (wave + j * S::NW) * 1024, k_b[j] < end ? off_b[j] : kRange);
    }
    if (i < S::D - 1) return;
    at_a += a_step * 2;
    at_b += b_step * 2;
    if constexpr (NP == 2) at_b2 += b_step * 2;
    if (++kt == nk) {  // (behind the last pair the first one's values are never asked for: `live` is off)
      kt = 0;
      pair = pair + 1 < a.pairs ? pair + 1 : 0;
      begin();
    }
  };

  using FragA = Frag<BK, S::BM, ADOWN, TM>;
  using FragB = Frag<BK, S::BN, BDOWN, TN>;
  FragA fa;
  FragB fb;
  fa.init(wm * TM * 32, lane);
  fb.init(wn * TN * 32, lane);
  f32x16 sums[S::SETS][NP][TM][TN];
#pragma unroll
  for (int h = 0; h < S::SETS; ++h)
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) sums[h][p][i][j] = f32x16{};
  typename FragA::Value ra[2][PARTS][TM];
  typename FragB::Value rb[2][PARTS][NP][TN];
  constexpr int NR = PARTS * (NP * TN + TM), NM = S::ORDERS * NP * TN * TM;  // fragment reads and MFMAs per k-step
  auto read = [&](const char* stage, int s, int r, int to) __attribute__((always_inline)) {
    // (what the first products need comes first)
    const int h = PARTS == 1 ? 0 : r / (NP * TN + TM), q = PARTS == 1 ? r : r % (NP * TN + TM);
    if (q < NP * TN) {
      const int part = PARTS == 1 ? 0 : h == 0 ? 0 : h == 1 ? 2 : 1;
      rb[to][part][q / TN][q % TN] = fb.read(stage + PARTS * S::A_BYTES + (q / TN) * PARTS * S::B_BYTES + part * S::B_BYTES, q % TN, s);
    } else {
      const int part = PARTS == 1 ? 0 : h == 0 ? 2 : h == 1 ? 0 : 1;
      ra[to][part][q - NP * TN] = fa.read(stage + part * S::A_BYTES, q - NP * TN, s);
    }
  };
  auto mma = [&](int q, int from) __attribute__((always_inline)) {
    const int i = q % TM, j = q / TM % TN, p = q / (TM * TN) % NP, o = q / (TM * TN * NP);
    const int pa = PARTS == 1 ? 0 : kOrder[o][0], pb = PARTS == 1 ? 0 : kOrder[o][1];
    f32x16& c = sums[o == S::ORDERS - 1 ? 0 : 1 % S::SETS][p][i][j];
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(FragB::value(rb[from][pb][p][j]), FragA::value(ra[from][pa][i]), c, 0, 0, 0);
  };
  // k-step s of the tile in `cur`: between its MFMAs the next step's fragments are read and, in the last step, the tile NS - 1
  // ahead is asked for, one instruction after each, so that neither the LDS nor the memory unit is asked for all at once.
  auto step_of = [&](const char* cur, const char* next, char* refill, int s, bool live) __attribute__((always_inline)) {
    const bool last = s == S::STEPS - 1;
#pragma unroll
    for (int q = 0; q < NM; ++q) {
      mma(q, s & 1);
#pragma unroll
      for (int r = q * NR / NM; r < (q + 1) * NR / NM; ++r) read(last ? next : cur, last ? 0 : s + 1, r, (s + 1) & 1);
      if (last) {
#pragma unroll
        for (int i = q * S::D / NM; i < (q + 1) * S::D / NM; ++i) issue(refill, live, i);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int s = 0; s < S::AHEAD; ++s)
#pragma unroll
    for (int i = 0; i < S::D; ++i) issue(smem + s * S::STAGE, s < steps, i);
  wait_vmcnt<(S::AHEAD - 1) * S::D>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int r = 0; r < NR; ++r) read(smem, 0, r, 0);
  int st = 0;
  for (int step = 0; step < steps; ++step) {
    const char* cur = smem + st * S::STAGE;
    const int nx = st + 1 == NS ? 0 : st + 1, pv = st == 0 ? NS - 1 : st - 1;
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
      if (s == S::STEPS - 1) {
        wait_vmcnt<(S::AHEAD - 2) * S::D>();  // this wave's part of the next tile has landed
        if (S::OWN) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();   // ... every wave's, and every wave is done with the tile before this one
        asm volatile("" ::: "memory");
      }
      step_of(cur, smem + nx * S::STAGE, smem + (S::OWN ? st : pv) * S::STAGE, s, step + S::AHEAD < steps);
    }
    st = nx;
  }
  static_assert(S::STEPS % 2 == 0, "a tile starts on the first fragments");
  wait_vmcnt<0>();  // the loads of zeros past the last tile: the slabs take the stages' place
  __syncthreads();

  // 32 rows at a time through the wave's own slab of float32
  char* slab = smem + wave * S::SLAB;
  const int64_t nb = n0 + wn * TN * 32;
  void* out = a.out;
  if (KIND == kProdPartial) out = static_cast<float*>(a.out) + static_cast<int64_t>(blockIdx.y) * a.M * a.N;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x16 c = sums[0][p][i][j];
          if constexpr (PARTS > 1) c += sums[1][p][i][j];
          *reinterpret_cast<float4*>(slab + p * 32 * S::PITCH + (lane & 31) * S::PITCH + (32 * j + 8 * g + 4 * (lane >> 5)) * 4) =
              make_float4(c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]);
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    const int64_t mb = m0 + (wm * TM + i) * 32;
    // (store kind: where this row goes)
    auto place = [&](int64_t& m, void*& to) {
      to = out;
      if (m >= a.M) return false;
      if (KIND == kProdStore && a.out2 && m >= a.cut) {
        if (m < a.fold) return false;
        m -= a.fold;
        to = a.out2;
      }
      return true;
    };
    if (a.vec) {
      constexpr int UPR = TN * 4;  // units of 8 columns per row
#pragma unroll
      for (int it = 0; it < 32 * UPR / 64; ++it) {
        const int idx = it * 64 + lane, row = idx / UPR, u = idx % UPR;
        int64_t m = mb + row;
        const int64_t n = nb + u * 8;
        void* to;
        if (!place(m, to) || n >= a.N) continue;
        float v[8], v2[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4 f = *reinterpret_cast<const float4*>(slab + row * S::PITCH + u * 32 + q * 16);
          v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
          if constexpr (NP == 2) {
            const float4 h = *reinterpret_cast<const float4*>(slab + 32 * S::PITCH + row * S::PITCH + u * 32 + q * 16);
            v2[4 * q] = h.x, v2[4 * q + 1] = h.y, v2[4 * q + 2] = h.z, v2[4 * q + 3] = h.w;
          }
        }
        store_eight<KIND, DT>(a, to, m, n, v, v2);
      }
    } else {  // a value per lane, along the rows
      constexpr int W = TN * 32;
#pragma unroll 4
      for (int it = 0; it < 32 * W / 64; ++it) {
        const int idx = it * 64 + lane, row = idx / W, col = idx % W;
        int64_t m = mb + row;
        const int64_t n = nb + col;
        void* to;
        if (!place(m, to) || n >= a.N) continue;
        const float v = *reinterpret_cast<const float*>(slab + row * S::PITCH + col * 4);
        float v2 = 0.0f;
        if constexpr (NP == 2) v2 = *reinterpret_cast<const float*>(slab + 32 * S::PITCH + row * S::PITCH + col * 4);
        store_one<KIND, DT>(a, to, m, n, v, v2);
      }
    }
  }
}

template <int KIND, int DT, int PARTS, bool ADOWN, bool BDOWN, int WM, int WN, int TM, int TN, int BK, int NS>
int run_product(const ProductArgs& a, hipStream_t st) {
  using S = Shape<KIND, PARTS, WM, WN, TM, TN, BK, NS>;
  const int64_t tiles = ((a.M + S::BM - 1) / S::BM) * ((a.N + S::BN - 1) / S::BN);
  TESM_REQUIRE(fits_grid(tiles, S::NT), kErrUnsupported, "dense product: too many tiles for one call");
  // offsets from a tile's first value stay inside the buffer's range
  TESM_REQUIRE(static_cast<int64_t>(ADOWN ? BK : S::BM) * a.lda * 2 + 1024 < static_cast<int64_t>(kRange) &&
                   static_cast<int64_t>(BDOWN ? BK : S::BN) * a.ldb * 2 + 1024 < static_cast<int64_t>(kRange) &&
                   a.K / BK * a.pairs < (1LL << 30),
               kErrUnsupported, "dense product: rows too long");
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(KIND == kProdPartial ? a.splits : 1));
  product_kernel<KIND, DT, PARTS, ADOWN, BDOWN, WM, WN, TM, TN, BK, NS>
      <<<grid, S::NT, 0, TESM_LOGGED(st, product_kernel<KIND, DT, PARTS, ADOWN, BDOWN, WM, WN, TM, TN, BK, NS>)>>>(a);
  return check_launch("dense product");
}

// Tile sizes.  Large: 256 x 256 results (a gated pair: 256 x 128 of each product) on 8 waves of 128 x 64, one workgroup per CU.
// Mid: 128 x 128 (128 x 64) on 4 waves of 64 x 64, two workgroups per CU.  Small: the same tiles with four stages, one per CU, for
// grids that have no second one anyway.  Tiny: 64 x 64 on 4 waves, two per CU.  In us per round of the CUs, with k thousand values of
// the contraction: 25 k + 8, 15 k + 5 (9 k + 5 where half the places stay empty), 7.6 k + 4 and 5.5 k + 4 (4 k + 3.5; a pair, which has
// 64 x 64 of each, 9 k + 4); a split adds the float32 results it writes and reads again.  Measured,
// bfloat16: 8192 x 16384 x 4096 879 us large (1.25 Pflop/s; the library's product 1.29), mid 1075, small 1240; 8192 x 4096 x 768 58,
// 69, 83; 8192 x 768 x 2048 47, 31, 39; 4096 x 768 x 8192 147, 77, 66; 512 x 768 x 2048 43, 23, 19, tiny 11; 1024 x 2048 x 768 23, 13, 11, 10.  Operands that lie down: 8192 x 16384 x 4096 864 us with one, 860
// with both (the library 950 and 1080).  Tiles of 32 values of k instead of 64 cost 20 % where rows run along k (64-byte
// pieces), stages of 128 x 256 with 8 waves of 64 x 64 another 10 %, 128 x 192 on 4 waves is no faster than mid where it fills the CUs.
//
// Operands of three parts: all parts of a tile lie in a stage and meet there in six products, so that values are loaded and read from
// LDS once, not twice (pairs of parts one after the other: 999 x 2 x 1030 x 515 36 us, now 28).  Large: 256 x 128 (128 x 128 of each) on 8
// waves, mid: 128 x 128 (128 x 64), small: 64 x 64 (of each) with six (four) stages, one per CU, tiny: the same with three (two),
// two per CU.  With what lays out the operands, large, mid and tiny: 4096 x 4096 x 4096 633, 725, 998 us (217 Tflop/s; the library's
// float32 product 137), 2048 x 768 x 2048 115, 84, 74, small 74; 999 x 515 x 1030 79, 54, 37, small 32.
enum Config : int { kLarge, kMid, kSmall, kTiny };
struct Plan {
  Config config = kSmall;
  int splits = 1;
  double us = 1e30;
};
Plan plan_product(ProductKind kind, bool parts, int64_t M, int64_t N, int64_t K, int pairs, bool split) {
  const int64_t cus = std::max(device_limits().cus, 1);
  const bool gated = kind == kProdGated;
  auto tiles = [&](int64_t bm, int64_t bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  // rounds of one workgroup per CU, of two (`half`: where only one is left)
  auto ones = [&](int64_t n, double us) { return static_cast<double>((n + cus - 1) / cus) * us; };
  auto twos = [&](int64_t n, double half, double us) {
    const int64_t rest = n % (2 * cus);
    return static_cast<double>(n / (2 * cus)) * us + (rest == 0 ? 0.0 : rest <= cus ? half : us);
  };
  const int64_t large = parts ? (gated ? tiles(128, 128) : tiles(256, 128)) : tiles(256, gated ? 128 : 256);
  const int64_t mid = tiles(128, gated ? 64 : 128), tiny = tiles(64, 64);
  const double all = static_cast<double>(K) * pairs / 1000.0;
  const int64_t steps = (K + 63) / 64 * pairs;
  Plan best;
  for (int s = 1; s <= (split ? 16 : 1) && (s == 1 || s * 4 <= steps); ++s) {
    const double k = all / s, joined = s == 1 ? 0.0 : 6.0 + 2.0 * s * 4.0 * static_cast<double>(M) * static_cast<double>(N) / 5.0e6;
    double cost[4];
    if (parts) {
      cost[kLarge] = ones(large * s, 72.0 * k + 5.0);
      cost[kMid] = ones(mid * s, 39.0 * k + 4.0);
      cost[kSmall] = ones(tiny * s, (gated ? 34.0 : 16.0) * k + 2.0);
      cost[kTiny] = gated ? twos(tiny * s, 45.0 * k + 3.0, 52.0 * k + 2.0) : twos(tiny * s, 20.0 * k + 2.0, 24.0 * k + 2.0);
    } else {
      cost[kLarge] = ones(large * s, 25.4 * k + 8.0);
      cost[kMid] = twos(mid * s, 9.4 * k + 5.0, 15.3 * k + 5.0);
      cost[kSmall] = ones(mid * s, 7.6 * k + 4.0);
      cost[kTiny] = gated ? twos(tiny * s, 6.5 * k + 4.0, 9.0 * k + 4.0) : twos(tiny * s, 4.0 * k + 3.5, 5.5 * k + 4.0);
    }
    for (int c = 0; c < 4; ++c)
      if (cost[c] + joined < best.us) best = {static_cast<Config>(c), s, cost[c] + joined};
  }
  return best;
}

template <int KIND, int DT, bool ADOWN, bool BDOWN>
int pick(const ProductArgs& a, hipStream_t st) {
  const bool parts = a.part_a != 0;
  // (a split product was planned by product_splits, with the same numbers)
  const Plan p = plan_product(static_cast<ProductKind>(KIND), parts, a.M, a.N, a.K, a.pairs, KIND == kProdPartial);
#define TESM_RUN(PARTS, ...) return run_product<KIND, DT, PARTS, ADOWN, BDOWN, __VA_ARGS__>(a, st)
  if constexpr (DT == kF32) {
    if (KIND != kProdPartial || parts) {
      if constexpr (KIND == kProdGated) {
        if (p.config == kLarge) TESM_RUN(3, 4, 2, 1, 2, 32, 2);
        if (p.config == kMid) TESM_RUN(3, 2, 2, 2, 1, 32, 3);
        if (p.config == kSmall) TESM_RUN(3, 2, 2, 1, 1, 32, 4);
        TESM_RUN(3, 2, 2, 1, 1, 32, 2);
      } else {
        if (p.config == kLarge) TESM_RUN(3, 4, 2, 2, 2, 32, 2);
        if (p.config == kMid) TESM_RUN(3, 2, 4, 2, 1, 32, 3);
        if (p.config == kSmall) TESM_RUN(3, 2, 2, 1, 1, 32, 6);
        TESM_RUN(3, 2, 2, 1, 1, 32, 3);
      }
    }
  }
  if constexpr (DT == kBF16 || KIND == kProdPartial) {
    if constexpr (KIND == kProdGated) {
      if (p.config == kLarge) TESM_RUN(1, 4, 2, 2, 2, 64, 2);
      if (p.config == kMid) TESM_RUN(1, 2, 2, 2, 1, 64, 2);
      if (p.config == kSmall) TESM_RUN(1, 2, 2, 2, 1, 64, 4);
      TESM_RUN(1, 2, 2, 1, 1, 64, 3);
    } else {
      if (p.config == kLarge) TESM_RUN(1, 2, 4, 4, 2, 64, 2);
      if (p.config == kMid) TESM_RUN(1, 2, 2, 2, 2, 64, 2);
      if (p.config == kSmall) TESM_RUN(1, 2, 2, 2, 2, 64, 4);
      TESM_RUN(1, 2, 2, 1, 1, 64, 4);
    }
  }
#undef TESM_RUN
  return fail(kErrUnsupported, "dense product: no kernel for these operands");  // (float32 results of one part)
}

}  // namespace

int product_splits(int64_t M, int64_t N, int64_t K, int pairs, bool parts) {
  return plan_product(kProdPartial, parts, M, N, K, pairs, true).splits;
}

double product_us(ProductKind kind, int64_t M, int64_t N, int64_t K) { return plan_product(kind, false, M, N, K, 1, false).us; }

int launch_product(ProductKind kind, int dt, bool adown, bool bdown, ProductArgs a, hipStream_t st) {
  if (a.M == 0 || a.N == 0) return kOk;
#define TESM_PICK(KIND, DT, AD, BD) return pick<KIND, DT, AD, BD>(a, st)
  if (kind == kProdGated && !adown && !bdown) {
    if (dt == kBF16) TESM_PICK(kProdGated, kBF16, false, false);
    TESM_PICK(kProdGated, kF32, false, false);
  }
  if (kind == kProdLinear && !adown && !bdown) {
    if (dt == kBF16) TESM_PICK(kProdLinear, kBF16, false, false);
    TESM_PICK(kProdLinear, kF32, false, false);
  }
  if (kind == kProdStore && !adown && bdown) {
    if (dt == kBF16) TESM_PICK(kProdStore, kBF16, false, true);
    TESM_PICK(kProdStore, kF32, false, true);
  }
  if (kind == kProdStore && adown && bdown) {
    if (dt == kBF16) TESM_PICK(kProdStore, kBF16, true, true);
    TESM_PICK(kProdStore, kF32, true, true);
  }
  if (kind == kProdPartial && !adown && bdown) TESM_PICK(kProdPartial, kF32, false, true);
  if (kind == kProdPartial && adown && bdown) TESM_PICK(kProdPartial, kF32, true, true);
#undef TESM_PICK
  return fail(kErrUnsupported, "dense product: no kernel for these layouts");
}

}  // namespace tesm
