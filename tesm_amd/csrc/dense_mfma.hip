// Products of bfloat16 matrices for the dense operators.
//
// A workgroup owns BM x BN results: WM x WN waves of TM x TN tiles of 32 x 32, with a gated pair two accumulators per tile and
// two weight tiles.  Weights are the MFMA's first operand, so that a lane holds 4 consecutive columns of one row.  Operand tiles of BK values of k go
// straight from memory to LDS in NS stages; a fragment's LDS reads are issued one k-step ahead of its MFMAs; one barrier per
// tile, before its last k-step but one, where the next tile has landed and the previous one's stage is refilled.
//
// A tile with k along its rows has rows of BK values, 16-byte chunk q of row r at q ^ (r / (16 / CPR)) % CPR (CPR chunks per
// row): 16 rows' reads of one chunk fall on 256 different bytes.  A tile with k down its rows has BK rows of BM (BN) values; its
// fragments come through the transposing read of 4 x 16 values (lane i of 16 gives the address of 4 columns of row i / 4 and
// gets column i of the 4 rows), with the 64-byte block index of row k turned by k % 4 so that 4 rows fall on different banks.
// What lies behind the end of the contraction is read as zeros (an offset beyond the buffer's range), what lies behind the last
// row or column repeats the last one and is never stored.
#include "dense_mfma.h"

namespace tesm {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kRange = 0x80000000u;  // bytes from a tile's first value that a load can reach; offsets from here on give zeros

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, kRange, 0x00027000);
}
__device__ __forceinline__ void to_lds(__amdgpu_buffer_rsrc_t buf, char* dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buf, (__attribute__((address_space(3))) void*)(dst), 16, off, 0, 0, 0);
}

template <int KIND, int WM_, int WN_, int TM_, int TN_, int BK_, int NS_>
struct Shape {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, BK = BK_, NS = NS_;
  static constexpr int NP = KIND == kProdGated ? 2 : 1;  // products
  static constexpr int NW = WM * WN, NT = NW * 64, BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE = A_BYTES + NP * B_BYTES;
  static constexpr int NA = A_BYTES / 1024, NB = B_BYTES / 1024, BLOCKS = NA + NP * NB;  // 1 KB per load instruction
  static constexpr int D = BLOCKS / NW;
  static_assert(BLOCKS % NW == 0 && NA % NW == 0 && NB % NW == 0, "every wave loads as many blocks of each operand");
  static constexpr int STEPS = BK / 16;
  static constexpr int PITCH = TN * 32 * 4 + 16, SLAB = NP * 32 * PITCH;
  static constexpr int SMEM = NS * STAGE > NW * SLAB ? NS * STAGE : NW * SLAB;
  static_assert(NS >= 3 && STEPS >= 2 && SMEM <= 160 * 1024, "stages");
};

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
    const int u = (lane % UPR) ^ ((k & 3) << 2);
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
        at[i] = row * BX * 2 + ((((x0 >> 5) + i) ^ kk) * 4 + low) * 16 + 8 * (i16 & 1);
      turn = 0;
    }
  }
  __device__ __forceinline__ b16x8 read(const char* tile, int i, int s) const {
    if constexpr (!DOWN) {
      return *reinterpret_cast<const b16x8*>(tile + at[i] + ((turn ^ (2 * s)) * 16));
    } else {
      const char* p = tile + at[i] + s * 16 * BX * 2;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * BX * 2));
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(b16x8, s16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    }
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
template <int KIND, int DT>
__device__ __forceinline__ void store_eight(const ProductArgs& a, void* out, int64_t m, int64_t n, float (&v)[8], float (&v2)[8]) {
  if constexpr (KIND == kProdGated) {
    if (a.z) {
      store8<DT>(a.z, m * a.N + n, v);
      store8<DT>(a.z2, m * a.N + n, v2);
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
    if (a.z) store8<DT>(a.z, m * a.N + n, v);
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

template <int KIND, int DT, bool ADOWN, bool BDOWN, int WM, int WN, int TM, int TN, int BK, int NS>
__global__ __launch_bounds__(WM* WN * 64) void product_kernel(ProductArgs a) {
  using S = Shape<KIND, WM, WN, TM, TN, BK, NS>;
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

  // this wave's loads
  constexpr int DA = S::NA / S::NW, DB = S::NB / S::NW;
  uint32_t off_a[DA], off_b[DB];
  int k_a[DA], k_b[DB];
#pragma unroll
  for (int i = 0; i < DA; ++i) load_place<BK, S::BM, ADOWN>(wave + i * S::NW, lane, a.lda, (ADOWN ? a.ext_a : a.M) - m0, off_a[i], k_a[i]);
#pragma unroll
  for (int i = 0; i < DB; ++i) load_place<BK, S::BN, BDOWN>(wave + i * S::NW, lane, a.ldb, (BDOWN ? a.ext_b : a.N) - n0, off_b[i], k_b[i]);
  const int64_t a_first = ADOWN ? m0 : m0 * a.lda, b_first = BDOWN ? n0 : n0 * a.ldb;
  const int64_t a_step = ADOWN ? BK * a.lda : BK, b_step = BDOWN ? BK * a.ldb : BK;
  const int nk = static_cast<int>((a.K + BK - 1) / BK);
  const int all = nk * a.pairs;
  int first = 0, steps = all;  // this split's run
  if (KIND == kProdPartial) {
    first = static_cast<int>(static_cast<int64_t>(all) * blockIdx.y / a.splits);
    steps = static_cast<int>(static_cast<int64_t>(all) * (blockIdx.y + 1) / a.splits) - first;
  }
  int pair = first / nk, kt = first % nk;
  auto issue = [&](char* stage, bool live) {
    const int64_t left = a.K - static_cast<int64_t>(kt) * BK;
    const bool whole = left >= BK && live;
    const int end = live ? static_cast<int>(left < BK ? left : BK) : 0;
    const __amdgpu_buffer_rsrc_t ba = buffer_at(a.A[pair] + a_first + kt * a_step);
    const __amdgpu_buffer_rsrc_t bb = buffer_at(a.B[pair] + b_first + kt * b_step);
#pragma unroll
    for (int i = 0; i < DA; ++i) to_lds(ba, stage + (wave + i * S::NW) * 1024, whole || k_a[i] < end ? off_a[i] : kRange);
#pragma unroll
    for (int i = 0; i < DB; ++i) to_lds(bb, stage + S::A_BYTES + (wave + i * S::NW) * 1024, whole || k_b[i] < end ? off_b[i] : kRange);
    if constexpr (NP == 2) {
      const __amdgpu_buffer_rsrc_t b2 = buffer_at(a.B2[pair] + b_first + kt * b_step);
#pragma unroll
      for (int i = 0; i < DB; ++i)
        to_lds(b2, stage + S::A_BYTES + S::B_BYTES + (wave + i * S::NW) * 1024, whole || k_b[i] < end ? off_b[i] : kRange);
    }
    if (++kt == nk) {  // (behind the last pair the first one's values are never asked for: `live` is off)
      kt = 0;
      pair = pair + 1 < a.pairs ? pair + 1 : 0;
    }
  };

  Frag<BK, S::BM, ADOWN, TM> fa;
  Frag<BK, S::BN, BDOWN, TN> fb;
  fa.init(wm * TM * 32, lane);
  fb.init(wn * TN * 32, lane);
  f32x16 acc[NP][TM][TN];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[p][i][j] = f32x16{};
  b16x8 ra[2][TM], rb[2][NP][TN];
  auto read = [&](const char* stage, int s, b16x8 (&x)[TM], b16x8 (&y)[NP][TN]) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int j = 0; j < TN; ++j) y[p][j] = fb.read(stage + S::A_BYTES + p * S::B_BYTES, j, s);
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = fa.read(stage, i, s);
  };
  auto mma = [&](const b16x8 (&x)[TM], const b16x8 (&y)[NP][TN]) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[p][i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(y[p][j], x[i], acc[p][i][j], 0, 0, 0);
  };

#pragma unroll
  for (int s = 0; s < NS - 1; ++s) issue(smem + s * S::STAGE, s < steps);
  wait_vmcnt<(NS - 2) * S::D>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read(smem, 0, ra[0], rb[0]);
  int st = 0;
  for (int step = 0; step < steps; ++step) {
    const char* cur = smem + st * S::STAGE;
    const int nx = st + 1 == NS ? 0 : st + 1, pv = st == 0 ? NS - 1 : st - 1;
#pragma unroll
    for (int s = 0; s < S::STEPS; ++s) {
      if (s == S::STEPS - 1)
        read(smem + nx * S::STAGE, 0, ra[(s + 1) & 1], rb[(s + 1) & 1]);
      else
        read(cur, s + 1, ra[(s + 1) & 1], rb[(s + 1) & 1]);
      if (s == S::STEPS - 2) {
        wait_vmcnt<(NS - 3) * S::D>();  // this wave's part of the next tile has landed
        __builtin_amdgcn_s_barrier();   // ... every wave's, and every wave is done with the tile before this one
        asm volatile("" ::: "memory");
        issue(smem + pv * S::STAGE, step + NS - 1 < steps);
      }
      __builtin_amdgcn_sched_barrier(0);
      mma(ra[s & 1], rb[s & 1]);
      __builtin_amdgcn_sched_barrier(0);
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
          const f32x16& c = acc[p][i][j];
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

template <int KIND, int DT, bool ADOWN, bool BDOWN, int WM, int WN, int TM, int TN, int BK, int NS>
int run_product(const ProductArgs& a, hipStream_t st) {
  using S = Shape<KIND, WM, WN, TM, TN, BK, NS>;
  const int64_t tiles = ((a.M + S::BM - 1) / S::BM) * ((a.N + S::BN - 1) / S::BN);
  TESM_REQUIRE(tiles < (1LL << 31), kErrUnsupported, "dense product: too many tiles");
  // offsets from a tile's first value stay inside the buffer's range
  TESM_REQUIRE(static_cast<int64_t>(ADOWN ? BK : S::BM) * a.lda * 2 + 1024 < static_cast<int64_t>(kRange) &&
                   static_cast<int64_t>(BDOWN ? BK : S::BN) * a.ldb * 2 + 1024 < static_cast<int64_t>(kRange) &&
                   a.K / BK * a.pairs < (1LL << 30),
               kErrUnsupported, "dense product: rows too long");
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(KIND == kProdPartial ? a.splits : 1));
  product_kernel<KIND, DT, ADOWN, BDOWN, WM, WN, TM, TN, BK, NS>
      <<<grid, S::NT, 0, TESM_LOGGED(st, product_kernel<KIND, DT, ADOWN, BDOWN, WM, WN, TM, TN, BK, NS>)>>>(a);
  return check_launch("dense product");
}

template <int KIND, int DT, bool ADOWN, bool BDOWN>
int pick(const ProductArgs& a, hipStream_t st) {
  auto tiles = [&](int64_t bm, int64_t bn) { return ((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn) * (KIND == kProdPartial ? a.splits : 1); };
  const int64_t cus = std::max(device_limits().cus, 1);
  if constexpr (KIND == kProdGated) {
    if (4 * tiles(256, 128) >= 3 * cus) return run_product<KIND, DT, ADOWN, BDOWN, 4, 2, 2, 2, 32, 4>(a, st);
    return run_product<KIND, DT, ADOWN, BDOWN, 2, 2, 2, 1, 32, 4>(a, st);
  } else {
    if (4 * tiles(256, 256) >= 3 * cus) return run_product<KIND, DT, ADOWN, BDOWN, 2, 4, 4, 2, 32, 4>(a, st);
    return run_product<KIND, DT, ADOWN, BDOWN, 2, 2, 2, 2, 32, 4>(a, st);
  }
}

}  // namespace

int product_splits(int64_t M, int64_t N, int64_t K, int pairs) {
  const int64_t cus = std::max(device_limits().cus, 1);
  const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128), steps = (K + 31) / 32 * pairs;
  if (tiles >= cus) return 1;
  const int64_t want = std::min<int64_t>(2 * cus / tiles, steps / 16);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, 16)));
}

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
