// The dense operators around the matrix product (dense_mfma.hip): operands brought into its form, few rows, gradients of the
// activations, sums over rows.
//
// Operands.  bfloat16 matrices whose rows start on 16 bytes and hold a multiple of 8 values are read where they lie; others are laid
// out so in the workspace first, padded with zeros.  float32 matrices are laid out as three bfloat16 parts, x = x0 + x1 + x2 with
// x0 = bf16(x), x1 = bf16(x - x0), x2 = x - x0 - x1 (8 bits each, together all 24 of x), and a product takes the six of their nine products
// that reach above 2^-26 of it, smallest first; the largest has a float32 sum of its own: bfloat16 products run at 16 times the
// float32 rate, so six of them are 2.7 times as fast as one in float32.  An infinite operand gives NaN where the formula may
// give an infinity.
//
// Gradients.  What stands before the activation is kept by the forward pass.  The gradient in front of the products is float32; an
// activation or a pair's factor leaves more bits in it than bfloat16 holds, and it goes into the products in two bfloat16 parts, 16 bits
// (float32: in three).  In one part its rounding alone was as large as the results' own (8192 x 768 x 2 x 2048: gradients 2.3e-3 of
// themselves off, the results' rounding 1.7e-3).
#include "dense_mfma.h"

namespace tesm {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(2)));  // at any alignment of its values
typedef uint32_t any8 __attribute__((ext_vector_type(2), aligned(1)));

int64_t size_of_dt(int dt) { return dt == kBF16 ? 2 : 4; }

// ---------------------------------------------------------------------------
// float32 as three bfloat16 parts
// ---------------------------------------------------------------------------
struct Parts3 {
  uint16_t p[3];
};
__device__ __forceinline__ Parts3 split3(float x) {
  uint16_t h = f32_to_bf16(x);
  if ((h & 0x7f80u) == 0x7f80u) {
    if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) return {{h, 0, 0}};  // an infinity or NaN
    h = static_cast<uint16_t>(__float_as_uint(x) >> 16);                       // (the largest values would round to infinity)
  }
  const float r = x - bf16_to_f32(h);
  const uint16_t m = f32_to_bf16(r);
  return {{h, m, f32_to_bf16(r - bf16_to_f32(m))}};
}
// Eight values to PARTS parts, `stride` apart (two parts: the first 16 bits).
template <int PARTS>
__device__ __forceinline__ void store_parts(uint16_t* to, int64_t stride, const float (&v)[8]) {
  if constexpr (PARTS == 1) {
    *reinterpret_cast<uint4*>(to) =
        make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  } else {
    uint32_t w[PARTS][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const Parts3 a = split3(v[2 * q]), b = split3(v[2 * q + 1]);
#pragma unroll
      for (int p = 0; p < PARTS; ++p) w[p][q] = a.p[p] | static_cast<uint32_t>(b.p[p]) << 16;
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) *reinterpret_cast<uint4*>(to + p * stride) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
  }
}
// Eight values at element i, of which `n` exist (the others are 0); whole ones by one or two loads, at any alignment.
template <int DT>
__device__ __forceinline__ void load_eight(const void* p, int64_t i, int n, float (&v)[8]) {
  if (n >= 8) {
    if constexpr (DT == kBF16) {
      const any16 u = *reinterpret_cast<const any16*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[2 * q] = __uint_as_float(u[q] << 16);
        v[2 * q + 1] = __uint_as_float(u[q] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const any16 u = *reinterpret_cast<const any16*>(static_cast<const float*>(p) + i + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = __uint_as_float(u[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? ld<DT>(p, i + e) : 0.0f;
  }
}

// Up to three matrices of R rows and C values per row into their parts, rows of Cp values, in one launch.
struct LayOut {
  const void* src = nullptr;
  int64_t ld = 0, R = 0, C = 0, Cp = 0;
  uint16_t* dst = nullptr;
  unsigned block0 = 0;  // first workgroup
};
struct LayOuts {
  LayOut m[3];
  int count = 0;
};
template <int DT>
__global__ __launch_bounds__(256) void lay_out_kernel(LayOuts t) {
  int k = 0;
  while (k + 1 < t.count && t.m[k + 1].block0 <= blockIdx.x) ++k;
  const LayOut& a = t.m[k];
  const int64_t i = static_cast<int64_t>(blockIdx.x - a.block0) * 256 + threadIdx.x, units = a.Cp / 8;
  if (i >= a.R * units) return;
  const int64_t r = i / units, c = i % units * 8;
  float v[8];
  load_eight<DT>(a.src, r * a.ld + c, static_cast<int>(a.C - c < 8 ? a.C - c : 8), v);
  store_parts<DT == kBF16 ? 1 : 3>(a.dst + r * a.Cp + c, a.R * a.Cp, v);
}

// ---------------------------------------------------------------------------
// few rows: the weights are read once, straight into the matrix unit's operands
// ---------------------------------------------------------------------------
// A workgroup owns 16 columns; its 8 waves share the contraction (chunks of 32 values, float32 of 16, taken in turn) and add
// their sums through LDS in order.  Lane l holds 16 bytes of weight row l % 16 and of x row l % 16.  Bound by the weights' bytes (4096 x
// 16384 bfloat16, 1 row: 23 us, 5.8 TB/s), for small ones by latency (768 x 2 x 2048: 4.9 us), above 16 rows by its reads of x.
constexpr int kSkinnyWaves = 8;

template <int DT>
__device__ __forceinline__ any16 chunk_at(const void* p, int64_t row, int64_t ld, int64_t k, int64_t K) {
  constexpr int EV = DT == kBF16 ? 8 : 4;
  const char* q = static_cast<const char*>(p) + (row * ld + k) * (16 / EV);
  if (k + EV <= K) return *reinterpret_cast<const any16*>(q);
  any16 v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < EV; ++e)
    if (k + e < K) {
      if constexpr (DT == kBF16)
        v[e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(q)[e]) << 16 * (e & 1);
      else
        v[e] = reinterpret_cast<const uint32_t*>(q)[e];
    }
  return v;
}
template <int DT>
__device__ __forceinline__ f32x4 chunk_mma(const any16& w, const any16& x, f32x4 c) {
  if constexpr (DT == kBF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, make_uint4(w[0], w[1], w[2], w[3])),
                                                   __builtin_bit_cast(b16x8, make_uint4(x[0], x[1], x[2], x[3])), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[j]), __uint_as_float(x[j]), c, 0, 0, 0);
    return c;
  }
}

template <int KIND, int DT, int MT>
__global__ __launch_bounds__(64 * kSkinnyWaves) void skinny_product_kernel(DenseArgs d, ProductArgs a) {
  constexpr int NP = KIND == kProdGated ? 2 : 1, EV = DT == kBF16 ? 8 : 4, CK = 4 * EV, U = 4;
  __shared__ float sums[kSkinnyWaves][NP][MT][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16, n = n0 + r < d.N ? n0 + r : d.N - 1;
  int64_t m[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) m[i] = i * 16 + r < d.M ? i * 16 + r : d.M - 1;
  f32x4 acc[NP][MT];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[p][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int64_t chunks = (d.K + CK - 1) / CK;
  for (int64_t c0 = wave; c0 < chunks; c0 += kSkinnyWaves * U) {
    any16 w[U][NP], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (chunks behind the end are zeros)
      const int64_t k = (c0 + u * kSkinnyWaves) * CK + g * EV;
      w[u][0] = chunk_at<DT>(d.w, n, d.ld_w, k, d.K);
      if constexpr (NP == 2) w[u][1] = chunk_at<DT>(d.w2, n, d.ld_w2, k, d.K);
#pragma unroll
      for (int i = 0; i < MT; ++i) x[u][i] = chunk_at<DT>(d.x, m[i], d.ld_x, k, d.K);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[p][i] = chunk_mma<DT>(w[u][p], x[u][i], acc[p][i]);
  }
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[wave][p][i][4 * g + e][r] = acc[p][i][e];
  __syncthreads();
  const int col = threadIdx.x & 15;
  if (n0 + col >= d.N) return;
  for (int row = threadIdx.x >> 4; row < d.M; row += 4 * kSkinnyWaves) {
    float v[2] = {0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int q = 0; q < kSkinnyWaves; ++q) v[p] += sums[q][p][row >> 4][col][row & 15];
    store_one<KIND, DT>(a, a.out, row, n0 + col, v[0], v[1]);
  }
}

// ---------------------------------------------------------------------------
// in front of the backward products
// ---------------------------------------------------------------------------
// Eight kept products.
template <int DT>
__device__ __forceinline__ void kept_eight(const void* z, int64_t all, int64_t i, int n, float (&v)[8]) {
  if constexpr (DT == kF32) {
    load_eight<kF32>(z, i, n, v);
  } else {
    const uint16_t* hi = static_cast<const uint16_t*>(z) + i;
    const uint8_t* lo = static_cast<const uint8_t*>(z) + 2 * all + i;
    if (n >= 8) {
      const any16 h = *reinterpret_cast<const any16*>(hi);
      const any8 l = *reinterpret_cast<const any8*>(lo);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[e] = __uint_as_float((e & 1 ? h[e / 2] & 0xffff0000u : h[e / 2] << 16) | (l[e / 4] >> 8 * (e & 3) & 0xffu) << 8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? __uint_as_float(static_cast<uint32_t>(hi[e]) << 16 | static_cast<uint32_t>(lo[e]) << 8) : 0.0f;
    }
  }
}
// dg = dh u act'(g) and du = dh act(g) beside each other in rows of 2 Np values.  Bound by HBM: 8192 x 2048 bfloat16 47 to 52 us for 268 MB.
template <int DT>
__global__ __launch_bounds__(256) void gated_grad_kernel(const void* grad, int64_t ld_g, const void* z, const void* z2, int64_t M, int64_t N,
                                                         int64_t Np, int act, uint16_t* dst) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, units = Np / 8;
  if (i >= M * units) return;
  const int64_t m = i / units, c = i % units * 8;
  const int n = static_cast<int>(N - c < 8 ? N - c : 8);
  float d[8], g[8], u[8];
  load_eight<DT>(grad, m * ld_g + c, n, d);
  kept_eight<DT>(z, M * N, m * N + c, n, g);
  kept_eight<DT>(z2, M * N, m * N + c, n, u);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float v, s;
    act_both(g[e], act, v, s);
    g[e] = e < n ? d[e] * u[e] * s : 0.0f;
    u[e] = e < n ? d[e] * v : 0.0f;
  }
  constexpr int P = DT == kBF16 ? 2 : 3;
  store_parts<P>(dst + m * 2 * Np + c, M * 2 * Np, g);
  store_parts<P>(dst + m * 2 * Np + Np + c, M * 2 * Np, u);
}

constexpr int kSumRows = 64;  // rows per sum
// dz = dy act'(z) into its parts (dst), and the sums of kSumRows rows of it (sums); either may be left out.  A workgroup takes every
// gridDim.y-th run of kSumRows rows.  8192 x 768 bfloat16 7 us without an activation, 23 with one (56 MB); its time is latency, three
// workgroups per two CUs.
template <int DT>
__global__ __launch_bounds__(256) void linear_grad_kernel(const void* grad, int64_t ld_g, const void* z, int64_t M, int64_t N, int64_t Np,
                                                          int act, uint16_t* dst, float* sums) {
  __shared__ float part[8][32][9];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int64_t c = (static_cast<int64_t>(blockIdx.x) * 32 + cx) * 8;
  const int col = threadIdx.x;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + col;
  for (int64_t run = blockIdx.y; run * kSumRows < M; run += gridDim.y) {
    const int64_t m0 = run * kSumRows;
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.0f;
    if (c < Np) {
      const int n = static_cast<int>(N - c < 8 ? N - c : 8);
      const int64_t end = m0 + kSumRows < M ? m0 + kSumRows : M;
#pragma unroll 4
      for (int64_t m = m0 + ry; m < end; m += 8) {
        float d[8];
        load_eight<DT>(grad, m * ld_g + c, n, d);
        if (act != kActNone) {
          float v[8];
          kept_eight<DT>(z, M * N, m * N + c, n, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a, b;
            act_both(v[e], act, a, b);
            d[e] = e < n ? d[e] * b : 0.0f;
          }
        }
        if (dst) {  // (without an activation the gradient is as it came)
          if (DT == kBF16 && act == kActNone)
            store_parts<1>(dst + m * Np + c, M * Np, d);
          else
            store_parts<DT == kBF16 ? 2 : 3>(dst + m * Np + c, M * Np, d);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += d[e];
      }
    }
    if (!sums) continue;
#pragma unroll
    for (int e = 0; e < 8; ++e) part[ry][cx][e] = s[e];
    __syncthreads();
    if (at < N) {
      float x = 0.0f;
#pragma unroll
      for (int q = 0; q < 8; ++q) x += part[q][col >> 3][col & 7];
      sums[run * N + at] = x;
    }
    __syncthreads();  // (`part` is written again)
  }
}
// The sums of all workgroups' rows, in 64 bits: 16 runs of them side by side, joined in order.
template <int DT>
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* sums, int64_t count, int64_t N, void* out) {
  __shared__ double part[16][64];
  const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  double x = 0.0;
  if (n < N) {
    const int64_t each = (count + 15) / 16, lo = run * each, hi = lo + each < count ? lo + each : count;
#pragma unroll 8
    for (int64_t s = lo; s < hi; ++s) x += sums[s * N + n];
  }
  part[run][lane] = x;
  __syncthreads();
  if (run == 0 && n < N) {
    for (int q = 1; q < 16; ++q) x += part[q][lane];
    st<DT>(out, n, static_cast<float>(x));
  }
}

// The runs of a split contraction added in order.
template <int DT>
__global__ __launch_bounds__(256) void join_splits_kernel(const float* part, int splits, int64_t M, int64_t N, int64_t cut, int64_t fold,
                                                          void* out, void* out2) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, all = M * N;
  if (i >= all) return;
  float x = 0.0f;
  for (int s = 0; s < splits; ++s) x += part[s * all + i];
  if (!out2 || i < cut * N)
    st<DT>(out, i, x);
  else if (i >= fold * N)
    st<DT>(out2, i - fold * N, x);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
struct Space {  // a workspace handed out in pieces (base null: only measured)
  char* base = nullptr;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += round_up(std::max<int64_t>(count, 1) * static_cast<int64_t>(sizeof(T)), 256);
    return base ? p : nullptr;
  }
};

struct Matrix {
  const uint16_t* p = nullptr;
  int64_t part = 0;  // values from part to part of float32 operands
  int64_t ld = 0, ext = 0;
};
bool lies_ready(int dt, const void* p, int64_t ld, int64_t C) { return dt == kBF16 && aligned(p, 16) && ld % 8 == 0 && C % 8 == 0; }

// The matrix as the product reads it: where it lies if `ready`, else laid out in `s` by `todo`'s launch.  Laid out, rows are whole cache
// lines (rows that begin inside one cost the product 10 to 25 %).
Matrix bring(Space& s, LayOuts& todo, int dt, const void* p, int64_t ld, int64_t R, int64_t C, bool ready) {
  if (ready) return {static_cast<const uint16_t*>(p), 0, ld, C};
  const int64_t Cp = round_up(C, 64);
  LayOut& m = todo.m[todo.count++];
  m.src = p, m.ld = ld, m.R = R, m.C = C, m.Cp = Cp;
  m.dst = s.take<uint16_t>(R * Cp * (dt == kBF16 ? 1 : 3));
  return {m.dst, dt == kBF16 ? 0 : R * Cp, Cp, Cp};
}
int lay_out(LayOuts& t, int dt, hipStream_t st) {
  int64_t blocks = 0;
  for (int k = 0; k < t.count; ++k) {
    t.m[k].block0 = static_cast<unsigned>(blocks);
    blocks += (t.m[k].R * t.m[k].Cp / 8 + 255) / 256;
    TESM_REQUIRE(fits_grid(blocks, 256), kErrUnsupported, "dense product: operands too large for one call");
  }
  if (blocks == 0) return kOk;
  const unsigned n = static_cast<unsigned>(blocks);
  if (dt == kBF16)
    lay_out_kernel<kBF16><<<n, 256, 0, TESM_LOGGED(st, lay_out_kernel<kBF16>)>>>(t);
  else
    lay_out_kernel<kF32><<<n, 256, 0, TESM_LOGGED(st, lay_out_kernel<kF32>)>>>(t);
  return kOk;
}

void add_pair(ProductArgs& a, const Matrix& A, int64_t a_off, const Matrix& B, const Matrix* B2) {
  a.A[a.pairs] = A.p + a_off;
  a.B[a.pairs] = B.p;
  a.B2[a.pairs] = B2 ? B2->p : nullptr;
  a.part_a = A.part, a.part_b = B.part;
  ++a.pairs;
}

int dense_check(const DenseArgs& a, const char* who) {
  const std::string w = std::string(who) + ": ";
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, w + "dtype must be 0 or 1");
  TESM_REQUIRE(a.act >= kActNone && a.act <= kActGelu, kErrInvalidArg, w + "no such activation");
  TESM_REQUIRE(a.M >= 0 && a.N >= 0 && a.K >= 1 && a.M < (1LL << 31) && a.N < (1LL << 24) && a.K < (1LL << 24), kErrInvalidArg,
               w + "bad sizes");
  return kOk;
}

ProductArgs epilogue_of(const DenseArgs& d) {
  ProductArgs a;
  a.M = d.M, a.N = d.N, a.K = d.K;
  a.act = d.act;
  a.bias = d.bias;
  a.residual = d.residual, a.ld_r = d.ld_r;
  a.out = d.y, a.ldo = d.ld_y;
  a.z = d.z, a.z2 = d.z2;
  const int64_t e = size_of_dt(d.dt);
  auto whole = [&](const void* p, int64_t ld) { return !p || (aligned(p, 16) && ld * e % 16 == 0); };
  a.vec = d.N % 8 == 0 && whole(d.y, d.ld_y) && whole(d.residual, d.ld_r) && whole(d.bias, 0) && whole(d.z, d.N) && whole(d.z2, d.N);
  return a;
}

template <int KIND>
int run_skinny(const DenseArgs& d, hipStream_t st) {
  const ProductArgs a = epilogue_of(d);
  const unsigned blocks = static_cast<unsigned>((d.N + 15) / 16);
  constexpr int T = 64 * kSkinnyWaves;
  const int64_t tiles = (d.M + 15) / 16;
#define TESM_SKINNY(DT, MT) skinny_product_kernel<KIND, DT, MT><<<blocks, T, 0, TESM_LOGGED(st, skinny_product_kernel<KIND, DT, MT>)>>>(d, a)
  if (d.dt == kBF16) {
    if (tiles == 1)
      TESM_SKINNY(kBF16, 1);
    else
      TESM_SKINNY(kBF16, 2);
  } else {
    if (tiles == 1)
      TESM_SKINNY(kF32, 1);
    else if (tiles == 2)
      TESM_SKINNY(kF32, 2);
    else
      TESM_SKINNY(kF32, 4);
  }
#undef TESM_SKINNY
  return check_launch("dense product of few rows");
}

// Whether the weights are streamed once, past the matrix product's tiles.  float32 ones up to 64 rows, since tiles need them laid out
// (768 x 2048: 64 rows 12.7 us, in tiles 21.6; 4096 x 16384: 198 and 216).  bfloat16 ones up to 32 rows, but not where the tiles read them where they lie and are expected to take
// less time: streaming, every wave reads x besides, and comes to 4.7 TB/s of weights up to 16 rows and 3.2 above (768 x 2048: 1 row 3.8 us,
// 32 rows 5.2, tiles 6.0; 4096 x 16384: 23, 45 and 22).
bool streams(const DenseArgs& d, bool ready) {
  if (d.dt == kF32) return d.M <= 64;
  if (d.M > 32) return false;
  const double us = 3.0 + 2.0 * static_cast<double>(d.N * d.K) * (d.w2 ? 2 : 1) / (d.M <= 16 ? 4.7e6 : 3.2e6);
  return !ready || us <= product_us(d.w2 ? kProdGated : kProdLinear, d.M, d.N, d.K);
}

int forward(const DenseArgs& d, Space s, bool run, int64_t* need, hipStream_t st) {
  const bool x_ready = lies_ready(d.dt, d.x, d.ld_x, d.K);
  const bool ready = lies_ready(d.dt, d.w, d.ld_w, d.K) && (!d.w2 || (lies_ready(d.dt, d.w2, d.ld_w2, d.K) && d.ld_w == d.ld_w2));
  if (streams(d, x_ready && ready)) {
    if (need) *need = 0;
    if (!run || d.M == 0 || d.N == 0) return kOk;
    return d.w2 ? run_skinny<kProdGated>(d, st) : run_skinny<kProdLinear>(d, st);
  }
  LayOuts todo;
  const Matrix x = bring(s, todo, d.dt, d.x, d.ld_x, d.M, d.K, x_ready);
  const Matrix w = bring(s, todo, d.dt, d.w, d.ld_w, d.N, d.K, ready);
  const Matrix w2 = d.w2 ? bring(s, todo, d.dt, d.w2, d.ld_w2, d.N, d.K, ready) : Matrix{};
  if (need) *need = s.used;
  if (!run || d.N == 0) return kOk;
  if (int rc = lay_out(todo, d.dt, st)) return rc;
  ProductArgs a = epilogue_of(d);
  a.pairs = 0;
  add_pair(a, x, 0, w, d.w2 ? &w2 : nullptr);
  a.lda = x.ld, a.ldb = w.ld;
  return launch_product(d.w2 ? kProdGated : kProdLinear, d.dt, false, false, a, st);
}

// A product whose results are gradients, its contraction split where there are few tiles.
int grad_product(Space& s, bool run, int dt, bool adown, ProductArgs a, hipStream_t st) {
  a.splits = a.K ? product_splits(a.M, a.N, a.K, a.pairs, a.part_a != 0) : 0;  // (nothing to add up: zeros)
  const int64_t e = size_of_dt(dt);
  if (a.splits == 1) {
    a.ldo = a.N;
    a.vec = a.N * e % 16 == 0 && a.N % 8 == 0 && aligned(a.out, 16) && (!a.out2 || aligned(a.out2, 16));
    return run ? launch_product(kProdStore, dt, adown, true, a, st) : kOk;
  }
  float* part = s.take<float>(a.splits * a.M * a.N);
  if (!run) return kOk;
  ProductArgs b = a;
  b.out = part, b.out2 = nullptr;
  b.ldo = a.N;
  b.vec = a.N % 8 == 0;
  if (a.splits)
    if (int rc = launch_product(kProdPartial, kF32, adown, true, b, st)) return rc;
  TESM_REQUIRE(fits_grid((a.M * a.N + 255) / 256, 256), kErrUnsupported, "dense product: too large for one call");
  const unsigned blocks = static_cast<unsigned>((a.M * a.N + 255) / 256);
  if (dt == kBF16)
    join_splits_kernel<kBF16><<<blocks, 256, 0, TESM_LOGGED(st, join_splits_kernel<kBF16>)>>>(part, a.splits, a.M, a.N, a.cut, a.fold, a.out, a.out2);
  else
    join_splits_kernel<kF32><<<blocks, 256, 0, TESM_LOGGED(st, join_splits_kernel<kF32>)>>>(part, a.splits, a.M, a.N, a.cut, a.fold, a.out, a.out2);
  return check_launch("dense product, joined");
}


int backward(const DenseBwdArgs& b, Space s, bool run, int64_t* need, hipStream_t st) {
  const DenseArgs& d = b.in;
  const int dt = d.dt;
  const int64_t M = d.M, N = d.N, K = d.K, Np = round_up(N, 64);  // (rows of whole cache lines)
  const bool gated = d.w2 != nullptr, products = b.dx || b.dw || b.dw2;
  const int parts = dt == kF32 ? 3 : gated || d.act != kActNone ? 2 : 1;  // of the gradient in front of the products
  Matrix dz;
  if (gated) {
    uint16_t* dst = s.take<uint16_t>(M * 2 * Np * parts);
    dz = {dst, dt == kBF16 ? 0 : M * 2 * Np, 2 * Np, 2 * Np};
    const int64_t threads = M * Np / 8;
    if (run && threads && products) {
      TESM_REQUIRE(fits_grid((threads + 255) / 256, 256), kErrUnsupported, "dense backward: too large for one call");
      const unsigned blocks = static_cast<unsigned>((threads + 255) / 256);
      if (dt == kBF16)
        gated_grad_kernel<kBF16><<<blocks, 256, 0, TESM_LOGGED(st, gated_grad_kernel<kBF16>)>>>(b.grad, b.ld_g, d.z, d.z2, M, N, Np, d.act, dst);
      else
        gated_grad_kernel<kF32><<<blocks, 256, 0, TESM_LOGGED(st, gated_grad_kernel<kF32>)>>>(b.grad, b.ld_g, d.z, d.z2, M, N, Np, d.act, dst);
    }
  } else {
    const bool direct = d.act == kActNone && lies_ready(dt, b.grad, b.ld_g, N);
    uint16_t* dst = nullptr;
    if (direct)
      dz = {static_cast<const uint16_t*>(b.grad), 0, b.ld_g, N};
    else {
      dst = s.take<uint16_t>(M * Np * parts);
      dz = {dst, dt == kBF16 ? 0 : M * Np, Np, Np};
    }
    const int64_t rows = (M + kSumRows - 1) / kSumRows;
    float* sums = b.dbias ? s.take<float>(rows * N) : nullptr;
    if (run && M && N && (sums || (dst && products))) {
      const dim3 grid(static_cast<unsigned>((Np + 255) / 256), static_cast<unsigned>(std::min<int64_t>(rows, 65535)));
      if (dt == kBF16)
        linear_grad_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, linear_grad_kernel<kBF16>)>>>(b.grad, b.ld_g, d.z, M, N, Np, d.act, dst, sums);
      else
        linear_grad_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, linear_grad_kernel<kF32>)>>>(b.grad, b.ld_g, d.z, M, N, Np, d.act, dst, sums);
    }
    if (run && b.dbias && N) {
      const unsigned blocks = static_cast<unsigned>((N + 63) / 64);
      if (dt == kBF16)
        column_sum_kernel<kBF16><<<blocks, 1024, 0, TESM_LOGGED(st, column_sum_kernel<kBF16>)>>>(sums, M ? rows : 0, N, b.dbias);
      else
        column_sum_kernel<kF32><<<blocks, 1024, 0, TESM_LOGGED(st, column_sum_kernel<kF32>)>>>(sums, M ? rows : 0, N, b.dbias);
    }
  }
  LayOuts todo;
  Matrix w, w2, x;
  const bool for_x = b.dx && M, for_w = (b.dw || b.dw2) && N;
  const int sums_of = dt == kF32 ? 1 : parts;  // (float32 parts meet inside the product, two bfloat16 ones as products that are added up)
  if (for_x) {
    const bool ready = lies_ready(dt, d.w, d.ld_w, K) && (!gated || (lies_ready(dt, d.w2, d.ld_w2, K) && d.ld_w == d.ld_w2));
    w = bring(s, todo, dt, d.w, d.ld_w, N, K, ready);
    if (gated) w2 = bring(s, todo, dt, d.w2, d.ld_w2, N, K, ready);
  }
  if (for_w) x = bring(s, todo, dt, d.x, d.ld_x, M, K, lies_ready(dt, d.x, d.ld_x, K));
  if (run)
    if (int rc = lay_out(todo, dt, st)) return rc;
  if (for_x) {
    ProductArgs a;
    a.M = M, a.N = K, a.K = N;
    a.pairs = 0;
    for (int p = 0; p < sums_of; ++p) {
      add_pair(a, dz, p * M * dz.ld, w, nullptr);
      if (gated) add_pair(a, dz, p * M * dz.ld + Np, w2, nullptr);
    }
    a.lda = dz.ld, a.ldb = w.ld, a.ext_b = w.ext;
    a.out = b.dx;
    if (int rc = grad_product(s, run, dt, false, a, st)) return rc;
  }
  if (for_w) {
    ProductArgs a;
    a.M = gated ? Np + N : N, a.N = K, a.K = M;
    a.pairs = 0;
    for (int p = 0; p < sums_of; ++p) add_pair(a, dz, p * M * dz.ld, x, nullptr);
    a.lda = dz.ld, a.ext_a = dz.ext, a.ldb = x.ld, a.ext_b = x.ext;
    a.out = b.dw, a.out2 = b.dw2;
    a.cut = N, a.fold = Np;
    if (int rc = grad_product(s, run, dt, true, a, st)) return rc;
  }
  if (need) *need = s.used;
  return run ? check_launch("dense backward") : kOk;
}

}  // namespace

int64_t dense_ws_bytes(const DenseArgs& a) {
  int64_t need = 0;
  if (dense_check(a, "dense product") != kOk || forward(a, Space{}, false, &need, nullptr) != kOk) return -1;
  return need;
}
int64_t dense_bwd_ws_bytes(const DenseBwdArgs& b) {
  int64_t need = 0;
  if (dense_check(b.in, "dense backward") != kOk || backward(b, Space{}, false, &need, nullptr) != kOk) return -1;
  return need;
}

int launch_dense(const DenseArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  const char* who = a.w2 ? "gated linear" : "fused linear";
  const std::string w = std::string(who) + ": ";
  if (int rc = dense_check(a, who)) return rc;
  if (a.M == 0 || a.N == 0) return kOk;
  TESM_REQUIRE(a.x && a.w && a.y, kErrInvalidArg, w + "need x, the weights and the output");
  TESM_REQUIRE(a.ld_x >= a.K && a.ld_w >= a.K && (!a.w2 || a.ld_w2 >= a.K) && a.ld_y >= a.N && (!a.residual || a.ld_r >= a.N),
               kErrInvalidArg, w + "a row pitch below the row's values");
  TESM_REQUIRE(!a.w2 || (a.act != kActNone && (a.z != nullptr) == (a.z2 != nullptr)), kErrInvalidArg,
               w + "need an activation, and both kept products or none");
  const int64_t need = dense_ws_bytes(a);
  TESM_REQUIRE(need == 0 || (ws && ws_bytes >= need && aligned(ws, 16)), kErrWorkspace, w + "workspace too small or not 16-byte aligned");
  return forward(a, Space{static_cast<char*>(ws), 0}, true, nullptr, st);
}

int launch_dense_bwd(const DenseBwdArgs& b, void* ws, int64_t ws_bytes, hipStream_t st) {
  const DenseArgs& a = b.in;
  const char* who = a.w2 ? "gated linear backward" : "fused linear backward";
  const std::string w = std::string(who) + ": ";
  if (int rc = dense_check(a, who)) return rc;
  TESM_REQUIRE(a.M == 0 || a.N == 0 || (b.grad && b.ld_g >= a.N), kErrInvalidArg, w + "need the gradient");
  TESM_REQUIRE(a.M == 0 || a.N == 0 || ((!b.dx || (a.w && a.ld_w >= a.K && (!a.w2 || a.ld_w2 >= a.K))) &&
                                        (!(b.dw || b.dw2) || (a.x && a.ld_x >= a.K))),
               kErrInvalidArg, w + "need the operands that the gradients asked for are made of");
  TESM_REQUIRE(!a.w2 || (b.dw != nullptr) == (b.dw2 != nullptr), kErrInvalidArg, w + "both weights' gradients or none");
  TESM_REQUIRE(!a.w2 || a.act != kActNone, kErrInvalidArg, w + "need an activation");
  TESM_REQUIRE(a.M == 0 || a.N == 0 || a.act == kActNone || (a.z && (!a.w2 || a.z2)), kErrInvalidArg,
               w + "need what the forward call kept");
  const int64_t need = dense_bwd_ws_bytes(b);
  TESM_REQUIRE(need == 0 || (ws && ws_bytes >= need && aligned(ws, 16)), kErrWorkspace, w + "workspace too small or not 16-byte aligned");
  return backward(b, Space{static_cast<char*>(ws), 0}, true, nullptr, st);
}

}  // namespace tesm
