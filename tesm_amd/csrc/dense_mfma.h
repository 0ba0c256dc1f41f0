// The matrix product that the dense operators share: bfloat16 operands, float32 sums on v_mfma_f32_32x32x16_bf16.
#pragma once

#include "dense.h"
#include "linear_dev.h"

namespace tesm {

constexpr int kMaxPairs = 4;

// out[m, n] = sum over pairs p and k of A_p[m, k] B_p[n, k] (a gradient in two bfloat16 parts is two pairs with one B).  An operand lies with k along its rows (m or n picks the row), or, where
// its layout is "down", with k picking the row.  All pairs share extents and pitches.  Rows start on 16 bytes; the contiguous
// extent is a multiple of 8.  With part_a set, operands are float32 values in three bfloat16 parts, part i lying i * part_a (part_b)
// values behind the first.
struct ProductArgs {
  int64_t M = 0, N = 0, K = 0;
  int pairs = 1;
  const uint16_t* A[kMaxPairs] = {};
  const uint16_t* B[kMaxPairs] = {};
  const uint16_t* B2[kMaxPairs] = {};  // the second weight of a gated pair
  int64_t part_a = 0, part_b = 0;
  int64_t lda = 0, ldb = 0;
  int64_t ext_a = 0, ext_b = 0;  // values per row of an operand that lies down, a multiple of 8 (not below M, N)
  int splits = 1;  // the contraction in this many runs of steps, each to its own float32 result at out + split * M * N
  // epilogue
  int act = kActNone;
  const void* bias = nullptr;
  const void* residual = nullptr;
  int64_t ld_r = 0;
  void* out = nullptr;
  int64_t ldo = 0;
  void* out2 = nullptr;   // rows from `fold` on go to out2, counted from `fold`; rows in [cut, fold) nowhere
  int64_t cut = 0, fold = 0;
  void* z = nullptr;
  void* z2 = nullptr;
  int vec = 0;  // every array of the epilogue takes 16-byte accesses at columns that are multiples of 8
};

enum ProductKind : int { kProdGated = 0, kProdLinear = 1, kProdStore = 2, kProdPartial = 3 };

// dt: type of the results (kProdPartial: float32).  adown, bdown: operand layouts.
int launch_product(ProductKind kind, int dt, bool adown, bool bdown, ProductArgs a, hipStream_t st);
// How many runs the contraction of such a product should be split into (1: none).
int product_splits(int64_t M, int64_t N, int64_t K, int pairs, bool parts);

// How long a product of bfloat16 operands that lie ready is expected to take.
double product_us(ProductKind kind, int64_t M, int64_t N, int64_t K);

// The normal distribution's Phi(z) = (1 + erf(z / sqrt 2)) / 2 and e = exp(-z^2 / 2), with erfc(x) = P(t) exp(-x^2), t = 1 / (1 + p x),
// the polynomial of Abramowitz and Stegun 7.1.26 (1.5e-7 off at most).  The library's erff takes three times as long: 8192 x 16384
// results of K = 4096 1101 us with it.
__device__ __forceinline__ float normal_phi(float z, float& e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.3275911f * 0.70710678118654752440f, 1.0f));
  float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  p = __builtin_fmaf(t, p, 1.421413741f);
  p = __builtin_fmaf(t, p, -0.284496736f);
  p = __builtin_fmaf(t, p, 0.254829592f);
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170368f);
  const float tail = 0.5f * p * t * e;
  return z < 0.0f ? tail : 1.0f - tail;
}
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == kActSilu) return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
  if (act == kActGelu) {
    float e;
    return z * normal_phi(z, e);
  }
  return z;
}
// act(z) and act'(z)
__device__ __forceinline__ void act_both(float z, int act, float& v, float& d) {
  if (act == kActSilu) {
    const float p = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f));
    v = z * p;
    d = __builtin_fmaf(v, 1.0f - p, p);
  } else if (act == kActGelu) {
    float e;
    const float p = normal_phi(z, e);
    v = z * p;
    d = __builtin_fmaf(z * 0.39894228040143267794f, e, p);
  } else {
    v = z;
    d = 1.0f;
  }
}

// What is kept of bfloat16 operands' products for the backward pass: the upper 24 bits of each (16 of its significand), the first 16 of
// all values, then the next 8 (`all` values further).  The gradients are products of a pair's kept ones and of an activation's slope at
// them, and with 16 bits of each they would be further off than their own rounding takes them.  float32 products are kept as they are.
__device__ __forceinline__ uint32_t to_24(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b & 0x7f800000u) == 0x7f800000u ? b | (b & 0x007fffffu ? 0x00400000u : 0u) : b + 0x80u;  // (infinities and NaNs keep their kind)
}
template <int DT>
__device__ __forceinline__ void keep_one(void* z, int64_t all, int64_t i, float v) {
  if constexpr (DT == kBF16) {
    const uint32_t b = to_24(v);
    static_cast<uint16_t*>(z)[i] = static_cast<uint16_t>(b >> 16);
    (static_cast<uint8_t*>(z) + 2 * all)[i] = static_cast<uint8_t>(b >> 8);
  } else {
    static_cast<float*>(z)[i] = v;
  }
}

// One value (two products v, v2 of a gated pair) to its places.
template <int KIND, int DT>
__device__ __forceinline__ void store_one(const ProductArgs& a, void* out, int64_t m, int64_t n, float v, float v2) {
  if constexpr (KIND == kProdGated) {
    if (a.z) {
      keep_one<DT>(a.z, a.M * a.N, m * a.N + n, v);
      keep_one<DT>(a.z2, a.M * a.N, m * a.N + n, v2);
    }
    st<DT>(out, m * a.ldo + n, act_value(v, a.act) * v2);
  } else if constexpr (KIND == kProdLinear) {
    if (a.bias) v += ld<DT>(a.bias, n);
    if (a.z) keep_one<DT>(a.z, a.M * a.N, m * a.N + n, v);
    v = act_value(v, a.act);
    if (a.residual) v += ld<DT>(a.residual, m * a.ld_r + n);
    st<DT>(out, m * a.ldo + n, v);
  } else {
    st<DT>(out, m * a.ldo + n, v);
  }
}

}  // namespace tesm
