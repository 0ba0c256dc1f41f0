// Beam search.  A beam k of a request with score s_k and logits l_k offers every token v at
//   s_k + l_k[v] - logsumexp(l_k),
// and the n best of all beams' offers are chosen, equal ones in the order of k * V + v.  Offers that are not a number
// (a NaN logit, a row with an infinite one) and all offers of a beam without a finite score count as -infinity; a
// finished beam offers its padding token alone, at its own score.
//
// Inside a beam the order of the offers is the order of the logits, so each row is reduced to its n largest logits
// and its logsumexp; requests then merge K lists of n, with the offers compared in 64 bits.
#include "beam.h"

namespace tesm {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// Larger first, equal ones by index.
__device__ __forceinline__ bool before(double v, int64_t i, double w, int64_t j) { return v > w || (v == w && i < j); }

template <int DT>
__device__ __forceinline__ float logit(const void* row, int64_t v) {
  const float x = ld<DT>(row, v);
  return x == x ? x : -__builtin_inff();
}

struct RowTop {
  float value;
  int32_t index;
};

template <int DT>
__global__ __launch_bounds__(256) void beam_row_kernel(BeamArgs a, int m, RowTop* top, double* lse) {
  __shared__ double red[4];
  __shared__ RowTop best[4];
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* row = static_cast<const char*>(a.logits) + r * a.ld * (DT == kBF16 ? 2 : 4);
  float mx = -__builtin_inff();
  for (int64_t v = tid; v < a.V; v += 256) mx = fmaxf(mx, logit<DT>(row, v));
  mx = wave_max<64>(mx);
  if (lane == 0) red[wave] = mx;
  __syncthreads();
  mx = static_cast<float>(fmax(fmax(red[0], red[1]), fmax(red[2], red[3])));
  __syncthreads();
  double sum = 0.0;
  for (int64_t v = tid; v < a.V; v += 256) sum += __builtin_amdgcn_exp2f((logit<DT>(row, v) - mx) * kLog2e);
  sum = wave_sum_d<64>(sum);
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  if (tid == 0) lse[r] = static_cast<double>(mx) + log((red[0] + red[1]) + (red[2] + red[3]));
  float pv = __builtin_inff();
  int64_t pi = -1;
  for (int i = 0; i < m; ++i) {  // the next one in order
    float bv = -__builtin_inff();
    int64_t bi = INT32_MAX;
    for (int64_t v = tid; v < a.V; v += 256) {
      const float x = logit<DT>(row, v);
      if (before(pv, pi, x, v) && before(x, v, bv, bi)) bv = x, bi = v;
    }
    for (int d = 32; d > 0; d >>= 1) {
      const float ov = __shfl_xor(bv, d);
      const int64_t oi = __shfl_xor(static_cast<int>(bi), d);
      if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
    }
    __syncthreads();
    if (lane == 0) best[wave] = {bv, static_cast<int32_t>(bi)};
    __syncthreads();
    for (int w = 0; w < 4; ++w)
      if (before(best[w].value, best[w].index, bv, bi)) bv = best[w].value, bi = best[w].index;
    if (tid == 0) top[r * m + i] = {bv, static_cast<int32_t>(bi)};
    pv = bv;
    pi = bi;
  }
}

// Offer i of beam k in the beam's own order: its value, and its token.
__device__ __forceinline__ double offer(const BeamArgs& a, int64_t r, int m, int i, const RowTop* top, const double* lse,
                                        int64_t& token) {
  const float s = a.scores[r];
  const double inf = __builtin_inf();
  const bool live = fabsf(s) < __builtin_inff();
  if (live && a.finished && a.finished[r]) {
    token = i == 0 ? a.pad : (i <= a.pad ? i - 1 : i);
    return i == 0 ? static_cast<double>(s) : -inf;
  }
  if (live && fabs(lse[r]) < inf) {
    token = top[r * m + i].index;
    return static_cast<double>(s) + (static_cast<double>(top[r * m + i].value) - lse[r]);
  }
  token = i;
  return -inf;
}

// One wave per request.
__global__ __launch_bounds__(64) void beam_merge_kernel(BeamArgs a, int m, const RowTop* top, const double* lse) {
  const int64_t b = blockIdx.x;
  const int lane = threadIdx.x;
  const int count = static_cast<int>(a.K) * m;
  double pv = __builtin_inf();
  int64_t pi = -1;
  for (int o = 0; o < static_cast<int>(a.n); ++o) {
    double bv = -__builtin_inf();
    int64_t bi = INT64_MAX;
    for (int c = lane; c < count; c += 64) {
      const int64_t k = c / m;
      int64_t token;
      const double v = offer(a, b * a.K + k, m, c % m, top, lse, token);
      const int64_t flat = k * a.V + token;
      if (before(pv, pi, v, flat) && before(v, flat, bv, bi)) bv = v, bi = flat;
    }
    for (int d = 32; d > 0; d >>= 1) {
      const double ov = __shfl_xor(bv, d);
      const int64_t oi = __shfl_xor(static_cast<long long>(bi), d);
      if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
    }
    if (lane == 0) {
      const int64_t k = bi / a.V, token = bi % a.V;
      a.out_scores[b * a.n + o] = static_cast<float>(bv);
      a.parents[b * a.n + o] = k;
      a.tokens[b * a.n + o] = token;
      if (a.finished_out)
        a.finished_out[b * a.n + o] = (a.finished && a.finished[b * a.K + k]) || (a.eos >= 0 && token == a.eos);
    }
    pv = bv;
    pi = bi;
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

// A thread moves one unit of all K rows of a request: every load before the first store, so a row may be the parent
// of several others and be overwritten itself.  Rows that stay are neither read nor written.
template <typename U, int KM>
__device__ __forceinline__ void reorder_unit(char* at, int64_t pitch, const int64_t* parents, int K) {
  U v[KM];
#pragma unroll
  for (int k = 0; k < KM; ++k) {
    if (k >= K) break;
    const int64_t p = parents[k];
    if (p != k && p >= 0 && p < K) v[k] = *reinterpret_cast<const U*>(at + p * pitch);
  }
#pragma unroll
  for (int k = 0; k < KM; ++k) {
    if (k >= K) break;
    const int64_t p = parents[k];
    if (p != k && p >= 0 && p < K) *reinterpret_cast<U*>(at + k * pitch) = v[k];
  }
}

template <int KM>
__global__ __launch_bounds__(256) void reorder_rows_kernel(ReorderTable tab, const int64_t* parents, int K) {
  const int64_t b = blockIdx.y;
  const int64_t* par = parents + b * K;
  int lo = 0, hi = tab.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].block0 <= blockIdx.x)
      lo = mid;
    else
      hi = mid;
  }
  const ReorderTable::Entry& e = tab.t[lo];
  const int64_t off = (static_cast<int64_t>(blockIdx.x - e.block0) * 256 + threadIdx.x) * e.unit;
  if (blockIdx.x == 0 && threadIdx.x < K && (par[threadIdx.x] < 0 || par[threadIdx.x] >= K))
    __hip_atomic_fetch_or(&g_reorder_status, 2u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (off >= e.bytes) return;
  char* at = e.p + b * K * e.pitch + off;
  if (e.unit == 16)
    reorder_unit<uint4, KM>(at, e.pitch, par, K);
  else if (e.unit == 4)
    reorder_unit<uint32_t, KM>(at, e.pitch, par, K);
  else
    reorder_unit<uint8_t, KM>(at, e.pitch, par, K);
}

int64_t round256(int64_t v) { return round_up(std::max<int64_t>(v, 1), 256); }

}  // namespace

int64_t beam_select_ws_bytes(const BeamArgs& a) {
  const int64_t m = std::min(a.n, a.V), rows = a.B * a.K;
  return round256(rows * m * static_cast<int64_t>(sizeof(RowTop))) + round256(rows * 8);
}

int launch_beam_select(const BeamArgs& a, void* ws, int64_t ws_bytes, hipStream_t st) {
  TESM_REQUIRE(a.dt == kF32 || a.dt == kBF16, kErrInvalidArg, "beam select: dtype must be 0 or 1");
  TESM_REQUIRE(a.B >= 0 && a.K >= 1 && a.V >= 1 && a.n >= 1 && a.B < (1LL << 24) && a.V < (1LL << 31) - 65536, kErrInvalidArg,
               "beam select: bad sizes");
  TESM_REQUIRE(a.K <= kBeamMaxN && a.n <= kBeamMaxN, kErrUnsupported,
               "beam select: at most 64 beams and 64 chosen candidates");
  TESM_REQUIRE(a.n <= a.K * a.V, kErrInvalidArg, "beam select: more candidates asked for than there are");
  TESM_REQUIRE(a.ld >= a.V, kErrInvalidArg, "beam select: ld < V");
  TESM_REQUIRE(!a.finished || (a.pad >= 0 && a.pad < a.V), kErrInvalidArg, "beam select: pad outside the vocabulary");
  TESM_REQUIRE(a.eos < a.V, kErrInvalidArg, "beam select: eos outside the vocabulary");
  if (a.B == 0) return kOk;
  TESM_REQUIRE(a.logits && a.scores && a.out_scores && a.parents && a.tokens, kErrInvalidArg,
               "beam select: need logits, scores and the three outputs");
  TESM_REQUIRE(ws && ws_bytes >= beam_select_ws_bytes(a) && aligned(ws, 8), kErrWorkspace,
               "beam select: workspace too small or not 8-byte aligned");
  const int m = static_cast<int>(std::min(a.n, a.V));
  const int64_t rows = a.B * a.K;
  RowTop* top = static_cast<RowTop*>(ws);
  double* lse = reinterpret_cast<double*>(static_cast<char*>(ws) + round256(rows * m * static_cast<int64_t>(sizeof(RowTop))));
  const unsigned grid = static_cast<unsigned>(rows);
  if (a.dt == kBF16)
    beam_row_kernel<kBF16><<<grid, 256, 0, TESM_LOGGED(st, beam_row_kernel<kBF16>)>>>(a, m, top, lse);
  else
    beam_row_kernel<kF32><<<grid, 256, 0, TESM_LOGGED(st, beam_row_kernel<kF32>)>>>(a, m, top, lse);
  beam_merge_kernel<<<static_cast<unsigned>(a.B), 64, 0, TESM_LOGGED(st, beam_merge_kernel)>>>(a, m, top, lse);
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
  if (B == 0 || K == 1) return kOk;
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
