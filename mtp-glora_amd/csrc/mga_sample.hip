// Token sampling from rows of logits with temperature, top-k, top-p and min-p,
// from one given uniform number a row.
//
// With the row's elements in order (value descending, column ascending) the three
// filters each keep a leading run of them, so what is kept is a threshold in that
// order; the token is the first column at which the kept weights, added by
// ascending column, pass u times their total.
//
// Neighbouring borders of that sum lie 2^-17 of it apart in a row of 151 936
// about equal tokens, so the weights e^{(x - max) / T} are taken in 64 bits and
// held as whole numbers of 2^-s of the largest (s = 45 at that width): their sums
// are exact and the same in whatever order they are formed.
//
// One workgroup a row, the row in registers (mga_vocab_row.hpp). Rows with
// 1 <= top_k <= 1024 are settled among the listed candidates; others take the
// weight of every element that is not filtered out.
#include "mga_internal.hpp"
#include "mga_vocab_row.hpp"

namespace mga {

namespace {

// round(2^s e^{(x - top) / T}) for x <= top; 0 for NaN and -inf.
struct Weight {
  float top;
  double topd, c;   // c = log2(e) / T
  int s;
  __device__ __forceinline__ Weight(float m, float temperature, int bits)
      : top(m), topd(m), c(1.4426950408889634074 / (double)temperature), s(bits) {}
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (x == top) return uint64_t(1) << s;   // +inf among them
    const double a = ((double)x - topd) * c;
    if (!(a > (double)(-s - 2))) return 0;
    const double n = __builtin_rint(a), t = (a - n) * 0.69314718055994530942;
    // e^t, |t| <= ln(2) / 2, by its series: the rest is below 2^-47 of it
    double p = 1.0 / 39916800;
    p = __builtin_fma(p, t, 1.0 / 3628800);
    p = __builtin_fma(p, t, 1.0 / 362880);
    p = __builtin_fma(p, t, 1.0 / 40320);
    p = __builtin_fma(p, t, 1.0 / 5040);
    p = __builtin_fma(p, t, 1.0 / 720);
    p = __builtin_fma(p, t, 1.0 / 120);
    p = __builtin_fma(p, t, 1.0 / 24);
    p = __builtin_fma(p, t, 1.0 / 6);
    p = __builtin_fma(p, t, 0.5);
    p = __builtin_fma(p, t, 1.0);
    p = __builtin_fma(p, t, 1.0);
    // 2^52 + p 2^{n + s}, rounded to a whole number by the addition
    const double v = __builtin_amdgcn_ldexp(p, (int)n + s) + 4503599627370496.0;
    return __builtin_bit_cast(uint64_t, v) & ((uint64_t(1) << 52) - 1);
  }
};

// What a running sum has to pass, as a whole number: the first sum >= this is the
// first > u total. u outside [0, 1) and NaN: the first or the last kept token.
__device__ __forceinline__ uint64_t target_of(float u, uint64_t total) {
  if (!(u > 0.f)) return 1;
  const double t = (double)u * (double)total;
  return t < (double)total ? min((uint64_t)t, total - 1) + 1 : total;
}

__device__ __forceinline__ uint64_t mass_needed(float p, uint64_t total) {
  const double t = __builtin_ceil((double)p * (double)total);
  return t >= 1.0 ? min((uint64_t)t, total) : 1;
}

}  // namespace

// The kept element of the smallest column at which the running sum of weights
// reaches its target, among all elements of at least `thr`.
template <typename T, int NB, typename WF>
__device__ int pick_in_row(const Row<T, NB> &row, RowShared &sh, uint64_t thr, WF weight, float u) {
  constexpr int W = RowElem<T>::W;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float least = thr >> 32 > 1 ? rank_value(thr) : kRowNegInf;
  auto kept = [&](float x, int col) { return x >= least && rank_of(x, col) >= thr ? weight(x) : uint64_t(0); };
  auto lane_sum = [&](const i32x4 &v, int col) {
    uint64_t s = 0;
    if (col < row.V) {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float x = RowElem<T>::get(v, e);
        if (x >= least) s += kept(x, col + e);
      }
    }
    return s;
  };
  // in order of the columns: the elements before the vectors, (vector, wave)
  // groups, the elements behind them
  row.each_vec([&](const i32x4 &v, int col, int i) {
    uint64_t s = lane_sum(v, col);
    if (__ballot(s != 0) != 0) s = wave_scan(s);
    if (lane == 63) sh.bins[i * kRowWaves + wave] = s;
  });
  const uint64_t mine = row.ecol >= 0 ? kept(row.edge, row.ecol) : 0;
  const uint64_t edges = wave_scan(mine);
  if (wave == 0 && lane == W - 1) sh.found[0] = edges;
  if (wave == 0 && lane == 2 * W - 1) sh.found[1] = edges;
  __syncthreads();
  const uint64_t before = sh.found[0], behind = sh.found[1] - before;
  __syncthreads();
  const int groups = (row.nvec + kRowThreads - 1) / kRowThreads * kRowWaves;
  const int per = (groups + kRowThreads - 1) / kRowThreads, g0 = min(groups, tid * per), g1 = min(groups, g0 + per);
  uint64_t s = 0, total;
  for (int g = g0; g < g1; ++g) s += sh.bins[g];
  uint64_t at = before + block_scan(s, sh, &total);
  const uint64_t target = target_of(u, before + total + behind);
  if (tid == 0) sh.count = -1;
  __syncthreads();
  if (target > before && target <= before + total) {
    if (at < target && target <= at + s)
      for (int g = g0; g < g1; ++g) {
        if (at + sh.bins[g] >= target) {
          sh.count = g;
          sh.found[0] = target - at;   // to be reached within the group
          break;
        }
        at += sh.bins[g];
      }
    __syncthreads();
    const int g = sh.count;
    if (wave == (g & (kRowWaves - 1))) {
      const int vi = (g / kRowWaves) * kRowThreads + tid;
      i32x4 v = {RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill};
      int col = row.V;
      if (vi < row.nvec) {
        v = reinterpret_cast<const i32x4 *>(row.p + row.head)[vi];
        col = row.head + vi * W;
      }
      const uint64_t in = lane_sum(v, col), upto = wave_scan(in), want = sh.found[0];
      if (upto >= want && upto - in < want) {
        uint64_t run = upto - in;
        int token = -1;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float x = RowElem<T>::get(v, e);
          run += kept(x, col + e);
          if (token < 0 && run >= want) token = col + e;
        }
        sh.count = token;
      }
    }
  } else if (wave == 0) {   // among the single elements
    const uint64_t want = target <= before ? target : target - total;
    if (mine && edges >= want && edges - mine < want) sh.count = row.ecol;
  }
  __syncthreads();
  return sh.count;
}

template <typename T, int NB>
__global__ __launch_bounds__(kRowThreads) void sample_kernel(const T *__restrict__ x, int64_t xs, int32_t V,
                                                             const float *__restrict__ uniform, SampleParams prm,
                                                             int s, int64_t *__restrict__ token) {
  __shared__ RowShared sh;
  const int64_t n = blockIdx.x;
  const int tid = threadIdx.x;
  const float temperature = prm.temperature ? prm.temperature[n] : prm.temperature_all;
  const int top_k = prm.top_k ? prm.top_k[n] : prm.top_k_all;
  const float top_p = prm.top_p ? prm.top_p[n] : prm.top_p_all;
  const float min_p = prm.min_p ? prm.min_p[n] : prm.min_p_all;
  const float u = uniform[n];
  Row<T, NB> row;
  row.load(x + n * xs, V);
  const float tmax = thread_max(row), top = block_max(tmax, sh);
  if (top == kRowNegInf) {   // nothing to draw from
    if (tid == 0) token[n] = -1;
    return;
  }
  if (!(temperature > 0.f)) {   // the first of the largest
    if (tid == 0) sh.count = V;
    __syncthreads();
    row.each_from(top, [&](float, int col) { atomicMin(&sh.count, col); });
    __syncthreads();
    if (tid == 0) token[n] = sh.count;
    return;
  }
  const Weight weight(top, temperature, s);
  // least value that min_p leaves: w >= min_p as (x - top) / T >= ln(min_p)
  float least = kRowNegInf;
  if (min_p > 0.f) {
    const double b = min_p < 1.f ? (double)top + (double)temperature * log((double)min_p) : (double)top;
    least = (float)b;
    if ((double)least < b) least = rank_value((uint64_t)(value_key(least) + 1) << 32);   // the next one up
  }
  const bool by_k = top_k > 0 && top_k < V, by_p = top_p < 1.f;
  if (by_k && top_k <= kMaxTop) {
    top_list(row, sh, tmax, top_k);
    // thread i has the i-th element in order
    const uint64_t r = tid < top_k ? sh.list[tid] : 0;
    const float v = rank_value(r);
    const uint64_t w = tid < top_k ? weight(v) : 0;
    uint64_t total;
    const uint64_t before = block_scan(w, sh, &total);
    const bool keep = tid < top_k && (tid == 0 || ((!by_p || before < mass_needed(top_p, total)) && v >= least));
    // the kept ones by column
    const int n_kept = __syncthreads_count(keep);
    if (keep) sh.list[tid] = (uint64_t)(uint32_t)~rank_col(r) << 32 | r >> 32;
    sort_list(sh, n_kept);
    const uint64_t e = tid < n_kept ? sh.list[tid] : 0;
    const uint64_t we = tid < n_kept ? weight(rank_value(e << 32)) : 0;
    const uint64_t upto = block_scan(we, sh, &total), target = target_of(u, total);
    if (we && upto < target && target <= upto + we) token[n] = ~(uint32_t)(e >> 32);
    return;
  }
  uint64_t thr = 0;
  if (by_k)
    thr = radix_threshold<true>(row, sh, 0, [](float) { return uint64_t(1); }, [&](uint64_t) { return (uint64_t)top_k; });
  if (by_p) thr = radix_threshold<false>(row, sh, thr, weight, [&](uint64_t total) { return mass_needed(top_p, total); });
  if (least > kRowNegInf) thr = max(thr, (uint64_t)value_key(least) << 32);
  const int t = pick_in_row(row, sh, thr, weight, u);
  if (tid == 0) token[n] = t;
}

template <typename T>
static void sample_typed(const void *x, int64_t xs, int32_t N, int32_t V, const float *u, const SampleParams &prm,
                         int s, int64_t *token, hipStream_t st) {
  with_row_blocks<T>(V, [&](auto nb) {
    hipLaunchKernelGGL((sample_kernel<T, decltype(nb)::value>), dim3(N), dim3(kRowThreads), 0, st, (const T *)x, xs, V,
                       u, prm, s, token);
  });
}

void launch_sample(const void *x, int64_t xs, int32_t N, int32_t V, int dtype, const float *u,
                   const SampleParams &prm, int64_t *token, hipStream_t st) {
  int bits = 0;
  while ((int64_t(1) << bits) < V) ++bits;
  const int s = 45 < 62 - bits ? 45 : 62 - bits;   // V weights of up to 2^s, below 2^63
  auto run = dtype == kDtF32 ? sample_typed<float> : dtype == kDtF16 ? sample_typed<f16_t> : sample_typed<bf16_t>;
  run(x, xs, N, V, u, prm, s, token, st);
}

}  // namespace mga
