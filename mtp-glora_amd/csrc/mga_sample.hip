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
// One workgroup a row (mga_vocab_row.hpp). Rows with 1 <= top_k <= 1024, or whose
// filters leave at most kListCap tokens, are settled among listed candidates;
// others add the weight of every token that is left. Such a weight is some 25
// double operations, 24 us for a row of 151 936 on its compute unit; bf16 logits
// take few values, so their weights are tabulated and a histogram of the values
// gives the thresholds.
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

// ---- bf16: the weights of the values that occur ----------------------------------

// Positions 0 .. kTable - 1 in descending order of the value: the positive values of
// kOctaves octaves, then the negative ones. The top octave is that of the largest
// magnitude with a weight; the values below the window (2^-27 of that) are few, and
// stand between the halves.
constexpr int kOctaves = 28, kHalf = kOctaves * 128, kTable = 2 * kHalf, kPerThread = kTable / kRowThreads;
static_assert(kTable == kPerThread * kRowThreads && kHalf % kPerThread == 0, "a thread's positions are of one sign");

struct TableShared {
  uint64_t weight[kTable + 1];   // the last: no weight
  uint32_t count[kTable];
  uint64_t small_weight;
  uint32_t small_count;
};

struct Window {
  uint32_t lo, gap;
  // values as whole numbers in descending order: 0 .. 0x7FFF positive, 0x8000 .. negative
  __device__ __forceinline__ static uint32_t descending(uint32_t bits) { return bits ^ (bits & 0x8000u ? 0u : 0x7FFFu); }
  // kTable: none (below the window, past its ends, NaN)
  __device__ __forceinline__ uint32_t position(uint32_t bits) const {
    const uint32_t e = descending(bits) - lo, neg = e - gap;
    return e < (uint32_t)kHalf ? e : neg - (uint32_t)kHalf < (uint32_t)kHalf ? neg : (uint32_t)kTable;
  }
  __device__ __forceinline__ bool small(uint32_t bits) const { return descending(bits) - lo - (uint32_t)kHalf < gap; }
  __device__ __forceinline__ float value(int pos) const {
    return __builtin_bit_cast(float, descending(lo + pos + (pos >= kHalf ? gap : 0)) << 16);
  }
};

__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x) >> 16; }

// Weight of a bf16 value from the table.
struct Tabulated {
  Weight weight;
  Window win;
  const TableShared *tab;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const uint32_t b = bits_of(x);
    return win.small(b) ? weight(x) : tab->weight[win.position(b)];
  }
};

// Weights of the window's values; the counts cleared. top is finite.
__device__ __forceinline__ Window make_table(TableShared &tab, const Weight &weight) {
  const double least = weight.topd - (weight.s + 2) / weight.c;   // nothing below it has a weight
  const float big = fminf(fmaxf(fabsf((float)least), fabsf(weight.top)), 3.3895314e38f);
  const uint32_t octave = max(__builtin_bit_cast(uint32_t, big) >> 23, (uint32_t)kOctaves);
  const uint32_t mag0 = (octave + 1 - kOctaves) << 7;   // the window's smallest magnitude
  const Window win{0x7FFFu - (mag0 + kHalf - 1), 2 * mag0};
#pragma unroll 1
  for (int j = 0; j < kPerThread; ++j) {
    const int pos = (int)threadIdx.x + j * kRowThreads;
    const float v = win.value(pos);
    tab.weight[pos] = v <= weight.top ? weight(v) : 0;
    tab.count[pos] = 0;
  }
  if (threadIdx.x == 0) {
    tab.weight[kTable] = 0;
    tab.small_weight = 0;
    tab.small_count = 0;
  }
  __syncthreads();
  return win;
}

// Threshold of top_k and top_p by the histogram of the row's values, and how many
// elements it leaves; what scan_row left stays. False where a cut falls among the values below the window.
__device__ bool table_threshold(const Row<bf16_t> &row, RowShared &sh, TableShared &tab, const Tabulated &t, bool by_k,
                                uint64_t top_k, bool by_p, float top_p, uint64_t *thr, uint64_t *kept) {
  const int tid = threadIdx.x;
  auto tally = [&](uint32_t bits) {
    const uint32_t pos = t.win.position(bits);
    if (pos < (uint32_t)kTable) atomicAdd(&tab.count[pos], 1u);
    else if (t.win.small(bits)) {
      atomicAdd(&tab.small_count, 1u);
      atomicAdd((unsigned long long *)&tab.small_weight,
                (unsigned long long)t.weight(__builtin_bit_cast(float, bits << 16)));
    }
  };
  row.each_vec([&](const i32x4 &v, int col, int) {
    if (col >= row.V) return;
#pragma unroll 2
    for (int d = 0; d < 4; ++d) {
      tally((uint32_t)v[d] & 0xFFFFu);
      tally((uint32_t)v[d] >> 16);
    }
  });
  if (row.ecol >= 0) tally(bits_of(row.edge));
  __syncthreads();
  // a thread's positions; the values below the window stand before thread kHalf / kPerThread's
  const int p0 = tid * kPerThread;
  const uint32_t between = p0 == kHalf ? tab.small_count : 0;
  uint32_t c[kPerThread];
  uint64_t cs = between, total;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) cs += c[j] = tab.count[p0 + j];
  const uint64_t before = block_scan(cs, sh, &total);
  int cut = kTable;        // position of the last kept value, -1: below the window
  uint64_t ties = 0;       // kept elements of it
  auto share = [&](int pos, uint64_t n, uint64_t left) {   // by the one thread that has it
    sh.count = pos;
    sh.found[0] = n;
    sh.found[1] = left;
  };
  auto shared = [&]() {
    __syncthreads();
    cut = sh.count;
    ties = sh.found[0];
    *kept = sh.found[1];
    __syncthreads();
  };
  *thr = 0;
  *kept = total;
  if (by_k && total > top_k) {
    if (before < top_k && top_k <= before + cs) {
      uint64_t run = before + between;
      int pos = run >= top_k ? -1 : -2;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        if (pos == -2 && run + c[j] >= top_k) {
          pos = p0 + j;
          share(pos, top_k - run, top_k);
        }
        run += c[j];
      }
      if (pos == -1) share(-1, 0, 0);
    }
    shared();
    if (cut < 0) return false;
  }
  if (by_p) {
    const uint64_t mid = between && cut >= kHalf ? tab.small_weight : 0;
    uint64_t ms = mid, z;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      if (p0 + j >= cut) c[j] = p0 + j == cut ? (uint32_t)ties : 0;
      ms += c[j] * tab.weight[p0 + j];
    }
    const uint64_t mb = block_scan(ms, sh, &z), want = mass_needed(top_p, z);
    if (mb < want && want <= mb + ms) {
      uint64_t run = mb + mid, left = before + between;
      int pos = run >= want ? -1 : -2;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        const uint64_t w = tab.weight[p0 + j], m = c[j] * w;
        if (pos == -2 && m && run + m >= want) {
          const uint64_t n = (want - run + w - 1) / w;
          pos = p0 + j;
          share(pos, n, left + n);
        }
        run += m;
        left += c[j];
      }
      if (pos == -1) share(-1, 0, 0);
    }
    shared();
    if (cut < 0) return false;
  }
  if (cut == kTable) return true;
  const uint32_t key = value_key(t.win.value(cut));
  *thr = ties >= tab.count[cut] ? (uint64_t)key << 32 : column_threshold(row, sh, 0, key, ties);
  return true;
}

}  // namespace

// The kept element of the smallest column at which the running sum of weights
// reaches its target, among the n <= kListCap ranks of sh.list: columns by two
// digits of ten bits.
template <typename WF>
__device__ int pick_in_list(RowShared &sh, int n, const WF &weight, float u) {
  constexpr int kEach = kListCap / kRowThreads;
  const int tid = threadIdx.x;
  uint64_t w[kEach];
  int col[kEach];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = tid + i * kRowThreads;
    w[i] = 0;
    if (at < n) {
      const uint64_t r = sh.list[at];
      col[i] = rank_col(r);
      w[i] = weight(rank_value(r));
    }
  }
  uint64_t target = 0, total;
  int token = 0;
#pragma unroll
  for (int digit = 0; digit < 2; ++digit) {
    sh.bins[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (w[i] && (digit == 0 || col[i] >> 10 == token))
        atomicAdd((unsigned long long *)&sh.bins[digit ? col[i] & 1023 : col[i] >> 10], (unsigned long long)w[i]);
    find_bin(sh, sh.bins, 1024, false, [&](uint64_t t) { return digit ? target : target_of(u, t); }, &total);
    if (digit == 0) target = target_of(u, total);
    target -= sh.found[1];
    token = token << 10 | (int)sh.found[0];
    __syncthreads();
  }
  return token;
}

// The same among all elements of at least `thr`.
template <typename T, typename WF>
__device__ int pick_in_row(const Row<T> &row, RowShared &sh, uint64_t thr, const WF &weight, float u) {
  constexpr int W = RowElem<T>::W;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float least = thr >> 32 > 1 ? rank_value(thr) : kRowNegInf;
  const int last = (uint32_t)thr ? rank_col(thr) : row.V;   // of the elements equal to least, the last column that counts
  auto kept = [&](float x, int col) {
    return x > least || (x == least && col <= last) ? weight(x) : uint64_t(0);
  };
  auto lane_sum = [&](const i32x4 &v, int col) {
    uint64_t s = 0;
    if (col < row.V) {
#pragma unroll
      for (int e = 0; e < W; ++e) s += kept(RowElem<T>::get(v, e), col + e);
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
  const int groups = row.blocks() * 4 * kRowWaves;
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
    const uint64_t want = sh.found[0];
    __syncthreads();
    if (wave == (g & (kRowWaves - 1))) {
      const int vi = (g / kRowWaves) * kRowThreads + tid;
      i32x4 v = {RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill};
      int col = row.V;
      if (vi < row.nvec) {
        v = reinterpret_cast<const i32x4 *>(row.p + row.head)[vi];
        col = row.head + vi * W;
      }
      const uint64_t in = lane_sum(v, col), upto = wave_scan(in);
      if (upto >= want && upto - in < want) {
        uint64_t run = upto - in;
        int token = -1;
#pragma unroll
        for (int e = 0; e < W; ++e) {
          run += kept(RowElem<T>::get(v, e), col + e);
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

// LDS of a type's kernel: the table for bf16.
template <typename T> struct SampleShared : RowShared {};
template <> struct SampleShared<bf16_t> : RowShared { TableShared tab; };

template <typename T>
__global__ __launch_bounds__(kRowThreads) void sample_kernel(const T *__restrict__ x, int64_t xs, int32_t V,
                                                             const float *__restrict__ uniform, SampleParams prm,
                                                             int s, int32_t group, int64_t *__restrict__ token) {
  __shared__ SampleShared<T> sh;
  const int64_t n = blockIdx.x;
  const int tid = threadIdx.x;
  const float temperature = prm.temperature ? prm.temperature[n] : prm.temperature_all;
  const int top_k = prm.top_k ? prm.top_k[n] : prm.top_k_all;
  const float top_p = prm.top_p ? prm.top_p[n] : prm.top_p_all;
  const float min_p = prm.min_p ? prm.min_p[n] : prm.min_p_all;
  const float u = uniform[n];
  Row<T> row;
  row.load(x + n * xs, V);
  RowSum none;
  const float tmax = scan_row<false>(row, sh, group, 0.f, none), top = block_max(tmax, sh);
  if (top == kRowNegInf) {   // nothing to draw from
    if (tid == 0) token[n] = -1;
    return;
  }
  if (!(temperature > 0.f)) {   // the first of the largest
    if (tid == 0) sh.count = V;
    __syncthreads();
    scan_hits(row, sh, group, top, [&](float, int col) { atomicMin(&sh.count, col); });
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
  int t;
  if (by_k && top_k <= kMaxTop) {
    top_list(row, sh, group, tmax, top_k);
    // thread i has the i-th element in order; the kept ones are the first ones
    const uint64_t r = tid < top_k ? sh.list[tid] : 0;
    const uint64_t w = tid < top_k && by_p ? weight(rank_value(r)) : 0;
    uint64_t total = 0, before = 0;
    if (by_p) before = block_scan(w, sh, &total);
    const bool keep = tid < top_k && (tid == 0 || ((!by_p || before < mass_needed(top_p, total)) && rank_value(r) >= least));
    t = pick_in_list(sh, __syncthreads_count(keep), weight, u);
  } else {
    uint64_t thr = 0, kept = by_k ? (uint64_t)top_k : (uint64_t)V;
    const uint64_t floor = least > kRowNegInf ? (uint64_t)value_key(least) << 32 : 0;
    // the elements of at least thr into the list; how many there are
    auto gather = [&]() {
      const float low = rank_value(thr);
      if (tid == 0) sh.count = 0;
      __syncthreads();
      scan_hits(row, sh, group, low, [&](float v, int col) {
        const uint64_t r = rank_of(v, col);
        if (r < thr) return;
        const int at = atomicAdd(&sh.count, 1);
        if (at < kListCap) sh.list[at] = r;
      });
      __syncthreads();
      return sh.count;
    };
    int listed = kListCap + 1;
    if (floor && !by_k && !by_p) {   // min_p alone: mostly few
      thr = floor;
      listed = gather();
    }
    auto threshold = [&]() {   // digit by digit
      if (by_k)
        thr = radix_threshold<true>(row, sh, 0, [](float) { return uint64_t(1); },
                                    [&](uint64_t) { return (uint64_t)top_k; });
      if (by_p)
        thr = radix_threshold<false>(row, sh, thr, weight, [&](uint64_t total) { return mass_needed(top_p, total); });
      thr = max(thr, floor);
    };
    if (listed <= kListCap) {
      t = pick_in_list(sh, listed, weight, u);
    } else if constexpr (sizeof(SampleShared<T>) > sizeof(RowShared)) {
      // up to kTable columns, their own weights are no more work than the table's
      if (top < -kRowNegInf && V > kTable) {
        const Tabulated tw{weight, make_table(sh.tab, weight), &sh.tab};
        bool found = true;
        if (by_k || by_p) {
          found = table_threshold(row, sh, sh.tab, tw, by_k, top_k, by_p, top_p, &thr, &kept);
          if (!found) threshold();
          thr = max(thr, floor);
        }
        if (found && kept <= kListCap && thr >> 32 > 1) listed = gather();
        t = listed <= kListCap ? pick_in_list(sh, listed, tw, u) : pick_in_row(row, sh, thr, tw, u);
      } else {
        threshold();
        t = pick_in_row(row, sh, thr, weight, u);
      }
    } else {
      threshold();
      t = pick_in_row(row, sh, thr, weight, u);
    }
  }
  if (tid == 0) token[n] = t;
}

template <typename T>
static void sample_typed(const void *x, int64_t xs, int32_t N, int32_t V, const float *u, const SampleParams &prm,
                         int s, int64_t *token, hipStream_t st) {
  hipLaunchKernelGGL(sample_kernel<T>, dim3(N), dim3(kRowThreads), 0, st, (const T *)x, xs, V, u, prm, s,
                     row_group<T>(V), token);
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
