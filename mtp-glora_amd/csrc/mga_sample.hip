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
// held as whole numbers of 2^-s of the largest (s = 44 at that width): their sums
// are exact and the same in whatever order they are formed.
//
// One workgroup a row (mga_vocab_row.hpp). Rows with 1 <= top_k <= 1024, or whose
// filters leave at most kListCap tokens, are settled among listed candidates; others
// add the weight of every token that is left. Such a weight is some 25 double
// operations, 24 us for a row of 151 936 on its compute unit, or seven by a table of
// roots; bf16 logits take few values, so their weights are tabulated and a histogram of
// the values gives the thresholds. 256 rows of 151 936 bf16, a workgroup and a compute
// unit each: the largest logit 17 us (4.5 TB/s), top-k 40 26, temperature alone 50,
// top-p 0.95 with thousands left 68, of which the histogram's and the table's reads of
// LDS at random bound the last two passes. fp16 and fp32, whose thresholds are found
// digit by digit: temperature alone 66 and 79, top-p 0.95 158 and 193. Of one row (14 us
// with top-k 50) the read is a third, the ordered list half.
#include "mga_internal.hpp"
#include "mga_vocab_row.hpp"

namespace mga {

namespace {

// 2^f for |f| <= 1 / 2 by the series of e^{f ln 2}: the rest is below 2^-47 of it.
__device__ __forceinline__ double exp2_part(double f) {
  double p = 4.44553827187081e-10;
  p = __builtin_fma(p, f, 7.054911620801121e-09);
  p = __builtin_fma(p, f, 1.0178086009239696e-07);
  p = __builtin_fma(p, f, 1.3215486790144305e-06);
  p = __builtin_fma(p, f, 1.5252733804059838e-05);
  p = __builtin_fma(p, f, 0.00015403530393381606);
  p = __builtin_fma(p, f, 0.0013333558146428441);
  p = __builtin_fma(p, f, 0.009618129107628477);
  p = __builtin_fma(p, f, 0.055504108664821576);
  p = __builtin_fma(p, f, 0.2402265069591007);
  p = __builtin_fma(p, f, 0.6931471805599453);
  return __builtin_fma(p, f, 1.0);
}

// 2^52: added to a smaller number, it leaves its nearest whole number in the low bits
constexpr double kTwo52 = 4503599627370496.0;
constexpr uint64_t kLow52 = (uint64_t(1) << 52) - 1;

// round(2^s e^{(x - top) / T}) for x <= top; 0 for NaN and -inf. Where top is +inf it
// counts as 2^128, 2^104 above the largest number: that and all others have weight 0.
struct Weight {
  double topd, c;   // c = log2(e) / T
  float top;
  int s;
  __device__ __forceinline__ Weight(float m, float temperature, int bits) : top(m), s(bits) {
    const bool inf = m == -kRowNegInf;
    c = inf ? 1.0 : 1.4426950408889634074 / (double)temperature;
    topd = inf ? 0x1p128 : (double)m;
  }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    constexpr double kMagic = 1.5 * kTwo52;
    const double v = (double)x > topd ? topd : (double)x;   // NaN stays
    // log2 of the weight; far below 2^-s (and NaN) at a value that rounds to 0
    const double a = __builtin_fmax((v - topd) * c, (double)(-s - 2));
    const double m = a + kMagic, f = a - (m - kMagic);   // m: the nearest whole number in its low bits
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, m) + (uint32_t)s;
    const double w = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, exp2_part(f)) + ((uint64_t)n << 52));
    return __builtin_bit_cast(uint64_t, w + kTwo52) & kLow52;
  }
};

// The same for whole rows. A double operation takes 16 cycles a wave here, four
// times a float one: with 2^{i / 256} from LDS seven of them are left of fourteen
// (32 003 weights a row: 21 -> 12 us). Of a row of 32 003 fp32 drawn by temperature alone,
// 38 000 cycles, the pass of the weights takes 21 600, the double operations 14 000 of
// those; the first look 4 800, the roots 2 400, the sums' joining and the draw 9 400.
struct RowWeight {
  double c, base;        // 768 + (x - top) c = x c + base: 43 bits of fraction in [512, 1024)
  float low, top;        // x <= low has no weight
  const double *roots;   // 2^{i / 256}
  int s, rough;
  __device__ __forceinline__ RowWeight(const Weight &w, const double *table) : top(w.top), roots(table), s(w.s) {
    // c so large that the number below top is 60 to 122 powers of two away: a larger one
    // changes no weight (+inf: the largest number is 60 away)
    c = fmin(w.c, 1020054733.0 / fabs(w.topd));
    base = 768.0 - w.topd * c;
    // top c + base is 768 where base has its 43 bits, else next to it
    rough = __builtin_amdgcn_readfirstlane(!(fabs(base) < 1024.0));
    const double l = w.topd - (s + 3) / c;
    low = (float)l;
    if ((double)low > l) low = rank_value((uint64_t)(value_key(low) - 1) << 32);   // the next one down
  }
  // x finite or +inf. The weight of top is 2^s itself: a share of equal largest elements
  // that is a whole number of them stays one.
  __device__ __forceinline__ uint64_t operator()(float x) const { return x >= top ? uint64_t(1) << s : fine(x); }
  // The same unless rough.
  __device__ __forceinline__ uint64_t fine(float x) const {
    const double m = __builtin_fma((double)fminf(fmaxf(x, low), top), c, base);
    const uint64_t bits = __builtin_bit_cast(uint64_t, m);
    const uint32_t hi = (uint32_t)(bits >> 32);   // 12 bits of exponent, 9 of whole part, 11 of fraction
    const double f = m - __builtin_bit_cast(double, (uint64_t)(hi & ~7u) << 32);   // below 2^-8
    double p = __builtin_fma(0.009618129107628477, f, 0.055504108664821576);
    p = __builtin_fma(p, f, 0.2402265069591007);
    p = __builtin_fma(p, f, 0.6931471805599453);
    p = __builtin_fma(p, f, 1.0);
    const uint32_t n = (hi >> 11 & 511u) - 256u + (uint32_t)s;
    const double r = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, roots[hi >> 3 & 255u]) + ((uint64_t)n << 52));
    return __builtin_bit_cast(uint64_t, __builtin_fma(r, p, kTwo52)) & kLow52;
  }
};
__device__ __forceinline__ void make_roots(double *roots) {
  if (threadIdx.x < 256) {
    const int i = threadIdx.x - (threadIdx.x > 128 ? 256 : 0);
    roots[threadIdx.x] = exp2_part(i / 256.0) * (threadIdx.x > 128 ? 2.0 : 1.0);
  }
  __syncthreads();
}

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

// The table has the positive values of kOctaves octaves at [0, kHalf) by magnitude,
// then the negative ones. The top octave is one above that of the largest magnitude
// that has a weight; what is larger still (-inf, NaN) shares its last entries, which
// have none. Values below the window (2^-31 of that magnitude) are few: they are
// computed.
constexpr int kOctaves = 32, kHalf = kOctaves * 128, kTable = 2 * kHalf, kPerThread = kTable / kRowThreads;

struct TableShared {
  uint64_t weight[kTable];
  uint64_t small_weight;
  uint32_t small_count;
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct Window {
  uint32_t mag0;   // the smallest magnitude, bits of a bf16
  // Two values' entries in the halves of a word. Where one is below the window its
  // bit 15 is set (13 bits are the entry).
  __device__ __forceinline__ uint32_t entries(uint32_t two) const {
    const u16x2 low = (u16x2)(uint16_t)mag0, high = (u16x2)(uint16_t)(mag0 + kHalf - 1);
    const u16x2 m = __builtin_elementwise_min(__builtin_bit_cast(u16x2, two & 0x7FFF7FFFu), high) - low;
    return __builtin_bit_cast(uint32_t, m) | (two >> 3 & 0x10001000u);
  }
  __device__ __forceinline__ float value(int entry) const {
    const uint32_t bits = mag0 + (entry & (kHalf - 1)) + (entry & kHalf ? 0x8000u : 0u);
    return __builtin_bit_cast(float, bits << 16);
  }
};
static_assert(kHalf == 0x1000, "the sign's place in entries()");
constexpr uint32_t kBelow = 0x80008000u;

// Entries in descending order of the value.
__device__ __forceinline__ int entry_at(int place) { return place < kHalf ? kHalf - 1 - place : place; }

constexpr float kLeastNumber = -3.402823466e38f;

// Weight of a value that is at least `least` (a number), computed.
struct Computed {
  RowWeight weight;
  float least;
  __device__ __forceinline__ uint64_t operator()(float x) const { return x >= least ? weight(x) : 0; }
};

// The same for bf16, from the table.
struct Tabulated {
  Weight weight;
  float least;
  Window win;
  const TableShared *tab;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    const uint32_t e = win.entries(__builtin_bit_cast(uint32_t, x) >> 16);
    return !(x >= least) ? 0 : e & 0x8000u ? weight(x) : tab->weight[e & (kTable - 1)];
  }
};

// The window for values up to weight.top; false where none will do.
__device__ __forceinline__ bool find_window(const Weight &weight, Window *win) {
  const double least = (double)weight.top - (weight.s + 2) / weight.c;   // nothing below it has a weight
  const float big = fmaxf(fabsf((float)least), fabsf(weight.top));
  const uint32_t octave = max((__builtin_bit_cast(uint32_t, big) >> 23) + 1, (uint32_t)kOctaves);   // zeros stay below it
  win->mag0 = ((octave + 1) << 7) - kHalf;
  return octave <= 254;   // no octave of infinities
}

__device__ __forceinline__ void make_table(TableShared &tab, const Weight &weight, const Window &win) {
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int e = (int)threadIdx.x + j * kRowThreads;
    const float v = win.value(e);
    const uint64_t w = weight(fminf(v, weight.top));
    tab.weight[e] = v <= weight.top ? w : 0;
  }
  if (threadIdx.x == 0) {
    tab.small_weight = 0;
    tab.small_count = 0;
  }
  __syncthreads();
}

// The rank of the element that is number `ties` by column of the `there` <= kFewTies
// ones that have this value: they are listed, and each counts those before it.
constexpr uint32_t kFewTies = 256;
__device__ __forceinline__ uint64_t tied_threshold(const Row<bf16_t> &row, RowShared &sh, float value, int there,
                                                   int ties) {
  uint64_t *list = sh.list;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  auto one = [&](float x, int col) {
    if (x == value) list[atomicAdd(&sh.count, 1)] = (uint32_t)~col;
  };
  row.template each_vec<3>([&](const i32x4 &v, int col) {
    if (col >= row.V) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) one(RowElem<bf16_t>::get(v, e), col + e);
  }, [](int) {});
  if (row.ecol >= 0) one(row.edge, row.ecol);
  __syncthreads();
  for (int i = threadIdx.x; i < there; i += kRowThreads) {
    const uint64_t mine = list[i];
    int above = 0;
    for (int j = 0; j < there; ++j) above += list[j] > mine;
    if (above == ties - 1) sh.found[0] = mine;
  }
  __syncthreads();
  const uint64_t col = sh.found[0];
  __syncthreads();
  return (uint64_t)value_key(value) << 32 | col;
}

// Threshold of top_k and top_p by the histogram of the row's values (counted in
// sh.list), and how many elements it leaves; what scan_row left stays. More than
// kListCap: its key alone, and how many elements of that key count (quota). False
// where a cut falls among the values below the window.
__device__ __forceinline__ bool table_threshold(const Row<bf16_t> &row, RowShared &sh, TableShared &tab,
                                                const Tabulated &t, bool by_k, uint64_t top_k, bool by_p, float top_p,
                                                uint64_t *thr, uint64_t *kept, uint64_t *quota) {
  const int tid = threadIdx.x;
  static_assert(sizeof(sh.list) >= kTable * sizeof(uint32_t), "the counts");
  uint32_t *count = reinterpret_cast<uint32_t *>(sh.list);
  for (int i = tid; i < kTable; i += kRowThreads) count[i] = 0;
  __syncthreads();
  auto tally = [&](uint32_t e) {   // the last entries have no weight, and may be most of a masked row
    if ((e & (kHalf - 1)) != kHalf - 1) atomicAdd(&count[e & (kTable - 1)], 1u);
  };
  auto one = [&](uint32_t bits) {
    const uint32_t e = t.win.entries(bits);
    if (!(e & 0x8000u)) return tally(e);
    atomicAdd(&tab.small_count, 1u);
    atomicAdd((unsigned long long *)&tab.small_weight,
              (unsigned long long)t.weight(__builtin_bit_cast(float, bits << 16)));
  };
  row.template each_vec<3>([&](const i32x4 &v, int col) {
    if (col >= row.V) return;
    uint32_t e[4], below = 0;
#pragma unroll
    for (int d = 0; d < 4; ++d) below |= e[d] = t.win.entries((uint32_t)v[d]);
    if (below & kBelow) {
#pragma unroll 1
      for (int d = 0; d < 8; ++d) one((uint32_t)v[d >> 1] >> (d & 1) * 16 & 0xFFFFu);
      return;
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      tally(e[d] & 0xFFFFu);
      tally(e[d] >> 16);
    }
  }, [](int) {});
  if (row.ecol >= 0) one(__builtin_bit_cast(uint32_t, row.edge) >> 16);
  __syncthreads();
  // a thread's entries, in descending order; the values below the window stand
  // before those of the first thread of the negative half
  const int p0 = tid * kPerThread;
  const uint32_t between = p0 == kHalf ? tab.small_count : 0;
  uint32_t c[kPerThread];
  uint64_t cs = between, total;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) cs += c[j] = count[entry_at(p0 + j)];
  const uint64_t before = block_scan(cs, sh, &total);
  int cut = kTable;        // place of the last kept value, -1: below the window
  uint64_t ties = 0;       // kept elements of it
  auto share = [&](int place, uint64_t n, uint64_t left) {   // by the one thread that has it
    sh.count = place;
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
      int place = run >= top_k ? -1 : -2;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        if (place == -2 && run + c[j] >= top_k) {
          place = p0 + j;
          share(place, top_k - run, top_k);
        }
        run += c[j];
      }
      if (place == -1) share(-1, 0, 0);
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
      ms += c[j] * tab.weight[entry_at(p0 + j)];
    }
    const uint64_t mb = block_scan(ms, sh, &z), want = mass_needed(top_p, z);
    if (mb < want && want <= mb + ms) {
      uint64_t run = mb + mid, left = before + between;
      int place = run >= want ? -1 : -2;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        const uint64_t w = tab.weight[entry_at(p0 + j)], m = c[j] * w;
        if (place == -2 && m && run + m >= want) {
          const uint64_t n = (want - run + w - 1) / w;
          place = p0 + j;
          share(place, n, left + n);
        }
        run += m;
        left += c[j];
      }
      if (place == -1) share(-1, 0, 0);
    }
    shared();
    if (cut < 0) return false;
  }
  if (cut == kTable) return true;
  const float value = t.win.value(entry_at(cut));
  const uint64_t key = (uint64_t)value_key(value) << 32;
  const uint32_t there = count[entry_at(cut)];
  __syncthreads();   // the counts are over
  *thr = key;
  if (ties >= there) return true;
  if (*kept > kListCap) *quota = ties;
  else *thr = there > kFewTies ? column_threshold(row, sh, 0, (uint32_t)(key >> 32), ties)
                               : tied_threshold(row, sh, value, (int)there, (int)ties);
  return true;
}

}  // namespace

// The kept element of the smallest column at which the running sum of weights
// reaches its target, among the n <= kListCap ranks of sh.list: columns by two
// digits of ten bits.
template <typename WF>
__device__ __forceinline__ int pick_in_list(RowShared &sh, int n, const WF &weight, float u) {
  constexpr int kEach = kListCap / kRowThreads;
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= 256) {   // each entry adds those of columns up to its own
    const uint64_t r = tid < n ? sh.list[tid] : 0;
    const int col = rank_col(r);
    const uint64_t w = tid < n ? weight(rank_value(r)) : 0;
    if (tid < 256) {
      sh.bins[2 * tid] = w;
      sh.bins[2 * tid + 1] = (uint64_t)col;
    }
    __syncthreads();
    if (tid < n) {
      uint64_t upto = 0, all = 0;
      for (int i = 0; i < n; i += 8)   // those past n have no weight
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const uint64_t o = sh.bins[2 * (i + u)];
          all += o;
          upto += (int)sh.bins[2 * (i + u) + 1] <= col ? o : 0;
        }
      const uint64_t target = target_of(u, all);
      if (w && upto >= target && upto - w < target) sh.count = col;
    }
    __syncthreads();
    return sh.count;
  }
  uint64_t w[kEach];
  int col[kEach];
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

// The weights of a vector's elements, added.
template <typename T>
__device__ __forceinline__ uint64_t vector_sum(const Computed &weight, const i32x4 &v) {
  uint64_t s = 0;
  if (weight.weight.rough) {   // of the whole row
#pragma unroll 1
    for (int e = 0; e < RowElem<T>::W; ++e) s += weight(RowElem<T>::get(v, e));
    return s;
  }
#pragma unroll
  for (int e = 0; e < RowElem<T>::W; ++e) {   // 96 rows of 32 003 fp32: 18.3 us, with the comparison to top 19.4
    const float x = RowElem<T>::get(v, e);
    s += x >= weight.least ? weight.weight.fine(x) : 0;
  }
  return s;
}
template <typename T>
__device__ __forceinline__ uint64_t vector_sum(const Tabulated &t, const i32x4 &v) {
  uint32_t e[4], below = 0;
  uint64_t s = 0;
#pragma unroll
  for (int d = 0; d < 4; ++d) below |= e[d] = t.win.entries((uint32_t)v[d]);
  // a random read of LDS by 64 lanes takes some 20 cycles, by few of them less
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (RowElem<T>::get(v, i) >= t.least) s += t.tab->weight[(e[i >> 1] >> (i & 1) * 16) & (kTable - 1)];
  if (below & kBelow) {
    s = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) s += t(RowElem<T>::get(v, i));
  }
  return s;
}

// The same among all elements of at least weight.least (`weight` is 0 for smaller
// ones), of those equal to it the first `quota` by column (~0: all).
template <typename T, typename WF>
__device__ __forceinline__ int pick_in_row(const Row<T> &row, RowShared &sh, uint64_t quota, const WF &weight, float u) {
  constexpr int W = RowElem<T>::W;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool some = quota != ~uint64_t(0);
  const uint64_t tie = weight(weight.least);
  uint32_t *tied = reinterpret_cast<uint32_t *>(sh.list);   // a group's elements equal to the least
  // the weight of the `n` of them, behind `before` others, that do not count
  auto over = [&](uint64_t before, uint64_t n) {
    return (before + n <= quota ? 0 : before >= quota ? n : before + n - quota) * tie;
  };
  // In order of the columns: the elements before the vectors, the (vector, wave)
  // groups, the elements behind them; within a group its lanes, within a lane its
  // elements.
  int i = 0;
  row.template each_vec<3>(
      [&](const i32x4 &v, int) {
        const uint64_t s = last_lane(wave_scan(vector_sum<T>(weight, v)));   // 0 of the -inf past the row's end
        uint32_t c = 0;
        if (some) {
#pragma unroll
          for (int e = 0; e < W; ++e) c += __popcll(__ballot(RowElem<T>::get(v, e) == weight.least));
        }
        if (lane == 0) {
          sh.bins[i * kRowWaves + wave] = s;
          tied[i * kRowWaves + wave] = c;
        }
        ++i;
      },
      [](int) {});
  const uint64_t edge_ties = __ballot(some && row.ecol >= 0 && row.edge == weight.least);   // of the first wave
  if (tid == 0) sh.found[0] = __popcll(edge_ties & ((uint64_t(1) << W) - 1));
  __syncthreads();
  const uint64_t first_ties = sh.found[0];
  const int groups = row.blocks() * 4 * kRowWaves;   // at most kBins
  const int per = (groups + kRowThreads - 1) / kRowThreads, g0 = min(groups, tid * per), g1 = min(groups, g0 + per);
  uint64_t ties = 0, all_ties = 0, s = 0, total;
  if (some) {
    for (int g = g0; g < g1; ++g) ties += tied[g];
    ties = first_ties + block_scan(ties, sh, &all_ties);
  }
  uint64_t run = ties;
  for (int g = g0; g < g1; ++g) {
    uint64_t w = sh.bins[g];
    if (some) {
      sh.bins[g] = w -= over(run, tied[g]);
      run += tied[g];
    }
    s += w;
  }
  uint64_t mine = row.ecol >= 0 ? weight(row.edge) : 0;
  if (edge_ties >> lane & 1) {
    const int below = __popcll(edge_ties & lanes_below());
    mine -= over(lane < W ? below : all_ties + below, 1);
  }
  const uint64_t edges = wave_scan(mine);
  __syncthreads();
  if (wave == 0 && lane == W - 1) sh.found[0] = edges;
  if (wave == 0 && lane == 2 * W - 1) sh.found[1] = edges;
  __syncthreads();
  const uint64_t before = sh.found[0], behind = sh.found[1] - before;
  __syncthreads();
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
          sh.found[1] = ties;          // equal to the least before it
          break;
        }
        at += sh.bins[g];
        if (some) ties += tied[g];
      }
    __syncthreads();
    const int g = sh.count;
    const uint64_t want = sh.found[0];
    ties = sh.found[1];
    __syncthreads();
    if (wave == (g & (kRowWaves - 1))) {
      const int vi = (g / kRowWaves) * kRowThreads + tid;
      i32x4 v = {RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill};
      if (vi < row.nvec) v = reinterpret_cast<const i32x4 *>(row.p + row.head)[vi];
      uint64_t in = vector_sum<T>(weight, v);
      if (some) {
        uint64_t c = 0;
#pragma unroll
        for (int e = 0; e < W; ++e) c += RowElem<T>::get(v, e) == weight.least;
        ties += wave_scan(c) - c;
        in -= over(ties, c);
      }
      const uint64_t upto = wave_scan(in);
      if (upto >= want && upto - in < want) {
        uint64_t sum = upto - in;
        int token = -1;
#pragma unroll 1
        for (int e = 0; e < W && token < 0; ++e) {
          const float x = RowElem<T>::get(v, e);
          sum += weight(x);
          if (some && x == weight.least) sum -= over(ties++, 1);
          if (sum >= want) token = row.head + vi * W + e;
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
struct SampleBase : RowShared { double roots[256]; };
template <typename T> struct SampleShared : SampleBase {};
template <> struct SampleShared<bf16_t> : SampleBase { TableShared tab; };

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
  const float tmax = scan_row<false, 5>(row, sh, group, 0.f, none), top = block_max(tmax, sh);
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
    const bool below = min_p < 1.f && top < -kRowNegInf;
    const double b = below ? (double)top + (double)temperature * log((double)min_p) : (double)top;
    least = (float)b;
    if ((double)least < b) least = rank_value((uint64_t)(value_key(least) + 1) << 32);   // the next one up
  }
  const bool by_k = top_k > 0 && top_k < V, by_p = top_p < 1.f;
  int t = -1;
  if (by_k && top_k <= kMaxTop) {
    top_list(row, sh, group, tmax, top_k);
    // thread i has the i-th element in order; the kept ones are the first ones
    const uint64_t r = tid < top_k ? sh.list[tid] : 0;
    const uint64_t w = tid < top_k && by_p ? weight(rank_value(r)) : 0;
    uint64_t total = 0, before = 0;
    if (by_p && top_k <= 64) {   // the first wave has them
      before = wave_scan(w);
      total = __shfl(before, 63, 64);
      before -= w;
    } else if (by_p) {
      before = block_scan(w, sh, &total);
    }
    const bool in = (!by_p || before < mass_needed(top_p, total)) && rank_value(r) >= least;
    const bool keep = tid < top_k && (tid == 0 || in);
    t = pick_in_list(sh, __syncthreads_count(keep), weight, u);
  } else {
    uint64_t thr = 0, quota = ~uint64_t(0), kept = by_k ? (uint64_t)top_k : (uint64_t)V;
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
    auto raise = [&]() {
      if (floor <= thr) return;
      thr = floor;
      quota = ~uint64_t(0);
    };
    int listed = kListCap + 1;
    if (floor && !by_k && !by_p) {   // min_p alone: mostly few
      thr = floor;
      listed = gather();
    }
    // bf16: by the table (up to kTable columns, their own weights are no more work)
    bool tabulated = false, found = false;
    Window win;
    if constexpr (sizeof(SampleShared<T>) > sizeof(SampleBase)) {
      if (listed > kListCap && top < -kRowNegInf && V > kTable && find_window(weight, &win)) {
        tabulated = true;
        make_table(sh.tab, weight, win);
        found = !by_k && !by_p;
        if (!found) {
          const Tabulated tw{weight, kRowNegInf, win, &sh.tab};
          found = table_threshold(row, sh, sh.tab, tw, by_k, top_k, by_p, top_p, &thr, &kept, &quota);
          raise();
          if (found && kept <= kListCap && thr >> 32 > 1) listed = gather();
        }
      }
    }
    const Computed row_weight{RowWeight(weight, sh.roots), kLeastNumber};
    if (listed > kListCap && !(tabulated && found)) make_roots(sh.roots);
    if (listed > kListCap && !found) {   // digit by digit
      thr = 0;
      quota = ~uint64_t(0);
      if (by_k)
        thr = radix_threshold<true>(row, sh, 0, [](float) { return uint64_t(1); },
                                    [&](uint64_t) { return (uint64_t)top_k; }, &quota);
      if (by_p) {
        // top_p counts among the first `quota` of top_k's key; where its own cut has that
        // key (and leaves them all: its quota is none), the smaller quota holds
        const uint64_t floor_k =
            quota != ~uint64_t(0) ? column_threshold(row, sh, 0, (uint32_t)(thr >> 32), quota) : thr;
        uint64_t quota_p = ~uint64_t(0);
        thr = radix_threshold<false>(row, sh, floor_k, row_weight,
                                     [&](uint64_t total) { return mass_needed(top_p, total); }, &quota_p);
        quota = thr < floor_k ? min(quota, quota_p) : quota_p;
      }
      // a cut among -inf or NaN leaves all that has a weight
      if (thr >> 32 <= value_key(kRowNegInf)) quota = ~uint64_t(0);
      raise();
    }
    const float low = thr >> 32 > 1 ? rank_value(thr) : kRowNegInf;
    if (listed <= kListCap) {
      t = pick_in_list(sh, listed, weight, u);
    } else if (!tabulated) {
      t = pick_in_row(row, sh, quota, Computed{row_weight.weight, fmaxf(low, kLeastNumber)}, u);
    } else if constexpr (sizeof(SampleShared<T>) > sizeof(SampleBase)) {
      t = pick_in_row(row, sh, quota, Tabulated{weight, low, win, &sh.tab}, u);
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
