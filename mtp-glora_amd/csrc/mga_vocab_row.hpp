// One row of vocabulary logits, held by one workgroup of kRowThreads threads:
// what the kernels that put a row's tokens in order (top logits, sampling) share.
//
// A row of 151 936 16-bit logits (304 KB) fits the register file of a compute
// unit (512 KB) and not its LDS (160 KB): it is loaded once, 16 bytes a thread
// and load, and every later pass over it reads registers. Longer rows (and fp32
// rows past 81 920 columns) are read again in each pass, from the caches.
//
// Order of a row's elements: value descending, then column ascending; -0 equals
// +0, NaN stands below -inf. As one number (rank_of): the value's bits made
// monotone, then the column's complement.
#pragma once

#include <algorithm>
#include <type_traits>

#include "mga_common.hpp"

namespace mga {

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
constexpr int kRowMaxCols = 1 << 20;       // columns' width in rank_of
constexpr int kListCap = 4096;             // candidates that are put in order in LDS
constexpr int kMaxTop = 1024;              // most elements that are asked for in order
constexpr float kRowNegInf = -__builtin_huge_valf();

typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---- elements ---------------------------------------------------------------

template <typename T> struct RowElem;
template <> struct RowElem<bf16_t> {
  static constexpr int W = 8, kFill = (int)0xFF80FF80u;   // two -inf
  static constexpr int kKeyBits = 16;                     // leading bits of the fp32 pattern that differ between values
  __device__ __forceinline__ static float get(const i32x4 &v, int e) {
    const uint32_t w = (uint32_t)v[e >> 1];
    return __builtin_bit_cast(float, e & 1 ? w & 0xFFFF0000u : w << 16);
  }
};
template <> struct RowElem<f16_t> {
  static constexpr int W = 8, kFill = (int)0xFC00FC00u;
  static constexpr int kKeyBits = 19;                     // 8 of the exponent, 10 of the mantissa, the sign
  __device__ __forceinline__ static float get(const i32x4 &v, int e) {
    const uint32_t w = (uint32_t)v[e >> 1];
    return e & 1 ? pair_hi<f16_t>(w) : pair_lo<f16_t>(w);
  }
};
template <> struct RowElem<float> {
  static constexpr int W = 4, kFill = (int)0xFF800000u;
  static constexpr int kKeyBits = 32;
  __device__ __forceinline__ static float get(const i32x4 &v, int e) { return __builtin_bit_cast(f32x4, v)[e]; }
};

// Monotone in the value; 1 for NaN, 0 for no element.
__device__ __forceinline__ uint32_t value_key(float x) {
  if (x != x) return 1u;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);   // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;            // -inf: 0x007FFFFF
}
__device__ __forceinline__ uint64_t rank_of(float x, int col) {
  return (uint64_t)value_key(x) << 32 | (uint32_t)~col;
}
__device__ __forceinline__ int rank_col(uint64_t r) { return (int)~(uint32_t)r; }
__device__ __forceinline__ float rank_value(uint64_t r) {   // NaN where the key is NaN's
  const uint32_t k = (uint32_t)(r >> 32);
  if (k == 1u) return __builtin_nanf("");
  return __builtin_bit_cast(float, (k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

// ---- the row ----------------------------------------------------------------

// NB > 0: NB blocks of four vectors a thread stay in registers; NB = 0: the
// blocks are loaded again by every pass. Loops over a block's vectors stay
// rolled (the vector is picked by a uniform index), so that a pass is a few KB
// of code: a single row's time would otherwise go into fetching instructions.
// Elements before the first 16-byte boundary and after the last are single
// ones of the threads 0 .. W-1 and W .. 2W-1.
template <typename T, int NB>
struct Row {
  static constexpr int W = RowElem<T>::W;
  const T *p;
  int V, head, nvec, ecol;   // ecol: column of this thread's single element, or -1
  float edge;
  i32x16 r[NB > 0 ? NB : 1];

  __device__ __forceinline__ i32x16 load_block(int b) const {
    const i32x4 *vp = reinterpret_cast<const i32x4 *>(p + head) + threadIdx.x;
    i32x16 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = (b * 4 + j) * kRowThreads;
      i32x4 v = {RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill};
      if (at + (int)threadIdx.x < nvec) v = vp[at];
      q[4 * j] = v[0]; q[4 * j + 1] = v[1]; q[4 * j + 2] = v[2]; q[4 * j + 3] = v[3];
    }
    return q;
  }

  __device__ __forceinline__ void load(const T *row, int n) {
    p = row;
    V = n;
    const int tid = threadIdx.x;
    const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = min(n, off ? W - off : 0);
    nvec = (n - head) / W;
    const int tail0 = head + nvec * W;
    ecol = tid < W ? (tid < head ? tid : -1) : (tid < 2 * W && tail0 + tid - W < n ? tail0 + tid - W : -1);
    edge = ecol >= 0 ? (float)row[ecol] : kRowNegInf;
    if constexpr (NB > 0) {
#pragma unroll
      for (int b = 0; b < NB; ++b) r[b] = load_block(b);
    }
  }

  // f(v, col, i): the i-th vector of every thread (all lanes take part; a thread
  // without one has -inf and a column of at least V), in ascending order of i.
  template <typename F>
  __device__ __forceinline__ void each_vec(F f) const {
    const int n = (nvec + kRowThreads - 1) / kRowThreads;
    auto block = [&](const i32x16 &q, int b) {
      const int left = min(4, n - 4 * b);
#pragma unroll 1
      for (int j = 0; j < left; ++j) {
        const int i = 4 * b + j, vi = i * kRowThreads + (int)threadIdx.x;
        const i32x4 v = {q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]};
        f(v, vi < nvec ? head + vi * W : V, i);
      }
    };
    if constexpr (NB > 0) {
#pragma unroll
      for (int b = 0; b < NB; ++b) block(r[b], b);
    } else {
      for (int b = 0; 4 * b < n; ++b) block(load_block(b), b);
    }
  }

  // f(x, col) of every element that there is.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each_vec([&](const i32x4 &v, int col, int) {
      if (col < V) {
#pragma unroll
        for (int e = 0; e < W; ++e) f(RowElem<T>::get(v, e), col + e);
      }
    });
    if (ecol >= 0) f(edge, ecol);
  }

  // f(x, col) of every element with x >= least (NaN: never).
  template <typename F>
  __device__ __forceinline__ void each_from(float least, F f) const {
    each_vec([&](const i32x4 &v, int col, int) {
      float m = RowElem<T>::get(v, 0);
#pragma unroll
      for (int e = 1; e < W; ++e) m = fmaxf(m, RowElem<T>::get(v, e));
      if (m >= least && col < V) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float x = RowElem<T>::get(v, e);
          if (x >= least) f(x, col + e);
        }
      }
    });
    if (ecol >= 0 && edge >= least) f(edge, ecol);
  }
};

// f(std::integral_constant NB) for the rows of V columns: the fewest blocks that
// hold them, 0 where five (80 registers) do not.
template <typename T, typename F>
void with_row_blocks(int32_t V, F f) {
  const int64_t block = 4 * (int64_t)kRowThreads * RowElem<T>::W;
  if (V <= block) f(std::integral_constant<int, 1>());
  else if (V <= 2 * block) f(std::integral_constant<int, 2>());
  else if (V <= 4 * block) f(std::integral_constant<int, 4>());
  else if (V <= 5 * block) f(std::integral_constant<int, 5>());
  else f(std::integral_constant<int, 0>());
}

// Largest element of this thread (-inf without one; NaN left out).
template <typename T, int NB>
__device__ __forceinline__ float thread_max(const Row<T, NB> &row) {
  float m = fmaxf(row.edge, kRowNegInf);
  row.each_vec([&](const i32x4 &v, int, int) {
#pragma unroll
    for (int e = 0; e < RowElem<T>::W; ++e) m = fmaxf(m, RowElem<T>::get(v, e));
  });
  return m;
}

// ---- the workgroup -----------------------------------------------------------

struct RowPart {
  float fpart[kRowWaves];
};
constexpr int kBins = 4096;
struct RowShared : RowPart {
  uint64_t list[kListCap];
  uint64_t bins[kBins];
  uint64_t part[kRowWaves];
  uint64_t found[2];
  int count;
};

template <typename F>
__device__ __forceinline__ float block_reduce(float v, RowPart &sh, F op) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = op(v, __shfl_xor(v, m, 64));
  if ((threadIdx.x & 63) == 0) sh.fpart[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.fpart[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) v = op(v, sh.fpart[w]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_max(float v, RowPart &sh) {
  return block_reduce(v, sh, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float block_sum(float v, RowPart &sh) {
  return block_reduce(v, sh, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
  const uint32_t lo = __shfl_up((uint32_t)v, d, 64), hi = __shfl_up((uint32_t)(v >> 32), d, 64);
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {   // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t o = shfl_up64(v, d);
    if ((int)(threadIdx.x & 63) >= d) v += o;
  }
  return v;
}
// Sum of v over the threads before this one and (*total) over all of them.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, RowShared &sh, uint64_t *total) {
  const uint64_t in = wave_scan(v);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) sh.part[wave] = in;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const uint64_t s = sh.part[w];
    before += w < wave ? s : 0;
    all += s;
  }
  __syncthreads();
  *total = all;
  return before + in - v;
}

// sh.list[0, n) in descending order. Up to 256 entries by counting those above
// each (n / 2 broadcast reads a thread), else by a bitonic network.
__device__ __forceinline__ void sort_list(RowShared &sh, int n) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= 256) {
    const uint64_t mine = tid < n ? sh.list[tid] : 0;
    int above = 0;
    if (tid < n)
      for (int i = 0; i < n; ++i) above += sh.list[i] > mine;
    __syncthreads();
    if (tid < n) sh.list[above] = mine;
    __syncthreads();
    return;
  }
  int size = 512;
  while (size < n) size <<= 1;
  for (int i = n + tid; i < size; i += kRowThreads) sh.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int t = tid; t < size / 2; t += kRowThreads) {
        const int a = 2 * t - (t & (j - 1)), b = a + j;
        const uint64_t x = sh.list[a], y = sh.list[b];
        if ((x < y) == ((a & k) == 0)) {
          sh.list[a] = y;
          sh.list[b] = x;
        }
      }
      __syncthreads();
    }
}

// Adds w to the bin of every calling lane; lanes that all have one bin add once
// (a masked row is tens of thousands of equal values). Sums are whole numbers:
// their order changes nothing.
__device__ __forceinline__ void add_bin(uint64_t *bins, uint32_t bin, uint64_t w, bool ones) {
  if (ones) {
    const uint32_t first = __builtin_amdgcn_readfirstlane(bin);
    const uint64_t all = __ballot(1);
    if (__ballot(bin == first) == all) {
      if (__builtin_ctzll(all) == (int)(threadIdx.x & 63))
        atomicAdd((unsigned long long *)&bins[first], (unsigned long long)__popcll(all));
      return;
    }
  }
  atomicAdd((unsigned long long *)&bins[bin], (unsigned long long)w);
}

// The bin in which the running sum of sh.bins[0, nbins) (from the top bin down,
// or from bin 0 up) reaches need, and the sum before it (sh.found). *total: of
// all bins. need(total) >= 1 gives what has to be reached, at most the total.
template <typename F>
__device__ __forceinline__ void find_bin(RowShared &sh, int nbins, bool down, F need, uint64_t *total) {
  const int tid = threadIdx.x, per = nbins <= kRowThreads ? 1 : nbins / kRowThreads;
  uint64_t s = 0;
  const int b0 = tid * per;
  __syncthreads();
  if (b0 < nbins)
    for (int i = 0; i < per; ++i) s += sh.bins[down ? nbins - 1 - b0 - i : b0 + i];
  uint64_t before = block_scan(s, sh, total);
  const uint64_t want = need(*total);
  if (before < want && want <= before + s)
    for (int i = 0; i < per; ++i) {
      const int b = down ? nbins - 1 - b0 - i : b0 + i;
      if (before + sh.bins[b] >= want) {
        sh.found[0] = b;
        sh.found[1] = before;
        break;
      }
      before += sh.bins[b];
    }
  __syncthreads();
}

// The largest rank such that the elements of at least that rank (among those of
// at least `floor`) weigh need(total) or more. weight(x) is 1 (ONES) or a whole
// number that depends on the value alone. Digits of the key from the top, 12
// bits at first, then of the columns of the elements that share the last key.
template <bool ONES, typename T, int NB, typename WF, typename NF>
__device__ uint64_t radix_threshold(const Row<T, NB> &row, RowShared &sh, uint64_t floor, WF weight, NF need) {
  uint64_t want = 0, total = 0;
  uint32_t prefix = 0;
  int shift = 32;
  uint64_t in_bin = 0;
  while (shift > 32 - RowElem<T>::kKeyBits) {
    const int width = min(12, shift - (32 - RowElem<T>::kKeyBits)), next = shift - width;
    for (int i = threadIdx.x; i < 1 << width; i += kRowThreads) sh.bins[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << width) - 1;
    row.each([&](float x, int col) {
      const uint64_t r = rank_of(x, col);
      const uint32_t key = (uint32_t)(r >> 32);
      if (r < floor || (shift < 32 && key >> shift != prefix)) return;
      const uint64_t w = ONES ? 1 : weight(x);
      if (ONES || w) add_bin(sh.bins, (key >> next) & mask, w, ONES);
    });
    const bool first = shift == 32;
    find_bin(sh, 1 << width, true, [&](uint64_t t) { return first ? need(t) : want; }, &total);
    if (first) want = need(total);
    want -= sh.found[1];
    in_bin = sh.bins[sh.found[0]];
    prefix = prefix << width | (uint32_t)sh.found[0];
    shift = next;
    __syncthreads();
  }
  uint32_t key = prefix;
  if constexpr (RowElem<T>::kKeyBits < 32) {
    constexpr int low = 32 - RowElem<T>::kKeyBits;
    key = prefix == 0 ? 1u : prefix << low | (key >> (RowElem<T>::kKeyBits - 1) ? 0u : (1u << low) - 1);
  }
  // elements of this key that are needed, of those there are
  const uint64_t w = ONES ? 1 : weight(rank_value((uint64_t)key << 32));
  uint64_t ties = (want + w - 1) / w;
  if (ties >= in_bin / w) return (uint64_t)key << 32;
  uint32_t cprefix = 0;
  for (int cshift = 20; cshift > 0; cshift -= 10) {
    for (int i = threadIdx.x; i < 1024; i += kRowThreads) sh.bins[i] = 0;
    __syncthreads();
    row.each([&](float x, int col) {
      const uint64_t r = rank_of(x, col);
      if ((uint32_t)(r >> 32) != key || r < floor || (cshift < 20 && (uint32_t)col >> cshift != cprefix)) return;
      add_bin(sh.bins, ((uint32_t)col >> (cshift - 10)) & 1023u, 1, true);
    });
    find_bin(sh, 1024, false, [&](uint64_t) { return ties; }, &total);
    ties -= sh.found[1];
    cprefix = cprefix << 10 | (uint32_t)sh.found[0];
    __syncthreads();
  }
  return (uint64_t)key << 32 | (uint32_t)~cprefix;
}

// The k <= kMaxTop first elements of the row in sh.list[0, k), in order (the
// row has k). tmax: this thread's largest element.
//
// Each wave puts its threads' largest in order; with j = ceil(k / 16) the least of
// the 16 waves' j-th ones has at least 16 j >= k elements at or above it, and for
// ordinary rows few more: those are taken into LDS and put in order there. A row
// with too many of them (equal values) has its threshold found digit by digit.
template <typename T, int NB>
__device__ void top_list(const Row<T, NB> &row, RowShared &sh, float tmax, int k) {
  const int tid = threadIdx.x, lane = tid & 63;
  float v = tmax;
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const float o = __shfl_xor(v, stride, 64);
      v = ((lane & stride) == 0) == ((lane & size) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
  const float least = -block_max(-__shfl(v, (k + kRowWaves - 1) / kRowWaves - 1, 64), sh);
  if (tid == 0) sh.count = 0;
  __syncthreads();
  row.each_from(least, [&](float x, int col) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kListCap) sh.list[at] = rank_of(x, col);
  });
  __syncthreads();
  int n = sh.count;
  __syncthreads();
  if (n > kListCap || n < k) {   // n < k: NaN among the first
    const uint64_t thr = radix_threshold<true>(row, sh, 0, [](float) { return uint64_t(1); },
                                               [&](uint64_t) { return (uint64_t)k; });
    if (tid == 0) sh.count = 0;
    __syncthreads();
    row.each([&](float x, int col) {
      const uint64_t r = rank_of(x, col);
      if (r >= thr) sh.list[atomicAdd(&sh.count, 1)] = r;
    });
    n = k;
  }
  sort_list(sh, n);
}

}  // namespace mga
