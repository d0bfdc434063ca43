// One row of vocabulary logits, taken by one workgroup of kRowThreads threads:
// what the kernels that put a row's tokens in order (top logits, sampling) share.
//
// A row of 151 936 16-bit logits (304 KB) does not fit LDS (160 KB). Holding it in
// the register file (512 KB a compute unit) leaves room for one workgroup there,
// whose read, arithmetic and latency then follow each other: 132 us for the top
// logits of 1 024 such rows. So a row is read in one pass that keeps what later
// steps need, the largest element of each run of vectors, and the few vectors that
// matter are read again from the caches.
//
// Order of a row's elements: value descending, then column ascending; -0 equals
// +0, NaN stands below -inf. As one number (rank_of): the value's bits made
// monotone, then the column's complement.
#pragma once

#include <algorithm>

#include "mga_common.hpp"

namespace mga {

constexpr int kRowThreads = 1024;
constexpr int kRowWaves = kRowThreads / 64;
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

// Vectors of 16 bytes, a block of four of them a thread and turn; elements before
// the first 16-byte boundary and after the last are single ones of the threads
// 0 .. W-1 and W .. 2W-1.
template <typename T>
struct Row {
  static constexpr int W = RowElem<T>::W;
  const T *p;
  int V, head, nvec, ecol;   // ecol: column of this thread's single element, or -1
  float edge;

  // This thread's vector i. Its address is a uniform base and the lane's own 32-bit
  // offset: one register a lane for all of them.
  __device__ __forceinline__ i32x4 load_vec(int i) const {
    const char *base = reinterpret_cast<const char *>(p + head);
    const int at = i * kRowThreads;
    i32x4 v = {RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill, RowElem<T>::kFill};
    if ((int)threadIdx.x < nvec - at) v = *reinterpret_cast<const i32x4 *>(base + (int64_t)at * 16 + threadIdx.x * 16u);
    return v;
  }
  __device__ __forceinline__ i32x16 load_block(int b) const {
    i32x16 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32x4 v = load_vec(4 * b + j);
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
  }

  // blocks of four vectors a thread that hold the row's vectors
  __device__ __forceinline__ int blocks() const { return (nvec + 4 * kRowThreads - 1) / (4 * kRowThreads); }

  // f(v, col): every thread's vectors in ascending order (all lanes take part; a
  // thread without one has -inf and a column of at least V); last(b) behind the
  // vectors of block b. K blocks are asked for before the first is used: a row is
  // few blocks, and each wait for memory is about 2 600 cycles. K = 5 is the whole of a
  // 16-bit row of up to 163 840 columns, in 80 registers a lane: for kernels that have
  // the compute unit to themselves anyway.
  template <int K, typename F, typename L>
  __device__ __forceinline__ void each_vec(F f, L last) const {
    const int n = blocks();
#pragma unroll 1
    for (int b0 = 0; b0 < n; b0 += K) {
      i32x16 q[K];
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (b0 + k < n) q[k] = load_block(b0 + k);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (b0 + k >= n) break;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int vi = (4 * (b0 + k) + j) * kRowThreads + (int)threadIdx.x;
          const i32x4 v = {q[k][4 * j], q[k][4 * j + 1], q[k][4 * j + 2], q[k][4 * j + 3]};
          f(v, vi < nvec ? head + vi * W : V);
        }
        last(b0 + k);
      }
    }
  }

  // f(x, col) of every element that there is.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each_vec<1>([&](const i32x4 &v, int col) {
      if (col < V) {
#pragma unroll
        for (int e = 0; e < W; ++e) f(RowElem<T>::get(v, e), col + e);
      }
    }, [](int) {});
    if (ecol >= 0) f(edge, ecol);
  }
};

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

// A value of another lane, by data-parallel operands (no LDS crossbar): `old` where
// there is none. kShr<n>: n lanes down in the row of 16; kLast15 / kLast31: the last
// lane of the row / of the half before, to the rows of MASK.
constexpr int kShr = 0x110, kLast15 = 0x142, kLast31 = 0x143;
template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ uint32_t dpp(uint32_t old, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)old, (int)v, CTRL, MASK, 0xF, false);
}
template <int CTRL, int MASK = 0xF>
__device__ __forceinline__ uint64_t dpp_add(uint64_t v) {
  return v + ((uint64_t)dpp<CTRL, MASK>(0u, (uint32_t)(v >> 32)) << 32 | dpp<CTRL, MASK>(0u, (uint32_t)v));
}
template <int CTRL, int MASK, typename F>
__device__ __forceinline__ float dpp_op(float v, F op) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  return op(v, __builtin_bit_cast(float, dpp<CTRL, MASK>(b, b)));
}

__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {   // inclusive; all lanes active
  v = dpp_add<kShr + 1>(v);
  v = dpp_add<kShr + 2>(v);
  v = dpp_add<kShr + 4>(v);
  v = dpp_add<kShr + 8>(v);
  v = dpp_add<kLast15, 0xA>(v);
  return dpp_add<kLast31, 0xC>(v);
}
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ float block_max(float v, RowPart &sh) {
  auto op = [](float a, float b) { return fmaxf(a, b); };
  v = dpp_op<kShr + 1, 0xF>(v, op);
  v = dpp_op<kShr + 2, 0xF>(v, op);
  v = dpp_op<kShr + 4, 0xF>(v, op);
  v = dpp_op<kShr + 8, 0xF>(v, op);
  v = dpp_op<kLast15, 0xA>(v, op);
  v = dpp_op<kLast31, 0xC>(v, op);
  if ((threadIdx.x & 63) == 63) sh.fpart[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.fpart[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) v = fmaxf(v, sh.fpart[w]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, RowPart &sh) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  if ((threadIdx.x & 63) == 0) sh.fpart[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.fpart[0];
#pragma unroll
  for (int w = 1; w < kRowWaves; ++w) v += sh.fpart[w];
  __syncthreads();
  return v;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
  const uint32_t lo = __shfl_xor((uint32_t)v, m, 64), hi = __shfl_xor((uint32_t)(v >> 32), m, 64);
  return (uint64_t)hi << 32 | lo;
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
// each, by all threads (360 of them: 22 000 cycles, 16 000 by the network); up to
// 1 024 by a bitonic network with an entry a thread, whose steps within a wave need
// no barrier; more by one in LDS. Uses sh.bins.
__device__ __forceinline__ void sort_list(RowShared &sh, int n) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= 256) {
    const int wide = n <= 128 ? 128 : 256, mine = tid & (wide - 1), parts = kRowThreads / wide;
    uint32_t *above = reinterpret_cast<uint32_t *>(sh.bins);
    if (tid < wide) above[tid] = 0;
    const uint64_t v = mine < n ? sh.list[mine] : 0;
    const int per = (n + parts - 1) / parts, i0 = tid / wide * per, i1 = min(n, i0 + per);
    int count = 0;
    for (int i = i0; i < i1; i += 8)
#pragma unroll
      for (int u = 0; u < 8; ++u) count += i + u < i1 && sh.list[i + u] > v;
    __syncthreads();
    if (mine < n) atomicAdd(&above[mine], (uint32_t)count);
    __syncthreads();
    if (tid < n) sh.list[above[tid]] = v;
    __syncthreads();
    return;
  }
  int size = 1024;
  while (size < n) size <<= 1;
  if (size == kRowThreads) {
    uint64_t v = tid < n ? sh.list[tid] : 0;
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        uint64_t o;
        if (j >= 64) {
          __syncthreads();
          sh.list[tid] = v;
          __syncthreads();
          o = sh.list[tid ^ j];
        } else {
          o = shfl_xor64(v, j);
        }
        const bool larger = ((tid & j) == 0) == ((tid & k) == 0);
        if ((v < o) == larger) v = o;
      }
    __syncthreads();
    sh.list[tid] = v;
    __syncthreads();
    return;
  }
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

// The bin in which the running sum of bins[0, nbins) (from the top bin down,
// or from bin 0 up) reaches need, and the sum before it (sh.found). *total: of
// all bins. need(total) >= 1 gives what has to be reached, at most the total.
template <typename F>
__device__ __forceinline__ void find_bin(RowShared &sh, const uint64_t *bins, int nbins, bool down, F need,
                                         uint64_t *total) {
  const int tid = threadIdx.x, per = nbins <= kRowThreads ? 1 : nbins / kRowThreads;
  uint64_t s = 0;
  const int b0 = tid * per;
  __syncthreads();
  if (b0 < nbins)
    for (int i = 0; i < per; ++i) s += bins[down ? nbins - 1 - b0 - i : b0 + i];
  uint64_t before = block_scan(s, sh, total);
  const uint64_t want = need(*total);
  if (before < want && want <= before + s)
    for (int i = 0; i < per; ++i) {
      const int b = down ? nbins - 1 - b0 - i : b0 + i;
      if (before + bins[b] >= want) {
        sh.found[0] = b;
        sh.found[1] = before;
        break;
      }
      before += bins[b];
    }
  __syncthreads();
}

// The rank of the element that is number `ties` by column among those of `key` (and
// of at least `floor`): more than that have the key. Uses sh.list.
template <typename T>
__device__ __forceinline__ uint64_t column_threshold(const Row<T> &row, RowShared &sh, uint64_t floor, uint32_t key,
                                                     uint64_t ties) {
  uint32_t prefix = 0;
  uint64_t total;
  for (int shift = 20; shift > 0; shift -= 10) {
    for (int i = threadIdx.x; i < 1024; i += kRowThreads) sh.list[i] = 0;
    __syncthreads();
    row.each([&](float x, int col) {
      const uint64_t r = rank_of(x, col);
      if ((uint32_t)(r >> 32) != key || r < floor || (shift < 20 && (uint32_t)col >> shift != prefix)) return;
      add_bin(sh.list, ((uint32_t)col >> (shift - 10)) & 1023u, 1, true);
    });
    find_bin(sh, sh.list, 1024, false, [&](uint64_t) { return ties; }, &total);
    ties -= sh.found[1];
    prefix = prefix << 10 | (uint32_t)sh.found[0];
    __syncthreads();
  }
  return (uint64_t)key << 32 | (uint32_t)~prefix;
}

// The largest rank such that the elements of at least that rank (among those of
// at least `floor`) weigh need(total) or more; with `quota` its key alone, and how
// many elements of that key count, by column (~0: all). weight(x) is 1 (ONES) or a whole
// number that depends on the value alone. Digits of the key from the top, 12
// bits at first, then of the columns of the elements that share the last key.
template <bool ONES, typename T, typename WF, typename NF>
__device__ __forceinline__ uint64_t radix_threshold(const Row<T> &row, RowShared &sh, uint64_t floor, WF weight,
                                                    NF need, uint64_t *quota = nullptr) {
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
    find_bin(sh, sh.bins, 1 << width, true, [&](uint64_t t) { return first ? need(t) : want; }, &total);
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
  const uint64_t ties = (want + w - 1) / w;
  if (ties >= in_bin / w) return (uint64_t)key << 32;
  if (!quota) return column_threshold(row, sh, floor, key, ties);
  *quota = ties;
  return (uint64_t)key << 32;
}

// A running maximum m and sum d = sum 2^{x c - mc}, mc = m c rounded: one fma an
// element for the exponent. What the rounding of mc does to d is taken out once, at
// the end (sum_at_max): a factor of at most 2^32 while |m c| < 2^30. Further out
// (a row masked with the type's lowest value) two different elements are at least 64
// octaves apart, and d is the number of those that equal m: counted when the maximum
// of the row is known (count_equal); until then mc = 0, and d is 0 below zero and
// of no use above.
constexpr float kFar = 1073741824.f;
__device__ __forceinline__ bool far(float m, float c) { return m != kRowNegInf && !(fabsf(m * c) < kFar); }
__device__ __forceinline__ float scaled(float m, float c) { return fabsf(m * c) < kFar ? m * c : 0.f; }
// What a sum at the maximum `part` counts at the maximum `whole`.
__device__ __forceinline__ float part_weight(float part, float whole, float c) {
  if (part == whole || part == kRowNegInf) return 1.f;   // a sum at -inf: 0, or NaN
  return far(part, c) || far(whole, c) ? 0.f : __builtin_amdgcn_exp2f(scaled(part, c) - scaled(whole, c));
}
struct RowSum {
  float m = kRowNegInf, mc = 0.f, d = 0.f;
  __device__ __forceinline__ void raise(float g, float c) {   // g > m
    const float n = scaled(g, c);
    if (d != 0.f) d *= __builtin_amdgcn_exp2f(mc - n);
    m = g;
    mc = n;
  }
  // elements of which g is the largest (NaN left out); every lane of the wave calls
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float g, float c) {
    if (__ballot(g > m) != 0) {   // seldom after the first vectors
      if (g > m) raise(g, c);
    }
    // four sums side by side: an add waits for the one before it
    float s[N < 4 ? 1 : 4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, -mc));
      if (i < (int)(sizeof(s) / sizeof(float))) s[i] = e;
      else s[i % (int)(sizeof(s) / sizeof(float))] += e;
    }
    if constexpr (N < 4) d += s[0];
    else d += (s[0] + s[1]) + (s[2] + s[3]);
  }
  __device__ __forceinline__ void merge(float om, float od, float c) {
    if (om > m) {
      d = d * part_weight(m, om, c) + od;
      m = om;
      mc = scaled(om, c);
    } else {
      d += od * part_weight(om, m, c);
    }
  }
};
// A part's sum at the whole's maximum m >= st.m.
__device__ __forceinline__ float sum_at(const RowSum &st, float m, float c) { return st.d * part_weight(st.m, m, c); }
// sum 2^{(x - m) c} from d = sum 2^{x c - mc}
__device__ __forceinline__ float sum_at_max(float m, float d, float c) {
  return m == kRowNegInf || far(m, c) ? d : d * __builtin_amdgcn_exp2f(-__builtin_fmaf(m, c, -scaled(m, c)));
}
// This thread's part of d of n elements whose maximum m is far: how many equal it. NaN
// where there is one.
template <int B, typename T>
__device__ __forceinline__ float count_equal(const T *p, int n, float m) {
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += B) {
    const float x = (float)p[i];
    s += x == m ? 1.f : x == x ? 0.f : x;
  }
  return s;
}

// ---- the first elements in order ------------------------------------------------

// A pass over the row that leaves, for each thread, the largest element of every
// `group` blocks of four vectors (sh.bins, as floats; the thread's own column)
// and of all its elements (the result). With those, the few vectors that hold an
// element above a bound are found, and read again, without another pass.
// With SUM the elements' exponentials are added too.
constexpr int kGroups = 8;
template <bool SUM, int K, typename T>
__device__ __forceinline__ float scan_row(const Row<T> &row, RowShared &sh, int group, float c, RowSum &st) {
  constexpr int W = RowElem<T>::W;
  float *tops = reinterpret_cast<float *>(sh.bins) + threadIdx.x;
  const int nblocks = row.blocks();
  float tmax = fmaxf(row.edge, kRowNegInf), gmax = kRowNegInf;
  if constexpr (SUM) {
    const float f[1] = {row.edge};   // -inf adds nothing
    st.add(f, tmax, c);
  }
  int g = 0, left = group;
  row.template each_vec<K>(
      [&](const i32x4 &v, int) {
        float f[W], m = kRowNegInf;
#pragma unroll
        for (int e = 0; e < W; ++e) m = fmaxf(m, f[e] = RowElem<T>::get(v, e));
        gmax = fmaxf(gmax, m);
        if constexpr (SUM) st.add(f, m, c);
      },
      [&](int b) {
        if (--left != 0 && b != nblocks - 1) return;
        tops[g * kRowThreads] = gmax;
        tmax = fmaxf(tmax, gmax);
        gmax = kRowNegInf;
        left = group;
        ++g;
      });
  return tmax;
}

// Blocks a group, for kGroups groups to hold any row of V columns.
template <typename T>
int row_group(int32_t V) {
  const int64_t block = 4 * (int64_t)kRowThreads * RowElem<T>::W;
  return (int)((((int64_t)V + block - 1) / block + kGroups - 1) / kGroups);
}

// f(x, col) of the elements that are >= least, by what scan_row left: each thread
// goes through its own groups that have one.
template <typename T, typename F>
__device__ __forceinline__ void scan_hits(const Row<T> &row, const RowShared &sh, int group, float least, F f) {
  constexpr int W = RowElem<T>::W;
  const float *tops = reinterpret_cast<const float *>(sh.bins) + threadIdx.x;
  const int nblocks = row.blocks(), ngroups = (nblocks + group - 1) / group;
  if (row.ecol >= 0 && row.edge >= least) f(row.edge, row.ecol);
  uint32_t groups = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
    if (g < ngroups && tops[g * kRowThreads] >= least) groups |= 1u << g;
  while (groups) {
    const int g = __builtin_ctz(groups);
    groups &= groups - 1;
    for (int b = g * group; b < min(nblocks, (g + 1) * group); ++b) {
      const i32x16 q = row.load_block(b);
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const i32x4 v = {q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]};
        uint32_t h = 0;
#pragma unroll
        for (int e = 0; e < W; ++e) h |= RowElem<T>::get(v, e) >= least ? 1u << e : 0u;
        if ((4 * b + j) * kRowThreads + (int)threadIdx.x < row.nvec) hits |= h << (j * W);
      }
      while (hits) {   // few: read once more instead of picked out of the registers
        const int i = __builtin_ctz(hits);
        hits &= hits - 1;
        const int col = row.head + ((4 * b + i / W) * kRowThreads + (int)threadIdx.x) * W + i % W;
        f((float)row.p[col], col);
      }
    }
  }
}

// The k <= kMaxTop first elements of the row in sh.list[0, k), in order (the
// row has k), after scan_row, which gave tmax.
//
// Each wave puts its threads' largest in order; with j = ceil(k / 16) the least of
// the 16 waves' j-th ones has at least 16 j >= k elements at or above it, and for
// ordinary rows few more: those are taken into LDS and put in order there. A row
// with too many of them (equal values) has its threshold found digit by digit. So
// has any row where k comes near the 1 024 threads (the least of all their largest lets
// some 4 % through), and one of 16-bit elements and 4 097 to about 7 700 columns, of which
// some waves hold no vector. 1 024 x 151 936 bf16, a call by itself: k = 64 89 us, 256 114,
// 512 139, 896 226, 1 024 427; 256 rows, k = 64: of 6 000 columns 23 us, of 8 192 14, of
// 3 000 (all in the list) 46.
template <typename T>
__device__ __forceinline__ void top_list(const Row<T> &row, RowShared &sh, int group, float tmax, int k) {
  const int tid = threadIdx.x, lane = tid & 63;
  float v = tmax;
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const float o = __shfl_xor(v, stride, 64);
      v = ((lane & stride) == 0) == ((lane & size) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
  if (tid == 0) sh.count = 0;
  const float least = -block_max(-__shfl(v, (k + kRowWaves - 1) / kRowWaves - 1, 64), sh);
  scan_hits(row, sh, group, least, [&](float x, int col) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < kListCap) sh.list[at] = rank_of(x, col);
  });
  __syncthreads();
  int n = sh.count;
  if (n > kListCap || n < k) {   // n < k: NaN among the first
    __syncthreads();
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
