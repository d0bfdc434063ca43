// Logits shaped before a token is drawn: penalties for repeated tokens, added
// biases, and a bit mask of the tokens that are allowed.
//
//   y = x;  seen in prompt or output: y = x > 0 ? x / r : x * r;
//   y -= f * count + (count > 0 ? p : 0), count over the output;
//   y += biases;  not allowed: y = -inf
//
// Bounded by HBM: each logit is read and written once (80 rows of 151 936 bf16: 8.3 us without lists, a copy 7.9;
// with 2048 tokens a row, 8 biases and a mask 16.8: the tiles' turns over the tokens). A workgroup takes a tile of
// one row's columns.
// While the tile's logits are on their way it counts the row's tokens that fall into it in LDS: a count of the
// output's in the low bits, a bit for the prompt's, a bit for columns with a bias (integer adds, so
// their order does not matter). Every tile reads the row's tokens, from L2, which asks for wide
// tiles where the rows alone fill the chip. Columns that nothing hit are copied as they are; the others find
// their biases in the tile's list, kept in the caller's order, so that equal ids add up in it.
// Counts of up to 2^14 - 1 tokens take 16 bits a column and biases of up to 1024 entries a list; longer ones
// (the wide form) 32 bits and a sum a column, added by the first entry of each column for those after it. What
// decides is the room for a row's tokens, not its length: the 80 rows in rows of 16 383 17.3 us, of 16 384 21.8.
#include <type_traits>

#include "mga_internal.hpp"
#include "mga_common.hpp"

namespace mga {
namespace {

constexpr int kListMax = 1024;
constexpr int kNarrowTokens = (1 << 14) - 1;

template <bool WIDE> struct Count;
template <> struct Count<false> { typedef uint16_t type; static constexpr int bits = 16; };
template <> struct Count<true> { typedef uint32_t type; static constexpr int bits = 32; };

struct RowSettings {
  float r, f, p;
};

// c: a column's count and, above it, whether it has a bias and whether the prompt holds it.
template <int BITS>
__device__ __forceinline__ float penalised(float x, uint32_t c, const RowSettings &s) {
  const uint32_t n = c & ((1u << (BITS - 2)) - 1);
  if (n || c >> (BITS - 1)) x = x > 0.f ? x / s.r : x * s.r;
  return n ? fmaf(-s.f, (float)n, x) - s.p : x;
}

// A tile of TC columns from `base` on, which may begin before column 0 by less than a vector
// (VEC: vectors of 16 bytes are aligned in x and out alike at base).
constexpr int NT = 256;   // threads

template <typename T, typename ID, int TC, bool VEC, bool WIDE>
__global__ __launch_bounds__(NT) void adjust_logits_kernel(AdjustArgs a, int tiles) {
  typedef typename Count<WIDE>::type CT;
  constexpr int VN = 16 / sizeof(T), BITS = Count<WIDE>::bits, NV = (TC + NT * VN - 1) / (NT * VN);
  constexpr uint32_t kPrompt = 1u << (BITS - 1), kBias = 1u << (BITS - 2);
  // counts; where there are biases, a column's sum (wide) or the entry that holds it, and the list
  extern __shared__ __attribute__((aligned(16))) char lds[];
  CT *count = reinterpret_cast<CT *>(lds);
  float *bias = reinterpret_cast<float *>(count + TC);
  uint16_t *owner = reinterpret_cast<uint16_t *>(count + TC);
  int32_t *list_col = reinterpret_cast<int32_t *>(WIDE ? (char *)(bias + TC) : (char *)(owner + TC));
  float *list_val = reinterpret_cast<float *>(list_col + (WIDE ? NT : a.K));
  __shared__ int32_t wave_n[NT / 64], twice;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int row = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const T *x = (const T *)a.x + (int64_t)row * a.xs;
  T *out = (T *)a.out + (int64_t)row * a.os;
  const int off = VEC ? (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % VN) : 0;
  const int base = tile * TC - off;
  const int c0 = max(base, 0), c1 = min(base + TC, a.V);
  if (c0 >= c1) return;

  i32x4 raw[VEC ? NV : 1];
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * NT + tid) * VN, col = base + i;
      raw[k] = i32x4{0, 0, 0, 0};
      if (i < TC && col >= 0 && col + VN <= a.V) raw[k] = *reinterpret_cast<const i32x4 *>(x + col);
    }
  }
  // the row's first tokens and biases and what says which count, all in flight before the first wait
  constexpr int TU = 8;
  const ID *tokens = (const ID *)a.tokens + (int64_t)row * a.tokens_rs;
  ID tok[TU], tnext[TU];
  auto load_tokens = [&](int i0, ID *tok) {   // of the TU * NT from i0 on every NT-th
    if (i0 + TU * NT <= a.L) {
#pragma unroll
      for (int u = 0; u < TU; ++u) tok[u] = tokens[i0 + tid + NT * u];
    } else {
#pragma unroll
      for (int u = 0; u < TU; ++u) tok[u] = tokens[min(i0 + tid + NT * u, a.L - 1)];
    }
  };
  int64_t id = -1;
  float val = 0.f;
  auto load_bias = [&](int i) {
    id = -1;
    if (i >= a.K) return;
    const int64_t at = (int64_t)row * a.bias_ids_rs + i;
    id = a.bias64 ? ((const int64_t *)a.bias_ids)[at] : ((const int32_t *)a.bias_ids)[at];
    val = a.bias[(int64_t)row * a.bias_rs + i];
  };
  if (a.L > 0) load_tokens(0, tok);
  load_bias(tid);
  const int n = a.lengths ? min(max(a.lengths[row], 0), a.L) : a.L;
  const int m = a.prompts ? min(max(a.prompts[row], 0), n) : 0;
  for (int i = tid; i < (int)(TC * sizeof(CT) / 16); i += NT) reinterpret_cast<i32x4 *>(count)[i] = i32x4{0, 0, 0, 0};
  if (WIDE && a.K > 0)
    for (int i = tid; i < TC; i += NT) bias[i] = 0.f;
  RowSettings s{a.repetition ? a.repetition[row] : a.repetition_all, a.frequency ? a.frequency[row] : a.frequency_all,
                a.presence ? a.presence[row] : a.presence_all};
  if (!(s.r > 0.f)) s.r = 1.f;
  if (tid == 0) twice = 0;
  __syncthreads();

  // two narrow counts share a word: neither can pass its bits, nor reach the other's
  auto shift = [&](int c) { return WIDE ? 0 : 16 * (c & 1); };
  auto word = [&](int c) { return reinterpret_cast<uint32_t *>(count) + (WIDE ? c : c >> 1); };
  // a token within the tile: of 64 bits, the high word has to be 0
  auto within = [&](ID t) {
    const bool low = (uint32_t)((uint32_t)t - (uint32_t)c0) < (uint32_t)(c1 - c0);
    if constexpr (sizeof(ID) == 8) return low && (uint32_t)((uint64_t)t >> 32) == 0;
    else return low;
  };
  for (int i0 = 0; i0 < n; i0 += NT * TU) {
    if (i0 + NT * TU < n) load_tokens(i0 + NT * TU, tnext);
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      const int i = i0 + tid + NT * u;
      if (within(tok[u]) && i < n) {
        const int c = (int)tok[u] - base;
        if (i < m) atomicOr(word(c), kPrompt << shift(c));
        else atomicAdd(word(c), 1u << shift(c));
      }
    }
#pragma unroll
    for (int u = 0; u < TU; ++u) tok[u] = tnext[u];
  }
  int listed = 0;
  for (int i0 = 0; i0 < a.K; i0 += NT) {
    if (i0) load_bias(i0 + tid);
    const bool mine = id >= c0 && id < c1;
    const uint64_t who = __ballot(mine);
    if (lane == 0) wave_n[w] = __popcll(who);
    __syncthreads();
    int at = (WIDE ? 0 : listed) + __popcll(who & lanes_below()), found = 0;
    for (int k = 0; k < NT / 64; ++k) {
      at += k < w ? wave_n[k] : 0;
      found += wave_n[k];
    }
    listed += found;
    if (mine) {
      const int c = (int)id - base;
      list_col[at] = c;
      list_val[at] = val;
      atomicOr(word(c), kBias << shift(c));
    }
    __syncthreads();
    if constexpr (WIDE) {
      if (tid < found) {
        const int c = list_col[tid];
        bool first = true;
        for (int k = 0; k < tid; ++k) first = first && list_col[k] != c;
        if (first) {
          float b = bias[c];
          for (int k = tid; k < found; ++k) b += list_col[k] == c ? list_val[k] : 0.f;
          bias[c] = b;
        }
      }
      __syncthreads();
    }
  }
  if (!WIDE && listed) {
    // one entry of each column, whichever, holds its sum
    for (int t = tid; t < listed; t += NT) owner[list_col[t]] = (uint16_t)t;
    __syncthreads();
    for (int t = tid; t < listed; t += NT)
      if (owner[list_col[t]] != t) twice = 1;
    __syncthreads();
    if (twice)   // of equal ids, added in their order
      for (int t = tid; t < listed; t += NT) {
        const int c = list_col[t];
        if (owner[c] != t) continue;
        float b = 0.f;
#pragma unroll 8
        for (int k = 0; k < listed; ++k) b += list_col[k] == c ? list_val[k] : 0.f;
        list_val[t] = b;   // read by no other column's sum
      }
  }
  __syncthreads();

  const uint32_t *ok = a.allowed ? (const uint32_t *)a.allowed + (int64_t)row * a.allowed_rs : nullptr;
  auto value = [&](float v, uint32_t c, int i) {   // of tile column i, c != 0
    v = penalised<BITS>(v, c, s);
    if (c & kBias) v += WIDE ? bias[i] : list_val[owner[i]];
    return v;
  };
  auto one = [&](int col) {
    const uint32_t c = count[col - base];
    T y = x[col];
    if (c) y = (T)value((float)y, c, col - base);
    out[col] = ok && !(ok[col >> 5] >> (col & 31) & 1) ? (T)-__builtin_huge_valf() : y;
  };
  if constexpr (VEC) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = (k * NT + tid) * VN, col = base + i;
      if (i >= TC) break;
      if (col >= 0 && col + VN <= a.V) {
        uint32_t bits = ~0u;
        if (ok) {
          const int word = col >> 5;
          const uint32_t lo = ok[word], hi = (col + VN - 1) >> 5 != word ? ok[word + 1] : 0;
          bits = (uint32_t)((((uint64_t)hi << 32) | lo) >> (col & 31));
        }
        uint32_t c[VN], any = 0;
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          c[e] = count[i + e];
          any |= c[e];
        }
        i32x4 put = raw[k];
        const T *src = reinterpret_cast<const T *>(&raw[k]);
        T *o = reinterpret_cast<T *>(&put);
        if (any) {
#pragma unroll
          for (int e = 0; e < VN; ++e)
            if (c[e]) o[e] = (T)value((float)src[e], c[e], i + e);
        }
        if (ok) {
#pragma unroll
          for (int e = 0; e < VN; ++e) o[e] = bits >> e & 1 ? o[e] : (T)-__builtin_huge_valf();
        }
        *reinterpret_cast<i32x4 *>(out + col) = put;
      } else {
        for (int e = 0; e < VN; ++e)
          if (col + e >= 0 && col + e < a.V) one(col + e);
      }
    }
  } else {
    for (int i = tid; i < c1 - base; i += NT) one(base + i);
  }
}

// Bytes of a tile's logits. Small tiles give few rows more workgroups; past the large ones' 8 KB a row's
// tokens would be read less often, but reads and writes overlap less: 80 rows of 151 936 bf16 with 2048 tokens
// at 8 KB by 256 threads, 16 KB by 512, 32 KB by 1024: 16.9 / 16.6 / 22.5 us; 256 rows of 32 003 fp32 with 4096
// tokens and 300 biases 29.7 / 32.7 / 41.7 us.
constexpr int kSmallTile = 2048, kLargeTile = 8192, kWideTile = 8192;

bool wide_form(int32_t L, int32_t K) { return L > kNarrowTokens || K > kListMax; }

// Large tiles where the rows fill the chip with them: two workgroups a CU and more.
int tile_bytes(int32_t N, int32_t V, int32_t L, int32_t K, int eb) {
  if (wide_form(L, K)) return kWideTile;
  const int64_t bytes = (int64_t)V * eb;
  return (bytes + kLargeTile - 1) / kLargeTile * N >= 2 * device_cu_count() ? kLargeTile : kSmallTile;
}

template <typename T>
void launch(const AdjustArgs &a, hipStream_t stream) {
  constexpr int VN = 16 / sizeof(T);
  const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p) / sizeof(T) % VN; };
  // rows that begin alike within a vector in x and out
  const bool vec = at(a.x) == at(a.out) && (a.N == 1 || a.xs % VN == a.os % VN);
  auto go = [&](auto id, auto bytes, auto v, auto wide) {
    constexpr int TC = decltype(bytes)::value / sizeof(T);
    constexpr bool W = decltype(wide)::value;
    const int tiles = (a.V + (decltype(v)::value ? VN - 1 : 0) + TC - 1) / TC;
    const int lds = TC * (W ? 4 : 2) + (a.K > 0 ? TC * (W ? 4 : 2) + 8 * (W ? NT : a.K) : 0);
    adjust_logits_kernel<T, decltype(id), TC, decltype(v)::value, W><<<(uint32_t)tiles * a.N, NT, lds, stream>>>(a, tiles);
  };
  auto go1 = [&](auto bytes, auto v, auto wide) {
    if (a.tokens64) go(int64_t{}, bytes, v, wide);
    else go(int32_t{}, bytes, v, wide);
  };
  auto go2 = [&](auto bytes, auto wide) {
    if (vec) go1(bytes, std::true_type{}, wide);
    else go1(bytes, std::false_type{}, wide);
  };
  const int tile = tile_bytes(a.N, a.V, a.L, a.K, sizeof(T));
  if (wide_form(a.L, a.K)) go2(std::integral_constant<int, kWideTile>{}, std::true_type{});
  else if (tile == kLargeTile) go2(std::integral_constant<int, kLargeTile>{}, std::false_type{});
  else go2(std::integral_constant<int, kSmallTile>{}, std::false_type{});
}

}  // namespace

int64_t adjust_blocks(int32_t N, int32_t V, int32_t L, int32_t K, int eb) {
  return ((int64_t)V * eb / tile_bytes(N, V, L, K, eb) + 2) * N;
}

void launch_adjust_logits(const AdjustArgs &a, int dtype, hipStream_t stream) {
  if (dtype == kDtBf16) launch<bf16_t>(a, stream);
  else if (dtype == kDtF16) launch<f16_t>(a, stream);
  else launch<float>(a, stream);
}

}  // namespace mga
