// Logits shaped before a token is drawn: penalties for repeated tokens, added
// biases, and a bit mask of the tokens that are allowed.
//
//   y = x;  seen in prompt or output: y = x > 0 ? x / r : x * r;
//   y -= f * count + (count > 0 ? p : 0), count over the output;
//   y += biases;  not allowed: y = -inf
//
// Bounded by HBM: each logit is read and written once. A workgroup takes a tile of
// one row's columns. It first counts the row's tokens that fall into the tile in
// LDS (a word a column: bits 0..30 count the output, bit 31 says that the prompt holds it;
// integer adds, so their order does not matter), which costs a read of the row's tokens
// for every tile, from L2, and so asks for wide tiles where the rows alone fill the chip.
// Biases are added by one thread a column, in the order of the list: the tile's
// entries are set in their order, 256 of the list at a time, and the first of each column
// adds up those that follow it.
#include <type_traits>

#include "mga_internal.hpp"
#include "mga_common.hpp"

namespace mga {
namespace {

constexpr uint32_t kInPrompt = 0x80000000u;

template <typename T>
__device__ __forceinline__ float as_float(T v) { return (float)v; }

struct RowSettings {
  float r, f, p;
};

__device__ __forceinline__ float adjusted(float x, uint32_t c, float b, const RowSettings &s) {
  if (c) {
    x = x > 0.f ? x / s.r : x * s.r;
    const uint32_t n = c & ~kInPrompt;
    if (n) x = fmaf(-s.f, (float)n, x) - s.p;
  }
  return x + b;
}

// A tile of TC columns from `base` on, which may begin before column 0 by less than a vector
// (VEC: vectors of 16 bytes are aligned in x and out alike at base).
template <typename T, int TC, bool VEC, bool BIAS>
__global__ __launch_bounds__(256) void adjust_logits_kernel(AdjustArgs a, int tiles) {
  constexpr int VN = 16 / sizeof(T);
  __shared__ uint32_t count[TC];
  __shared__ float bias[BIAS ? TC : 1];
  __shared__ int32_t list_col[BIAS ? 256 : 1];
  __shared__ float list_val[BIAS ? 256 : 1];
  __shared__ int32_t wave_n[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int row = blockIdx.x / tiles, tile = blockIdx.x % tiles;
  const T *x = (const T *)a.x + (int64_t)row * a.xs;
  T *out = (T *)a.out + (int64_t)row * a.os;
  const int off = VEC ? (int)(reinterpret_cast<uintptr_t>(x) / sizeof(T) % VN) : 0;
  const int base = tile * TC - off;
  const int c0 = max(base, 0), c1 = min(base + TC, a.V);
  if (c0 >= c1) return;

  for (int i = tid * 4; i < TC; i += 1024) {
    *reinterpret_cast<i32x4 *>(&count[i]) = i32x4{0, 0, 0, 0};
    if constexpr (BIAS) *reinterpret_cast<f32x4 *>(&bias[i]) = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  RowSettings s{a.repetition ? a.repetition[row] : a.repetition_all, a.frequency ? a.frequency[row] : a.frequency_all,
                a.presence ? a.presence[row] : a.presence_all};
  if (!(s.r > 0.f)) s.r = 1.f;
  __syncthreads();

  if (a.L > 0) {
    const int n = a.lengths ? min(max(a.lengths[row], 0), a.L) : a.L;
    const int m = a.prompts ? min(max(a.prompts[row], 0), n) : 0;
    auto scan = [&](const auto *tok) {
      for (int i0 = tid; i0 < n; i0 += 1024) {
        int64_t t[4];   // four loads in flight, clamped instead of skipped past the end
#pragma unroll
        for (int u = 0; u < 4; ++u) t[u] = tok[min(i0 + 256 * u, n - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int i = i0 + 256 * u;
          if (i < n && t[u] >= c0 && t[u] < c1) {
            uint32_t *c = &count[(int)t[u] - base];
            if (i < m) atomicOr(c, kInPrompt);
            else atomicAdd(c, 1u);
          }
        }
      }
    };
    if (a.tokens64) scan((const int64_t *)a.tokens + (int64_t)row * a.tokens_rs);
    else scan((const int32_t *)a.tokens + (int64_t)row * a.tokens_rs);
  }
  if constexpr (BIAS) {
    const float *val = a.bias + (int64_t)row * a.bias_rs;
    for (int i0 = 0; i0 < a.K; i0 += 256) {
      const int i = i0 + tid;
      int64_t id = -1;
      if (i < a.K)
        id = a.bias64 ? ((const int64_t *)a.bias_ids)[(int64_t)row * a.bias_ids_rs + i]
                      : ((const int32_t *)a.bias_ids)[(int64_t)row * a.bias_ids_rs + i];
      const bool mine = id >= c0 && id < c1;
      const uint64_t who = __ballot(mine);
      if (lane == 0) wave_n[w] = __popcll(who);
      __syncthreads();
      int at = __popcll(who & lanes_below()), n = 0;
      for (int k = 0; k < 4; ++k) {
        at += k < w ? wave_n[k] : 0;
        n += wave_n[k];
      }
      if (mine) {
        list_col[at] = (int)id - base;
        list_val[at] = val[i];
      }
      __syncthreads();
      if (tid < n) {
        const int c = list_col[tid];
        bool first = true;
        for (int k = 0; k < tid; ++k) first = first && list_col[k] != c;
        if (first) {
          float b = bias[c];
          for (int k = tid; k < n; ++k) b += list_col[k] == c ? list_val[k] : 0.f;
          bias[c] = b;
        }
      }
      __syncthreads();
    }
  }
  __syncthreads();

  const uint32_t *ok = a.allowed ? (const uint32_t *)a.allowed + (int64_t)row * a.allowed_rs : nullptr;
  auto one = [&](int col) {
    const float y = adjusted(as_float(x[col]), count[col - base], BIAS ? bias[col - base] : 0.f, s);
    out[col] = (T)(ok && !(ok[col >> 5] >> (col & 31) & 1) ? -__builtin_huge_valf() : y);
  };
  if constexpr (VEC) {
    for (int i = tid * VN; i < TC; i += 256 * VN) {
      const int col = base + i;
      if (col >= 0 && col + VN <= a.V) {
        const i32x4 raw = *reinterpret_cast<const i32x4 *>(x + col);
        const T *e = reinterpret_cast<const T *>(&raw);
        i32x4 put;
        T *o = reinterpret_cast<T *>(&put);
        uint32_t bits = ~0u;
        if (ok) {
          const int word = col >> 5;
          const uint32_t lo = ok[word], hi = (col + VN - 1) >> 5 != word ? ok[word + 1] : 0;
          bits = (uint32_t)((((uint64_t)hi << 32) | lo) >> (col & 31));
        }
#pragma unroll
        for (int k = 0; k < VN; ++k) {
          const float y = adjusted(as_float(e[k]), count[i + k], BIAS ? bias[i + k] : 0.f, s);
          o[k] = (T)(bits >> k & 1 ? y : -__builtin_huge_valf());
        }
        *reinterpret_cast<i32x4 *>(out + col) = put;
      } else {
        for (int k = 0; k < VN; ++k)
          if (col + k >= 0 && col + k < a.V) one(col + k);
      }
    }
  } else {
    for (int i = tid; i < c1 - base; i += 256) one(base + i);
  }
}

constexpr int kSmallTile = 1024, kLargeTile = 4096;

int tile_of(int32_t N, int32_t V) {
  return (int64_t)(V / kLargeTile) * N >= 4 * device_cu_count() ? kLargeTile : kSmallTile;
}

template <typename T>
void launch(const AdjustArgs &a, hipStream_t stream) {
  constexpr int VN = 16 / sizeof(T);
  const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p) / sizeof(T) % VN; };
  // rows that begin alike within a vector in x and out
  const bool vec = at(a.x) == at(a.out) && (a.N == 1 || a.xs % VN == a.os % VN);
  auto go = [&](auto tc, auto v, auto b) {
    constexpr int TC = decltype(tc)::value;
    const int tiles = (a.V + (decltype(v)::value ? VN - 1 : 0) + TC - 1) / TC;
    adjust_logits_kernel<T, TC, decltype(v)::value, decltype(b)::value><<<(uint32_t)tiles * a.N, 256, 0, stream>>>(a, tiles);
  };
  auto go2 = [&](auto tc, auto v) {
    if (a.K > 0) go(tc, v, std::true_type{});
    else go(tc, v, std::false_type{});
  };
  auto go3 = [&](auto tc) {
    if (vec) go2(tc, std::true_type{});
    else go2(tc, std::false_type{});
  };
  if (tile_of(a.N, a.V) == kLargeTile) go3(std::integral_constant<int, kLargeTile>{});
  else go3(std::integral_constant<int, kSmallTile>{});
}

}  // namespace

int64_t adjust_blocks(int32_t N, int32_t V) { return ((int64_t)V / tile_of(N, V) + 2) * N; }

void launch_adjust_logits(const AdjustArgs &a, int dtype, hipStream_t stream) {
  if (dtype == kDtBf16) launch<bf16_t>(a, stream);
  else if (dtype == kDtF16) launch<f16_t>(a, stream);
  else launch<float>(a, stream);
}

}  // namespace mga
