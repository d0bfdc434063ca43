// Scaled embedding lookup, out[n] = T(scale W[id_n]), and its gradient by sorted
// tokens, dW[v] = T(scale sum_{n: id_n = v} dY[n]).
//
// In an MTP chunk D of every 1 + D tokens can be the one mask token: a scatter of
// atomic additions queues hundreds to thousands of rows up at one row of dW. Here
// the tokens are put in order of (id, position) and summed in that order, in fp32,
// with one rounding: every run is bit-for-bit repeatable. Both directions are bound
// by memory, the gradient by writing dW (1.2 GB at 151 936 x 4 096 bf16).
//
//   embed_sort_kernel    - a workgroup per kTile tokens sorts its (id, position)
//       pairs in LDS; the other workgroups clear dW meanwhile;
//   embed_merge_kernel   - more than one tile: every pair's place among all;
//   embed_sum_kernel     - grid (chunk of sorted tokens, column slice): sums the
//       runs of equal ids; a run that lies within its chunk is written, the parts
//       of one that crosses chunks go to the workspace;
//   embed_join_kernel    - adds the parts of each crossing run, in order;
//   embed_few_kernel     - all of it for up to kFew tokens.
#include <algorithm>

#include "mga_common.hpp"
#include "mga_internal.hpp"

namespace mga {

namespace {

constexpr int kTile = 8192;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64, kRounds = kTile / kSortThreads;
constexpr int kThreads = 256;
constexpr uint32_t kNoId = 0xFFFFFFFFu;   // padding and ids outside the table: last in order, summed nowhere

template <typename T> constexpr int kW = 16 / (int)sizeof(T);

__device__ __forceinline__ int64_t token_id(const void *ids, bool ids64, int64_t n) {
  return ids64 ? static_cast<const int64_t *>(ids)[n] : static_cast<const int32_t *>(ids)[n];
}

// kW<T> elements from p as fp32: one 16-byte load (VEC), or those of the n <= kW
// that there are.
template <typename T, bool VEC>
__device__ __forceinline__ void load_elems(const T *p, int n, float *f) {
  if constexpr (VEC) {
    const i32x4 v = *reinterpret_cast<const i32x4 *>(p);
    if constexpr (sizeof(T) == 4) {
      const f32x4 x = __builtin_bit_cast(f32x4, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = x[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = pair_lo<T>((uint32_t)v[e]);
        f[2 * e + 1] = pair_hi<T>((uint32_t)v[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kW<T>; ++e) f[e] = e < n ? (float)p[e] : 0.f;
  }
}
// N elements f to p in TO's type; n of them where not VEC
template <typename TO, bool VEC, int N>
__device__ __forceinline__ void store_elems(TO *p, int n, const float *f) {
  if constexpr (VEC) {
#pragma unroll
    for (int e = 0; e < N; e += 4) store4(p + e, f[e], f[e + 1], f[e + 2], f[e + 3]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) p[e] = (TO)f[e];
  }
}

}  // namespace

// A wave per part of up to 256 vectors of a token's row, all loads in flight.
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void embed_fwd_kernel(EmbedArgs a, int32_t parts) {
  constexpr int W = kW<T>, U = 4;
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const int64_t n = unit / parts;
  if (n >= a.N) return;
  const int part = (int)(unit - n * parts);
  const int64_t id = token_id(a.ids, a.ids64, n);
  const bool ok = id >= 0 && id < a.V;
  const T *w = static_cast<const T *>(a.w) + (ok ? id : 0) * a.w_rs;
  T *o = static_cast<T *>(a.out) + n * a.out_rs;
  float f[U][W];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = ((part * U + u) * 64 + lane) * W;
    if (c < a.H && ok) load_elems<T, VEC>(w + c, a.H - c, f[u]);
    else
#pragma unroll
      for (int e = 0; e < W; ++e) f[u][e] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = ((part * U + u) * 64 + lane) * W;
    if (c >= a.H) continue;
#pragma unroll
    for (int e = 0; e < W; ++e) f[u][e] *= ok ? a.scale : 0.f;
    store_elems<T, VEC, W>(o + c, a.H - c, f[u]);
  }
}

// Clears [V, H] (row stride rs): kClear bytes a workgroup where the rows follow each
// other, 16 KB at a time (1.24 GB: 204 us, 6.1 TB/s; past the cache or by workgroups
// that go on to a next part 210 to 350 us), else a row a wave.
constexpr int64_t kClear = 16 * 16 * kSortThreads;
template <typename TO, bool VEC>
__device__ __forceinline__ void clear_rows(TO *out, int64_t rs, int32_t V, int32_t H, int64_t block, int64_t blocks) {
  const i32x4 zero = {0, 0, 0, 0};
  if (VEC && rs == H) {
    const int64_t n = (int64_t)V * H * (int64_t)sizeof(TO) / 16;
    i32x4 *o = reinterpret_cast<i32x4 *>(out);
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      const int64_t i = (block * 16 + u) * kSortThreads + threadIdx.x;
      if (i < n) o[i] = zero;
    }
    return;
  }
  const int lane = threadIdx.x & 63;
  for (int64_t v = block * (kSortThreads / 64) + (threadIdx.x >> 6); v < V; v += blocks * (kSortThreads / 64)) {
    TO *o = out + v * rs;
    if constexpr (VEC) {
      for (int c = lane * kW<TO>; c < H; c += 64 * kW<TO>) *reinterpret_cast<i32x4 *>(o + c) = zero;
    } else {
      for (int c = lane; c < H; c += 64) o[c] = (TO)0.f;
    }
  }
}

template <typename TO, bool VEC>
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(EmbedArgs a, int32_t tiles, bool clear,
                                                                  uint64_t *__restrict__ sorted) {
  __shared__ uint64_t key[kTile];
  __shared__ uint32_t count[kSortThreads], sums[kSortWaves];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= tiles) {
    if (clear)
      clear_rows<TO, VEC>(static_cast<TO *>(a.out), a.out_rs, a.V, a.H, blockIdx.x - tiles, gridDim.x - tiles);
    return;
  }
  const int64_t n0 = (int64_t)blockIdx.x * kTile;
  const int n = (int)min((int64_t)kTile, a.N - n0);
  // the tile in order of position: a wave's part is contiguous, 64 pairs a round
  const int rounds = (n + kSortThreads - 1) / kSortThreads, lane = tid & 63, wave = tid >> 6;
  const int at0 = wave * rounds * 64 + lane;
  uint64_t k[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = at0 + r * 64;
    k[r] = (uint64_t)kNoId << 32;
    if (r < rounds && i < n) {
      const int64_t id = token_id(a.ids, a.ids64, n0 + i);
      const bool ok = id >= 0 && id < a.V && id != a.padding_idx;
      k[r] = (uint64_t)(ok ? (uint32_t)id : kNoId) << 32 | (uint32_t)(n0 + i);
    }
  }
  // By digits of six bits from the lowest, each pass stable: lane d of a wave counts
  // digit d, and a pair's place is what has its digit in earlier waves, earlier
  // rounds and lower lanes, behind all lower digits. The pairs that are none, and
  // the places past n, have the digit 63 in every pass and stay last (the last
  // pass has a spare bit for them).
  const int bits = 33 - __builtin_clz(a.V);
  for (int shift = 0; shift < bits; shift += 6) {
    uint32_t place[kRounds], mine = 0;   // mine: of digit `lane`, in the rounds so far
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (r >= rounds) break;
      const uint32_t d = (uint32_t)(k[r] >> (32 + shift)) & 63;
      uint64_t same = ~uint64_t(0), own = ~uint64_t(0);   // lanes of my digit, of the digit I count
#pragma unroll
      for (int b = 0; b < 6; ++b) {
        const uint64_t set = __ballot((d >> b) & 1);
        same &= (d >> b) & 1 ? set : ~set;
        own &= (lane >> b) & 1 ? set : ~set;
      }
      place[r] = __shfl(mine, d, 64) + __popcll(same & lanes_below());
      mine += __popcll(own);
    }
    count[lane * kSortWaves + wave] = mine;
    __syncthreads();
    // sums over (digit, wave) in that order, an entry a thread
    const uint32_t c = count[tid];
    uint32_t in = c;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t o = __shfl_up(in, s, 64);
      if (lane >= s) in += o;
    }
    if (lane == 63) sums[wave] = in;
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) before += w < wave ? sums[w] : 0;
    count[tid] = before + in - c;
    __syncthreads();
    const uint32_t base = count[lane * kSortWaves + wave];
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (r < rounds) key[__shfl(base, (int)(k[r] >> (32 + shift)) & 63, 64) + place[r]] = k[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (r < rounds) k[r] = key[at0 + r * 64];
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (r < rounds && at0 + r * 64 < n) sorted[n0 + at0 + r * 64] = k[r];
}

// Each pair's place: those before it in its own tile and in the others.
__global__ __launch_bounds__(kThreads) void embed_merge_kernel(const uint64_t *__restrict__ tiles_in, int32_t N,
                                                               int32_t tiles, uint64_t *__restrict__ sorted) {
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= N) return;
  const uint64_t k = tiles_in[i];
  const int own = (int)(i / kTile);
  int64_t place = i - (int64_t)own * kTile;
  for (int t = 0; t < tiles; ++t) {
    if (t == own) continue;
    const uint64_t *p = tiles_in + (int64_t)t * kTile;
    int lo = 0, hi = (int)min((int64_t)kTile, N - (int64_t)t * kTile);
    while (lo < hi) {   // pairs are all different
      const int mid = (lo + hi) >> 1;
      if (p[mid] < k) lo = mid + 1;
      else hi = mid;
    }
    place += lo;
  }
  sorted[place] = k;
}

namespace {

__device__ __forceinline__ uint32_t id_at(const uint64_t *sorted, int64_t i) { return (uint32_t)(sorted[i] >> 32); }

// scale f into out[id], added to what is there where ADD
template <typename TO, bool VEC, bool ADD, int N>
__device__ __forceinline__ void put_row(const EmbedArgs &a, uint32_t id, int col, float *f) {
  TO *o = static_cast<TO *>(a.out) + (int64_t)id * a.out_rs + col;
  const int n = a.H - col;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    f[e] *= a.scale;
    if constexpr (ADD)
      if (VEC || e < n) f[e] += (float)o[e];
  }
  store_elems<TO, VEC, N>(o, n, f);
}

}  // namespace

constexpr int kMaxChunk = 64;

template <typename T, typename TO, bool VEC, bool ADD>
__global__ __launch_bounds__(kThreads) void embed_sum_kernel(EmbedArgs a, const uint64_t *__restrict__ sorted,
                                                             int32_t chunk, float *__restrict__ part) {
  constexpr int W = kW<T>, U = 8;
  __shared__ uint64_t key[kMaxChunk + 2];   // the chunk's, with its neighbours on both sides
  const int tid = threadIdx.x;
  const int64_t n0 = (int64_t)blockIdx.x * chunk;
  const int n = (int)min((int64_t)chunk, a.N - n0);
  if (tid < n + 2) {
    const int64_t i = n0 - 1 + tid;
    key[tid] = i >= 0 && i < a.N ? sorted[i] : (uint64_t)kNoId << 32;
  }
  __syncthreads();
  const int col = (blockIdx.y * kThreads + tid) * W;
  if (col >= a.H) return;
  auto id = [&](int i) { return (uint32_t)(key[i + 1] >> 32); };
  const T *dy = static_cast<const T *>(a.dy) + col;
  float acc[W];
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = 0.f;
  bool whole = id(0) != id(-1);   // the run began in this chunk
  for (int i0 = 0; i0 < n && id(i0) != kNoId; i0 += U) {
    float f[U][W];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = (uint32_t)key[min(i0 + u, n - 1) + 1];   // past the end: the last one again
      load_elems<T, VEC>(dy + at * a.dy_rs, a.H - col, f[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= n || id(i) == kNoId) break;
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] += f[u][e];
      const bool ends = id(i + 1) != id(i);
      if (!ends && i + 1 < n) continue;
      if (whole && ends) {
        put_row<TO, VEC, ADD, W>(a, id(i), col, acc);
      } else {   // slot 0: came from the chunk before, 1: began here
        float *p = part + ((int64_t)blockIdx.x * 2 + (whole ? 1 : 0)) * a.part_rs + col;
        store_elems<float, true, W>(p, W, acc);
      }
#pragma unroll
      for (int e = 0; e < W; ++e) acc[e] = 0.f;
      whole = true;
    }
  }
}

// grid (kLook chunks, slice of 256 columns): where a run begins in a chunk and goes on
// behind it, the sum of its parts, shared by the waves. Most chunks have no such run:
// a workgroup looks at several, since those that end at once cost their dispatch
// (6 144 tokens x 2 560 and 5 120 x 4 096: four chunks 9.8 and 9.9 us, two 10.3 and
// 13.0, eight 11.9 and 11.2, sixteen waves 16.7 and 18.9).
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64, kLook = 4;
template <typename TO, bool VEC, bool ADD>
__global__ __launch_bounds__(kJoinThreads) void embed_join_kernel(EmbedArgs a, const uint64_t *__restrict__ sorted,
                                                                  int32_t chunk, const float *__restrict__ part) {
  __shared__ f32x4 sums[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.y * 256 + lane * 4;
  const int64_t chunks = ((int64_t)a.N + chunk - 1) / chunk, first = (int64_t)blockIdx.x * kLook;
  auto goes_on = [&](int64_t c) {   // the run at the end of chunk c
    const int64_t at = (c + 1) * chunk;
    const uint32_t id = id_at(sorted, at);
    if (id == kNoId || id_at(sorted, at - 1) != id) return false;
    const int64_t n0 = c * chunk;
    return !(n0 > 0 && id_at(sorted, n0) == id && id_at(sorted, n0 - 1) == id);   // began further back
  };
  uint64_t found = __ballot(lane < kLook && first + lane + 1 < chunks && goes_on(first + lane));
  for (; found; found &= found - 1) {
    const int64_t c0 = first + __builtin_ctzll(found);
    const uint32_t id = id_at(sorted, (c0 + 1) * chunk);
    int64_t lo = c0 + 1, hi = chunks;   // the last chunk that begins with the run: 64 probes a turn
    while (hi - lo > 1) {
      const int64_t step = (hi - lo + 63) / 64, c = lo + (lane + 1) * step;
      lo += step * __popcll(__ballot(c < hi && id_at(sorted, c * chunk) == id));
      hi = min(hi, lo + step);
    }
    const int64_t count = lo - c0 + 1;   // slot 1 of c0, slot 0 of the others
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (col < a.H) {
      const int64_t per = (count + kJoinWaves - 1) / kJoinWaves, to = min(count, (wave + 1) * per);
      auto slot = [&](int64_t i) {
        return *reinterpret_cast<const f32x4 *>(part + ((c0 + i) * 2 + (i == 0)) * a.part_rs + col);
      };
      int64_t i = wave * per;
      for (; i + 8 <= to; i += 8) {
        f32x4 f[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) f[u] = slot(i + u);
#pragma unroll
        for (int u = 0; u < 8; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += f[u][e];
      }
      for (; i < to; ++i) {
        const f32x4 f = slot(i);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += f[e];
      }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && col < a.H) {
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[e] = sums[0][lane][e];
#pragma unroll
        for (int w = 1; w < kJoinWaves; ++w) f[e] += sums[w][lane][e];
      }
      put_row<TO, VEC, ADD, 4>(a, id, col, f);
    }
    __syncthreads();
  }
}

// Few tokens in one launch, unsorted. Workgroups [0, N slices): token n and a slice of
// columns; where n is the first with its id, the sum of all with it, shared by the
// waves in order. The others: clear those of `rows` rows that no token has. 323
// tokens, half of one id, new and added to: 1 024 x 256 fp32 5.8 and 5.5 us, sorted
// 15.6 and 17.1; 32 003 x 2 560 fp16 27 and 8, sorted 34 and 20; all 512 of one id
// 35 and 16, sorted 33 and 18. A large table is cleared faster beside the sort (parts
// of 256 KB that look no row up); 323 tokens x 4 096 bf16, few against sorted: 131 MB 29
// and 32 us, 213 MB 49 and 50, 262 MB 59 and 59, 426 MB 91 and 87, 1.2 GB 233 and 221
// (64 tokens: even at 524 MB; 512: 33 MB 23 and 27, 131 MB 34 and 31).
constexpr int kFew = 512, kFewThreads = 512, kFewWaves = kFewThreads / 64, kFewRows = 4096;
constexpr int64_t kFewClear = 64 << 10, kFewTable = 256 << 20;   // bytes a workgroup clears; of the table
template <typename T, typename TO, bool VEC, bool ADD>
__global__ __launch_bounds__(kFewThreads) void embed_few_kernel(EmbedArgs a, int32_t slices, int32_t rows) {
  constexpr int W = kW<T>, U = 8, kEach = kFew / 64;
  __shared__ uint32_t ids[kFew], list[kFew];
  __shared__ float sums[kFewWaves][64 * W];
  static_assert(kFewThreads == kFew && sizeof(sums) >= kFewRows, "a token a thread; the flags in sums");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t own = tid < a.N ? token_id(a.ids, a.ids64, tid) : -1;
  ids[tid] = own >= 0 && own < a.V && own != a.padding_idx ? (uint32_t)own : kNoId;
  const int64_t unit = blockIdx.x;
  if (unit >= (int64_t)a.N * slices) {
    bool *used = reinterpret_cast<bool *>(sums);
    const int64_t v0 = (unit - (int64_t)a.N * slices) * rows, v1 = min((int64_t)a.V, v0 + rows);
    for (int i = tid; i < rows; i += kFewThreads) used[i] = false;
    __syncthreads();
    if (ids[tid] != kNoId && own >= v0 && own < v1) used[own - v0] = true;
    __syncthreads();
    TO *o = static_cast<TO *>(a.out) + v0 * a.out_rs;
    constexpr int S = VEC ? kW<TO> : 1;   // elements a store
    const uint32_t wide = (uint32_t)a.H / S, all = (uint32_t)(v1 - v0) * wide;
#pragma unroll 4
    for (uint32_t i = tid; i < all; i += kFewThreads) {
      const uint32_t v = i / wide;
      if (used[v]) continue;
      TO *p = o + (int64_t)v * a.out_rs + (i - v * wide) * S;
      if constexpr (VEC) *reinterpret_cast<i32x4 *>(p) = i32x4{0, 0, 0, 0};
      else *p = (TO)0.f;
    }
    return;
  }
  __syncthreads();
  const int n = (int)(unit / slices), col = ((int)(unit - (int64_t)n * slices) * 64 + lane) * W;
  const uint32_t id = ids[n];
  if (id == kNoId) return;
  int count = 0, place = 0, before = 0;   // tokens with the id; of them before mine, before n
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const uint64_t same = __ballot(ids[j * 64 + lane] == id);
    if (j == wave) place = count + __popcll(same & lanes_below());
    if (j * 64 < n) before += __popcll(n - j * 64 >= 64 ? same : same & ((uint64_t(1) << (n - j * 64)) - 1));
    count += __popcll(same);
  }
  if (before) return;   // not the first
  if (ids[tid] == id) list[place] = tid;
  __syncthreads();
  const int per = (count + kFewWaves - 1) / kFewWaves, to = min(count, (wave + 1) * per);
  const T *dy = static_cast<const T *>(a.dy) + col;
  float acc[W];
#pragma unroll
  for (int e = 0; e < W; ++e) acc[e] = 0.f;
  if (col < a.H) {
    for (int i0 = wave * per; i0 < to; i0 += U) {
      float f[U][W];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < to) load_elems<T, VEC>(dy + (int64_t)list[i0 + u] * a.dy_rs, a.H - col, f[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < to)
#pragma unroll
          for (int e = 0; e < W; ++e) acc[e] += f[u][e];
    }
  }
  const int waves = (count + per - 1) / per;   // that have tokens
  if (waves > 1) {
    if (wave > 0)
#pragma unroll
      for (int e = 0; e < W; ++e) sums[wave][e * 64 + lane] = acc[e];
    __syncthreads();
    if (wave == 0)
      for (int w = 1; w < waves; ++w)
#pragma unroll
        for (int e = 0; e < W; ++e) acc[e] += sums[w][e * 64 + lane];
  }
  if (wave == 0 && col < a.H) put_row<TO, VEC, ADD, W>(a, id, col, acc);
}

namespace {

// Sorted tokens a chunk: about a thousand workgroups over all slices.
int chunk_of(int32_t N, int32_t H, int W) {
  const int64_t slices = ((int64_t)H + kThreads * W - 1) / (kThreads * W);
  return (int)std::min<int64_t>(kMaxChunk, std::max<int64_t>(16, (int64_t)N * slices / 1024));
}

template <typename T, bool VEC>
void fwd_typed(const EmbedArgs &a, hipStream_t st) {
  const int32_t parts = (a.H + 256 * kW<T> - 1) / (256 * kW<T>);
  const int64_t units = (int64_t)a.N * parts;
  hipLaunchKernelGGL((embed_fwd_kernel<T, VEC>), dim3((unsigned)((units + 3) / 4)), dim3(kThreads), 0, st, a, parts);
}

template <typename T, typename TO, bool VEC>
void bwd_typed(EmbedArgs a, bool add, char *ws, hipStream_t st) {
  const int32_t slices = (a.H + 64 * kW<T> - 1) / (64 * kW<T>);
  if (a.N > 0 && a.N <= kFew && (int64_t)a.N * slices < 1 << 20 &&
      (add || (int64_t)a.V * a.H * (int64_t)sizeof(TO) < kFewTable)) {
    const int64_t fit = kFewClear / ((int64_t)a.H * (int64_t)sizeof(TO));
    const int32_t rows = (int32_t)std::max<int64_t>(1, std::min<int64_t>(kFewRows, fit));
    const int64_t units = (int64_t)a.N * slices + (add ? 0 : ((int64_t)a.V + rows - 1) / rows);
    auto run = [&](auto few) {
      hipLaunchKernelGGL(few, dim3((unsigned)units), dim3(kFewThreads), 0, st, a, slices, rows);
    };
    if (add) run(embed_few_kernel<T, TO, VEC, true>);
    else run(embed_few_kernel<T, TO, VEC, false>);
    return;
  }
  const int tiles = (a.N + kTile - 1) / kTile;
  uint64_t *sorted = reinterpret_cast<uint64_t *>(ws), *raw = sorted;
  ws += ((int64_t)a.N * 8 + 15) / 16 * 16;
  if (tiles > 1) {
    raw = reinterpret_cast<uint64_t *>(ws);
    ws += ((int64_t)a.N * 8 + 15) / 16 * 16;
  }
  float *part = reinterpret_cast<float *>(ws);
  // workgroups that clear: one a part, or each for several rows
  int64_t clear = 0;
  if (!add) {
    clear = ((int64_t)a.V * a.H * (int64_t)sizeof(TO) + kClear - 1) / kClear;
    if (!VEC || a.out_rs != a.H) clear = std::min<int64_t>(((int64_t)a.V + 15) / 16, 4096);
  }
  if (tiles + clear == 0) return;
  hipLaunchKernelGGL((embed_sort_kernel<TO, VEC>), dim3((unsigned)(tiles + clear)), dim3(kSortThreads), 0, st, a, tiles,
                     !add, raw);
  if (a.N == 0) return;
  if (tiles > 1)
    hipLaunchKernelGGL(embed_merge_kernel, dim3((a.N + kThreads - 1) / kThreads), dim3(kThreads), 0, st, raw, a.N,
                       tiles, sorted);
  const int chunk = chunk_of(a.N, a.H, kW<T>);
  const unsigned chunks = (a.N + chunk - 1) / chunk;
  const dim3 grid(chunks, (a.H + kThreads * kW<T> - 1) / (kThreads * kW<T>));
  const dim3 join((chunks + kLook - 1) / kLook, (a.H + 255) / 256);
  auto run = [&](auto sum, auto joined) {
    hipLaunchKernelGGL(sum, grid, dim3(kThreads), 0, st, a, sorted, chunk, part);
    if (chunks > 1) hipLaunchKernelGGL(joined, join, dim3(kJoinThreads), 0, st, a, sorted, chunk, part);
  };
  if (add) run(embed_sum_kernel<T, TO, VEC, true>, embed_join_kernel<TO, VEC, true>);
  else run(embed_sum_kernel<T, TO, VEC, false>, embed_join_kernel<TO, VEC, false>);
}

}  // namespace

int64_t embed_part_stride(int32_t H) { return ((int64_t)H + 15) / 16 * 16; }

int64_t embed_workspace_bytes(int32_t N, int32_t H) {
  const int64_t keys = ((int64_t)N * 8 + 15) / 16 * 16;
  const int chunk = std::min(chunk_of(N, H, 4), chunk_of(N, H, 8));
  return keys * (N > kTile ? 2 : 1) + ((int64_t)N + chunk - 1) / chunk * 2 * embed_part_stride(H) * 4;
}

void launch_embed_fwd(const EmbedArgs &a, int dtype, bool vec, hipStream_t st) {
  auto run = dtype == kDtF32   ? (vec ? fwd_typed<float, true> : fwd_typed<float, false>)
             : dtype == kDtF16 ? (vec ? fwd_typed<f16_t, true> : fwd_typed<f16_t, false>)
                               : (vec ? fwd_typed<bf16_t, true> : fwd_typed<bf16_t, false>);
  run(a, st);
}

void launch_embed_bwd(const EmbedArgs &a, int dtype, int out_dtype, bool vec, bool add, void *ws, hipStream_t st) {
  EmbedArgs b = a;
  b.part_rs = embed_part_stride(a.H);
  auto run = dtype == kDtF32 ? (vec ? bwd_typed<float, float, true> : bwd_typed<float, float, false>)
             : dtype == kDtF16
                 ? (out_dtype == kDtF32 ? (vec ? bwd_typed<f16_t, float, true> : bwd_typed<f16_t, float, false>)
                                        : (vec ? bwd_typed<f16_t, f16_t, true> : bwd_typed<f16_t, f16_t, false>))
                 : (out_dtype == kDtF32 ? (vec ? bwd_typed<bf16_t, float, true> : bwd_typed<bf16_t, float, false>)
                                        : (vec ? bwd_typed<bf16_t, bf16_t, true> : bwd_typed<bf16_t, bf16_t, false>));
  run(b, add, static_cast<char *>(ws), st);
}

}  // namespace mga
