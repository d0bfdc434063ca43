// Attention of new tokens over a paged 8-bit cache (layout: mga_paged.hpp):
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   j <= length + i of i's sequence,
// for a ragged batch of 1 .. thousands of new tokens a sequence.
//
// Work. A tile is up to 16 NT query rows of one sequence and KV head: TM tokens (a
// power of two) times the G query heads of the group. It visits the cache in steps
// of 64 keys. The steps of all tiles, sequences and heads form one list, cut into
// equal shares, one a workgroup: ragged batches and few long sequences fill the chip
// alike. A tile that a cut goes through leaves fp32 partial results (at most two
// a workgroup), joined in a fixed order by a second launch. Each workgroup finds its
// share from the lengths on the device (a scan over the sequences; a tile's place
// within its sequence has a closed form, as TM divides 64), so the launch depends on
// no length and can be captured.
//
// Step. Each of the 4 waves takes every fourth step of the share and keeps its own
// running maximum, sum and output; they meet in LDS at the tile's end. K and V go from
// memory to registers to the matrix unit, 16 bytes a lane, with nothing in between
// but the conversion of two codes an instruction, under the page's scale, to bf16
// (exact). S^T = K Q^T by v_mfma_f32_16x16x32_bf16: key m of tile t of the step is key
// 16 (m / 4) + 4 t + m % 4, so that lane group g holds the probabilities of keys
// 16 g .. 16 g + 15, which is what it needs as the second operand of O^T += V^T P^T
// against 16 consecutive bytes of a value page. The channels of a K row are dealt to the
// lane groups 16 at a time, and those of Q likewise.
// Probabilities are taken against a running offset; a step is accepted while
// every lane's partial row sum stays <= 2^20, else the offset moves to the exact
// maximum and the step is redone from its scores.
//
// Precision: scores, statistics and outputs in fp32. bf16 queries: P is rounded to
// bf16 for its product, the row sum is not. fp16 and fp32 queries are split into 2 or 3
// bf16 parts and P into as many (K and V are exact in bf16): 16 and 24 bits.
//
// Where a value that a row may not see is NaN (a masked place), its products would be
// NaN although p = 0: see put_nan.
#include <algorithm>

#include "mga_internal.hpp"
#include "mga_paged.hpp"

namespace mga {
namespace {

template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int n = 1; };
template <> struct Parts<f16_t> { static constexpr int n = 2; };
template <> struct Parts<float> { static constexpr int n = 3; };

constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Eight codes (two dwords) under a power-of-two scale.
__device__ __forceinline__ bf16x8 decode8(uint32_t a, uint32_t b, float s) {
  const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false),
               q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true),
               r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false),
               t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true);
  return bf16x8{p[0], p[1], q[0], q[1], r[0], r[1], t[0], t[1]};
}

// x = the sum of N bf16 parts, up to the last one's rounding.
template <int N>
__device__ __forceinline__ void split8(const float *x, bf16x8 *part) {
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[n][i] = (bf16_t)rest[i];
      if (n + 1 < N) rest[i] -= (float)part[n][i];
    }
  }
}

// Bit 7 of each byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_bits(uint32_t c) { return ((c & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The bytes of a dword before byte n.
__device__ __forceinline__ uint32_t first_bytes(int n) { return n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1; }

// ---- tiles and steps -----------------------------------------------------------

// Sum over i < n of floor(i / 2^r).
__device__ __forceinline__ int64_t floor_sum(int64_t n, int r) {
  const int64_t q = n >> r, m = n - (q << r);
  return ((q * (q - 1) / 2) << r) + m * q;
}

// A sequence's tiles of 2^tmshift tokens: tile t takes ceil((len + min(n, (t + 1) TM)) / 64) steps.
struct SeqTiles {
  int n, len, tmshift;
  __device__ __forceinline__ int tiles() const { return (n + (1 << tmshift) - 1) >> tmshift; }
  __device__ __forceinline__ int steps(int t) const { return (len + min(n, (t + 1) << tmshift) + 63) >> 6; }
  // of the tiles before t <= tiles() - 1
  __device__ __forceinline__ int64_t before(int t) const {
    if (t == 0) return 0;
    const int64_t x = ((int64_t)len + 63 + (1 << tmshift)) >> tmshift;
    return floor_sum(x + t, 6 - tmshift) - floor_sum(x, 6 - tmshift);
  }
  __device__ __forceinline__ int64_t all() const {
    const int t = tiles();
    return t ? before(t - 1) + steps(t - 1) : 0;
  }
};

// Tokens of a tile: the largest power of two (at most 64) of which a tile holds the query heads.
inline int tm_shift(int rows, int G) {
  int s = 0;
  while (((2 << s) * G <= rows) && s < 6) ++s;
  return s;
}

// One tile: `b`'s tokens tok0 .. tok0 + ntok - 1 and the G query heads of KV head h.
struct Tile {
  int b, h, t;
  SeqSpan q;
  int tok0, ntok, rows, steps;
  __device__ __forceinline__ void set(const SeqTiles &st, int tile, int G) {
    t = tile;
    tok0 = t << st.tmshift;
    ntok = min(1 << st.tmshift, q.n - tok0);
    rows = ntok * G;
    steps = st.steps(t);
  }
};

// Tiles are also numbered without a scan: sequence b owns the slots from (cu[b] >> tmshift) + b
// on, as many as n tokens can make tiles.
__device__ __forceinline__ int tile_slot(const SeqSpan &q, int b, int t, int tmshift) {
  return (q.first >> tmshift) + b + t;
}
__host__ __device__ __forceinline__ int tile_slots(int T, int B, int tmshift) { return (T >> tmshift) + B; }

// The tile of a slot; false: none. All lanes of the wave take part.
__device__ __forceinline__ bool tile_of_slot(const PagedAttnArgs &a, int slot, int tmshift, int G, Tile &x) {
  int b = 0;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = i0 + (threadIdx.x & 63) + 1;
    b += __popcll(__ballot(i <= a.B && (min(max(a.cu[min(i, a.B)], 0), a.T) >> tmshift) + i <= slot));
  }
  x.b = __builtin_amdgcn_readfirstlane(b);
  if (x.b >= a.B) return false;
  x.q = seq_span(a.cu, a.lengths, x.b, a.T, a.width << a.pshift);
  const SeqTiles st{x.q.n, x.q.len, tmshift};
  const int t = slot - tile_slot(x.q, x.b, 0, tmshift);
  if (t < 0 || t >= st.tiles()) return false;
  x.set(st, t, G);
  return true;
}

// A row of a tile in q and out.
template <typename T>
__device__ __forceinline__ T *row_of(const Tile &x, int G, int r, const void *base, int64_t ss, int64_t hs) {
  const int tk = r / G;
  return (T *)base + (int64_t)(x.q.first + x.tok0 + tk) * ss + (int64_t)(x.h * G + r - tk * G) * hs;
}

// 16 bytes at a wave-uniform address plus a lane offset; the address stays in scalar registers.
__device__ __forceinline__ i32x4 load16(const uint8_t *base, uint32_t off) {
  typedef const __attribute__((address_space(1))) uint8_t *global_u8;
  typedef const __attribute__((address_space(1))) i32x4 *global_v4;
  global_u8 b = (global_u8)base;
  asm("" : "+s"(b));
  return *(global_v4)(b + off);
}

// ---- the steps of one wave ------------------------------------------------------

// UNI: pages of 64 tokens or more, so that a step lies in one page: its id and scales are
// wave-uniform (read for 64 steps at a time, one a lane), and the loads take a scalar base with
// a lane offset that never changes.
template <int HD, int NT, typename T, bool UNI>
struct Steps {
  static constexpr int NQ = Parts<T>::n, KS = HD / 32, ND = HD / 16, KL = HD / 64;
  const PagedAttnArgs &a;
  const Tile &x;
  const int lane, col, g;
  bf16x8 qf[NT][NQ][KS];
  int lim[NT];          // each row's last key
  f32x4 o[NT][ND];
  float m[NT], l[NT];   // l: this lane's part of the row sum

  __device__ __forceinline__ Steps(const PagedAttnArgs &a_, const Tile &x_, int G)
      : a(a_), x(x_), lane(threadIdx.x & 63), col(lane & 15), g(lane >> 4) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 16 + col;
      lim[nt] = r < x.rows ? x.q.len + x.tok0 + r / G : -1;
      const T *qp = row_of<const T>(x, G, r, a.q, a.q_ss, a.q_hs);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int c = 64 * (ks >> 1) + 16 * g + 8 * (ks & 1);
        if constexpr (NQ == 1) {
          qf[nt][0][ks] = r < x.rows ? load8(qp + c) : bf16x8{};
        } else {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
          if (r < x.rows) {
            if constexpr (NQ == 2) {
              const f16x8 e = __builtin_bit_cast(f16x8, load8(qp + c));
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = (float)e[i];
            } else {
              const f32x4 e = *reinterpret_cast<const f32x4 *>(qp + c), f = *reinterpret_cast<const f32x4 *>(qp + c + 4);
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] = e[i], v[i + 4] = f[i];
            }
          }
          bf16x8 part[NQ];
          split8<NQ>(v, part);
#pragma unroll
          for (int n = 0; n < NQ; ++n) qf[nt][n][ks] = part[n];
        }
      }
      m[nt] = kNegInf;
      l[nt] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // steps p0, p0 + stride, .. below p1
  __device__ __forceinline__ void run(int p0, int p1, int stride) {
    if (p0 >= p1) return;
    const int n = (p1 - p0 + stride - 1) / stride;
    const int PS = 1 << a.pshift, kg = col >> 2;
    const int32_t *trow = a.table + (int64_t)x.b * a.table_rs;
    const int first_lim = x.q.len + x.tok0;   // the last key that the tile's first token sees
    const int end_key = x.q.len + x.q.n;

    auto page_at = [&](int i) {   // -1: none
      const int id = i < a.width ? trow[i] : -1;
      return (uint32_t)id < (uint32_t)a.num_pages ? id : -1;
    };
    // UNI: lane i holds what step 64 k + i needs
    int tpage = -1;
    float tks = 0.f, tvs = 0.f;
    auto refill = [&](int i0) {
      const int i = i0 + lane;
      tpage = i < n ? page_at((p0 + i * stride) >> (a.pshift - 6)) : -1;
      const int64_t ph = (int64_t)max(tpage, 0) * a.Hkv + x.h;
      tks = a.ks[ph];
      tvs = a.vs[ph];
      // wait here, once in 64 steps: left to the reads of a lane, the wait would be in every step
      // and drain the tiles in flight
      __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));   // vmcnt(0) only
    };
    // else: the ids of the lane's key group (K) and of its value group, two steps ahead
    int kid[2] = {-1, -1}, vid[2] = {-1, -1};
    auto ids = [&](int i, int at) {
      const int k0 = (p0 + i * stride) * 64;
      kid[at] = i < n ? page_at((k0 + 16 * kg) >> a.pshift) : -1;
      vid[at] = i < n ? page_at((k0 + 16 * g) >> a.pshift) : -1;
    };

    i32x4 kc[4][KL], vc[ND];
    float ksc = 0.f, vsc = 0.f;
    int vpage = -1;
    const uint32_t koff = (uint32_t)((16 * kg + (col & 3)) * HD + 16 * g), voff = (uint32_t)(col * PS + 16 * g);
    // Step i's loads. Past the last step they still issue (a branch around them would make the
    // compiler wait for all loads where its paths meet), for a few bytes of page 0.
    auto load_k = [&](int i) {
      const int p = p0 + i * stride;
      if constexpr (UNI) {
        const int page = max(__builtin_amdgcn_readlane(tpage, i & 63), 0);
        const uint8_t *base = a.kp + (((int64_t)page * a.Hkv + x.h) * PS + ((p * 64) & (PS - 1))) * HD;
        ksc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, tks), i & 63));
        const uint32_t off = i < n ? koff : 0;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < KL; ++j) kc[t][j] = load16(base + (4 * t * HD + 64 * j), off);
      } else {
        const int64_t ph = (int64_t)max(kid[0], 0) * a.Hkv + x.h;
        const uint8_t *base = a.kp + (ph * PS + ((p * 64 + 16 * kg) & (PS - 1)) + (col & 3)) * HD + 16 * g;
        ksc = a.ks[ph];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < KL; ++j) kc[t][j] = *reinterpret_cast<const i32x4 *>(base + 4 * t * HD + 64 * j);
      }
      __builtin_amdgcn_sched_barrier(0);   // keys before values, here and in the loop
    };
    auto load_v = [&](int i, int at) {   // at: the lane that holds step i's page
      const int p = p0 + i * stride;
      if constexpr (UNI) {
        vpage = __builtin_amdgcn_readlane(tpage, at);
        const uint8_t *base = a.vp + ((int64_t)max(vpage, 0) * a.Hkv + x.h) * HD * PS + ((p * 64) & (PS - 1));
        vsc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, tvs), at));
        const uint32_t off = i < n ? voff : 0;
#pragma unroll
        for (int d = 0; d < ND; ++d) vc[d] = load16(base + 16 * d * PS, off);
      } else {
        vpage = vid[0];
        const int64_t ph = (int64_t)max(vpage, 0) * a.Hkv + x.h;
        const uint8_t *base = a.vp + (ph * HD + col) * PS + ((p * 64 + 16 * g) & (PS - 1));
        vsc = a.vs[ph];
#pragma unroll
        for (int d = 0; d < ND; ++d) vc[d] = *reinterpret_cast<const i32x4 *>(base + 16 * d * PS);
      }
      __builtin_amdgcn_sched_barrier(0);
    };

    if constexpr (UNI) {
      refill(0);
    } else {
      ids(0, 0);
      ids(1, 1);
    }
    int nan_from = n;
    load_k(0);
    load_v(0, 0);
    for (int i = 0; i < n; ++i) {
      const int p = p0 + i * stride;
      f32x4 s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[nt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
      // four independent sums a turn; the fences keep the compiler from converting the whole
      // step first, which would take 64 registers each for K and V
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const i32x4 c = kc[t][ks >> 1];
          const bf16x8 kf = decode8(c[2 * (ks & 1)], c[2 * (ks & 1) + 1], ksc);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < NQ; ++q) s[nt][t] = mfma16(kf, qf[nt][q][ks], s[nt][t]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      const int vnow = vpage;
      if constexpr (UNI) {
        if (((i + 1) & 63) == 0) refill(i + 1);
      } else {
        kid[0] = kid[1];
        vid[0] = vid[1];
        ids(i + 2, 1);
      }
      load_k(i + 1);

      // this lane's keys: key0 + 4 t + r
      const int key0 = p * 64 + 16 * g;
      const bool edge = p * 64 + 63 > first_lim || (UNI ? vnow < 0 : (bool)__any(vnow < 0));
      bf16x8 pf[NT][NQ][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (edge) {
          const int last = vnow < 0 ? -1 : lim[nt];
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[nt][t][r] = key0 + 4 * t + r <= last ? s[nt][t][r] : kNegInf;
        }
        float e[16], sum = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          e[k] = __builtin_amdgcn_exp2f(fmaf(s[nt][k >> 2][k & 3], a.scale_log2, -m[nt]));
          sum += e[k];
        }
        if (__any(!(sum <= 0x1p20f))) {
          float mx = kNegInf;
#pragma unroll
          for (int k = 0; k < 16; ++k) mx = fmaxf(mx, s[nt][k >> 2][k & 3]);
          mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float now = fmaxf(m[nt], mx * a.scale_log2);
          const float off = now == kNegInf ? 0.f : now;
          const float alpha = __builtin_amdgcn_exp2f(m[nt] - off);   // 0 from -inf
          l[nt] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) o[nt][d] *= alpha;
          m[nt] = now;
          sum = 0.f;
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            e[k] = __builtin_amdgcn_exp2f(fmaf(s[nt][k >> 2][k & 3], a.scale_log2, -off));
            sum += e[k];
          }
        }
        l[nt] += sum;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          bf16x8 part[NQ];
          split8<NQ>(e + 8 * c, part);
#pragma unroll
          for (int q = 0; q < NQ; ++q) pf[nt][q][c] = part[q];
        }
      }

      if (edge && cut_values(vc, vnow < 0 ? 0 : end_key - key0)) nan_from = min(nan_from, i);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const bf16x8 vf = decode8(vc[d][2 * c], vc[d][2 * c + 1], vsc);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < NQ; ++q) o[nt][d] = mfma16(vf, pf[nt][q][c], o[nt][d]);
          if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
      load_v(i + 1, (i + 1) & 63);
    }

    // NaNs that were taken out of an edge step's values (rare)
    for (int i = nan_from; i < n; ++i) {
      const int p = p0 + i * stride;
      if constexpr (UNI) refill(i);
      else ids(i, 0);
      load_v(i, 0);
      if (p * 64 + 63 > first_lim || __any(vpage < 0)) put_nan(vc, p * 64 + 16 * g, vpage);
    }
  }

  // Of an edge step's values: zeros from row `valid` on and for NaN, whose product with a
  // probability of 0 would be NaN. Whether there was a NaN.
  __device__ __forceinline__ bool cut_values(i32x4 *vc, int valid) const {
    uint32_t nan = 0;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t c = (uint32_t)vc[d][k] & first_bytes(valid - 4 * k), bad = nan_bits(c);
        nan |= bad;
        vc[d][k] = (int)(c & ~((bad >> 7) * 0xffu));
      }
    return __any(nan);
  }

  // The NaNs of an edge step's values count for the rows that see them, and only for those: an
  // output becomes NaN where a product of the NaNs' places with the mask is not 0.
  __device__ __forceinline__ void put_nan(const i32x4 *vc, int key0, int vnow) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      bf16x8 sees[2];
#pragma unroll
      for (int k = 0; k < 16; ++k) sees[k >> 3][k & 7] = (bf16_t)(key0 + k <= lim[nt] && vnow >= 0 ? 1.f : 0.f);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        uint32_t one[4];   // 1.0 (0x38) where the code is NaN
#pragma unroll
        for (int k = 0; k < 4; ++k) one[k] = (nan_bits((uint32_t)vc[d][k]) >> 7) * 0x38u;
        f32x4 hit = {0.f, 0.f, 0.f, 0.f};
        hit = mfma16(decode8(one[0], one[1], 1.f), sees[0], hit);
        hit = mfma16(decode8(one[2], one[3], 1.f), sees[1], hit);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[nt][d][r] = hit[r] > 0.f ? __builtin_nanf("") : o[nt][d][r];
      }
    }
  }

  __device__ __forceinline__ float row_sum(int nt) const {
    float s = l[nt];
    s += __shfl_xor(s, 16, 64);
    return s + __shfl_xor(s, 32, 64);
  }
};

// Rows behind the last sequence.
template <int HD, typename T>
__device__ __forceinline__ void zero_rest(const PagedAttnArgs &a) {
  if (!a.zero_rest) return;
  const int used = min(max(a.cu[a.B], 0), a.T);
  for (int64_t t = used + (int64_t)blockIdx.x; t < a.T; t += gridDim.x)
    for (int i = threadIdx.x * 4; i < a.Hq * HD; i += blockDim.x * 4)
      store4((T *)a.out + t * a.o_ss + (int64_t)(i / HD) * a.o_hs + i % HD, 0.f, 0.f, 0.f, 0.f);
}

// ---- equal shares of all steps, a wave each ----------------------------------------

constexpr int kMinShare = 1;

// Workgroups a CU: what the registers of a wave allow.
constexpr int share_occupancy(int NT, int parts) { return parts == 1 || (NT == 1 && parts == 2) ? 2 : 1; }

// Partial results of a worker's first (0) and last (1) tile: rows of HD values, then (max, sum) pairs.
__host__ __device__ __forceinline__ int64_t slot_floats(int rows, int HD) { return (int64_t)rows * (HD + 2); }

struct JoinNote {   // of a tile: the worker that begins it, how many go through it, the first one's slot
  int worker, n, slot, pad;
};

// Inclusive sums of the sequences' steps (all heads) in LDS; returns the total.
__device__ __forceinline__ int scan_steps(const PagedAttnArgs &a, int tmshift, int32_t *pre, int32_t *wave_sum) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int carry = 0;
  for (int b0 = 0; b0 < a.B; b0 += 256) {
    const int b = b0 + tid;
    int s = 0;
    if (b < a.B) {
      const SeqSpan q = seq_span(a.cu, a.lengths, b, a.T, a.width << a.pshift);
      s = (int)(SeqTiles{q.n, q.len, tmshift}.all() * a.Hkv);
    }
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(s, m, 64);
      s += lane >= m ? o : 0;
    }
    if (lane == 63) wave_sum[w] = s;
    __syncthreads();
    int add = carry;
    for (int i = 0; i < 4; ++i) {
      add += i < w ? wave_sum[i] : 0;
      carry += wave_sum[i];
    }
    if (b < a.B) pre[b] = s + add;
    __syncthreads();
  }
  return carry;
}

// The tile that holds step u, and u's place in it.
__device__ __forceinline__ int locate(const PagedAttnArgs &a, int tmshift, int G, const int32_t *pre, int u, Tile &x) {
  int b = 0;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = i0 + (threadIdx.x & 63);
    b += __popcll(__ballot(i < a.B && pre[min(i, a.B - 1)] <= u));
  }
  x.b = __builtin_amdgcn_readfirstlane(min(b, a.B - 1));
  const int rest = u - (x.b ? __builtin_amdgcn_readfirstlane(pre[x.b - 1]) : 0);
  x.q = seq_span(a.cu, a.lengths, x.b, a.T, a.width << a.pshift);
  const SeqTiles st{x.q.n, x.q.len, tmshift};
  const int each = (int)st.all();
  x.h = rest / each;
  const int in = rest - x.h * each;
  int lo = 0, hi = st.tiles() - 1;
  while (lo < hi) {   // the last tile that begins at or before `in`
    const int mid = (lo + hi + 1) >> 1;
    if (st.before(mid) <= in) lo = mid;
    else hi = mid - 1;
  }
  x.set(st, lo, G);
  return in - (int)st.before(lo);
}

template <int HD, int NT, typename T, bool UNI>
__global__ __launch_bounds__(256, share_occupancy(NT, Parts<T>::n)) void paged_share_kernel(PagedAttnArgs a, int tmshift, int G) {
  constexpr int ND = HD / 16, ROWS = 16 * NT;
  __shared__ int32_t pre[kMaxSeqs];
  __shared__ int32_t wave_sum[4];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int workers = gridDim.x * 4;
  const int me = xcd_swizzle(blockIdx.x, gridDim.x) * 4 + wave_id();
  const int total = scan_steps(a, tmshift, pre, wave_sum);
  const int share = max((total + workers - 1) / workers, kMinShare);
  const int u0 = (int)min((int64_t)me * share, (int64_t)total), u1 = (int)min((int64_t)u0 + share, (int64_t)total);
  JoinNote *notes = reinterpret_cast<JoinNote *>(a.ws + (int64_t)workers * 2 * slot_floats(ROWS, HD));

  for (int u = u0; u < u1;) {
    Tile x;
    const int p0 = locate(a, tmshift, G, pre, u, x), p1 = min(x.steps, p0 + u1 - u);
    const bool whole = p0 == 0 && p1 == x.steps;
    const int slot = 2 * me + (u > u0 ? 1 : 0);
    if (p0 == 0 && lane == 0)
      notes[tile_slot(x.q, x.b, x.t, tmshift) * a.Hkv + x.h] =
          JoinNote{me, whole ? 0 : (u + x.steps - 1) / share - me + 1, slot, 0};
    Steps<HD, NT, T, UNI> st(a, x, G);
    st.run(p0, p1, 1);
    float *pp = a.ws + slot * slot_floats(ROWS, HD);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float sum = st.row_sum(nt);
      const int r = nt * 16 + col;
      if (r < x.rows) {
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no visible key: zeros
          T *op = row_of<T>(x, G, r, a.out, a.o_ss, a.o_hs) + 4 * g;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const f32x4 v = st.o[nt][d] * inv;
            store4(op + 16 * d, v[0], v[1], v[2], v[3]);
          }
        } else {
#pragma unroll
          for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(pp + r * HD + 16 * d + 4 * g) = st.o[nt][d];
          if (g == 0) {
            pp[ROWS * HD + 2 * r] = st.m[nt];
            pp[ROWS * HD + 2 * r + 1] = sum;
          }
        }
      }
    }
    u += p1 - p0;
  }
  zero_rest<HD, T>(a);
}

// The partial results of a tile that more than one worker went through, joined in a fixed
// order: a workgroup a row, its waves a quarter of every 64 parts each.
template <int HD, int NT, typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, int tmshift, int G, int workers) {
  constexpr int ROWS = 16 * NT, C = HD / 64;
  __shared__ float acc4[4][HD];
  const int lane = threadIdx.x & 63, w = wave_id();
  const int slot = blockIdx.x / a.Hkv, h = blockIdx.x - slot * a.Hkv, r = blockIdx.y;
  const JoinNote *notes = reinterpret_cast<const JoinNote *>(a.ws + (int64_t)workers * 2 * slot_floats(ROWS, HD));
  JoinNote n = notes[blockIdx.x];   // of a slot without a tile: anything, and not used
  Tile x;
  x.h = h;
  if (!tile_of_slot(a, slot, tmshift, G, x) || n.n == 0 || r >= x.rows) return;
  auto part = [&](int i) { return a.ws + (int64_t)(i == 0 ? n.slot : 2 * (n.worker + i)) * slot_floats(ROWS, HD); };
  float m = kNegInf;
  for (int i = lane; i < n.n; i += 64) m = fmaxf(m, part(i)[ROWS * HD + 2 * r]);
  for (int k = 32; k; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
  const float off = m == kNegInf ? 0.f : m;
  float l = 0.f, acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  for (int i0 = 0; i0 < n.n; i0 += 64) {
    float f = 0.f;
    if (i0 + lane < n.n) {
      const float *pp = part(i0 + lane) + ROWS * HD + 2 * r;
      f = __builtin_amdgcn_exp2f(pp[0] - off);
      l += f * pp[1];
    }
    const int k1 = min(16 * (w + 1), n.n - i0);
#pragma unroll 8
    for (int k = 16 * w; k < k1; ++k) {
      const float fk = __shfl(f, k, 64);
      const float *pp = part(i0 + k) + r * HD + lane * C;
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] += fk * pp[c];
    }
  }
  for (int k = 32; k; k >>= 1) l += __shfl_xor(l, k, 64);
#pragma unroll
  for (int c = 0; c < C; ++c) acc4[w][lane * C + c] = acc[c];
  __syncthreads();
  const int d = threadIdx.x;
  if (d < HD) {
    const float v = (acc4[0][d] + acc4[1][d]) + (acc4[2][d] + acc4[3][d]);
    row_of<T>(x, G, r, a.out, a.o_ss, a.o_hs)[d] = (T)(l == 0.f ? 0.f : v * (1.f / l));
  }
}

// ---- a workgroup a tile, for short sequences ------------------------------------------

// The waves take every NW-th step and meet in LDS: one launch, no partial results.
template <int HD, int NT, typename T, bool UNI, int NW>
__global__ __launch_bounds__(64 * NW) void paged_tile_kernel(PagedAttnArgs a, int tmshift, int G) {
  constexpr int ND = HD / 16;
  __shared__ float om[NW][16][HD + 4];
  __shared__ float ml[NW][2][16];
  const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), col = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.Hkv;
  Tile x;
  x.h = blockIdx.x - slot * a.Hkv;
  if (tile_of_slot(a, slot, tmshift, G, x)) {
    Steps<HD, NT, T, UNI> st(a, x, G);
    st.run(w, x.steps, NW);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 16 >= x.rows) break;
      const float sum = st.row_sum(nt);
      if (nt) __syncthreads();   // om and ml are free again
      if (g == 0) {
        ml[w][0][col] = st.m[nt];
        ml[w][1][col] = sum;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&om[w][col][16 * d + 4 * g]) = st.o[nt][d];
      __syncthreads();
      // 4 channels a thread
      for (int i = tid; i < 16 * HD / 4; i += 64 * NW) {
        const int r16 = i / (HD / 4), r = nt * 16 + r16, c0 = i % (HD / 4) * 4;
        if (r >= x.rows) break;
        float mt = kNegInf, lt = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) mt = fmaxf(mt, ml[v][0][r16]);
        const float off = mt == kNegInf ? 0.f : mt;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NW; ++v) {
          const float f = __builtin_amdgcn_exp2f(ml[v][0][r16] - off);
          lt += ml[v][1][r16] * f;
          acc += *reinterpret_cast<const f32x4 *>(&om[v][r16][c0]) * f;
        }
        const float inv = lt == 0.f ? 0.f : 1.f / lt;   // no visible key: zeros
        store4(row_of<T>(x, G, r, a.out, a.o_ss, a.o_hs) + c0, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      }
    }
  }
  zero_rest<HD, T>(a);
}

enum Mode { kShares, kTiles };

struct Shape {
  Mode mode;
  int NT, tmshift, nwg;
};

// Keys up to which a sequence is one workgroup's.
constexpr int kShortKeys = 4096;

// The narrowest tile that holds an average sequence's query rows: a wide one's empty
// columns cost matrix work only, a narrow one reads the cache once more a tile.
Shape shape_of(int T, int B, int Hq, int Hkv, int64_t keys, int dtype) {
  const int G = Hq / Hkv;
  const int64_t rows = ((int64_t)T * G + B - 1) / B;
  const int NT = rows <= 16 && G <= 16 ? 1 : 2, parts = dtype == kDtBf16 ? 1 : dtype == kDtF16 ? 2 : 3;
  return {keys <= kShortKeys ? kTiles : kShares, NT, tm_shift(16 * NT, G), share_occupancy(NT, parts) * device_cu_count()};
}

template <int HD, int NT, typename T, bool UNI>
void launch3(const PagedAttnArgs &a, const Shape &s, hipStream_t stream) {
  const int G = a.Hq / a.Hkv, tiles = tile_slots(a.T, a.B, s.tmshift) * a.Hkv;
  if (s.mode == kTiles) {
    constexpr int NW = NT == 1 || Parts<T>::n == 1 ? 8 : 4;   // by the registers of a wave
    paged_tile_kernel<HD, NT, T, UNI, NW><<<tiles, 64 * NW, 0, stream>>>(a, s.tmshift, G);
  } else {
    paged_share_kernel<HD, NT, T, UNI><<<s.nwg, 256, 0, stream>>>(a, s.tmshift, G);
    const int rows = std::min(1 << s.tmshift, a.T) * G;
    paged_join_kernel<HD, NT, T><<<dim3(tiles, rows), 256, 0, stream>>>(a, s.tmshift, G, s.nwg * 4);
  }
}

template <int HD, typename T>
void launch1(const PagedAttnArgs &a, const Shape &s, hipStream_t stream) {
  if (a.pshift >= 6) {
    if (s.NT == 1) launch3<HD, 1, T, true>(a, s, stream);
    else launch3<HD, 2, T, true>(a, s, stream);
  } else {
    if (s.NT == 1) launch3<HD, 1, T, false>(a, s, stream);
    else launch3<HD, 2, T, false>(a, s, stream);
  }
}

}  // namespace

int64_t paged_attn_ws_bytes(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int head_dim, int64_t keys, int dtype) {
  const Shape s = shape_of(T, B, Hq, Hkv, keys, dtype);
  if (s.mode != kShares) return 0;
  return (int64_t)s.nwg * 4 * 2 * slot_floats(16 * s.NT, head_dim) * 4 +
         (int64_t)tile_slots(T, B, s.tmshift) * Hkv * sizeof(JoinNote);
}

int64_t paged_attn_steps(const PagedAttnArgs &a, int dtype) {
  const int64_t keys = (int64_t)a.width << a.pshift;
  const Shape s = shape_of(a.T, a.B, a.Hq, a.Hkv, keys, dtype);
  return (int64_t)tile_slots(a.T, a.B, s.tmshift) * a.Hkv * ((keys + a.T + 63) / 64 + 1);
}

void launch_paged_attn(const PagedAttnArgs &a, int head_dim, int dtype, hipStream_t stream) {
  const Shape s = shape_of(a.T, a.B, a.Hq, a.Hkv, (int64_t)a.width << a.pshift, dtype);
  if (head_dim == 128) {
    if (dtype == kDtBf16) launch1<128, bf16_t>(a, s, stream);
    else if (dtype == kDtF16) launch1<128, f16_t>(a, s, stream);
    else launch1<128, float>(a, s, stream);
  } else {
    if (dtype == kDtBf16) launch1<64, bf16_t>(a, s, stream);
    else if (dtype == kDtF16) launch1<64, f16_t>(a, s, stream);
    else launch1<64, float>(a, s, stream);
  }
}

}  // namespace mga
