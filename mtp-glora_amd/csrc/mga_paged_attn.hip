// Attention of new tokens over a paged 8-bit cache (layout: mga_paged.hpp):
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j,   j <= length + i of i's sequence,
// for a ragged batch of 1 .. thousands of new tokens a sequence.
//
// Work. A tile is up to 16 NT query rows of one sequence and KV head: TM tokens (a
// power of two) times the G query heads of the group. It visits the cache in steps
// of 64 keys. The steps of all tiles, sequences and heads form one list, cut into
// equal shares, one a wave: ragged batches and few long sequences fill the chip
// alike. A tile that a cut goes through leaves fp32 partial results (at most two
// a wave), joined in a fixed order by a second launch. Each workgroup finds its
// shares from the lengths on the device (a scan over the sequences; a tile's place
// within its sequence has a closed form, as TM divides 64), so the launch depends on
// no length and can be captured. The K and V loads run one step ahead and on across
// the tiles of a share.
//
// Bounds and times (32 / 8 heads of 128, bf16, pages of 64). Few rows: HBM. A plain read of as many
// bytes in this pattern reaches 5.85 TB/s here. 64 sequences of 177 385 tokens in all, a token each
// (364 MB): 75 us + 5 us joining, 4.5 TB/s; 2 of 212 590 (435 MB): 81 + 7 us, 4.9 TB/s; what is left is
// the start (cu, lengths, pages, first keys: 4 us), the join's launch, and waves that end up to 15% apart
// with equal shares. Prompts: the matrix unit and the softmax's vector work beside it, and the last tiles, which leave
// a part of the chip idle: 10 075 new tokens behind up to 15 399, 1175 GFLOP visible, 1.24 ms, 945 TFLOP/s,
// in the orders of the same four sequences 1.11 to 1.26 ms.
//
// Three forms share this: few rows a sequence over long ones by equal shares (paged_share_kernel), short
// sequences by a workgroup a tile (paged_tile_kernel), prompts by 128 rows (paged_prompt_kernel, further
// below).
//
// Step. A wave keeps its own running maximum, sum and output. K and V go from
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
// Precision: scores, statistics and outputs in fp32; K and V are exact in bf16. fp16 queries meet the
// codes in fp16, exact too without the scale, which the scores take (16 x 5 tokens over 47 000: 32.8 us,
// by two bf16 parts of the queries 38.3); for prompts they are split into 2 bf16
// parts, fp32 queries into 3. P is held in 2 parts (16 bits; fp32: 3, 24 bits) where the
// cache's bytes bound the kernel and the matrix unit waits for them; a single part's rounding is as
// large as that of the bf16 output. Prompts with bf16 queries are bound by the matrix unit and take one. The row
// sum is of the unrounded P.
//
// Where a value that a row may not see is NaN (a masked place), its products would be
// NaN although p = 0: see put_nan.
#include <algorithm>
#include <type_traits>

#include "mga_internal.hpp"
#include "mga_paged.hpp"

namespace mga {
namespace {

// bf16 parts of the queries (n; fp16's: of prompts), and of the probabilities over a streamed cache (p).
template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int n = 1, p = 2; };
template <> struct Parts<f16_t> { static constexpr int n = 2, p = 2; };
template <> struct Parts<float> { static constexpr int n = 3, p = 3; };

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

// The same without a scale, in fp16 (exact).
__device__ __forceinline__ f16x8 decode8_f16(uint32_t a, uint32_t b) {
  const auto two = [](uint32_t c, auto high) {
    return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, decltype(high)::value));
  };
  const std::false_type lo;
  const std::true_type hi;
  const i32x4 r = {two(a, lo), two(a, hi), two(b, lo), two(b, hi)};
  return __builtin_bit_cast(f16x8, r);
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

// Tokens of a tile: the largest power of two (at most 2^most) of which a tile holds the query heads.
inline int tm_shift(int rows, int G, int most = 6) {
  int s = 0;
  while (((2 << s) * G <= rows) && s < most) ++s;
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

// Tiles are also numbered without sums over the sequences: b owns the slots from (cu[b] >> tmshift) + b
// on, as many as n tokens can make tiles.
__device__ __forceinline__ int tile_slot(const SeqSpan &q, int b, int t, int tmshift) {
  return (q.first >> tmshift) + b + t;
}
__host__ __device__ __forceinline__ int tile_slots(int T, int B, int tmshift) { return (T >> tmshift) + B; }

// The tile of a slot; false: none. All lanes of the wave take part. The lanes' loads find the
// sequence, 64 a turn, and hold what is needed of it. (A token each over 100 keys, 32 / 8 heads of 128: 12.6 us for
// 64 sequences, 95 for 512, 220 for 1024, 1496 for 4096, 760 at the rate of 512.)
__device__ __forceinline__ bool tile_of_slot(const PagedAttnArgs &a, int slot, int tmshift, int G, Tile &x) {
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = min(i0 + (int)(threadIdx.x & 63), a.B - 1);
    const SeqSpan q = seq_span(a.cu, a.lengths, i, a.T, a.width << a.pshift);
    // the sequences whose slots end at or before this one
    const uint64_t done = __ballot((min(max(a.cu[i + 1], 0), a.T) >> tmshift) + i + 1 <= slot);
    if (~done) {
      const int at = __ffsll((unsigned long long)~done) - 1;
      x.b = i0 + at;
      x.q.first = __builtin_amdgcn_readlane(q.first, at);
      x.q.n = __builtin_amdgcn_readlane(q.n, at);
      x.q.len = __builtin_amdgcn_readlane(q.len, at);
      const SeqTiles st{x.q.n, x.q.len, tmshift};
      const int t = slot - tile_slot(x.q, x.b, 0, tmshift);
      if (x.b >= a.B || t < 0 || t >= st.tiles()) return false;
      x.set(st, t, G);
      return true;
    }
  }
  return false;
}

// A row of a tile in q and out.
template <typename T>
__device__ __forceinline__ T *row_of(const Tile &x, int G, int r, const void *base, int64_t ss, int64_t hs) {
  const int tk = r / G;
  return (T *)base + (int64_t)(x.q.first + x.tok0 + tk) * ss + (int64_t)(x.h * G + r - tk * G) * hs;
}

// s_waitcnt's operand: at most n vector memory operations in flight.
constexpr int wait_vm(int n) { return (n & 15) | (n >> 4) << 14 | 7 << 4 | 15 << 8; }

// 16 bytes at a wave-uniform address plus a lane offset; the address stays in scalar registers.
__device__ __forceinline__ i32x4 load16(const uint8_t *base, uint32_t off) {
  typedef const __attribute__((address_space(1))) uint8_t *global_u8;
  typedef const __attribute__((address_space(1))) i32x4 *global_v4;
  global_u8 b = (global_u8)base;
  asm("" : "+s"(b));
  return *(global_v4)(b + off);
}

// ---- the steps of one wave ------------------------------------------------------

// The K and V loads of a wave's steps, whatever tiles they belong to, one step ahead of their
// use. The lanes hold the pages (page * Hkv + head, -1: none), places and scales of the next steps:
// 64 steps of one page each, or 64 / 2^pps of 2^pps pages each.
// UNI: pages of 64 tokens or more, so that a step lies in one page: its id and scales are
// wave-uniform, and the loads take a scalar base with a lane offset that never changes.
// F16: scores take the scales, not keys.
template <int HD, bool UNI, bool F16>
struct Stream {
  static constexpr int ND = HD / 16, KL = HD / 64;
  const PagedAttnArgs &a;
  const int n;   // steps
  const int lane, col, g, kg, PS, pps, hold;
  const uint32_t koff, voff;
  int tph = -1, tp = 0;
  float tks = 0.f, tvs = 0.f;
  i32x4 kc[4][KL], vc[ND];   // 16 channels of keys 16 kg + 4 t + col % 4; 16 keys of channels 16 d + col
  float ksc = 0.f, vsc = 0.f;
  int vph = -1;

  __device__ __forceinline__ Stream(const PagedAttnArgs &a_, int n_)
      : a(a_), n(n_), lane(threadIdx.x & 63), col(lane & 15), g(lane >> 4), kg(col >> 2), PS(1 << a_.pshift),
        pps(UNI ? 0 : 6 - a_.pshift), hold(64 >> pps), koff((16 * kg + (col & 3)) * HD + 16 * g),
        voff(col * PS + 16 * g) {}

  // step p of sequence b and head h: the page of this lane's part of it; none past the sequence's end,
  // where the table may name one that was never written
  __device__ __forceinline__ int page_of(int b, int h, int p, int end) const {
    const int at = UNI ? p >> (a.pshift - 6) : (p << pps) + (lane & ((1 << pps) - 1));
    const int id = a.table[(int64_t)b * a.table_rs + min(at, a.width - 1)];
    const bool there = at < a.width && (UNI || at << a.pshift < end);
    return there && (uint32_t)id < (uint32_t)a.num_pages ? id * a.Hkv + h : -1;
  }
  __device__ __forceinline__ void scales() {
    tks = a.ks[max(tph, 0)];
    tvs = a.vs[max(tph, 0)];
  }
  // what lane group `grp` needs of a held value at step i
  template <typename V>
  __device__ __forceinline__ V held(V v, int i, int grp) const {
    if constexpr (UNI)
      return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i & 63));
    else
      return __shfl(v, ((i & (hold - 1)) << pps) + (grp >> (2 - pps)), 64);
  }
  // of step i's values, whose page vph is; where there is none, 1: zeros under any scale could be NaN
  __device__ __forceinline__ float v_scale(int i) const {
    const float s = held(tvs, i, g);
    return vph < 0 ? 1.f : s;
  }
  // a held value that a step's lanes share
  __device__ __forceinline__ int step_of(int v, int i) const {
    return __builtin_amdgcn_readlane(v, (i & (hold - 1)) << pps);
  }
  // Step i's loads. Past the last step they still issue (a branch around them would make the
  // compiler wait for all loads where its paths meet), for a few bytes of page 0.
  __device__ __forceinline__ void load_k(int i) {
    const int64_t ph = max(held(tph, i, kg), 0);
    if constexpr (UNI) {
      const uint8_t *base = a.kp + (ph * PS + ((step_of(tp, i) * 64) & (PS - 1))) * HD;
      const uint32_t off = i < n ? koff : 0;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < KL; ++j) kc[t][j] = load16(base + (4 * t * HD + 64 * j), off);
    } else {
      const uint8_t *base = a.kp + (ph * PS + ((16 * kg) & (PS - 1)) + (col & 3)) * HD + 16 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < KL; ++j) kc[t][j] = *reinterpret_cast<const i32x4 *>(base + 4 * t * HD + 64 * j);
    }
    __builtin_amdgcn_sched_barrier(0);   // keys before values, here and in the loop
  }
  __device__ __forceinline__ void load_v(int i) {
    vph = held(tph, i, g);
    const int64_t ph = max(vph, 0);
    if constexpr (UNI) {
      const uint8_t *base = a.vp + ph * HD * PS + ((step_of(tp, i) * 64) & (PS - 1));
      const uint32_t off = i < n ? voff : 0;
#pragma unroll
      for (int d = 0; d < ND; ++d) vc[d] = load16(base + 16 * d * PS, off);
    } else {
      const uint8_t *base = a.vp + (ph * HD + col) * PS + ((16 * g) & (PS - 1));
#pragma unroll
      for (int d = 0; d < ND; ++d) vc[d] = *reinterpret_cast<const i32x4 *>(base + 16 * d * PS);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  // find(lane's step, tp) -> tph, for the steps from i0 on
  template <typename F>
  __device__ __forceinline__ void find_steps(int i0, F find) {
    const int i = i0 + (lane >> pps);
    tph = -1;
    if (i < n) tph = find(i, tp);
  }
  template <typename F>
  __device__ __forceinline__ void start(F find) {
    find_steps(0, find);
    scales();
    load_k(0);
    load_v(0);
    __builtin_amdgcn_s_waitcnt(wait_vm(4 * KL + ND));   // the scales
    ksc = held(tks, 0, F16 ? g : kg);   // of the keys that a lane converts, or has scores of
    vsc = v_scale(0);
  }
  template <typename F>
  __device__ __forceinline__ void next_k(int i, F find) {
    if ((i & (hold - 1)) == 0 && i < n) {
      find_steps(i, find);
      scales();
      // wait here, once for all these steps: left to the reads of a lane, the wait would be in
      // every step and drain the tiles in flight
      __builtin_amdgcn_s_waitcnt(wait_vm(0));
    }
    load_k(i);
    ksc = held(tks, i, F16 ? g : kg);
  }
  __device__ __forceinline__ void next_v(int i) {
    load_v(i);
    vsc = v_scale(i);
  }
};

// One tile's queries and results.
template <int HD, int NT, typename T, bool UNI>
struct Rows {
  // fp16 queries meet the codes in fp16 and the scale in the scores
  static constexpr bool F16 = std::is_same<T, f16_t>::value;
  static constexpr int NQ = F16 ? 1 : Parts<T>::n, NP = Parts<T>::p, KS = HD / 32, ND = HD / 16;
  const PagedAttnArgs &a;
  const Tile &x;
  const int col, g;
  bf16x8 qf[NT][NQ][KS];
  int lim[NT];          // each row's last key
  f32x4 o[NT][ND];
  float m[NT], l[NT];   // l: this lane's part of the row sum
  int nan_from;         // the first edge step with a NaN among its values

  __device__ __forceinline__ Rows(const PagedAttnArgs &a_, const Tile &x_, int G)
      : a(a_), x(x_), col(threadIdx.x & 15), g((threadIdx.x & 63) >> 4), nan_from(x_.steps) {
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
            const f32x4 e = *reinterpret_cast<const f32x4 *>(qp + c), f = *reinterpret_cast<const f32x4 *>(qp + c + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = e[i], v[i + 4] = f[i];
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

  // Step p of the tile, the stream's step i; the stream's loads go on to its next one.
  template <typename F>
  __device__ __forceinline__ void step(Stream<HD, UNI, F16> &st, int i, int p, F find) {
    f32x4 s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int t = 0; t < 4; ++t) s[nt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // four independent sums a turn; the fences keep the compiler from converting the whole step
    // first, which would take 64 registers each for K and V
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const i32x4 c = st.kc[t][ks >> 1];
        const uint32_t c0 = c[2 * (ks & 1)], c1 = c[2 * (ks & 1) + 1];
        if constexpr (F16) {
          const f16x8 kf = decode8_f16(c0, c1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            s[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, __builtin_bit_cast(f16x8, qf[nt][0][ks]), s[nt][t], 0, 0, 0);
        } else {
          const bf16x8 kf = decode8(c0, c1, st.ksc);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < NQ; ++q) s[nt][t] = mfma16(kf, qf[nt][q][ks], s[nt][t]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (F16) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[nt][t] *= st.ksc;
    }
    st.next_k(i + 1, find);

    // this lane's keys: key0 + 4 t + r
    const int key0 = p * 64 + 16 * g;
    const bool edge = p * 64 + 63 > x.q.len + x.tok0 || (UNI ? st.vph < 0 : (bool)__any(st.vph < 0));
    bf16x8 pf[NT][NP][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (edge) {
        const int last = st.vph < 0 ? -1 : lim[nt];
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
        bf16x8 part[NP];
        split8<NP>(e + 8 * c, part);
#pragma unroll
        for (int q = 0; q < NP; ++q) pf[nt][q][c] = part[q];
      }
    }

    if (edge && cut_values(st.vc, st.vph < 0 ? 0 : x.q.len + x.q.n - key0)) nan_from = min(nan_from, p);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const bf16x8 vf = decode8(st.vc[d][2 * c], st.vc[d][2 * c + 1], st.vsc);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < NP; ++q) o[nt][d] = mfma16(vf, pf[nt][q][c], o[nt][d]);
        if (d % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    st.next_v(i + 1);
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

  // The NaNs taken out of the edge steps below p1 count for the rows that see them, and only for
  // those: an output becomes NaN where a product of the NaNs' places with the mask is not 0. Rare; the
  // values are read again.
  __device__ __forceinline__ void put_nan(const Stream<HD, UNI, F16> &st, int p1, int stride) {
    for (int p = nan_from; p < p1; p += stride) {
      const int key0 = p * 64 + 16 * g, at = key0 >> a.pshift;
      const int id = at < a.width ? a.table[(int64_t)x.b * a.table_rs + at] : -1;
      const bool there = (uint32_t)id < (uint32_t)a.num_pages;
      if (p * 64 + 63 <= x.q.len + x.tok0 && !__any(!there)) continue;
      const uint8_t *base =
          a.vp + (((int64_t)(there ? id : 0) * a.Hkv + x.h) * HD + col) * st.PS + (key0 & (st.PS - 1));
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const i32x4 c = *reinterpret_cast<const i32x4 *>(base + 16 * d * st.PS);
        uint32_t one[4];   // 1.0 (0x38) where the code is NaN
#pragma unroll
        for (int k = 0; k < 4; ++k)
          one[k] = (nan_bits((uint32_t)c[k] & first_bytes(x.q.len + x.q.n - key0 - 4 * k)) >> 7) * 0x38u;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          bf16x8 sees[2];
#pragma unroll
          for (int k = 0; k < 16; ++k) sees[k >> 3][k & 7] = (bf16_t)(key0 + k <= lim[nt] && there ? 1.f : 0.f);
          f32x4 hit = {0.f, 0.f, 0.f, 0.f};
          hit = mfma16(decode8(one[0], one[1], 1.f), sees[0], hit);
          hit = mfma16(decode8(one[2], one[3], 1.f), sees[1], hit);
#pragma unroll
          for (int r = 0; r < 4; ++r) o[nt][d][r] = hit[r] > 0.f ? __builtin_nanf("") : o[nt][d][r];
        }
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

// Workgroups a CU: what the registers of a wave allow (2 x 5 tokens over 220 000, 32 / 8 heads of 64, bf16: one 65
// us, two 55; heads of 128 by two would spill: 33 and 44 us for 16 x 5 tokens over 47 000).
constexpr int share_occupancy(int HD, int NT, int parts) { return (NT == 1 || HD == 64) && parts < 3 ? 2 : 1; }

// Partial results of a worker's first (0) and last (1) tile: rows of HD values, then (max, sum) pairs.
__host__ __device__ __forceinline__ int64_t slot_floats(int rows, int HD) { return (int64_t)rows * (HD + 2); }

struct JoinNote {   // of a tile: the workers that begin and end it, the first one's slot
  int first, last, slot, pad;
};

// Where worker me's share begins: shares differ by one step at most and none is empty. (A CU serves
// its older workgroup first, which ends in 5/6 of the other's time; shares of 11 : 9 for the two were
// within 2% either way.)
__device__ __forceinline__ int share_begin(int me, int workers, int total) {
  const int w = min(workers, total);
  return me >= w ? total : (int)((int64_t)me * total / w);
}

// Most steps of a call. The sums stop there, so that they do not wrap for a cu_tokens that goes
// down, whose sequences overlap.
constexpr int kMaxSteps = 1 << 30;

// Inclusive sums of the sequences' steps (all heads) and the sequences themselves in LDS;
// returns the total.
__device__ __forceinline__ int scan_steps(const PagedAttnArgs &a, int tmshift, int32_t *pre, SeqSpan *seqs,
                                          int32_t *wave_sum) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int carry = 0;
  for (int b0 = 0; b0 < a.B; b0 += 256) {
    const int b = b0 + tid;
    int s = 0;
    if (b < a.B) {
      const SeqSpan q = seq_span(a.cu, a.lengths, b, a.T, a.width << a.pshift);
      s = (int)min(SeqTiles{q.n, q.len, tmshift}.all() * a.Hkv, (int64_t)kMaxSteps);
      seqs[b] = q;
    }
    for (int m = 1; m < 64; m <<= 1) {
      const int o = __shfl_up(s, m, 64);
      s = min(s + (lane >= m ? o : 0), kMaxSteps);
    }
    if (lane == 63) wave_sum[w] = s;
    __syncthreads();
    int add = carry;
    for (int i = 0; i < 4; ++i) {
      add = min(add + (i < w ? wave_sum[i] : 0), kMaxSteps);
      carry = min(carry + wave_sum[i], kMaxSteps);
    }
    if (b < a.B) pre[b] = min(s + add, kMaxSteps);
    __syncthreads();
  }
  return carry;
}

// The tile that holds step u (u differs from lane to lane) and u's place in it.
struct Place {
  int b, h, t, p;
};
__device__ __forceinline__ Place locate(const PagedAttnArgs &a, int tmshift, const int32_t *pre, const SeqSpan *seqs,
                                        int u) {
  Place r;
  int lo = 0, hi = a.B - 1;
  while (lo < hi) {   // the first sequence that ends behind u
    const int mid = (lo + hi) >> 1;
    if (pre[mid] > u) hi = mid;
    else lo = mid + 1;
  }
  r.b = lo;
  const SeqSpan q = seqs[lo];
  const SeqTiles st{q.n, q.len, tmshift};
  const int rest = u - (lo ? pre[lo - 1] : 0), each = max((int)st.all(), 1);
  r.h = rest / each;
  const int in = rest - r.h * each;
  lo = 0;
  hi = st.tiles() - 1;
  while (lo < hi) {   // the last tile that begins at or before `in`
    const int mid = (lo + hi + 1) >> 1;
    if (st.before(mid) <= in) lo = mid;
    else hi = mid - 1;
  }
  r.t = lo;
  r.p = in - (int)st.before(lo);
  return r;
}

template <int HD, int NT, typename T, bool UNI>
__global__ __launch_bounds__(256, share_occupancy(HD, NT, Parts<T>::n)) void paged_share_kernel(PagedAttnArgs a, int tmshift,
                                                                                            int G) {
  constexpr int ND = HD / 16, ROWS = 16 * NT;
  __shared__ int32_t pre[kMaxSeqs];
  __shared__ SeqSpan seqs[kMaxSeqs];
  __shared__ int32_t wave_sum[4];
  const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
  const int workers = gridDim.x * 4;
  const int me = xcd_swizzle(blockIdx.x, gridDim.x) * 4 + wave_id();
  const int total = scan_steps(a, tmshift, pre, seqs, wave_sum);
  const int u0 = share_begin(me, workers, total), u1 = share_begin(me + 1, workers, total);
  JoinNote *notes = reinterpret_cast<JoinNote *>(a.ws + (int64_t)workers * 2 * slot_floats(ROWS, HD));

  if (u0 < u1) {
    Stream<HD, UNI, std::is_same<T, f16_t>::value> st(a, u1 - u0);
    int tb = 0, th = 0, tt = 0;   // a lane holds the tile of its step, too
    auto find = [&](int i, int &p) {
      const Place pl = locate(a, tmshift, pre, seqs, u0 + i);
      tb = pl.b;
      th = pl.h;
      tt = pl.t;
      p = pl.p;
      return st.page_of(pl.b, pl.h, pl.p, seqs[pl.b].len + seqs[pl.b].n);
    };
    st.start(find);
    int nb = st.step_of(tb, 0), nh = st.step_of(th, 0), nt_ = st.step_of(tt, 0), np = st.step_of(st.tp, 0);
    for (int i = 0; i < st.n;) {
      Tile x;
      x.b = nb;
      x.h = nh;
      x.q.first = __builtin_amdgcn_readfirstlane(seqs[nb].first);
      x.q.n = __builtin_amdgcn_readfirstlane(seqs[nb].n);
      x.q.len = __builtin_amdgcn_readfirstlane(seqs[nb].len);
      x.set(SeqTiles{x.q.n, x.q.len, tmshift}, nt_, G);
      const int p0 = np, p1 = min(x.steps, p0 + st.n - i), slot = 2 * me + (i > 0 ? 1 : 0);
      const bool whole = p0 == 0 && p1 == x.steps;
      JoinNote &note = notes[tile_slot(x.q, x.b, x.t, tmshift) * a.Hkv + x.h];
      if (st.lane == 0) {
        if (p0 == 0) note.first = me, note.slot = slot;
        if (p1 == x.steps) note.last = me;
      }
      Rows<HD, NT, T, UNI> rows(a, x, G);
      // here for the queries and all before them: left to their first use, the wait would be in every step and
      // drain the values in flight (64 tokens over 177 385: 80.6 us, 82.2 without). With one wave a SIMD, which
      // its own instructions bound, it takes 114 us without and 119 with it (64 x 5 tokens over 197 000)
      if constexpr (share_occupancy(HD, NT, Parts<T>::n) == 2) __builtin_amdgcn_s_waitcnt(wait_vm(0));
      for (int p = p0; p < p1; ++p, ++i) rows.step(st, i, p, find);
      // the next tile, whose first step's page is held by now
      nb = st.step_of(tb, i);
      nh = st.step_of(th, i);
      nt_ = st.step_of(tt, i);
      np = st.step_of(st.tp, i);
      if (rows.nan_from < p1) rows.put_nan(st, p1, 1);
      float *pp = a.ws + slot * slot_floats(ROWS, HD);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float sum = rows.row_sum(nt);
        const int r = nt * 16 + col;
        if (r < x.rows) {
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no visible key: zeros
            T *op = row_of<T>(x, G, r, a.out, a.o_ss, a.o_hs) + 4 * g;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              const f32x4 v = rows.o[nt][d] * inv;
              store4(op + 16 * d, v[0], v[1], v[2], v[3]);
            }
          } else {
#pragma unroll
            for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(pp + r * HD + 16 * d + 4 * g) = rows.o[nt][d];
            if (g == 0) {
              pp[ROWS * HD + 2 * r] = rows.m[nt];
              pp[ROWS * HD + 2 * r + 1] = sum;
            }
          }
        }
      }
    }
  }
  zero_rest<HD, T>(a);
}

// The partial results of the tiles that more than one worker went through, joined in a fixed order.
// WPR waves take a row's parts, groups of HD / 4 lanes a part each (4 channels a lane), U of them in
// flight before their maximum is known: 1 where there are rows enough to fill the chip, else 4.
template <int HD, int NT, typename T, int WPR>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, int tmshift, int G, int workers) {
  constexpr int ROWS = 16 * NT, TPP = HD / 4, PG = 64 / TPP, U = 8;
  __shared__ f32x4 accs[4][64];
  const int lane = threadIdx.x & 63, w = wave_id(), sub = w % WPR, pg = sub * PG + lane / TPP, c = lane % TPP;
  const int slot = blockIdx.x / a.Hkv;
  const JoinNote *notes = reinterpret_cast<const JoinNote *>(a.ws + (int64_t)workers * 2 * slot_floats(ROWS, HD));
  JoinNote n = notes[blockIdx.x];   // of a slot without a tile: anything, and not used
  // so are parts of the notes where sequences of a cu_tokens that goes down overlap until the steps end at
  // kMaxSteps: tiles behind that have no worker. Whatever they say stays among the workers' partial results
  n.first = min(max(n.first, 0), workers - 1);
  n.last = min(max(n.last, n.first), workers - 1);
  n.slot = min(max(n.slot, 0), 2 * workers - 1);
  Tile x;
  x.h = blockIdx.x - slot * a.Hkv;
  if (!tile_of_slot(a, slot, tmshift, G, x) || n.first == n.last) return;
  const int parts = n.last - n.first + 1;
  auto part = [&](int i) { return a.ws + (int64_t)(i == 0 ? n.slot : 2 * (n.first + i)) * slot_floats(ROWS, HD); };
  for (int r0 = blockIdx.y * (4 / WPR); r0 < x.rows; r0 += gridDim.y * (4 / WPR)) {
    const int r = min(r0 + w / WPR, x.rows - 1);   // past the last row: the same once more, not stored
    float m = kNegInf, l = 0.f;   // l: of this lane's parts
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < parts; i0 += 64) {
      const int k = min(64, parts - i0);
      float pm = kNegInf, pl = 0.f;
      if (lane < k) {
        const float *pp = part(i0 + lane) + ROWS * HD + 2 * r;
        pm = pp[0];
        pl = pp[1];
      }
      f32x4 v[U];
      auto load = [&](int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          v[u] = *reinterpret_cast<const f32x4 *>(part(i0 + min(j0 + u * PG * WPR + pg, k - 1)) + r * HD + 4 * c);
      };
      load(0);
      float mx = pm;
      for (int s = 32; s; s >>= 1) mx = fmaxf(mx, __shfl_xor(mx, s, 64));
      const float now = fmaxf(m, mx), off = now == kNegInf ? 0.f : now, alpha = __builtin_amdgcn_exp2f(m - off);
      const float f = __builtin_amdgcn_exp2f(pm - off);
      l = l * alpha + pl * f;
      acc *= alpha;
      m = now;
      for (int j0 = 0; j0 < k; j0 += U * PG * WPR) {
        if (j0) load(j0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = j0 + u * PG * WPR + pg;
          const float fj = __shfl(f, min(j, 63), 64);
          acc += v[u] * (j < k ? fj : 0.f);
        }
      }
    }
    for (int s = 32; s; s >>= 1) l += __shfl_xor(l, s, 64);
    // the groups of the row's waves
    accs[w][lane] = acc;
    __syncthreads();
    if (sub == 0 && lane < TPP && r0 + w / WPR < x.rows) {
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < WPR; ++v)
#pragma unroll
        for (int i = 0; i < PG; ++i) sum += accs[w + v][i * TPP + lane];
      const float inv = l == 0.f ? 0.f : 1.f / l;   // no visible key: zeros
      store4(row_of<T>(x, G, r, a.out, a.o_ss, a.o_hs) + 4 * lane, sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
    }
    __syncthreads();
  }
}

// ---- a workgroup a tile, for short sequences ------------------------------------------

// The waves take every NW-th step and meet in LDS: one launch, no partial results.
template <int HD, int NT, typename T, bool UNI, int NW>
__global__ __launch_bounds__(64 * NW) void paged_tile_kernel(PagedAttnArgs a, int tmshift, int G) {
  constexpr int ND = HD / 16;
  __shared__ __attribute__((aligned(16))) float om[NW][16][HD + 4];
  __shared__ float ml[NW][2][16];
  const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), col = lane & 15, g = lane >> 4;
  const int slot = blockIdx.x / a.Hkv;
  Tile x;
  x.h = blockIdx.x - slot * a.Hkv;
  if (tile_of_slot(a, slot, tmshift, G, x)) {
    Rows<HD, NT, T, UNI> rows(a, x, G);
    Stream<HD, UNI, std::is_same<T, f16_t>::value> st(a, (x.steps - w + NW - 1) / NW);   // 0 or less: none
    if (st.n > 0) {
      auto find = [&](int i, int &p) {
        p = w + i * NW;
        return st.page_of(x.b, x.h, p, x.q.len + x.q.n);
      };
      st.start(find);
      for (int i = 0; i < st.n; ++i) rows.step(st, i, w + i * NW, find);
      if (rows.nan_from < x.steps) rows.put_nan(st, x.steps, NW);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 16 >= x.rows) break;
      const float sum = rows.row_sum(nt);
      if (nt) __syncthreads();   // om and ml are free again
      if (g == 0) {
        ml[w][0][col] = rows.m[nt];
        ml[w][1][col] = sum;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&om[w][col][16 * d + 4 * g]) = rows.o[nt][d];
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

// ---- prompts: 128 query rows a workgroup ----------------------------------------------

// Four waves of 32 rows share the keys and values, which are converted once for all of them: step
// j + 1's codes go from registers to bf16 tiles in LDS (rows XOR-swizzled, mga_common.hpp) and step
// j + 2's are loaded while step j is computed, one barrier a step. S^T = K Q^T and O^T += V^T P^T by
// v_mfma_f32_32x32x16_bf16; key m of a 32-key tile is read from row 16 (m / 16) + 8 (m / 4 % 2)
// + 4 (m / 8 % 2) + m % 4, so that a lane's scores are those of 8 consecutive keys twice and meet V rows of 16
// bytes as they lie. Bounded by the matrix unit and the softmax's vector work beside it.
constexpr int kPromptRows = 128;

template <int HD, typename T, bool UNI>
__global__ __launch_bounds__(256, Parts<T>::n == 1 ? 2 : 1) void paged_prompt_kernel(PagedAttnArgs a, int tmshift, int G,
                                                                                     int slots) {
  constexpr int NQ = Parts<T>::n, KS = HD / 16, DT = HD / 32;
  constexpr int NL = HD / 64;            // 16-byte loads a thread and step, for keys and for values
  constexpr int VR = 256 / HD;           // threads a value row
  __shared__ __attribute__((aligned(16))) bf16_t kt[2][64 * HD];
  __shared__ __attribute__((aligned(16))) bf16_t vt[2][HD * 64];
  __shared__ __attribute__((aligned(16))) int there[2][4];   // whether a 16-key group has a page
  __shared__ int nan_step;               // the first edge step with a NaN among its values
  const int tid = threadIdx.x, lane = tid & 63, w = wave_id(), l32 = lane & 31, hi = lane >> 5;
  const int PS = 1 << a.pshift;
  Tile x;
  x.h = blockIdx.x % a.Hkv;
  const int slot = slots - 1 - (int)blockIdx.x / a.Hkv;   // the last sequence first, of each its longest tiles
  if (tile_of_slot(a, slot, tmshift, G, x)) {
    const int row = w * 32 + l32, first_lim = x.q.len + x.tok0, end_key = x.q.len + x.q.n;
    const int lim = row < x.rows ? first_lim + row / G : -1;
    // of the wave's rows: the last key of the first and of the last one
    const int wave_first = w * 32 < x.rows ? first_lim + w * 32 / G : -1;
    const int wave_last = w * 32 < x.rows ? first_lim + min(w * 32 + 31, x.rows - 1) / G : -1;
    bf16x8 qf[NQ][KS];
    {
      const T *qp = row_of<const T>(x, G, row, a.q, a.q_ss, a.q_hs);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * hi;
        if constexpr (NQ == 1) {
          qf[0][ks] = row < x.rows ? load8(qp + c) : bf16x8{};
        } else {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
          if (row < x.rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (float)qp[c + i];
          }
          bf16x8 part[NQ];
          split8<NQ>(v, part);
#pragma unroll
          for (int n = 0; n < NQ; ++n) qf[n][ks] = part[n];
        }
      }
    }
    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = zero16();
    float m = kNegInf, l = 0.f;

    // this thread's part of a step: NL * 16 bytes of key row kr, and of value row vr; every other row
    // (pair of rows) takes its two in the other order, so that a write's lanes meet in no bank
    const int kr = tid >> 2, vr = tid / VR;
    int kat[NL], vat[NL];   // 16-byte pieces of a row
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      kat[i] = (tid & 3) * NL + (NL == 2 ? i ^ (kr & 1) : i);
      vat[i] = tid % VR * NL + (NL == 2 ? i ^ (vr >> 1 & 1) : i);
    }
    const int32_t *trow = a.table + (int64_t)x.b * a.table_rs;
    auto checked = [&](int id, int key) {
      return (uint32_t)id < (uint32_t)a.num_pages && (key >> a.pshift) < a.width && key < end_key ? id * a.Hkv + x.h : -1;
    };
    // UNI: the lanes hold the pages (page * Hkv + head, -1: none) and scales of 64 steps; else each
    // thread its own pages of the step after the one in registers, not checked yet
    int tph = -1, kid = 0, vid[NL];
    float tks = 0.f, tvs = 0.f;
    auto ids = [&](int p) {
      if constexpr (UNI) {
        if (p & 63) return;
        const int key = (p + lane) * 64;
        tph = checked(trow[min(key >> a.pshift, a.width - 1)], key);
        tks = a.ks[max(tph, 0)];
        tvs = a.vs[max(tph, 0)];
        __builtin_amdgcn_s_waitcnt(wait_vm(0));   // once in 64 steps, see Stream
        tvs = tph < 0 ? 1.f : tvs;                // likewise
      } else {
        kid = trow[min((p * 64 + kr) >> a.pshift, a.width - 1)];
#pragma unroll
        for (int i = 0; i < NL; ++i) vid[i] = trow[min((p * 64 + 16 * vat[i]) >> a.pshift, a.width - 1)];
      }
    };
    uint32_t klo[NL], vlo[NL];   // UNI: this thread's pieces within a page
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      klo[i] = kr * HD + 16 * kat[i];
      vlo[i] = (vr << a.pshift) + 16 * vat[i];
    }
    i32x4 kc[NL], vc[NL];
    float ksc, vsc[NL];
    int kph, vph[NL];
    auto load = [&](int p) {
      if constexpr (UNI) {
        kph = __builtin_amdgcn_readlane(tph, p & 63);
        const int64_t ph = max(kph, 0);
        const int in = (p * 64) & (PS - 1);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          kc[i] = load16(a.kp + ((ph << a.pshift) + in) * HD, klo[i]);
          vc[i] = load16(a.vp + (ph * HD << a.pshift) + in, vlo[i]);
          vph[i] = kph;
          vsc[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, tvs), p & 63));
        }
        ksc = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, tks), p & 63));
      } else {
        kph = checked(kid, p * 64 + kr);
        const uint8_t *kb = a.kp + (((int64_t)max(kph, 0) << a.pshift) + ((p * 64 + kr) & (PS - 1))) * HD;
#pragma unroll
        for (int i = 0; i < NL; ++i) kc[i] = *reinterpret_cast<const i32x4 *>(kb + 16 * kat[i]);
        ksc = a.ks[max(kph, 0)];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int key = p * 64 + 16 * vat[i];
          vph[i] = checked(vid[i], key);
          vc[i] = *reinterpret_cast<const i32x4 *>(
              a.vp + (((int64_t)max(vph[i], 0) * HD + vr) << a.pshift) + (key & (PS - 1)));
          vsc[i] = a.vs[max(vph[i], 0)];   // of no page: see put
        }
      }
    };
    // lane offsets in the tiles, bytes: formed once
    uint32_t kw[NL], vw[NL], ko[KS], vo[4];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      kw[i] = opaque_u32(2u * tile_off<HD>(kr, 2 * kat[i]));
      vw[i] = opaque_u32(2u * tile_off<64>(vr, 2 * vat[i]));
    }
    const int pm = (l32 & 16) + ((l32 & 4) << 1) + ((l32 & 8) >> 1) + (l32 & 3);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ko[ks] = opaque_u32(2u * tile_off<HD>(pm, 2 * ks + hi));
#pragma unroll
    for (int u = 0; u < 4; ++u) vo[u] = opaque_u32(2u * tile_off<64>(l32, 2 * u + hi));
    auto at = [](const bf16_t *tile, uint32_t off) {
      return reinterpret_cast<bf16x8 *>(const_cast<char *>(lds_at(tile, off)));
    };
    // the step in registers to LDS, converted
    auto put = [&](int p, int buf) {
      if ((tid & 63) == 0) there[buf][kr >> 4] = kph >= 0;
      // a piece's second 8 codes: the neighbouring granule
#pragma unroll
      for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) *at(kt[buf], kw[i] ^ 16 * k) = decode8(kc[i][2 * k], kc[i][2 * k + 1], ksc);
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if (p * 64 + 63 > first_lim || vph[i] < 0) {   // zeros for what is not there, and for NaN (put back at the end)
          const int valid = vph[i] < 0 ? 0 : end_key - (p * 64 + 16 * vat[i]);
          uint32_t nan = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t c = (uint32_t)vc[i][k] & first_bytes(valid - 4 * k), bad = nan_bits(c);
            nan |= bad;
            vc[i][k] = (int)(c & ~((bad >> 7) * 0xffu));
          }
          if (nan) atomicMin(&nan_step, p);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *at(vt[buf], vw[i] ^ 16 * k) = decode8(vc[i][2 * k], vc[i][2 * k + 1], UNI || vph[i] >= 0 ? vsc[i] : 1.f);
      }
    };

    if (tid == 0) nan_step = x.steps;
    ids(0);
    load(0);
    ids(1);
    __syncthreads();
    put(0, 0);
    load(1);
    ids(2);
    __syncthreads();
    // one step out of buffer BUF (a constant: the tiles' addresses are lane offsets plus immediates)
    auto turn = [&](int p, auto which) {
      constexpr int buf = decltype(which)::value;
      if (p + 1 < x.steps) put(p + 1, buf ^ 1);
      load(p + 2);   // past the last step: some page's, not used
      ids(p + 3);
      if (p * 64 <= wave_last) {
        f32x16 s[2] = {zero16(), zero16()};
        // the products first: a SIMD's other wave fills what they leave with its softmax (5%)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const bf16x8 kf = *at(kt[buf] + 32 * t * HD, ko[ks]);
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[t] = mfma32<bf16_t>(kf, qf[n][ks], s[t]);
          }
        __builtin_amdgcn_s_setprio(0);
        const i32x4 have = *reinterpret_cast<const i32x4 *>(there[buf]);
        const bool all = have[0] && have[1] && have[2] && have[3];
        if (p * 64 + 63 > wave_first || !all) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int key = p * 64 + 32 * t + 16 * (r >> 3) + 8 * hi + (r & 7);
              s[t][r] = key <= lim && have[2 * t + (r >> 3)] ? s[t][r] : kNegInf;
            }
        }
        float e[32], sum = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          e[k] = __builtin_amdgcn_exp2f(fmaf(s[k >> 4][k & 15], a.scale_log2, -m));
          sum += e[k];
        }
        if (__any(!(sum <= 0x1p20f))) {
          float mx = kNegInf;
#pragma unroll
          for (int k = 0; k < 32; ++k) mx = fmaxf(mx, s[k >> 4][k & 15]);
          mx = fmaxf(mx, xor32(mx));
          const float now = fmaxf(m, mx * a.scale_log2);
          const float off = now == kNegInf ? 0.f : now;
          const float alpha = __builtin_amdgcn_exp2f(m - off);   // 0 from -inf
          l *= alpha;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] *= alpha;
          m = now;
          sum = 0.f;
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            e[k] = __builtin_amdgcn_exp2f(fmaf(s[k >> 4][k & 15], a.scale_log2, -off));
            sum += e[k];
          }
        }
        l += sum;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          bf16x8 pf[NQ];
          split8<NQ>(e + 8 * u, pf);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            const bf16x8 vf = *at(vt[buf] + 32 * d * 64, vo[u]);
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[d] = mfma32<bf16_t>(vf, pf[n], o[d]);
          }
        }
        __builtin_amdgcn_s_setprio(0);
      }
      __syncthreads();
    };
    for (int p = 0; p < x.steps; p += 2) {
      turn(p, std::integral_constant<int, 0>{});
      if (p + 1 < x.steps) turn(p + 1, std::integral_constant<int, 1>{});
    }

    // NaNs taken out of the edge steps: for the rows that see them (see put_nan)
    for (int p = nan_step; p < x.steps; ++p)
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {
        const int key = p * 64 + 16 * u + 8 * hi;
        const int ph = checked(trow[min(key >> a.pshift, a.width - 1)], key);
        bf16x8 sees;
#pragma unroll
        for (int k = 0; k < 8; ++k) sees[k] = (bf16_t)(key + k <= lim && ph >= 0 ? 1.f : 0.f);
        const uint8_t *vb = a.vp + ((int64_t)max(ph, 0) * HD << a.pshift) + (key & (PS - 1));
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const i32x2 c = *reinterpret_cast<const i32x2 *>(vb + (32 * d + l32) * PS);
          uint32_t one[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            one[k] = (nan_bits((uint32_t)c[k] & first_bytes(end_key - key - 4 * k)) >> 7) * 0x38u;
          const f32x16 hit = mfma32<bf16_t>(decode8(one[0], one[1], 1.f), sees, zero16());
#pragma unroll
          for (int r = 0; r < 16; ++r) o[d][r] = hit[r] > 0.f ? __builtin_nanf("") : o[d][r];
        }
      }
    const float sum = l + xor32(l), inv = sum == 0.f ? 0.f : 1.f / sum;   // no visible key: zeros
    if (row < x.rows) {
      T *op = row_of<T>(x, G, row, a.out, a.o_ss, a.o_hs) + 4 * hi;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          store4(op + 32 * d + 2 * r, o[d][r] * inv, o[d][r + 1] * inv, o[d][r + 2] * inv, o[d][r + 3] * inv);
    }
  }
  zero_rest<HD, T>(a);
}

enum Mode { kShares, kTiles, kPrompts };

struct Shape {
  Mode mode;
  int NT, tmshift, nwg;
};

// Keys up to which a sequence is one workgroup's: 1 x 1 token, 32 / 8 heads of 128, over 1000 keys 10.4 us in
// one launch, 12.4 by shares; a CU's rate bounds it from there (20 ns a key). They are those that the table has
// room for: lengths are not known on the host.
constexpr int kShortKeys = 1024;

// The narrowest tile that holds an average sequence's query rows: a wide one's empty
// columns cost matrix work only, a narrow one reads the cache once more a tile.
Shape shape_of(int T, int B, int Hq, int Hkv, int HD, int64_t keys, int dtype) {
  const int G = Hq / Hkv;
  const int64_t rows = ((int64_t)T * G + B - 1) / B;
  const int NT = rows <= 16 && G <= 16 ? 1 : 2, parts = dtype == kDtBf16 ? 1 : dtype == kDtF16 ? 2 : 3;
  // prompts by 128 rows where those tiles fill the chip: 32 / 8 heads of 128, shares / prompts, behind 2000
  // and 30 000 cached tokens: 1 x 512 new tokens (136 tiles) 63 / 62 and 535 / 645 us, 4 x 128 (160) 62 / 55
  // and 562 / 644, 4 x 256 (288) 106 / 69 and 1097 / 802, 4 x 512 (544) 194 / 92 and 2131 / 988
  const int pm = tm_shift(kPromptRows, G, 7);
  if (rows >= kPromptRows / 2 && (int64_t)tile_slots(T, B, pm) * Hkv >= device_cu_count())
    return {kPrompts, 0, pm, 0};
  return {keys <= kShortKeys ? kTiles : kShares, NT, tm_shift(16 * NT, G),
          share_occupancy(HD, NT, parts) * device_cu_count()};
}

template <int HD, int NT, typename T, bool UNI>
void launch3(const PagedAttnArgs &a, const Shape &s, hipStream_t stream) {
  const int G = a.Hq / a.Hkv, tiles = tile_slots(a.T, a.B, s.tmshift) * a.Hkv;
  if (s.mode == kTiles) {
    constexpr int NW = NT == 1 || sizeof(T) == 2 ? 8 : 4;   // by the registers of a wave
    paged_tile_kernel<HD, NT, T, UNI, NW><<<tiles, 64 * NW, 0, stream>>>(a, s.tmshift, G);
  } else {
    paged_share_kernel<HD, NT, T, UNI><<<s.nwg, 256, 0, stream>>>(a, s.tmshift, G);
    // for the rows of an average sequence's tile
    const int rows = std::min(1 << s.tmshift, (a.T + a.B - 1) / a.B) * G;
    if ((int64_t)tiles * rows >= 8 * device_cu_count())
      paged_join_kernel<HD, NT, T, 1><<<dim3(tiles, (rows + 3) / 4), 256, 0, stream>>>(a, s.tmshift, G, s.nwg * 4);
    else
      paged_join_kernel<HD, NT, T, 4><<<dim3(tiles, rows), 256, 0, stream>>>(a, s.tmshift, G, s.nwg * 4);
  }
}

template <int HD, typename T>
void launch1(const PagedAttnArgs &a, const Shape &s, hipStream_t stream) {
  if (s.mode == kPrompts) {
    const int slots = tile_slots(a.T, a.B, s.tmshift);
    if (a.pshift >= 6)
      paged_prompt_kernel<HD, T, true><<<slots * a.Hkv, 256, 0, stream>>>(a, s.tmshift, a.Hq / a.Hkv, slots);
    else
      paged_prompt_kernel<HD, T, false><<<slots * a.Hkv, 256, 0, stream>>>(a, s.tmshift, a.Hq / a.Hkv, slots);
    return;
  }
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
  const Shape s = shape_of(T, B, Hq, Hkv, head_dim, keys, dtype);
  if (s.mode != kShares) return 0;
  return (int64_t)s.nwg * 4 * 2 * slot_floats(16 * s.NT, head_dim) * 4 +
         (int64_t)tile_slots(T, B, s.tmshift) * Hkv * sizeof(JoinNote);
}

int64_t paged_attn_tiles(const PagedAttnArgs &a, int dtype) {
  const Shape s = shape_of(a.T, a.B, a.Hq, a.Hkv, 128, (int64_t)a.width << a.pshift, dtype);   // of any head_dim
  return (int64_t)tile_slots(a.T, a.B, s.tmshift) * a.Hkv;
}

void launch_paged_attn(const PagedAttnArgs &a, int head_dim, int dtype, hipStream_t stream) {
  const Shape s = shape_of(a.T, a.B, a.Hq, a.Hkv, head_dim, (int64_t)a.width << a.pshift, dtype);
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
