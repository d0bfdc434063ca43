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
// NaN although p = 0: see edge_nan.
#include <algorithm>

#include "mga_internal.hpp"
#include "mga_paged.hpp"

namespace mga {
namespace {

constexpr int kMinShare = 4;   // steps: one a wave

template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int n = 1; };
template <> struct Parts<f16_t> { static constexpr int n = 2; };
template <> struct Parts<float> { static constexpr int n = 3; };

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
      rest[i] -= (float)part[n][i];
    }
  }
}

// ---- the list of steps -------------------------------------------------------

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
    const int64_t x = ((int64_t)len + 63 + (1 << tmshift)) >> tmshift;
    return floor_sum(x + t, 6 - tmshift) - floor_sum(x, 6 - tmshift);
  }
  __device__ __forceinline__ int64_t all() const {
    const int t = tiles();
    return t ? before(t - 1) + steps(t - 1) : 0;
  }
};

// Tokens of a tile: the largest power of two of which a tile holds the query heads.
inline int tm_shift(int rows, int G) {
  int s = 0;
  while (((2 << s) * G <= rows) && s < 6) ++s;
  return s;
}

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

struct Place {
  int b, h, t, p, steps;   // sequence, KV head, tile, step within the tile, the tile's steps
  SeqSpan q;
};

__device__ __forceinline__ Place locate(const PagedAttnArgs &a, int tmshift, const int32_t *pre, int u) {
  Place r;
  r.b = 0;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = i0 + (threadIdx.x & 63);
    r.b += __popcll(__ballot(i < a.B && pre[i] <= u));
  }
  r.b = __builtin_amdgcn_readfirstlane(min(r.b, a.B - 1));
  const int rest = u - (r.b ? pre[r.b - 1] : 0);
  r.q = seq_span(a.cu, a.lengths, r.b, a.T, a.width << a.pshift);
  const SeqTiles st{r.q.n, r.q.len, tmshift};
  const int each = (int)st.all();
  r.h = rest / each;
  const int in = rest - r.h * each;
  int lo = 0, hi = st.tiles() - 1;
  while (lo < hi) {   // the last tile that begins at or before `in`
    const int mid = (lo + hi + 1) >> 1;
    if (st.before(mid) <= in) lo = mid;
    else hi = mid - 1;
  }
  r.t = lo;
  r.p = in - (int)st.before(lo);
  r.steps = st.steps(lo);
  return r;
}

// Where the partial results of a workgroup's first (0) and last (1) tile lie.
__device__ __forceinline__ int64_t slot_floats(int rows, int HD) { return (int64_t)rows * (HD + 2); }

struct JoinNote {   // a tile that begins in a workgroup's share and goes on past it
  int b, h, t, n;   // n: the workgroups that it goes through, 0: no such tile
  int slot;         // of the first
  int pad[3];
};

template <typename T>
__device__ __forceinline__ void store_out(T *p, float v) { *p = (T)v; }

template <int HD, int NT, typename T>
__global__ __launch_bounds__(256, NT == 1 ? 2 : 1) void paged_attn_kernel(PagedAttnArgs a, int tmshift, int G) {
  constexpr int NQ = Parts<T>::n, KS = HD / 32, ND = HD / 16, KL = HD / 64;
  constexpr int ROWS = 16 * NT;
  __shared__ int32_t pre[kMaxSeqs];
  __shared__ int32_t wave_sum[4];
  __shared__ float om[4][16][HD + 4];
  __shared__ float ml[4][2][16];

  const int tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const int col = lane & 15, g = lane >> 4, kg = col >> 2;
  const int nwg = gridDim.x;
  const int wg = xcd_swizzle(blockIdx.x, nwg);
  const int total = scan_steps(a, tmshift, pre, wave_sum);
  const int share = max((total + nwg - 1) / nwg, kMinShare);
  const int u0 = (int)min((int64_t)wg * share, (int64_t)total), u1 = (int)min((int64_t)u0 + share, (int64_t)total);
  const int PS = 1 << a.pshift;
  float *parts = a.ws;
  JoinNote *notes = reinterpret_cast<JoinNote *>(a.ws + (int64_t)nwg * 2 * slot_floats(ROWS, HD));
  int noted = 0;

  for (int u = u0; u < u1;) {
    const Place pl = locate(a, tmshift, pre, u);
    const int p0 = pl.p, p1 = min(pl.steps, pl.p + u1 - u);
    const int tok0 = pl.t << tmshift, ntok = min(1 << tmshift, pl.q.n - tok0);
    const int rows = ntok * G;
    const int32_t *trow = a.table + (int64_t)pl.b * a.table_rs;
    const int first_lim = pl.q.len + tok0;   // the last key that the tile's first token sees
    const int end_key = pl.q.len + pl.q.n;

    // queries, and each row's last key
    bf16x8 qf[NT][NQ][KS];
    int lim[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 16 + col, tk = r / G, hd = pl.h * G + r - tk * G;
      lim[nt] = r < rows ? first_lim + tk : -1;
      const T *qp = (const T *)a.q + (int64_t)(pl.q.first + tok0 + tk) * a.q_ss + (int64_t)hd * a.q_hs;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int c = 64 * (ks >> 1) + 16 * g + 8 * (ks & 1);
        if constexpr (NQ == 1) {
          qf[nt][0][ks] = r < rows ? load8(qp + c) : bf16x8{};
        } else {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = r < rows ? (float)qp[c + i] : 0.f;
          bf16x8 part[NQ];
          split8<NQ>(x, part);
#pragma unroll
          for (int n = 0; n < NQ; ++n) qf[nt][n][ks] = part[n];
        }
      }
    }

    f32x4 o[NT][ND];
    float m[NT], l[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt] = -__builtin_huge_valf();
      l[nt] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[nt][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // page of a 16-key group of a step, -1 where there is none
    auto page_of = [&](int p, int grp) {
      const int i = (p * 64 + 16 * grp) >> a.pshift;
      const int id = i < a.width ? trow[i] : -1;
      return (uint32_t)id < (uint32_t)a.num_pages ? id : -1;
    };
    i32x4 kc[4][KL], vc[ND];
    float ksc, vsc;
    auto load_k = [&](int p, int page) {
      const int64_t ph = (int64_t)max(page, 0) * a.Hkv + pl.h;
      const uint8_t *base = a.kp + (ph * PS + ((p * 64 + 16 * kg) & (PS - 1)) + (col & 3)) * HD + 16 * g;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < KL; ++i) kc[t][i] = *reinterpret_cast<const i32x4 *>(base + 4 * t * HD + 64 * i);
      ksc = a.ks[ph];
    };
    auto load_v = [&](int p, int page) {
      const int64_t ph = (int64_t)max(page, 0) * a.Hkv + pl.h;
      const uint8_t *base = a.vp + (ph * HD + col) * PS + ((p * 64 + 16 * g) & (PS - 1));
#pragma unroll
      for (int d = 0; d < ND; ++d) vc[d] = *reinterpret_cast<const i32x4 *>(base + 16 * d * PS);
      vsc = a.vs[ph];
    };

    int p = p0 + w;
    int kpage = -1, vpage = -1, kpage1 = -1, vpage1 = -1;
    if (p < p1) {
      kpage = page_of(p, kg);
      vpage = page_of(p, g);
      if (p + 4 < p1) {
        kpage1 = page_of(p + 4, kg);
        vpage1 = page_of(p + 4, g);
      }
      load_k(p, kpage);
      load_v(p, vpage);
    }
    for (; p < p1; p += 4) {
      f32x4 s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < 4; ++t) s[nt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const i32x4 c = kc[t][ks >> 1];
          const bf16x8 kf = decode8(c[2 * (ks & 1)], c[2 * (ks & 1) + 1], ksc);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[nt][t] = mfma16(kf, qf[nt][n][ks], s[nt][t]);
        }
      const bool more = p + 4 < p1;
      int kpage2 = -1, vpage2 = -1;
      if (more) {
        if (p + 8 < p1) {
          kpage2 = page_of(p + 8, kg);
          vpage2 = page_of(p + 8, g);
        }
        load_k(p + 4, kpage1);
      }

      // keys of this lane: key0 + 4 t + r
      const int key0 = p * 64 + 16 * g;
      const bool edge = p * 64 + 63 > first_lim || __any(vpage < 0);
      bf16x8 pf[NT][NQ][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (edge) {
          const int last = vpage < 0 ? -1 : lim[nt];
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[nt][t][r] = key0 + 4 * t + r <= last ? s[nt][t][r] : -__builtin_huge_valf();
        }
        float e[16], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          e[i] = __builtin_amdgcn_exp2f(fmaf(s[nt][i >> 2][i & 3], a.scale_log2, -m[nt]));
          sum += e[i];
        }
        if (__any(!(sum <= 0x1p20f))) {
          float mx = -__builtin_huge_valf();
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[nt][i >> 2][i & 3]);
          mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          const float now = fmaxf(m[nt], mx * a.scale_log2);
          const float off = now == -__builtin_huge_valf() ? 0.f : now;
          const float alpha = __builtin_amdgcn_exp2f(m[nt] - off);   // 0 from -inf
          l[nt] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) o[nt][d] *= alpha;
          m[nt] = now;
          sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            e[i] = __builtin_amdgcn_exp2f(fmaf(s[nt][i >> 2][i & 3], a.scale_log2, -off));
            sum += e[i];
          }
        }
        l[nt] += sum;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          bf16x8 part[NQ];
          split8<NQ>(e + 8 * c, part);
#pragma unroll
          for (int n = 0; n < NQ; ++n) pf[nt][n][c] = part[n];
        }
      }

      if (edge) {   // values behind the sequence or of no page: zeros
        const int valid = vpage < 0 ? 0 : end_key - key0;
        uint32_t nan = 0;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = valid - 4 * i;
            const uint32_t keep = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
            vc[d][i] &= (int)keep;
            nan |= ((uint32_t)vc[d][i] & 0x7f7f7f7fu) + 0x01010101u;
          }
        if (__any(nan & 0x80808080u)) {   // edge_nan: a NaN counts for the rows that see it, and only for them
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            bf16x8 sees[2];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              sees[i >> 3][i & 7] = (bf16_t)(key0 + i <= lim[nt] && vpage >= 0 ? 1.f : 0.f);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
              uint32_t one[4];   // 1.0 (0x38) where the code is NaN
#pragma unroll
              for (int i = 0; i < 4; ++i)
                one[i] = (((((uint32_t)vc[d][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0x38u;
              f32x4 hit = {0.f, 0.f, 0.f, 0.f};
              hit = mfma16(decode8(one[0], one[1], 1.f), sees[0], hit);
              hit = mfma16(decode8(one[2], one[3], 1.f), sees[1], hit);
#pragma unroll
              for (int r = 0; r < 4; ++r) o[nt][d][r] = hit[r] > 0.f ? __builtin_nanf("") : o[nt][d][r];
            }
          }
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t bad = ((((uint32_t)vc[d][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
              vc[d][i] &= (int)~(bad * 0xffu);
            }
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const bf16x8 vf = decode8(vc[d][2 * c], vc[d][2 * c + 1], vsc);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[nt][d] = mfma16(vf, pf[nt][n][c], o[nt][d]);
        }
      if (more) load_v(p + 4, vpage1);
      kpage = kpage1;
      vpage = vpage1;
      kpage1 = kpage2;
      vpage1 = vpage2;
    }

    // the waves' results together: sixteen rows at a time
    const bool whole = p0 == 0 && p1 == pl.steps;
    const int slot = 2 * wg + (u > u0 ? 1 : 0);
    if (p0 == 0 && p1 < pl.steps) {
      noted = 1;
      if (tid == 0) {
        const int last = (u - p0 + pl.steps - 1) / share;
        notes[wg] = JoinNote{pl.b, pl.h, pl.t, last - wg + 1, slot, {0, 0, 0}};
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 16 >= rows) break;
      float lsum = l[nt];
      lsum += __shfl_xor(lsum, 16, 64);
      lsum += __shfl_xor(lsum, 32, 64);
      __syncthreads();   // om and ml are free again
      if (g == 0) {
        ml[w][0][col] = m[nt];
        ml[w][1][col] = lsum;
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&om[w][col][16 * d + 4 * g]) = o[nt][d];
      __syncthreads();
      const int r16 = tid >> 4, r = nt * 16 + r16, c0 = (tid & 15) * (HD / 16);
      float mt = -__builtin_huge_valf(), lt = 0.f, acc[HD / 16];
#pragma unroll
      for (int i = 0; i < 4; ++i) mt = fmaxf(mt, ml[i][0][r16]);
      const float off = mt == -__builtin_huge_valf() ? 0.f : mt;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) acc[i] = 0.f;
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float f = __builtin_amdgcn_exp2f(ml[v][0][r16] - off);
        lt += ml[v][1][r16] * f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) acc[i] += om[v][r16][c0 + i] * f;
      }
      if (r < rows) {
        if (whole) {
          const int tk = r / G, hd = pl.h * G + r - tk * G;
          T *op = (T *)a.out + (int64_t)(pl.q.first + tok0 + tk) * a.o_ss + (int64_t)hd * a.o_hs + c0;
          const float inv = lt == 0.f ? 0.f : 1.f / lt;   // no visible key: zeros
#pragma unroll
          for (int i = 0; i < HD / 16; i += 4) store4(op + i, acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
        } else {
          float *pp = parts + slot * slot_floats(ROWS, HD);
#pragma unroll
          for (int i = 0; i < HD / 16; i += 4) store4(pp + r * HD + c0 + i, acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
          if ((tid & 15) == 0) {
            pp[ROWS * HD + 2 * r] = mt;
            pp[ROWS * HD + 2 * r + 1] = lt;
          }
        }
      }
    }
    u += p1 - p0;
  }
  if (!noted && tid == 0) notes[wg].n = 0;

  if (a.zero_rest) {   // rows behind the last sequence
    const int used = min(max(a.cu[a.B], 0), a.T);
    for (int64_t t = used + (int64_t)blockIdx.x; t < a.T; t += nwg)
      for (int i = tid * 4; i < a.Hq * HD; i += 1024)
        store4((T *)a.out + t * a.o_ss + (int64_t)(i / HD) * a.o_hs + i % HD, 0.f, 0.f, 0.f, 0.f);
  }
}

// The partial results of one tile, joined in their order: a wave a row.
template <int HD, int NT, typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a, int tmshift, int G, int nwg) {
  constexpr int ROWS = 16 * NT;
  const JoinNote *notes = reinterpret_cast<const JoinNote *>(a.ws + (int64_t)nwg * 2 * slot_floats(ROWS, HD));
  const int wg = blockIdx.x, lane = threadIdx.x & 63;
  const JoinNote n = notes[wg];
  if (n.n == 0) return;
  const SeqSpan q = seq_span(a.cu, a.lengths, n.b, a.T, a.width << a.pshift);
  const int tok0 = n.t << tmshift, rows = min(1 << tmshift, q.n - tok0) * G;
  const int r = blockIdx.y * 4 + wave_id();
  if (r >= rows) return;
  auto part = [&](int i) { return a.ws + (int64_t)(i == 0 ? n.slot : 2 * (wg + i)) * slot_floats(ROWS, HD); };
  float m = -__builtin_huge_valf();
  for (int i = lane; i < n.n; i += 64) m = fmaxf(m, part(i)[ROWS * HD + 2 * r]);
  for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const float off = m == -__builtin_huge_valf() ? 0.f : m;
  float l = 0.f, acc[HD / 64];
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) acc[c] = 0.f;
  for (int i0 = 0; i0 < n.n; i0 += 64) {
    float f = 0.f;
    if (i0 + lane < n.n) {
      const float *pp = part(i0 + lane) + ROWS * HD + 2 * r;
      f = __builtin_amdgcn_exp2f(pp[0] - off);
      l += f * pp[1];
    }
    const int k = min(64, n.n - i0);
#pragma unroll 4
    for (int i = 0; i < k; ++i) {
      const float fi = __shfl(f, i, 64);
      const float *pp = part(i0 + i) + r * HD + lane * (HD / 64);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) acc[c] += fi * pp[c];
    }
  }
  for (int x = 32; x; x >>= 1) l += __shfl_xor(l, x, 64);
  const int tk = r / G, hd = n.h * G + r - tk * G;
  T *op = (T *)a.out + (int64_t)(q.first + tok0 + tk) * a.o_ss + (int64_t)hd * a.o_hs + lane * (HD / 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < HD / 64; ++c) store_out(op + c, acc[c] * inv);
}

struct Shape {
  int NT, tmshift, nwg;
};

// The narrowest tile that holds an average sequence's query rows: a wide one's empty
// columns cost matrix work only, a narrow one reads the cache once more a tile.
Shape shape_of(int T, int B, int Hq, int Hkv, int dtype) {
  const int G = Hq / Hkv;
  const int64_t rows = ((int64_t)T * G + B - 1) / B;
  int NT = rows <= 16 && G <= 16 ? 1 : rows <= 32 || dtype != kDtBf16 ? 2 : 4;
  const int per_cu = NT == 1 ? 2 : 1;
  return {NT, tm_shift(16 * NT, G), per_cu * device_cu_count()};
}

template <int HD, int NT, typename T>
void launch2(const PagedAttnArgs &a, const Shape &s, hipStream_t stream) {
  const int G = a.Hq / a.Hkv;
  paged_attn_kernel<HD, NT, T><<<s.nwg, 256, 0, stream>>>(a, s.tmshift, G);
  const int rows = std::min((1 << s.tmshift), a.T) * G;
  paged_join_kernel<HD, NT, T><<<dim3(s.nwg, (rows + 3) / 4), 256, 0, stream>>>(a, s.tmshift, G, s.nwg);
}

template <int HD, typename T>
void launch1(const PagedAttnArgs &a, const Shape &s, hipStream_t stream) {
  if (s.NT == 1) return launch2<HD, 1, T>(a, s, stream);
  if (s.NT == 2) return launch2<HD, 2, T>(a, s, stream);
  if constexpr (Parts<T>::n == 1) launch2<HD, 4, T>(a, s, stream);
}

}  // namespace

int64_t paged_attn_ws_bytes(int32_t T, int32_t B, int32_t Hq, int32_t Hkv, int head_dim, int dtype) {
  const Shape s = shape_of(T, B, Hq, Hkv, dtype);
  return (int64_t)s.nwg * (2 * 16 * s.NT * (head_dim + 2) * 4 + sizeof(JoinNote));
}

int64_t paged_attn_steps(const PagedAttnArgs &a, int dtype) {
  const Shape s = shape_of(a.T, a.B, a.Hq, a.Hkv, dtype);
  const int64_t tiles = ((int64_t)a.T >> s.tmshift) + std::min(a.B, a.T);
  return tiles * a.Hkv * ((((int64_t)a.width << a.pshift) + a.T + 63) / 64 + 1);
}

void launch_paged_attn(const PagedAttnArgs &a, int head_dim, int dtype, hipStream_t stream) {
  const Shape s = shape_of(a.T, a.B, a.Hq, a.Hkv, dtype);
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
