// New tokens' keys and values into a paged 8-bit cache (layout: mga_paged.hpp),
// with q / k normalisation and the rotary embedding on the way, in one launch.
//
//   y = x * rsqrt(mean(x^2) + eps) * w            (where norm weights are given)
//   r = y * cos + rotate_half(y) * sin            (where cos / sin are given)
// from the projections' values; the query rows in fp32, rounded once to their type.
// Keys are prepared in fp64 (half the rate of fp32; 4 us of the 29) and go on in fp32
// rounded to odd (to_float): prepared or rounded to nearest in fp32, a value next to the middle
// between two codes takes the wrong one about once in 2^20 values.
// Keys and values are rounded once to e4m3 under the scale of their (page, head): the
// least power of two of which 448 hold every value the page has taken
// since a row 0 was written. Where new rows make it grow, the rows kept from before
// are rounded again under the new scale (a shift of their exponents: exact unless a
// code falls below e4m3's normal range).
// Values that are not finite become NaN codes and count in no scale.
//
// Bounded by HBM for prompts (5006 tokens, 32 / 8 heads of 128, bf16, with norm: 115 MB
// in 29 us, 3.9 TB/s; a copy reaches 5.1), by the chain cu -> page and rows -> scale ->
// store for a token a sequence (64 sequences: 7.3 us). Occupancy is what the first needs:
// at 170 registers instead of 125 it took 39 us.
// A workgroup takes the new rows of one page, of one head's
// keys or values, so that a scale is one workgroup's maximum and no page has two
// writers; further workgroups rotate the query rows. The pages are numbered without
// sums over the sequences: b owns the slots from cu[b] / PS + 2b on, as many as n tokens can
// touch pages. A slot's sequence is found by a walk over the sequences, 64 a
// turn, which many sequences pay for: a token each for 64 / 512 / 1024 / 4096 of them 13 / 24 / 50 / 349 us.
#include "mga_internal.hpp"
#include "mga_paged.hpp"

namespace mga {
namespace {

// Eight consecutive elements as fp32.
__device__ __forceinline__ void load8f(const bf16_t *p, bool vec, float *x) {
  if (vec) {
    const bf16x8 v = load8(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
  }
}
__device__ __forceinline__ void load8f(const f16_t *p, bool vec, float *x) {
  if (vec) {
    const f16x8 v = __builtin_bit_cast(f16x8, load8(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
  }
}
__device__ __forceinline__ void load8f(const float *p, bool vec, float *x) {
  if (vec) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = a[i], x[i + 4] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
  }
}

// A lane's 16 channels of a row: 8j .. 8j + 7 and D/2 past them, so that the
// partners of rotate_half meet in one lane.
template <typename T, int D>
__device__ __forceinline__ void load_row(const T *row, int j, bool vec, float *x) {
  load8f(row + 8 * j, vec, x);
  load8f(row + D / 2 + 8 * j, vec, x + 8);
}

__device__ __forceinline__ float inv_root(float x) { return rsqrtf(x); }
__device__ __forceinline__ double inv_root(double x) { return 1.0 / sqrt(x); }

// A lane's 16 channels of a row as they lie in memory.
template <typename T>
struct RawRow {
  T v[16];
  template <int D>
  __device__ __forceinline__ void load(const T *row, int j, bool vec) {
    const T *p[2] = {row + 8 * j, row + D / 2 + 8 * j};
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (vec) {
#pragma unroll
        for (int i = 0; i < 8; i += V) *reinterpret_cast<i32x4 *>(v + 8 * h + i) = *reinterpret_cast<const i32x4 *>(p[h] + i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * h + i] = p[h][i];
      }
  }
};

__device__ __forceinline__ float to_float(float x) { return x; }

// d in fp32, rounded to odd: towards zero, with the last bit set where anything was lost. A middle between two
// codes and 448 times a power of two are even numbers of fp32: what is rounded to e4m3's 4 bits from the
// result, or compared with those, comes out as from d itself. (The nearest fp32 number may be the middle.)
__device__ __forceinline__ float to_float(double d) {
  const float f = (float)d;
  int bits = __builtin_bit_cast(int, f);
  bits -= fabs(d) < fabs((double)f) ? 1 : 0;   // from infinity, too
  bits |= (double)__builtin_bit_cast(float, bits) != d ? 1 : 0;
  return __builtin_bit_cast(float, bits);
}

// x <- x * rsqrt(mean(x^2) + eps) * w, then x * cos + rotate_half(x) * sin, computed in F. C: the type of cos
// and sin.
template <typename F, int D, typename T, typename C>
__device__ __forceinline__ void prepare(bool norm, bool turn, float eps, const RawRow<T> &w, const RawRow<C> &c,
                                        const RawRow<C> &s, float *x) {
  F rs = 1;
  if (norm) {
    F sum = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += (F)x[i] * (F)x[i];
    for (int m = 1; m < D / 16; m <<= 1) sum += __shfl_xor(sum, m, 64);
    rs = inv_root(sum * (F)(1.f / D) + (F)eps);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    F lo = x[i], hi = x[i + 8];
    if (norm) {
      lo = lo * rs * (F)(float)w.v[i];
      hi = hi * rs * (F)(float)w.v[i + 8];
    }
    if (turn) {
      const F a = lo * (F)(float)c.v[i] - hi * (F)(float)s.v[i];
      hi = hi * (F)(float)c.v[i + 8] + lo * (F)(float)s.v[i + 8];
      lo = a;
    }
    x[i] = to_float(lo);
    x[i + 8] = to_float(hi);
  }
}

__device__ __forceinline__ void store8f(bf16_t *p, bool vec, const float *x) {
  if (vec) {
    *reinterpret_cast<bf16x8 *>(p) = pack8<bf16_t>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (bf16_t)x[i];
  }
}
__device__ __forceinline__ void store8f(f16_t *p, bool vec, const float *x) {
  if (vec) {
    *reinterpret_cast<bf16x8 *>(p) = pack8<f16_t>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (f16_t)x[i];
  }
}
__device__ __forceinline__ void store8f(float *p, bool vec, const float *x) {
  if (vec) {
    store4(p, x[0], x[1], x[2], x[3]);
    store4(p + 4, x[4], x[5], x[6], x[7]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
  }
}

// Four values as e4m3 codes, to the nearest; past 448 the largest, not finite NaN.
__device__ __forceinline__ uint32_t encode4(const float *x, float inv) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = fminf(fmaxf(x[i] * inv, -448.f), 448.f);
    y[i] = fabsf(x[i]) < __builtin_huge_valf() ? c : __builtin_nanf("");
  }
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
}

// Four codes times a power of two <= 1.
__device__ __forceinline__ uint32_t requant4(uint32_t c, float ratio) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, r, true);
}

// Bytes lo <= i < hi of a dword whose first byte is number 0.
__device__ __forceinline__ uint32_t byte_mask(int lo, int hi) {
  const uint32_t h = hi >= 4 ? ~0u : hi <= 0 ? 0u : (1u << (8 * hi)) - 1;
  const uint32_t l = lo >= 4 ? ~0u : lo <= 0 ? 0u : (1u << (8 * lo)) - 1;
  return h & ~l;
}

// Which page, and which rows of which tokens, a workgroup writes.
struct PageRows {
  int b, pg, r0, r1;    // sequence, its page, the rows [r0, r1)
  int64_t tok0;         // the token of row r0
};

// The page of a slot; false: none. All lanes of the wave take part: their loads find the sequence and
// hold what is needed of it.
__device__ __forceinline__ bool page_of_slot(const PagedAppendArgs &a, int slot, PageRows &x) {
  const int PS = 1 << a.pshift;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = min(i0 + (int)(threadIdx.x & 63), a.B - 1);
    const SeqSpan q = seq_span(a.cu, a.lengths, i, a.T, a.width << a.pshift);
    // the sequences whose slots end at or before this one
    const uint64_t done = __ballot((min(max(a.cu[i + 1], 0), a.T) >> a.pshift) + 2 * (i + 1) <= slot);
    if (~done) {
      const int at = __ffsll((unsigned long long)~done) - 1;
      x.b = i0 + at;
      const int first = __builtin_amdgcn_readlane(q.first, at), n = __builtin_amdgcn_readlane(q.n, at),
                len = __builtin_amdgcn_readlane(q.len, at);
      const int nth = slot - ((first >> a.pshift) + 2 * x.b);
      const int64_t end = (int64_t)len + n;
      x.pg = (len >> a.pshift) + nth;
      if (x.b >= a.B || n == 0 || nth < 0 || x.pg >= a.width || (int64_t)x.pg << a.pshift >= end) return false;
      x.r0 = nth == 0 ? len & (PS - 1) : 0;
      x.r1 = (int)min((int64_t)PS, end - ((int64_t)x.pg << a.pshift));
      x.tok0 = first + ((int64_t)x.pg << a.pshift) + x.r0 - len;
      return true;
    }
  }
  return false;
}

// The page's scale: old and new exponent from the rows' largest magnitude.
struct Scaling {
  int was, now;
  bool grown;
  float inv, ratio;
};
__device__ __forceinline__ Scaling scaling(float amax, float old_scale, bool kept) {
  Scaling s;
  const int need = scale_exp(amax);
  s.was = exp_of(old_scale);
  s.now = kept ? max(s.was, need) : need;
  s.grown = kept && s.now > s.was;
  s.inv = pow2(-s.now);
  s.ratio = pow2(max(s.was - s.now, -126));
  return s;
}

__device__ __forceinline__ Scaling rescale(float amax, float old_scale, bool kept) {   // of all waves
  __shared__ float wave_max[4];
  for (int m = 32; m; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
  if ((threadIdx.x & 63) == 0) wave_max[threadIdx.x >> 6] = amax;
  __syncthreads();
  return scaling(fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3])), old_scale, kept);
}

__device__ __forceinline__ float finite_magnitude(float x) {
  const float v = fabsf(x);
  return v < __builtin_huge_valf() ? v : 0.f;
}

// Query rows: block qb's lane groups take every slots_per_token-th head of a token.
template <typename T, typename C, int D>
__device__ __forceinline__ void query_rows(const PagedAppendArgs &a, int qb, int slots_per_token) {
  constexpr int LR = D / 16, RP = 256 / LR;
  const int tid = threadIdx.x, j = tid % LR;
  const int slot = tid / LR;
  const int per = RP / slots_per_token;
  const int tok = qb * per + slot / slots_per_token;
  if (tok >= a.T) return;
  const bool live = tok < min(a.cu[a.B], a.T);
  RawRow<T> w = {};
  RawRow<C> c = {}, s = {};
  if (a.qw) w.template load<D>((const T *)a.qw, j, a.vec);
  if (a.cos) {
    c.template load<D>((const C *)a.cos + tok * a.cs_ss, j, a.vec);
    s.template load<D>((const C *)a.sin + tok * a.cs_ss, j, a.vec);
  }
  for (int h0 = slot % slots_per_token; h0 < a.Hq; h0 += 2 * slots_per_token) {
    float x[2][16];   // the rows of two heads in flight
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int h = min(h0 + u * slots_per_token, a.Hq - 1);
      load_row<T, D>((const T *)a.q + tok * a.q_ss + h * a.q_hs, j, a.vec, x[u]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int h = h0 + u * slots_per_token;
      if (h >= a.Hq) break;
      prepare<float, D>(a.qw != nullptr, a.cos != nullptr, a.eps, w, c, s, x[u]);
      if (!live) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
      }
      T *o = (T *)a.qo + tok * a.qo_ss + h * a.qo_hs;
      store8f(o + 8 * j, a.vec, x[u]);
      store8f(o + D / 2 + 8 * j, a.vec, x[u] + 8);
    }
  }
}

// NK: passes over a page's key rows (256 / (D / 16) rows each), NV: over its value rows (4 * 256 / (D / 8)).
template <typename T, typename C, int D, int NK, int NV>
__global__ __launch_bounds__(256, NK == 4 ? 2 : NK == 2 && sizeof(T) + sizeof(C) > 4 ? 3 : 4) void paged_append_kernel(
    PagedAppendArgs a, int32_t slots, int32_t slots_per_token) {
  constexpr int LR = D / 16, RP = 256 / LR;   // lanes a row, rows a pass
  const int tid = threadIdx.x, j = tid % LR;
  const int items = slots * a.Hkv * 2;
  const int blk = (int)blockIdx.x;

  if (blk >= items) return query_rows<T, C, D>(a, blk - items, slots_per_token);
  const bool is_v = blk & 1;
  const int head = (blk >> 1) % a.Hkv, slot = (blk >> 1) / a.Hkv;
  const int PS = 1 << a.pshift;
  PageRows pr;
  if (!page_of_slot(a, slot, pr)) return;
  const int r0 = pr.r0, r1 = pr.r1;
  const int page = a.table[(int64_t)pr.b * a.table_rs + pr.pg];   // in flight beside the rows' loads
  float amax = 0.f;

  if (!is_v) {
    float x[NK][16];
    RawRow<T> w = {};
    if (a.kw) w.template load<D>((const T *)a.kw, j, a.vec);
#pragma unroll
    for (int p = 0; p < NK; ++p) {
      const int r = r0 + p * RP + tid / LR;
      if (r < r1) load_row<T, D>((const T *)a.k + (pr.tok0 + (r - r0)) * a.k_ss + head * a.k_hs, j, a.vec, x[p]);
    }
    if ((uint32_t)page >= (uint32_t)a.num_pages) return;
    const int64_t ph = (int64_t)page * a.Hkv + head;
    uint8_t *codes = a.kp + ph * PS * D;
    const float old_scale = a.ks[ph];
#pragma unroll
    for (int p = 0; p < NK; ++p) {
      const int r = r0 + p * RP + tid / LR;
      if (r < r1) {
        if (a.kw || a.cos) {
          RawRow<C> c = {}, s = {};
          if (a.cos) {
            c.template load<D>((const C *)a.cos + (pr.tok0 + (r - r0)) * a.cs_ss, j, a.vec);
            s.template load<D>((const C *)a.sin + (pr.tok0 + (r - r0)) * a.cs_ss, j, a.vec);
          }
          prepare<double, D>(a.kw != nullptr, a.cos != nullptr, a.eps, w, c, s, x[p]);
          __builtin_amdgcn_sched_barrier(0);   // one pass's fp64 at a time
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, finite_magnitude(x[p][i]));
      }
    }
    const Scaling s = rescale(amax, old_scale, r0 > 0);
    if (tid == 0) a.ks[ph] = pow2(s.now);
#pragma unroll
    for (int p = 0; p < NK; ++p) {
      const int r = r0 + p * RP + tid / LR;
      if (r < r1) {
        uint8_t *o = codes + r * D + 8 * j;
        *reinterpret_cast<i32x2 *>(o) = i32x2{(int)encode4(x[p], s.inv), (int)encode4(x[p] + 4, s.inv)};
        *reinterpret_cast<i32x2 *>(o + D / 2) = i32x2{(int)encode4(x[p] + 8, s.inv), (int)encode4(x[p] + 12, s.inv)};
      }
    }
    if (s.grown)
      for (int i = tid * 16; i < r0 * D; i += 256 * 16) {
        i32x4 c = *reinterpret_cast<const i32x4 *>(codes + i);
#pragma unroll
        for (int w = 0; w < 4; ++w) c[w] = (int)requant4((uint32_t)c[w], s.ratio);
        *reinterpret_cast<i32x4 *>(codes + i) = c;
      }
    return;
  }

  // Values: a thread takes 8 channels of 4 rows, so that a channel's four codes are one dword of the
  // transposed tile in LDS; then 16 rows of a channel at a time go out.
  constexpr int CG = D / 8, RV = 4 * (256 / CG);
  const int cg = tid % CG, rg = tid / CG;
  float x[NV][4][8];
#pragma unroll
  for (int p = 0; p < NV; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = p * RV + 4 * rg + k;
      if (r >= r0 && r < r1)
        load8f((const T *)a.v + (pr.tok0 + (r - r0)) * a.v_ss + head * a.v_hs + 8 * cg, a.vec, x[p][k]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[p][k][i] = 0.f;
    }
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int64_t ph = (int64_t)page * a.Hkv + head;
  uint8_t *codes = a.vp + ph * PS * D;
  const float old_scale = a.vs[ph];
  // the chunk of 16 rows that a thread will complete first, read ahead: with one new row all there is
  const int d0 = tid % D, first0 = r0 >> 4;
  i32x4 ahead = {0, 0, 0, 0};
  if (tid < D) ahead = *reinterpret_cast<const i32x4 *>(codes + d0 * PS + first0 * 16);
#pragma unroll
  for (int p = 0; p < NV; ++p)
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_magnitude(x[p][k][i]));
  const Scaling s = rescale(amax, old_scale, r0 > 0);
  if (tid == 0) a.vs[ph] = pow2(s.now);
  const int first = s.grown ? 0 : first0, chunks = ((r1 + 15) >> 4) - first, ts = PS / 4 + 1;
  __shared__ uint32_t tile[D * (128 / 4 + 1)];
#pragma unroll
  for (int p = 0; p < NV; ++p)
    if (p * RV + 4 * rg < PS)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v[4] = {x[p][0][i], x[p][1][i], x[p][2][i], x[p][3][i]};
        tile[(8 * cg + i) * ts + p * RV / 4 + rg] = encode4(v, s.inv);
      }
  __syncthreads();
  for (int i = tid; i < D * chunks; i += 256) {
    const int d = i % D, c = first + i / D, base = c * 16;
    uint8_t *o = codes + d * PS + base;
    i32x4 w = {0, 0, 0, 0};
    if (base < r0 || base + 16 > r1) w = i < D && c == first0 ? ahead : *reinterpret_cast<const i32x4 *>(o);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t v = (uint32_t)w[k];
      if (s.grown) {
        const uint32_t kept = byte_mask(0, r0 - base - 4 * k);
        v = (v & ~kept) | (requant4(v, s.ratio) & kept);
      }
      const uint32_t put = byte_mask(r0 - base - 4 * k, r1 - base - 4 * k);
      w[k] = (int)((v & ~put) | (tile[d * ts + base / 4 + k] & put));
    }
    *reinterpret_cast<i32x4 *>(o) = w;
  }
}

// The same for few new tokens a sequence: a wave a page, head and keys or values, with no barrier and no
// LDS (64 sequences, a token each: 7.3 us, by a workgroup each 10.8). More rows than a wave holds at once
// are read twice.
template <typename T, typename C, int D>
__global__ __launch_bounds__(256) void paged_append_few_kernel(PagedAppendArgs a, int32_t slots, int32_t slots_per_token) {
  constexpr int LR = D / 16, RW = 64 / LR;   // lanes a row, rows at once
  const int lane = threadIdx.x & 63, j = lane % LR;
  const int items = slots * a.Hkv * 2, iblocks = (items + 3) / 4;
  if ((int)blockIdx.x >= iblocks) return query_rows<T, C, D>(a, blockIdx.x - iblocks, slots_per_token);
  const int item = blockIdx.x * 4 + wave_id();
  if (item >= items) return;
  const bool is_v = item & 1;
  const int head = (item >> 1) % a.Hkv, slot = (item >> 1) / a.Hkv;
  const int PS = 1 << a.pshift;
  PageRows pr;
  if (!page_of_slot(a, slot, pr)) return;
  const int r0 = pr.r0, r1 = pr.r1;
  const int page = a.table[(int64_t)pr.b * a.table_rs + pr.pg];   // in flight beside the rows' loads
  const T *src = is_v ? (const T *)a.v + head * a.v_hs : (const T *)a.k + head * a.k_hs;
  const int64_t ss = is_v ? a.v_ss : a.k_ss;
  const bool turn = !is_v && a.cos, norm = !is_v && a.kw;
  RawRow<T> w = {};
  if (norm) w.template load<D>((const T *)a.kw, j, a.vec);
  float x[16];
  auto rows_at = [&](int at) {   // this lane's row of RW from `at` on, prepared
    const int r = at + lane / LR;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
    if (r >= r1) return;
    const int64_t tok = pr.tok0 + (r - r0);
    load_row<T, D>(src + tok * ss, j, a.vec, x);
    RawRow<C> c = {}, s = {};
    if (turn) {
      c.template load<D>((const C *)a.cos + tok * a.cs_ss, j, a.vec);
      s.template load<D>((const C *)a.sin + tok * a.cs_ss, j, a.vec);
    }
    if (norm || turn) prepare<double, D>(norm, turn, a.eps, w, c, s, x);
  };
  rows_at(r0);
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int64_t ph = (int64_t)page * a.Hkv + head;
  uint8_t *codes = (is_v ? a.vp : a.kp) + ph * PS * D;
  float *scale = (is_v ? a.vs : a.ks) + ph;
  const float old_scale = *scale;
  float amax = 0.f;
  for (int at = r0;;) {
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, finite_magnitude(x[i]));
    at += RW;
    if (at >= r1) break;
    rows_at(at);
  }
  for (int m = 32; m; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
  const Scaling sc = scaling(amax, old_scale, r0 > 0);
  if (lane == 0) *scale = pow2(sc.now);
  if (r1 - r0 > RW) rows_at(r0);
  for (int at = r0;;) {
    const int r = at + lane / LR;
    if (r < r1) {
      uint32_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = encode4(x + 4 * i, sc.inv);
      if (!is_v) {
        uint8_t *o = codes + r * D + 8 * j;
        *reinterpret_cast<i32x2 *>(o) = i32x2{(int)c[0], (int)c[1]};
        *reinterpret_cast<i32x2 *>(o + D / 2) = i32x2{(int)c[2], (int)c[3]};
      } else {
        uint8_t *o = codes + 8 * j * PS + r;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          o[((i & 7) + (i >> 3) * (D / 2)) * PS] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
      }
    }
    at += RW;
    if (at >= r1) break;
    rows_at(at);
  }
  if (!sc.grown) return;
  if (!is_v) {
    for (int i = lane * 4; i < r0 * D; i += 256) {
      uint32_t *o = reinterpret_cast<uint32_t *>(codes + i);
      *o = requant4(*o, sc.ratio);
    }
  } else {
    // whole dwords of a channel's old rows, then the bytes beside the new ones
    const int q = r0 >> 2;
    for (int i = lane; i < D * q; i += 64) {
      uint32_t *o = reinterpret_cast<uint32_t *>(codes + i / q * PS) + i % q;
      *o = requant4(*o, sc.ratio);
    }
    for (int i = lane; i < D * (r0 & 3); i += 64) {
      uint8_t *o = codes + i / (r0 & 3) * PS + 4 * q + i % (r0 & 3);
      *o = (uint8_t)requant4(*o, sc.ratio);
    }
  }
}

// New tokens a sequence, on average, up to which a wave takes a page.
constexpr int kFewTokens = 8;

template <typename T, typename C>
void launch(const PagedAppendArgs &a, int D, hipStream_t stream) {
  const int PS = 1 << a.pshift;
  const int64_t slots = (a.T >> a.pshift) + 2 * (int64_t)a.B;
  const int rp = 256 / (D / 16);
  // a lane group takes several heads of a token, so that cos and sin are read once for them, where
  // there are rows enough to fill the chip
  const int spt = (int64_t)a.T * a.Hq >= 65536 ? 8 : 32;
  const int64_t qblocks = a.q ? (a.T + rp / spt - 1) / (rp / spt) : 0;
  if (a.T <= (int64_t)kFewTokens * a.B) {
    const dim3 grid((uint32_t)((slots * a.Hkv * 2 + 3) / 4 + qblocks));
    if (D == 128) paged_append_few_kernel<T, C, 128><<<grid, 256, 0, stream>>>(a, (int32_t)slots, spt);
    else paged_append_few_kernel<T, C, 64><<<grid, 256, 0, stream>>>(a, (int32_t)slots, spt);
    return;
  }
  const dim3 grid((uint32_t)(slots * a.Hkv * 2 + qblocks));
#define MGA_APPEND(DD, NK, NV) paged_append_kernel<T, C, DD, NK, NV><<<grid, 256, 0, stream>>>(a, (int32_t)slots, spt)
  if (D == 128) {
    if (PS <= 32) MGA_APPEND(128, 1, 1);
    else if (PS == 64) MGA_APPEND(128, 2, 1);
    else MGA_APPEND(128, 4, 2);
  } else {
    if (PS <= 64) MGA_APPEND(64, 1, 1);
    else MGA_APPEND(64, 2, 1);
  }
#undef MGA_APPEND
}

}  // namespace

int64_t paged_append_blocks(const PagedAppendArgs &a) {
  return ((a.T >> a.pshift) + 2 * (int64_t)a.B) * a.Hkv * 2 + a.T;
}

void launch_paged_append(const PagedAppendArgs &a, int head_dim, int dtype, hipStream_t stream) {
  if (dtype == kDtF32) launch<float, float>(a, head_dim, stream);
  else if (dtype == kDtBf16) a.cs32 ? launch<bf16_t, float>(a, head_dim, stream) : launch<bf16_t, bf16_t>(a, head_dim, stream);
  else a.cs32 ? launch<f16_t, float>(a, head_dim, stream) : launch<f16_t, f16_t>(a, head_dim, stream);
}

}  // namespace mga
