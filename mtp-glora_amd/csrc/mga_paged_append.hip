// New tokens' keys and values into a paged 8-bit cache (layout: mga_paged.hpp),
// with q / k normalisation and the rotary embedding on the way, in one launch.
//
//   y = x * rsqrt(mean(x^2) + eps) * w            (where norm weights are given)
//   r = y * cos + rotate_half(y) * sin            (where cos / sin are given)
// from the projections' values; the query rows in fp32, rounded once to their type.
// Keys are prepared in fp64 (half the rate of fp32, in a kernel that memory bounds): an
// fp32 value next to the middle between two codes takes the wrong one about once in 2^20
// values. Keys and values are rounded once to e4m3 under the scale of their (page, head): the least power of two of which 448 hold every value the page has taken
// since a row 0 was written. Where new rows make it grow, the rows kept from before
// are rounded again under the new scale (a shift of their exponents: exact unless a
// code falls below e4m3's normal range).
// Values that are not finite become NaN codes and count in no scale.
//
// Bounded by HBM for prompts, by the chain cu -> table -> rows -> maximum -> store
// for a token a sequence. A workgroup takes the new rows of one page, of one head's
// keys or values, so that a scale is one workgroup's maximum and no page has two
// writers; further workgroups rotate the query rows. The page of a workgroup is
// found without a scan: sequence b owns the slots from cu[b] / PS + 2b on, as many
// as n tokens can touch pages, so that a slot's sequence is a count of compares.
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

// y = x * rsqrt(mean(x^2) + eps) * w, then y * cos + rotate_half(y) * sin, in F.
template <typename T, int D, typename F>
__device__ __forceinline__ void norm_rotate(const PagedAppendArgs &a, const void *weight, int64_t tok, int j, F *x) {
  constexpr int LR = D / 16;
  if (weight) {
    float w[16];
    F s = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += x[i] * x[i];
    for (int m = 1; m < LR; m <<= 1) s += __shfl_xor(s, m, 64);
    load_row<T, D>((const T *)weight, j, a.vec, w);
    const F rs = inv_root(s * (F)(1.f / D) + (F)a.eps);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = x[i] * rs * (F)w[i];
  }
  if (a.cos) {
    float c[16], s[16];
    if (a.cs32) {
      load_row<float, D>((const float *)a.cos + tok * a.cs_ss, j, a.vec, c);
      load_row<float, D>((const float *)a.sin + tok * a.cs_ss, j, a.vec, s);
    } else {
      load_row<T, D>((const T *)a.cos + tok * a.cs_ss, j, a.vec, c);
      load_row<T, D>((const T *)a.sin + tok * a.cs_ss, j, a.vec, s);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const F lo = x[i], hi = x[i + 8];
      x[i] = lo * (F)c[i] - hi * (F)s[i];
      x[i + 8] = hi * (F)c[i + 8] + lo * (F)s[i + 8];
    }
  }
}

// fp32 next to d on the side of d: what is rounded to e4m3 from it is what d would be.
__device__ __forceinline__ float beside(double d) {
  const float f = (float)d;
  const double r = (double)f;
  const int bits = __builtin_bit_cast(int, f);
  const bool more = fabs(d) > fabs(r), less = fabs(d) < fabs(r);
  return fabsf(f) < __builtin_huge_valf() ? __builtin_bit_cast(float, bits + (more ? 1 : less ? -1 : 0)) : f;
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

template <typename T, int D, int NPASS>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, int32_t slots, int32_t slots_per_token) {
  constexpr int LR = D / 16, RP = 256 / LR;   // lanes a row, rows a pass
  const int tid = threadIdx.x, lane = tid & 63, j = tid % LR;
  const int items = slots * a.Hkv * 2;
  const int blk = (int)blockIdx.x;

  if (blk >= items) {   // query rows: a lane group takes every slots_per_token-th head of a token
    const int slot = tid / LR;
    const int per = RP / slots_per_token;
    const int tok = (blk - items) * per + slot / slots_per_token;
    if (tok >= a.T) return;
    const bool live = tok < min(a.cu[a.B], a.T);
    for (int h = slot % slots_per_token; h < a.Hq; h += slots_per_token) {
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.f;
      if (live) {
        load_row<T, D>((const T *)a.q + tok * a.q_ss + h * a.q_hs, j, a.vec, x);
        norm_rotate<T, D>(a, a.qw, tok, j, x);
      }
      T *o = (T *)a.qo + tok * a.qo_ss + h * a.qo_hs;
      store8f(o + 8 * j, a.vec, x);
      store8f(o + D / 2 + 8 * j, a.vec, x + 8);
    }
    return;
  }

  const bool is_v = blk & 1;
  const int head = (blk >> 1) % a.Hkv, slot = (blk >> 1) / a.Hkv;
  const int PS = 1 << a.pshift;
  // the slot's sequence: how many begin and end before it
  int b = 0;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = i0 + lane + 1;
    const bool before = i <= a.B && ((min(max(a.cu[i], 0), a.T) >> a.pshift) + 2 * i) <= slot;
    b += __popcll(__ballot(before));
  }
  b = __builtin_amdgcn_readfirstlane(b);
  if (b >= a.B) return;
  const SeqSpan sq = seq_span(a.cu, a.lengths, b, a.T, a.width << a.pshift);
  const int nth = slot - ((sq.first >> a.pshift) + 2 * b);
  const int pg = (sq.len >> a.pshift) + nth;   // which of the sequence's pages
  const int64_t end = (int64_t)sq.len + sq.n;
  if (sq.n == 0 || nth < 0 || pg >= a.width || (int64_t)pg << a.pshift >= end) return;
  const int page = a.table[(int64_t)b * a.table_rs + pg];
  if ((uint32_t)page >= (uint32_t)a.num_pages) return;
  const int r0 = nth == 0 ? sq.len & (PS - 1) : 0;
  const int r1 = (int)min((int64_t)PS, end - ((int64_t)pg << a.pshift));
  const int64_t tok0 = sq.first + ((int64_t)pg << a.pshift) + r0 - sq.len;   // of row r0
  const int64_t ph = (int64_t)page * a.Hkv + head;
  uint8_t *codes = (is_v ? a.vp : a.kp) + ph * PS * D;
  float *scale = (is_v ? a.vs : a.ks) + ph;
  const float old_scale = *scale;
  const T *src = (const T *)(is_v ? a.v : a.k);
  const int64_t ss = is_v ? a.v_ss : a.k_ss, hs = is_v ? a.v_hs : a.k_hs;

  float x[NPASS][16], amax = 0.f;
#pragma unroll
  for (int p = 0; p < NPASS; ++p) {
    const int r = r0 + p * RP + tid / LR;
    if (r < r1) {
      const int64_t tok = tok0 + (r - r0);
      load_row<T, D>(src + tok * ss + head * hs, j, a.vec, x[p]);
      if (!is_v && (a.kw || a.cos)) {
        double y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = x[p][i];
        norm_rotate<T, D>(a, a.kw, tok, j, y);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[p][i] = beside(y[i]);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = fabsf(x[p][i]);
        amax = fmaxf(amax, v < __builtin_huge_valf() ? v : 0.f);
      }
    }
  }
  for (int m = 32; m; m >>= 1) amax = fmaxf(amax, __shfl_xor(amax, m, 64));
  __shared__ float wave_max[4];
  if (lane == 0) wave_max[tid >> 6] = amax;
  __syncthreads();
  amax = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
  const int was = exp_of(old_scale), need = scale_exp(amax);
  const int now = r0 ? max(was, need) : need;
  const bool grown = r0 && now > was;
  const float inv = pow2(-now), ratio = pow2(max(was - now, -126));
  if (tid == 0) *scale = pow2(now);

  if (!is_v) {
#pragma unroll
    for (int p = 0; p < NPASS; ++p) {
      const int r = r0 + p * RP + tid / LR;
      if (r < r1) {
        uint8_t *o = codes + r * D + 8 * j;
        *reinterpret_cast<i32x2 *>(o) = i32x2{(int)encode4(x[p], inv), (int)encode4(x[p] + 4, inv)};
        *reinterpret_cast<i32x2 *>(o + D / 2) = i32x2{(int)encode4(x[p] + 8, inv), (int)encode4(x[p] + 12, inv)};
      }
    }
    if (grown)
      for (int i = tid * 16; i < r0 * D; i += 256 * 16) {
        i32x4 c = *reinterpret_cast<const i32x4 *>(codes + i);
#pragma unroll
        for (int w = 0; w < 4; ++w) c[w] = (int)requant4((uint32_t)c[w], ratio);
        *reinterpret_cast<i32x4 *>(codes + i) = c;
      }
    return;
  }

  // values: the rows' codes transposed in LDS, then 16 rows of a channel at a time
  __shared__ uint32_t tile[D * (128 + 4) / 4];
  uint8_t *t8 = reinterpret_cast<uint8_t *>(tile);
  const int ts = PS + 4;
#pragma unroll
  for (int p = 0; p < NPASS; ++p) {
    const int r = r0 + p * RP + tid / LR;
    if (r < r1) {
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const uint32_t c = encode4(x[p] + i, inv);
        const int d = (i < 8 ? 8 * j + i : D / 2 + 8 * j + i - 8);
#pragma unroll
        for (int w = 0; w < 4; ++w) t8[(d + w) * ts + r] = (uint8_t)(c >> (8 * w));
      }
    }
  }
  __syncthreads();
  const int first = (grown ? 0 : r0) >> 4, chunks = ((r1 + 15) >> 4) - first;
  for (int i = tid; i < D * chunks; i += 256) {
    const int d = i / chunks, c = first + i % chunks, base = c * 16;
    uint8_t *o = codes + d * PS + base;
    i32x4 w = {0, 0, 0, 0};
    if (base < r0 || base + 16 > r1) w = *reinterpret_cast<const i32x4 *>(o);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t fresh = tile[(d * ts + base) / 4 + k];
      uint32_t v = (uint32_t)w[k];
      if (grown) {
        const uint32_t kept = byte_mask(0, r0 - base - 4 * k);
        v = (v & ~kept) | (requant4(v, ratio) & kept);
      }
      const uint32_t put = byte_mask(r0 - base - 4 * k, r1 - base - 4 * k);
      w[k] = (int)((v & ~put) | (fresh & put));
    }
    *reinterpret_cast<i32x4 *>(o) = w;
  }
}

template <typename T>
void launch(const PagedAppendArgs &a, int D, hipStream_t stream) {
  const int PS = 1 << a.pshift;
  const int64_t slots = (a.T >> a.pshift) + 2 * (int64_t)a.B;
  const int rp = 256 / (D / 16);
  // a lane group takes several heads of a token, so that cos and sin are read once for them, where
  // there are rows enough to fill the chip
  const int spt = (int64_t)a.T * a.Hq >= 65536 ? 8 : 32;
  const int64_t qblocks = a.q ? (a.T + rp / spt - 1) / (rp / spt) : 0;
  const dim3 grid((uint32_t)(slots * a.Hkv * 2 + qblocks));
  const int passes = (PS + rp - 1) / rp;
#define MGA_APPEND(DD, NP) paged_append_kernel<T, DD, NP><<<grid, 256, 0, stream>>>(a, (int32_t)slots, spt)
  if (D == 128) {
    if (passes <= 1) MGA_APPEND(128, 1);
    else if (passes == 2) MGA_APPEND(128, 2);
    else MGA_APPEND(128, 4);
  } else {
    if (passes <= 1) MGA_APPEND(64, 1);
    else MGA_APPEND(64, 2);
  }
#undef MGA_APPEND
}

}  // namespace

int64_t paged_append_blocks(const PagedAppendArgs &a) {
  return ((a.T >> a.pshift) + 2 * (int64_t)a.B) * a.Hkv * 2 + a.T;
}

void launch_paged_append(const PagedAppendArgs &a, int head_dim, int dtype, hipStream_t stream) {
  if (dtype == kDtBf16) launch<bf16_t>(a, head_dim, stream);
  else if (dtype == kDtF16) launch<f16_t>(a, head_dim, stream);
  else launch<float>(a, head_dim, stream);
}

}  // namespace mga
