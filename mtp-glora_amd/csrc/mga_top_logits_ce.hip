// Cross-entropy of student logits x against the top logits that were kept of a
// teacher's row (K values t with their columns), forward and backward.
//
//   q_k = e^{t_k / tau - lse}, or the softmax of t / tau over the row's K;
//   Q = sum_k q_k; p = softmax(x / tau);
//   row loss = tau^2 (Q log sum_j e^{x_j / tau} - sum_k q_k x_{id_k} / tau)
//            = sum_k q_k (tau (m - x_{id_k}) + tau^2 log d),
//              m = max x, d = sum_j e^{(x_j - m) / tau} (no difference of large
//              numbers where student and teacher agree);
//   grad_j = go tau (Q p_j - sum_{k: id_k = j} q_k).
// The K columns are a few cache lines; all three kernels are bound by the rows of
// x (read) and of the gradient (written).
//
// Forward of few rows: column ranges of the rows to (m, d), then a wave per row joins
// them, forms q and the row's loss; the last workgroup adds the rows in a fixed order.
// Of more: a workgroup a row, and a launch that adds them. Backward: one more pass
// over x. Both in one (step): a workgroup a row, which reads it twice.
#include "mga_internal.hpp"
#include "mga_vocab_row.hpp"

namespace mga {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float ex2(float v) { return __builtin_amdgcn_exp2f(v); }

__device__ __forceinline__ void merge_lanes(RowSum &st, float c) {
#pragma unroll
  for (int s = 32; s >= 1; s >>= 1) st.merge(__shfl_xor(st.m, s, 64), __shfl_xor(st.d, s, 64), c);
}

// Four vectors of x a turn of the workgroup of B threads, upwards; f(vector).
template <int B, typename F>
__device__ __forceinline__ void vectors_up(const i32x4 *vp, int nvec, const i32x4 &none, F f) {
  const int tid = threadIdx.x, nturn = nvec / (4 * B);
  i32x4 a[4], b[4];
  if (nturn > 0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = vp[tid + u * B];
  }
  for (int i = 1; i <= nturn; ++i) {   // the next turn's loads before this turn's arithmetic
    if (i < nturn) {
#pragma unroll
      for (int u = 0; u < 4; ++u) b[u] = vp[(i * 4 + u) * B + tid];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) f(a[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = b[u];
  }
  // every lane of a wave calls f, with -inf where it has none
  for (int i = nturn * 4 * B + tid; i - (tid & 63) < nvec; i += B) f(i < nvec ? vp[i] : none);
}
// The same downwards; f(index, vector).
template <int B, typename F>
__device__ __forceinline__ void vectors_down(const i32x4 *vp, int nvec, F f) {
  const int tid = threadIdx.x, nturn = nvec / (4 * B);
  for (int i = nturn * 4 * B + tid; i < nvec; i += B) f(i, vp[i]);
  i32x4 a[4], b[4];
  if (nturn > 0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = vp[((nturn - 1) * 4 + u) * B + tid];
  }
  for (int i = nturn - 1; i >= 0; --i) {
    if (i > 0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) b[u] = vp[((i - 1) * 4 + u) * B + tid];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) f((i * 4 + u) * B + tid, a[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) a[u] = b[u];
  }
}

// Running sum over the n elements at p by a workgroup of B threads.
template <int B, typename T>
__device__ __forceinline__ RowSum sum_elements(const T *p, int n, float c) {
  constexpr int W = RowElem<T>::W;
  const int tid = threadIdx.x, off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
  const int head = min(n, off ? W - off : 0), nvec = (n - head) / W, tail0 = head + nvec * W;
  RowSum st;
  auto one = [&](float x) {   // every lane, -inf where there is none
    const float f[1] = {x};
    st.add(f, fmaxf(x, kRowNegInf), c);
  };
  constexpr int fill = RowElem<T>::kFill;
  const i32x4 none = {fill, fill, fill, fill};
  vectors_up<B>(reinterpret_cast<const i32x4 *>(p + head), nvec, none, [&](const i32x4 &v) {
    float f[W], g = kRowNegInf;
#pragma unroll
    for (int e = 0; e < W; ++e) g = fmaxf(g, f[e] = RowElem<T>::get(v, e));
    st.add(f, g, c);
  });
  one(tid < head ? (float)p[tid] : kRowNegInf);
  one(tid < n - tail0 ? (float)p[tail0 + tid] : kRowNegInf);
  return st;
}

template <typename T>
__device__ __forceinline__ i32x4 pack_vec(const float *v) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(i32x4, f32x4{v[0], v[1], v[2], v[3]});
  else
    return i32x4{(int)cvt2<T>(v[0], v[1]), (int)cvt2<T>(v[2], v[3]), (int)cvt2<T>(v[4], v[5]), (int)cvt2<T>(v[6], v[7])};
}

__device__ __forceinline__ float teacher_value(const TopLogitsCeArgs &a, int64_t row, int k) {
  const int64_t at = row * a.values_rs + k;
  return a.values_dtype == kDtF32 ? static_cast<const float *>(a.values)[at]
         : a.values_dtype == kDtF16 ? (float)static_cast<const f16_t *>(a.values)[at]
                                    : (float)static_cast<const bf16_t *>(a.values)[at];
}
// -1 outside the row
__device__ __forceinline__ int teacher_id(const TopLogitsCeArgs &a, int64_t row, int k) {
  const int64_t at = row * a.ids_rs + k;
  const int64_t id = a.ids64 ? static_cast<const int64_t *>(a.ids)[at] : static_cast<const int32_t *>(a.ids)[at];
  return id >= 0 && id < a.V ? (int)id : -1;
}
// q of a teacher value before the division by its sum (no lse; norm: the largest value)
// or as it is (lse). Without lse the values' difference is taken before the quotient by
// tau: a value's own may be past fp32 (the type's lowest at tau < 1).
struct TeacherWeight {
  float before, behind;
  __device__ __forceinline__ TeacherWeight(const TopLogitsCeArgs &a, float itau)
      : before(a.lse ? itau : 1.f), behind(a.lse ? kLog2e : itau * kLog2e) {}
  __device__ __forceinline__ float operator()(float t, int id, float norm) const {
    const float s = t * before;
    if (id < 0 || s == kRowNegInf || norm == kRowNegInf) return 0.f;
    return ex2((s - norm) * behind);
  }
};

// tau^2 q ((m - x) / tau + log d); tau2logd: tau^2 log d
__device__ __forceinline__ float loss_term(float q, float x, float m, float tau, float tau2logd) {
  if (q == 0.f) return 0.f;
  if (x == kRowNegInf && tau2logd == tau2logd) return -kRowNegInf;   // all of the row among them (m = -inf)
  return q * ((m - x) * tau + tau2logd);
}

// What the gradient's elements of a row have in common: a 2^{x c - mc}; zeros,
// whatever x holds, where nothing of the teacher's row is left (dead).
struct GradRow {
  float mc, c, a;
  bool dead;
  __device__ __forceinline__ GradRow(float m, float d, float Q, float c_, float coef)
      : mc(scaled(m, c_)), c(c_), a(d == 0.f ? 0.f : sum_at_max(m, coef * Q / d, c_)), dead(Q == 0.f) {
    if (far(m, c_)) {   // a where x is m and 0 elsewhere: m c and x c exact, |m c| up to 2^60
      c = ldexpf(1.f, 60 - __builtin_amdgcn_frexp_expf(m));
      mc = m * c;
    }
  }
  __device__ __forceinline__ float operator()(float x) const { return a * ex2(__builtin_fmaf(x, c, -mc)); }
};
struct ZeroRow {
  __device__ __forceinline__ float operator()(float) const { return 0.f; }
};

// Sum of q[j] over the j with ids[j] == id, in order; 0 where an earlier j than k has it.
__device__ __forceinline__ bool owned_sum(const int *ids, const float *q, int K, int k, float *sum) {
  const int id = ids[k];
  float s = 0.f;
  for (int j = 0; j < K; ++j) {
    if (ids[j] != id) continue;
    if (j < k) return false;
    s += q[j];
  }
  *sum = s;
  return true;
}

}  // namespace

template <typename T>
__global__ __launch_bounds__(kThreads) void top_ce_partial_kernel(const T *__restrict__ x, int64_t xs, int32_t V,
                                                                  float c, int32_t chunk, int32_t nsplit,
                                                                  float *__restrict__ part, int *__restrict__ done) {
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / nsplit;
  const int sp = blockIdx.x - row * nsplit, c0 = sp * chunk, n = min(V, c0 + chunk) - c0;
  if (blockIdx.x == 0 && tid == 0) *done = 0;   // for the combine kernel
  const T *xr = x + row * xs + c0;
  RowSum st = sum_elements<kThreads>(xr, n, c);
  merge_lanes(st, c);
  __shared__ float wm[kThreads / 64], wd[kThreads / 64];
  if ((tid & 63) == 0) {
    wm[tid >> 6] = st.m;
    wd[tid >> 6] = st.d;
  }
  __syncthreads();
  float m = wm[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) m = fmaxf(m, wm[w]);
  if (far(m, c)) {
    float s = count_equal<kThreads>(xr, n, m) + (m - m);   // NaN for +inf
#pragma unroll
    for (int i = 32; i >= 1; i >>= 1) s += __shfl_xor(s, i, 64);
    __syncthreads();
    if ((tid & 63) == 0) {
      wm[tid >> 6] = m;
      wd[tid >> 6] = s;
    }
    __syncthreads();
  }
  if (tid == 0) {
    float d = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) d += wd[w] * part_weight(wm[w], m, c);
    part[2 * blockIdx.x] = m;
    part[2 * blockIdx.x + 1] = d;
  }
}

// The losses added in a fixed order by one workgroup of kThreads; on thread 0.
__device__ __forceinline__ float sum_rows(const float *loss, int N) {
  float s = 0.f;
  for (int64_t r0 = 0; r0 < N; r0 += 8 * kThreads) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int64_t r = r0 + u * kThreads + threadIdx.x;
      v[u] = r < N ? __hip_atomic_load(loss + r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) s += v[u];
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
  __shared__ float ws[kThreads / 64];
  if ((threadIdx.x & 63) == 0) ws[threadIdx.x >> 6] = s;
  __syncthreads();
  return threadIdx.x ? 0.f : (ws[0] + ws[1]) + (ws[2] + ws[3]);
}

// A wave per row. Latency-bound (a few hundred bytes a row): everything that does
// not depend on another load is asked for first, two entries a lane (K <= 128).
template <typename T>
__global__ __launch_bounds__(kThreads) void top_ce_combine_kernel(TopLogitsCeArgs a, const float *__restrict__ part,
                                                                  int32_t nsplit, int *__restrict__ done) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  const float itau = 1.f / a.tau, c = itau * kLog2e;
  const TeacherWeight weight(a, itau);
  if (row < a.N) {
    const T *xr = static_cast<const T *>(a.x) + row * a.xs;
    const float2 *pr = reinterpret_cast<const float2 *>(part) + row * nsplit;
    float2 p = {kRowNegInf, 0.f};
    if (lane < nsplit) p = pr[lane];
    constexpr int kEach = 2;
    int id[kEach];
    float t[kEach], xk[kEach], q[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = lane + 64 * i;
      id[i] = k < a.K ? teacher_id(a, row, k) : -1;
      t[i] = k < a.K ? teacher_value(a, row, k) : kRowNegInf;
    }
    float norm = a.lse ? a.lse[row] : kRowNegInf;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      xk[i] = id[i] >= 0 ? (float)xr[id[i]] : 0.f;
      t[i] = id[i] >= 0 ? t[i] : kRowNegInf;
    }
    float inv = 1.f;
    if (!a.lse) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) norm = fmaxf(norm, t[i]);
      for (int k = lane + 64 * kEach; k < a.K; k += 64)
        if (teacher_id(a, row, k) >= 0) norm = fmaxf(norm, teacher_value(a, row, k));
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) norm = fmaxf(norm, __shfl_xor(norm, m, 64));
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) q[i] = weight(t[i], id[i], norm);
    if (!a.lse) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < kEach; ++i) s += q[i];
      for (int k = lane + 64 * kEach; k < a.K; k += 64)
        s += weight(teacher_value(a, row, k), teacher_id(a, row, k), norm);
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
      inv = s == 0.f ? 0.f : 1.f / s;
    }
    RowSum st;
    st.merge(p.x, p.y, c);
    for (int sp = lane + 64; sp < nsplit; sp += 64) st.merge(pr[sp].x, pr[sp].y, c);
    merge_lanes(st, c);
    const float d = sum_at_max(st.m, st.d, c), tau2logd = a.tau * a.tau * logf(d);
    float loss = 0.f, Q = 0.f;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = lane + 64 * i;
      q[i] *= inv;
      if (a.q && k < a.K) a.q[row * a.K + k] = q[i];
      Q += q[i];
      loss += loss_term(q[i], xk[i], st.m, a.tau, tau2logd);
    }
    for (int k = lane + 64 * kEach; k < a.K; k += 64) {
      const int at = teacher_id(a, row, k);
      const float w = weight(teacher_value(a, row, k), at, norm) * inv;
      if (a.q) a.q[row * a.K + k] = w;
      Q += w;
      if (at >= 0) loss += loss_term(w, (float)xr[at], st.m, a.tau, tau2logd);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      loss += __shfl_xor(loss, m, 64);
      Q += __shfl_xor(Q, m, 64);
    }
    if (lane == 0) {
      __hip_atomic_store(a.loss + row, loss, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      a.stats[row] = st.m;
      a.stats[a.N + row] = d;
      a.stats[2 * (int64_t)a.N + row] = Q;
    }
  }
  // the workgroup that finishes last adds the rows
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(done, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float s = sum_rows(a.loss, a.N);
  if (threadIdx.x == 0) *a.sum = s;
}

__global__ __launch_bounds__(kThreads) void top_ce_sum_kernel(const float *__restrict__ loss, int32_t N,
                                                              float *__restrict__ sum) {
  const float s = sum_rows(loss, N);
  if (threadIdx.x == 0) *sum = s;
}

// The gradient of the n elements at x to g.
template <int B, bool NT, typename T, typename G>
__device__ __forceinline__ void write_gradient(const G &gradient, const T *x, T *g, int n) {
  constexpr int W = RowElem<T>::W;
  const int tid = threadIdx.x, off = (int)((reinterpret_cast<uintptr_t>(g) & 15) / sizeof(T));
  const int head = min(n, off ? W - off : 0), nvec = (n - head) / W, tail0 = head + nvec * W;
  if (tid < head) g[tid] = (T)gradient((float)x[tid]);
  if (tid < n - tail0) g[tail0 + tid] = (T)gradient((float)x[tail0 + tid]);
  auto put = [&](int i, const float *v) {
    float f[W];
#pragma unroll
    for (int e = 0; e < W; ++e) f[e] = gradient(v[e]);
    i32x4 *out = reinterpret_cast<i32x4 *>(g + head) + i;
    if constexpr (NT) __builtin_nontemporal_store(pack_vec<T>(f), out);
    else *out = pack_vec<T>(f);
  };
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0) {
    vectors_down<B>(reinterpret_cast<const i32x4 *>(x + head), nvec, [&](int i, const i32x4 &v) {
      float f[W];
#pragma unroll
      for (int e = 0; e < W; ++e) f[e] = RowElem<T>::get(v, e);
      put(i, f);
    });
  } else {
    for (int i = tid; i < nvec; i += B) {
      float f[W];
#pragma unroll
      for (int e = 0; e < W; ++e) f[e] = (float)x[head + i * W + e];
      put(i, f);
    }
  }
}

// Walks the columns as the forward does, from the end: what the last-level cache
// still holds of x are its last columns.
template <typename T, bool NT>
__global__ __launch_bounds__(kThreads) void top_ce_bwd_kernel(TopLogitsCeArgs a, int32_t chunk, int32_t nsplit) {
  __shared__ int ids[kMaxTop];
  __shared__ float qs[kMaxTop];
  const int tid = threadIdx.x;
  const unsigned b = gridDim.x - 1 - blockIdx.x;
  const int64_t row = b / nsplit;
  const int sp = b - row * nsplit, c0 = sp * chunk, c1 = min(a.V, c0 + chunk), n = c1 - c0;
  for (int k = tid; k < a.K; k += kThreads) {
    ids[k] = teacher_id(a, row, k);
    qs[k] = a.q[row * a.K + k];
  }
  const float coef = a.scale * a.tau * (a.go ? *a.go : 1.f);
  const GradRow gradient(a.stats[row], a.stats[a.N + row], a.stats[2 * (int64_t)a.N + row], kLog2e / a.tau, coef);
  const T *xr = static_cast<const T *>(a.x) + row * a.xs + c0;
  T *gr = static_cast<T *>(a.grad) + row * a.gs + c0;
  if (gradient.dead) return write_gradient<kThreads, NT>(ZeroRow(), xr, gr, n);
  write_gradient<kThreads, NT>(gradient, xr, gr, n);
  // the teacher's columns over what was just written
  __syncthreads();
  for (int k = tid; k < a.K; k += kThreads) {
    const int id = ids[k];
    float s;
    if (id >= c0 && id < c1 && owned_sum(ids, qs, a.K, k, &s))
      gr[id - c0] = (T)(gradient((float)xr[id - c0]) - coef * s);
  }
}

// ---- loss and gradient in one kernel --------------------------------------------

// Largest of two values each, and sums of three, over a workgroup of B threads.
template <int B>
__device__ __forceinline__ float2 block_max2(float2 v, float4 *part) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    v.x = fmaxf(v.x, __shfl_xor(v.x, m, 64));
    v.y = fmaxf(v.y, __shfl_xor(v.y, m, 64));
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = {v.x, v.y, 0.f, 0.f};
  __syncthreads();
  v = {part[0].x, part[0].y};
#pragma unroll
  for (int w = 1; w < B / 64; ++w) v = {fmaxf(v.x, part[w].x), fmaxf(v.y, part[w].y)};
  __syncthreads();
  return v;
}
template <int B>
__device__ __forceinline__ float3 block_sum3(float3 v, float4 *part) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    v.x += __shfl_xor(v.x, m, 64);
    v.y += __shfl_xor(v.y, m, 64);
    v.z += __shfl_xor(v.z, m, 64);
  }
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = {v.x, v.y, v.z, 0.f};
  __syncthreads();
  v = {part[0].x, part[0].y, part[0].z};
#pragma unroll
  for (int w = 1; w < B / 64; ++w) v = {v.x + part[w].x, v.y + part[w].y, v.z + part[w].z};
  __syncthreads();
  return v;
}

template <int B>
struct StepShared {
  int ids[kMaxTop];
  float q[kMaxTop];
  float4 part[B / 64];
};

// A teacher's row, entries tid, tid + B, .. a thread.
template <int B>
struct TeacherRow {
  static constexpr int kEach = kMaxTop / B;
  int id[kEach];
  float t[kEach], x[kEach], q[kEach];   // values, the student's logits there, weights

  template <typename T>
  __device__ __forceinline__ void load(const TopLogitsCeArgs &a, int64_t n, const T *xr) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = threadIdx.x + i * B;
      id[i] = k < a.K ? teacher_id(a, n, k) : -1;
      t[i] = id[i] >= 0 ? teacher_value(a, n, k) : kRowNegInf;
      x[i] = id[i] >= 0 ? (float)xr[id[i]] : 0.f;
    }
  }

  // From this thread's part of the student's row xr: the row's loss and what its
  // gradient has in common; the entries in LDS, or (SAVE) all that the backward
  // reads in memory.
  template <bool SAVE, typename T>
  __device__ __forceinline__ GradRow finish(const TopLogitsCeArgs &a, int64_t n, const T *xr, const RowSum &st,
                                            float itau, float c, StepShared<B> &sh) {
    float top = kRowNegInf;
#pragma unroll
    for (int i = 0; i < kEach; ++i) top = fmaxf(top, t[i]);
    const float2 most = block_max2<B>({st.m, top}, sh.part);
    const float m = most.x, norm = a.lse ? a.lse[n] : most.y;
    const TeacherWeight weight(a, itau);
    // d (NaN for m = +inf); of the weights; of their part of the loss
    float3 sums = {far(m, c) ? count_equal<B>(xr, a.V, m) + (m - m) : sum_at(st, m, c), 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      q[i] = weight(t[i], id[i], norm);
      sums.y += q[i];
      sums.z += q[i] == 0.f ? 0.f : x[i] == kRowNegInf ? -kRowNegInf : q[i] * ((m - x[i]) * a.tau);
    }
    sums = block_sum3<B>(sums, sh.part);
    const float d = sum_at_max(m, sums.x, c), inv = a.lse ? 1.f : sums.y == 0.f ? 0.f : 1.f / sums.y;
    const float Q = sums.y * inv;
    if (threadIdx.x == 0)
      a.loss[n] = Q == 0.f ? 0.f : m == kRowNegInf && d == d ? -kRowNegInf : sums.z * inv + a.tau * a.tau * Q * logf(d);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = threadIdx.x + i * B;
      q[i] *= inv;
      if (k >= a.K) continue;
      if constexpr (SAVE) {
        if (a.q) a.q[n * a.K + k] = q[i];
      } else {
        sh.ids[k] = id[i];
        sh.q[k] = q[i];
      }
    }
    if (SAVE && threadIdx.x == 0) {
      a.stats[n] = m;
      a.stats[a.N + n] = d;
      a.stats[2 * (int64_t)a.N + n] = Q;
    }
    return GradRow(m, d, Q, c, a.scale * a.tau);
  }

  // The teacher's columns over the gradient that was just written.
  template <typename T>
  __device__ __forceinline__ void patch(const TopLogitsCeArgs &a, const GradRow &gradient, T *gr,
                                        const StepShared<B> &sh) const {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      float s;
      if (id[i] >= 0 && owned_sum(sh.ids, sh.q, a.K, threadIdx.x + i * B, &s))
        gr[id[i]] = (T)(gradient(x[i]) - a.scale * a.tau * s);
    }
  }
};

constexpr int kAloneThreads = 512;

// The forward with a workgroup a row.
template <typename T>
__global__ __launch_bounds__(kAloneThreads, 8) void top_ce_row_kernel(TopLogitsCeArgs a) {
  __shared__ StepShared<kAloneThreads> sh;
  const int64_t n = blockIdx.x;
  const float itau = 1.f / a.tau, c = itau * kLog2e;
  const T *xr = static_cast<const T *>(a.x) + n * a.xs;
  TeacherRow<kAloneThreads> teacher;
  teacher.load(a, n, xr);
  const RowSum st = sum_elements<kAloneThreads>(xr, a.V, c);
  teacher.template finish<true>(a, n, xr, st, itau, c, sh);
}

// A workgroup a row, whose second reading follows its first, from the end, and comes
// from the caches; four workgroups share a compute unit, so that one's arithmetic
// (the exponentials, twice) runs beside the others' memory. 1 024 x 151 936 bf16:
// 160 us, 933 MB past the L2 at 5.8 TB/s. Holding the row in registers instead, so
// that it is read once, leaves room for one workgroup a compute unit: 191 us, and
// 231 us where that one takes the next row's vectors as it writes this one's.
template <typename T, bool NT>
__global__ __launch_bounds__(kAloneThreads, 8) void top_ce_step_kernel(TopLogitsCeArgs a) {
  __shared__ StepShared<kAloneThreads> sh;
  const int64_t n = blockIdx.x;
  const float itau = 1.f / a.tau, c = itau * kLog2e;
  const T *xr = static_cast<const T *>(a.x) + n * a.xs;
  T *gr = static_cast<T *>(a.grad) + n * a.gs;
  TeacherRow<kAloneThreads> teacher;
  teacher.load(a, n, xr);
  const RowSum st = sum_elements<kAloneThreads>(xr, a.V, c);
  const GradRow gradient = teacher.template finish<false>(a, n, xr, st, itau, c, sh);
  if (gradient.dead) return write_gradient<kAloneThreads, NT>(ZeroRow(), xr, gr, a.V);
  write_gradient<kAloneThreads, NT>(gradient, xr, gr, a.V);
  teacher.patch(a, gradient, gr, sh);
}

namespace {

// Column split of the rows: enough workgroups to fill the chip (about 1024).
void split_plan(int32_t N, int32_t V, int32_t *nsplit, int32_t *chunk) {
  const int64_t want = (1024 + (int64_t)N - 1) / N, most = ((int64_t)V + 4095) / 4096;
  const int64_t s = std::max<int64_t>(1, std::min(want, most));
  const int64_t c = ((V + s - 1) / s + 2047) / 2048 * 2048;
  *chunk = (int32_t)std::min<int64_t>(c, V);
  *nsplit = (int32_t)((V + c - 1) / c);
}

// Bytes of x and its gradient up to which the last-level cache holds both; the
// gradient is then written into it, where the next operation finds it.
constexpr int64_t kCachedBytes = 200 << 20;
template <typename T>
bool past_cache(const TopLogitsCeArgs &a) { return 2 * (int64_t)a.N * a.V * (int64_t)sizeof(T) > kCachedBytes; }

// Rows from which a workgroup a row beats the column ranges and their joining. The
// forward of 128 256 fp16, ranges against rows with their sum: 64 rows 16 and 18 us,
// 96 rows 18.7 and 17.9, 333 rows 33 and 24. The step of 151 936 bf16: 64 rows 31 and
// 35 us, 100 rows 39 and 36, 512 rows 109 and 89.
constexpr int kRowsAlone = 96;

template <typename T>
void fwd_typed(const TopLogitsCeArgs &a, float *ws, hipStream_t st) {
  if (a.N >= kRowsAlone) {
    hipLaunchKernelGGL(top_ce_row_kernel<T>, dim3(a.N), dim3(kAloneThreads), 0, st, a);
    hipLaunchKernelGGL(top_ce_sum_kernel, dim3(1), dim3(kThreads), 0, st, a.loss, a.N, a.sum);
    return;
  }
  int32_t ns, ch;
  split_plan(a.N, a.V, &ns, &ch);
  int *done = reinterpret_cast<int *>(ws);
  hipLaunchKernelGGL((top_ce_partial_kernel<T>), dim3((unsigned)((int64_t)a.N * ns)), dim3(kThreads), 0, st,
                     static_cast<const T *>(a.x), a.xs, a.V, kLog2e / a.tau, ch, ns, ws + 4, done);
  hipLaunchKernelGGL((top_ce_combine_kernel<T>), dim3((a.N + 3) / 4), dim3(kThreads), 0, st, a, ws + 4, ns, done);
}

template <typename T>
void bwd_typed(const TopLogitsCeArgs &a, hipStream_t st) {
  int32_t ns, ch;
  split_plan(a.N, a.V, &ns, &ch);
  const dim3 grid((unsigned)((int64_t)a.N * ns));
  if (past_cache<T>(a)) hipLaunchKernelGGL((top_ce_bwd_kernel<T, true>), grid, dim3(kThreads), 0, st, a, ch, ns);
  else hipLaunchKernelGGL((top_ce_bwd_kernel<T, false>), grid, dim3(kThreads), 0, st, a, ch, ns);
}

template <typename T>
void step_typed(const TopLogitsCeArgs &a, float *ws, hipStream_t st) {
  if (a.N < kRowsAlone) {
    fwd_typed<T>(a, ws, st);
    bwd_typed<T>(a, st);
    return;
  }
  if (past_cache<T>(a)) hipLaunchKernelGGL((top_ce_step_kernel<T, true>), dim3(a.N), dim3(kAloneThreads), 0, st, a);
  else hipLaunchKernelGGL((top_ce_step_kernel<T, false>), dim3(a.N), dim3(kAloneThreads), 0, st, a);
  hipLaunchKernelGGL(top_ce_sum_kernel, dim3(1), dim3(kThreads), 0, st, a.loss, a.N, a.sum);
}

}  // namespace

int64_t top_ce_workspace_floats(int32_t N, int32_t V) {
  int32_t ns, ch;
  split_plan(N, V, &ns, &ch);
  return 4 + 2 * (int64_t)N * ns;
}

void launch_top_ce_fwd(const TopLogitsCeArgs &a, int dtype, float *ws, hipStream_t st) {
  (dtype == kDtF32 ? fwd_typed<float> : dtype == kDtF16 ? fwd_typed<f16_t> : fwd_typed<bf16_t>)(a, ws, st);
}
void launch_top_ce_bwd(const TopLogitsCeArgs &a, int dtype, hipStream_t st) {
  (dtype == kDtF32 ? bwd_typed<float> : dtype == kDtF16 ? bwd_typed<f16_t> : bwd_typed<bf16_t>)(a, st);
}
void launch_top_ce_step(const TopLogitsCeArgs &a, int dtype, float *ws, hipStream_t st) {
  (dtype == kDtF32 ? step_typed<float> : dtype == kDtF16 ? step_typed<f16_t> : step_typed<bf16_t>)(a, ws, st);
}

}  // namespace mga
