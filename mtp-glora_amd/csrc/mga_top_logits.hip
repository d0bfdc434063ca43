// The k largest logits of each row, their columns and the row's log-sum-exp: what
// is kept of a teacher's row for the distillation loss.
//
// One workgroup holds one row in registers (mga_vocab_row.hpp): the row is read
// once, its maximum, the sum of exponentials and the candidates come from passes
// over registers. Bound by the read.
#include "mga_internal.hpp"
#include "mga_vocab_row.hpp"

namespace mga {

template <typename T, int NB>
__global__ __launch_bounds__(kRowThreads) void top_logits_kernel(const T *__restrict__ x, int64_t xs, int32_t V,
                                                                 int32_t k, float itau, T *__restrict__ values,
                                                                 int32_t *__restrict__ ids, float *__restrict__ lse) {
  __shared__ RowShared sh;
  const int64_t n = blockIdx.x;
  Row<T, NB> row;
  row.load(x + n * xs, V);
  const float tmax = thread_max(row);
  if (lse) {
    const float m = block_max(tmax, sh);
    // exp((x - m) / tau); a row of -inf alone: exponents of -inf, not of -inf + inf
    const float c = itau * kLog2e, mc = m == kRowNegInf ? 0.f : m;
    float d = row.ecol >= 0 ? __builtin_amdgcn_exp2f((row.edge - mc) * c) : 0.f;
    row.each_vec([&](const i32x4 &v, int, int) {
#pragma unroll
      for (int e = 0; e < RowElem<T>::W; ++e) d += __builtin_amdgcn_exp2f((RowElem<T>::get(v, e) - mc) * c);
    });
    d = block_sum(d, sh);
    if (threadIdx.x == 0) lse[n] = m == -kRowNegInf ? m : m * itau + logf(d);
  }
  top_list(row, sh, tmax, k);
  if ((int)threadIdx.x < k) {
    const uint64_t r = sh.list[threadIdx.x];
    const int col = rank_col(r);
    values[n * k + threadIdx.x] = x[n * xs + col];
    ids[n * k + threadIdx.x] = col;
  }
}

template <typename T>
static void top_logits_typed(const void *x, int64_t xs, int32_t N, int32_t V, int32_t k, float itau, void *values,
                             int32_t *ids, float *lse, hipStream_t st) {
  with_row_blocks<T>(V, [&](auto nb) {
    hipLaunchKernelGGL((top_logits_kernel<T, decltype(nb)::value>), dim3(N), dim3(kRowThreads), 0, st, (const T *)x,
                       xs, V, k, itau, (T *)values, ids, lse);
  });
}

void launch_top_logits(const void *x, int64_t xs, int32_t N, int32_t V, int dtype, int32_t k, float tau, void *values,
                       int32_t *ids, float *lse, hipStream_t st) {
  auto run = dtype == kDtF32 ? top_logits_typed<float> : dtype == kDtF16 ? top_logits_typed<f16_t> : top_logits_typed<bf16_t>;
  run(x, xs, N, V, k, 1.f / tau, values, ids, lse, st);
}

}  // namespace mga
