// The k largest logits of each row, their columns and the row's log-sum-exp: what
// is kept of a teacher's row for the distillation loss.
//
// One workgroup takes a row in one pass (mga_vocab_row.hpp): the running maximum
// and sum, and the largest element of each run of vectors, from which the few
// vectors that hold a candidate are known and read again. Two workgroups share a
// compute unit, one's exponentials (152 a thread, 16 cycles a wave each: half of a
// row's time) beside the other's loads: 61 of the 64 registers that leaves a lane, none
// spilled. 1 024 x 151 936 bf16, k = 64: 78 us where call follows call, 4.0 TB/s (a copy
// moves 5.2); under the tracer 80 to 98.
#include "mga_internal.hpp"
#include "mga_vocab_row.hpp"

namespace mga {

template <typename T>
__global__ __launch_bounds__(kRowThreads, 8) void top_logits_kernel(const T *__restrict__ x, int64_t xs, int32_t V,
                                                                    int32_t k, float itau, int32_t group,
                                                                    T *__restrict__ values, int32_t *__restrict__ ids,
                                                                    float *__restrict__ lse) {
  __shared__ RowShared sh;
  const int64_t n = blockIdx.x;
  Row<T> row;
  row.load(x + n * xs, V);
  RowSum st;
  const float c = itau * kLog2e;
  float tmax;
  if (lse) {
    tmax = scan_row<true, 2>(row, sh, group, c, st);
    const float m = block_max(st.m, sh);
    const float d = block_sum(far(m, c) ? count_equal<kRowThreads>(x + n * xs, V, m) : sum_at(st, m, c), sh);
    if (threadIdx.x == 0) lse[n] = m * itau + logf(sum_at_max(m, d, c));
  } else {
    tmax = scan_row<false, 2>(row, sh, group, c, st);
  }
  top_list(row, sh, group, tmax, k);
  if ((int)threadIdx.x < k) {
    const int col = rank_col(sh.list[threadIdx.x]);
    values[n * k + threadIdx.x] = x[n * xs + col];
    ids[n * k + threadIdx.x] = col;
  }
}

template <typename T>
static void top_logits_typed(const void *x, int64_t xs, int32_t N, int32_t V, int32_t k, float itau, void *values,
                             int32_t *ids, float *lse, hipStream_t st) {
  hipLaunchKernelGGL(top_logits_kernel<T>, dim3(N), dim3(kRowThreads), 0, st, (const T *)x, xs, V, k, itau,
                     row_group<T>(V), (T *)values, ids, lse);
}

void launch_top_logits(const void *x, int64_t xs, int32_t N, int32_t V, int dtype, int32_t k, float tau, void *values,
                       int32_t *ids, float *lse, hipStream_t st) {
  auto run = dtype == kDtF32   ? top_logits_typed<float>
             : dtype == kDtF16 ? top_logits_typed<f16_t>
                               : top_logits_typed<bf16_t>;
  run(x, xs, N, V, k, 1.f / tau, values, ids, lse, st);
}

}  // namespace mga
