// Adapter projections of rows that follow different adapters: t[row] = A_a x[row].
//
// The second half, y += s_a B_a t, runs in the epilogue of the shared projection's kernels
// (grouped_simt.cu, grouped_tc.cu), so y is written once and t stays in fp32.
#include "grouped.h"

namespace moe {
namespace {

constexpr int kWarps = 8;

// Any type and alignment: one CTA per row, a warp per rank entry, the lanes striding over
// K.  The row comes from L1 after the first warp's pass; A_a is read once per row.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
lora_shrink_simt_kernel(const T* __restrict__ x, const T* __restrict__ a,
                        const int32_t* __restrict__ ids, int K, int rank, int adapters,
                        float* __restrict__ t) {
  const int64_t row = blockIdx.x;
  const int ad = ids[row];
  if (ad < 0 || ad >= adapters) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* xr = x + row * K;
  for (int j = warp; j < rank; j += kWarps) {
    const T* ar = a + (static_cast<int64_t>(ad) * rank + j) * K;
    float sum = 0.f;
#pragma unroll 4
    for (int k = lane; k < K; k += 32) sum = fmaf(to_f(ar[k]), to_f(xr[k]), sum);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) t[row * rank + j] = sum;
  }
}

template <typename T>
cudaError_t shrink_simt(const LoraShrink& l, cudaStream_t s) {
  lora_shrink_simt_kernel<T><<<static_cast<unsigned>(l.rows), kWarps * 32, 0, s>>>(
      static_cast<const T*>(l.x), static_cast<const T*>(l.a), l.ids, l.K, l.rank, l.adapters, l.t);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_lora_shrink_simt(const LoraShrink& l, cudaStream_t s) {
  if (l.dtype == kDtF32) return shrink_simt<float>(l, s);
  if (l.dtype == kDtF16) return shrink_simt<__half>(l, s);
  if (l.dtype == kDtBF16) return shrink_simt<__nv_bfloat16>(l, s);
  return cudaErrorInvalidValue;
}

}  // namespace moe
