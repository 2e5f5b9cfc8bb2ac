// dtypes.cuh -- element types of the training-step entries (f32, f16, bf16) and
// the conversions, block sums and row views their kernels share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace spmdb200 {

// Codes of the header's SPMDB200_F32 / F16 / BF16.
enum DType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// Rows of a rank 1-3 view whose last dimension is the row: row i starts at
// (i / n1) * s0 + (i % n1) * s1 elements; its elements lie sc apart.
struct Rows {
  int64_t n1, s0, s1, sc;
};

#ifdef __CUDACC__

__device__ __forceinline__ int64_t row_offset(const Rows &r, int64_t i) {
  if (i < r.n1) return i * r.s1;  // every row, where the leading dimensions collapse
  const int64_t a = i / r.n1;
  return a * r.s0 + (i - a * r.n1) * r.s1;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float load_as_f32(const void *p, int type, int64_t i) {
  if (type == kF32) return static_cast<const float *>(p)[i];
  if (type == kF16) return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void *p, int type, int64_t i, float v) {
  if (type == kF32) static_cast<float *>(p)[i] = v;
  else if (type == kF16) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

#endif  // __CUDACC__

}  // namespace spmdb200
