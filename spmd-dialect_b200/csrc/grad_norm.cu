// grad_norm.cu -- the 2-norm over every element of a list of tensors, and the
// factor min(1, max_norm / norm) that clips it.
//
// Squares are exact products of f32 values held in f64 (an f32 square
// overflows from 1.8e19 on and loses bits below 1e-19), partial sums are one
// f64 per block in a fixed order: the result does not depend on timing.
#include "dtypes.cuh"
#include "internal.h"
#include "tensor_list.cuh"

namespace spmdb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 8192;  // elements
constexpr int kMaxGrid = 592;
constexpr int kTableCap = 1024;

struct NormTable {
  int64_t first[kTableCap + 1];
  const void *p[kTableCap];
  int64_t n[kTableCap];
  uint8_t type[kTableCap];
  int count;
};

__device__ __forceinline__ double block_sum(double v, double *sh) {
  v = warp_sum_f64(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x < 32) t = warp_sum_f64(threadIdx.x < kThreads / 32 ? sh[threadIdx.x] : 0.0);
  return t;
}

__global__ void __launch_bounds__(kThreads) norm_parts(const __grid_constant__ NormTable t, double *parts) {
  __shared__ double sh[kThreads / 32];
  const int64_t pieces = t.first[t.count];
  double acc = 0.0;
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    const int k = tensor_of(t.first, t.count, piece);
    const int64_t lo = (piece - t.first[k]) * kPiece, left = t.n[k] - lo;
    const int64_t hi = lo + (left < kPiece ? left : kPiece);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
      const double g = (double)load_as_f32(t.p[k], t.type[k], i);
      acc = fma(g, g, acc);
    }
  }
  acc = block_sum(acc, sh);
  if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(kThreads) norm_finish(const double *parts, int count, float max_norm, float *norm,
                                                        float *scale) {
  __shared__ double sh[kThreads / 32];
  double acc = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) acc += parts[i];
  acc = block_sum(acc, sh);
  if (threadIdx.x == 0) {
    const double len = sqrt(acc);
    *norm = (float)len;
    // A norm that is not finite gives NaN, not 0: 0 times an infinite gradient
    // would be NaN anyway, and a step that sees a NaN factor leaves all as it was.
    if (scale) *scale = isfinite(len) ? (len > (double)max_norm ? (float)((double)max_norm / len) : 1.0f) : nanf("");
  }
}

}  // namespace

size_t grad_norm_workspace_bytes(int count) {
  const size_t tables = count < 1 ? 1 : ((size_t)count + kTableCap - 1) / kTableCap;
  return tables * kMaxGrid * sizeof(double);
}

cudaError_t launch_grad_norm(const GradNormProblem &p, cudaStream_t s) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const int most = num_sms(dev) * 4 < kMaxGrid ? num_sms(dev) * 4 : kMaxGrid;
  int parts = 0;
  NormTable t;
  t.count = 0;
  t.first[0] = 0;
  for (int k = 0; k <= p.count; ++k) {
    if (t.count == kTableCap || (k == p.count && t.count > 0)) {
      const int64_t pieces = t.first[t.count];
      const int grid = (int)(pieces < most ? pieces : most);
      norm_parts<<<grid, kThreads, 0, s>>>(t, p.ws + parts);
      if (cudaError_t e = cudaGetLastError()) return e;
      parts += grid;
      t.count = 0;
    }
    if (k == p.count) break;
    if (p.sizes[k] == 0) continue;
    t.p[t.count] = p.grads[k];
    t.n[t.count] = p.sizes[k];
    t.type[t.count] = (uint8_t)p.types[k];
    t.first[t.count + 1] = t.first[t.count] + (p.sizes[k] + kPiece - 1) / kPiece;
    ++t.count;
  }
  norm_finish<<<1, kThreads, 0, s>>>(p.ws, parts, p.max_norm, p.norm, p.scale);
  return cudaGetLastError();
}

}  // namespace spmdb200
