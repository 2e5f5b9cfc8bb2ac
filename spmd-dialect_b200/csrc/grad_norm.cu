// grad_norm.cu -- the 2-norm over every element of a list of tensors, and the
// factor min(1, max_norm / norm) that clips it.
//
// The sum is held in f64, a thread's and the block's, in a fixed order: the
// result does not depend on timing.  Eight squares at a time are added up in f32
// first (four roundings of 2^-24), because converting each to f64 would take
// longer than reading it; where their sum has left f32's range (it overflows
// from values of 1e19 on, and loses what is below 1e-12) they are taken again in f64.
#include "dtypes.cuh"
#include "internal.h"
#include "tensor_list.cuh"

namespace spmdb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // vectors of eight elements that a thread has in flight
constexpr int kPiece = kThreads * kUnroll * 8;  // elements
constexpr int kMaxGrid = 1184;
constexpr int kTableCap = 1024;

template <int CAP>
struct NormTable {
  int64_t first[CAP + 1];
  const void *p[CAP];
  int64_t n[CAP];
  uint8_t type[CAP];
  int count;
};
constexpr int kSmallCap = 128;

__device__ __forceinline__ double block_sum(double v, double *sh) {
  v = warp_sum_f64(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x < 32) t = warp_sum_f64(threadIdx.x < kThreads / 32 ? sh[threadIdx.x] : 0.0);
  return t;
}

__device__ __forceinline__ void add_squares(const float v[8], double &acc) {
  F2 a = mul2({v[0], v[1]}, {v[0], v[1]}), b = mul2({v[2], v[3]}, {v[2], v[3]});
  a = fma2({v[4], v[5]}, {v[4], v[5]}, a);
  b = fma2({v[6], v[7]}, {v[6], v[7]}, b);
  a = add2(a, b);
  const float s = a.x + a.y;
  if (s >= 0x1p-80f && s <= 0x1.fffffep127f) {
    acc += (double)s;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = fma((double)v[e], (double)v[e], acc);
  }
}

// A piece of a tensor at aligned addresses: all of a thread's vectors are loaded
// before the first is used.
template <class T>
__device__ __forceinline__ void whole_piece(const T *p, double &acc) {
  float v[kUnroll][8];
#pragma unroll
  for (int q = 0; q < kUnroll; ++q) load8(p + 8 * (q * kThreads + (int)threadIdx.x), v[q]);
#pragma unroll
  for (int q = 0; q < kUnroll; ++q) add_squares(v[q], acc);
}
// The rest: what is before the first aligned vector and past the last one element
// a thread.
template <class T>
__device__ __forceinline__ void odd_piece(const T *p, int n, double &acc) {
  int front = (int)((-(uintptr_t)p / sizeof(T)) % 8);
  front = front < n ? front : n;
  const int vectors = (n - front) / 8, back = front + 8 * vectors;
  for (int q = threadIdx.x; q < vectors; q += kThreads) {
    float v[8];
    load8(p + front + 8 * q, v);
    add_squares(v, acc);
  }
  const int t = threadIdx.x;
  const int i = t < front ? t : t >= 8 && t - 8 + back < n ? t - 8 + back : -1;
  if (i >= 0 && t < 16) {
    const double g = (double)to_f32(p[i]);
    acc = fma(g, g, acc);
  }
}
template <class T>
__device__ __forceinline__ void any_piece(const void *tensor, int64_t lo, int64_t left, double &acc) {
  const T *p = static_cast<const T *>(tensor) + lo;
  if (left >= kPiece && (uintptr_t)p % (8 * sizeof(T)) == 0) whole_piece(p, acc);
  else odd_piece(p, left < kPiece ? (int)left : kPiece, acc);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, 4) norm_parts(const __grid_constant__ NormTable<CAP> t, double *parts) {
  __shared__ double sh[kThreads / 32];
  const int64_t pieces = t.first[t.count];
  double acc = 0.0;
  pdl_trigger();
  int k = tensor_of(t.first, t.count, blockIdx.x);
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    while (piece >= t.first[k + 1]) ++k;
    const int64_t lo = (piece - t.first[k]) * kPiece;
    if (t.type[k] == kF32) any_piece<float>(t.p[k], lo, t.n[k] - lo, acc);
    else if (t.type[k] == kF16) any_piece<__half>(t.p[k], lo, t.n[k] - lo, acc);
    else any_piece<__nv_bfloat16>(t.p[k], lo, t.n[k] - lo, acc);
  }
  acc = block_sum(acc, sh);
  pdl_wait();  // for the list's tables before: the last kernel's end is the call's
  if (threadIdx.x == 0) parts[blockIdx.x] = acc;
}

__global__ void __launch_bounds__(kThreads) norm_finish(const double *parts, int count, float max_norm, float *norm,
                                                        float *scale) {
  __shared__ double sh[kThreads / 32];
  double acc = 0.0;
  pdl_wait();
  for (int i = threadIdx.x; i < count; i += kThreads) acc += parts[i];
  acc = block_sum(acc, sh);
  if (threadIdx.x == 0) {
    const double len = sqrt(acc);
    const float f = (float)len;
    *norm = f;
    // A norm that is not finite, as f32 holds it, gives NaN, not 0: 0 times an infinite gradient
    // would be NaN anyway, and a step that sees a NaN factor leaves all as it was.
    if (scale) *scale = isfinite(f) ? (len > (double)max_norm ? (float)((double)max_norm / len) : 1.0f) : nanf("");
  }
}

}  // namespace

size_t grad_norm_workspace_bytes(int count) {
  const size_t tables = count < 1 ? 1 : ((size_t)count + kTableCap - 1) / kTableCap;
  return tables * kMaxGrid * sizeof(double);
}

template <int CAP>
static cudaError_t launch_lists(const GradNormProblem &p, int most, cudaStream_t s) {
  int parts = 0;
  NormTable<CAP> t;
  t.count = 0;
  t.first[0] = 0;
  for (int k = 0; k <= p.count; ++k) {
    if (t.count == CAP || (k == p.count && t.count > 0)) {
      const int64_t pieces = t.first[t.count];
      const int grid = (int)(pieces < most ? pieces : most);
      // Tables after the first, and the sum of the parts, start while the one before ends.
      if (parts == 0) {
        norm_parts<<<grid, kThreads, 0, s>>>(t, p.ws);
        if (cudaError_t e = cudaGetLastError()) return e;
      } else if (cudaError_t e = launch_pdl(norm_parts<CAP>, grid, kThreads, 0, s, t, p.ws + parts)) {
        return e;
      }
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
  if (parts > 0) return launch_pdl(norm_finish, 1, kThreads, 0, s, (const double *)p.ws, parts, p.max_norm, p.norm, p.scale);
  norm_finish<<<1, kThreads, 0, s>>>(p.ws, parts, p.max_norm, p.norm, p.scale);
  return cudaGetLastError();
}

cudaError_t launch_grad_norm(const GradNormProblem &p, cudaStream_t s) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const int most = num_sms(dev) * 8 < kMaxGrid ? num_sms(dev) * 8 : kMaxGrid;
  // A short list's table has fewer bytes to send.
  return p.count <= kSmallCap ? launch_lists<kSmallCap>(p, most, s) : launch_lists<kTableCap>(p, most, s);
}

}  // namespace spmdb200
