// layer_norm.cuh -- what the two directions of the layer norm share.
//
// A row is taken by `lanes` threads (a power of two), each with NV vectors of W
// elements.  W is what 16 bytes of the wider type hold.  VEC: rows at vector
// alignment, thread t's vectors t, t + lanes, ...; otherwise (any strides and
// addresses) single elements t, t + lanes, ...  Columns are 32-bit numbers: a
// block holds at most a few thousand, longer rows are cut into runs.
#pragma once

#include "dtypes.cuh"
#include "internal.h"

namespace spmdb200 {

namespace {

constexpr int kThreads = 256;

template <class TX, class TY>
constexpr int kWidth = sizeof(TX) == 4 || sizeof(TY) == 4 ? 4 : 8;

// Sum over a row's lanes, in a fixed order; each of them gets it.  `sh` holds
// one float per warp of the block, and two uses in turn of two of them need no
// barrier in between.
__device__ __forceinline__ float row_sum(float v, int lanes, float *sh) {
  if (lanes <= 32) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = lanes >> 5;
  v = warp_sum_f32(v);
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  return warp_sum_f32(lane < warps ? sh[(warp & ~(warps - 1)) + lane] : 0.0f);
}

// Which column element e of a thread's vector k is.
template <int W, bool VEC>
__device__ __forceinline__ int column(int k, int e, int lane, int lanes) {
  return VEC ? (k * lanes + lane) * W + e : (k * W + e) * lanes + lane;
}

// A thread's part of a row of n columns; `rest` past the end.
template <int W, int NV, bool VEC, class T>
__device__ __forceinline__ void load_row(const T *p, int64_t stride, int n, int lane, int lanes, float rest, float (&v)[NV][W]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = column<W, VEC>(k, 0, lane, lanes);
    if (VEC && j + W <= n) {
      load_vec<W>(p + j, v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int c = column<W, VEC>(k, e, lane, lanes);
        v[k][e] = c < n ? to_f32(p[c * stride]) : rest;
      }
    }
  }
}
template <int W, int NV, bool VEC, class T>
__device__ __forceinline__ void store_row(T *p, int64_t stride, int n, int lane, int lanes, const float (&v)[NV][W]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = column<W, VEC>(k, 0, lane, lanes);
    if (VEC && j + W <= n) {
      store_vec<W>(p + j, v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int c = column<W, VEC>(k, e, lane, lanes);
        if (c < n) p[c * stride] = from_f32<T>(v[k][e]);
      }
    }
  }
}
// The same of weight or bias, elements `first` on; `rest` without one.
template <int W, bool VEC>
__device__ __forceinline__ void load_weight(const void *p, int type, int64_t first, int n, int k, int lane, int lanes,
                                            float rest, float (&v)[W]) {
  const int j = column<W, VEC>(k, 0, lane, lanes);
  if (VEC && p && j + W <= n) {
    load_kept<W>(p, type, first + j, v);
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, VEC>(k, e, lane, lanes);
      v[e] = p && c < n ? load_as_f32(p, type, first + c) : rest;
    }
  }
}

inline int device_sms() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? num_sms(dev) : 148;
}
inline unsigned grid_for(int64_t items) { return (unsigned)(items < INT32_MAX ? items : INT32_MAX); }

// Rows whose every vector of w elements is aligned to its size.
inline bool vec_rows(const void *p, const Rows &r, int64_t rows, int size, int w) {
  const uint64_t unit = (uint64_t)w * size;
  return r.sc == 1 && (uintptr_t)p % unit == 0 &&
         (rows < 2 || ((uint64_t)r.s1 * size % unit == 0 && (rows <= r.n1 || (uint64_t)r.s0 * size % unit == 0)));
}
inline bool vec_weight(const void *p) { return (uintptr_t)p % 16 == 0; }

// Lanes of a row: as few as hold it at `most` elements each, which leaves a
// thread several loads in flight; more, down to one vector each, where that
// leaves the GPU unfilled (a few rows: latency counts).
inline int row_lanes(int64_t rows, int64_t cols, int w, int most) {
  int lanes = 1;
  while (lanes < kThreads && (int64_t)lanes * most < cols) lanes *= 2;
  const int64_t fill = (int64_t)device_sms() * 1024;
  while (lanes < kThreads && (int64_t)lanes * w < cols && rows * lanes < fill) lanes *= 2;
  return lanes;
}
inline int row_vectors(int64_t cols, int lanes, int w) {
  int nv = 1;
  while ((int64_t)lanes * nv * w < cols) nv *= 2;
  return nv;
}

// The type pairs (x, y): equal, or one of the two f32.
template <class F>
cudaError_t by_types(int xt, int yt, F f) {
  if (xt == kF32 && yt == kF32) return f(float{}, float{});
  if (xt == kF16 && yt == kF16) return f(__half{}, __half{});
  if (xt == kBF16 && yt == kBF16) return f(__nv_bfloat16{}, __nv_bfloat16{});
  if (xt == kF32 && yt == kF16) return f(float{}, __half{});
  if (xt == kF32 && yt == kBF16) return f(float{}, __nv_bfloat16{});
  if (xt == kF16 && yt == kF32) return f(__half{}, float{});
  return f(__nv_bfloat16{}, float{});
}

}  // namespace

}  // namespace spmdb200
