// layer_norm.cuh -- what the two directions of the layer norm share.
//
// A row is taken by `lanes` threads (a power of two), each with NV vectors of W
// elements; W is what 16 bytes of the wider type hold.  Three layouts:
// - Streamed rows (up to a few thousand columns, last dimension contiguous): a
//   block goes through rows with stride, the next rows on their way to shared
//   memory while one is computed.  Thread t copies and reads the aligned vectors
//   t, t + lanes, ... that cover the row.  A row may start `shift` elements into
//   its first vector (odd lengths, odd addresses): the stride of rows is a
//   multiple of W, so that a thread's rows all have one shift, and its columns,
//   with their weights and sums in registers, are the same in all of them.
// - VEC: rows at vector alignment, thread t's vectors t, t + lanes, ...
// - Any strides and addresses: single elements t, t + lanes, ...
// Columns are 32-bit numbers: a block holds at most a few thousand, longer rows
// are cut into runs.
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

// Two such sums at once, for rows of one block; `sh` as above, of pairs.  The
// first exchange gives either half of the lanes one of the two to go on with.
__device__ __forceinline__ F2 row_sum2(F2 v, int lanes, F2 *sh) {
  const int lane = threadIdx.x & 31;
  if (lanes == 1) return v;
  int o = lanes < 32 ? lanes >> 1 : 16;
  const int half = o;
  const bool upper = lane & half;
  float s = (upper ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, o);
  for (o >>= 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lanes <= 32) {
    const float t = __shfl_xor_sync(0xffffffffu, s, half);
    return upper ? F2{t, s} : F2{s, t};
  }
  const int warp = threadIdx.x >> 5, warps = lanes >> 5;
  if ((lane & 15) == 0) (upper ? sh[warp].y : sh[warp].x) = s;
  __syncthreads();
  const float4 *two = reinterpret_cast<const float4 *>(sh + (warp & ~(warps - 1)));
  F2 t{0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 8; ++q)
    if (q < warps / 2) {
      const float4 f = two[q];
      t = add2(t, add2({f.x, f.y}, {f.z, f.w}));
    }
  return t;
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

// ---- streamed rows ------------------------------------------------------------------
// A view as a block goes through its rows: `step` elements from one to the next,
// or, where the rows are not at one stride (wraps), each row's own offset.
struct RowWalk {
  Rows r;
  int64_t step;
  bool wraps;
};
inline RowWalk row_walk(const Rows &r, int64_t rows, int64_t step) { return {r, step * r.s1, rows > r.n1}; }
template <class T>
__device__ __forceinline__ T *next_row(T *row, T *view, const RowWalk &w, int64_t i) {
  return w.wraps ? view + row_offset(w.r, i) : row + w.step;
}
// Rows i, i + step, ... below `rows`.
__device__ __forceinline__ int row_count(int64_t i, int64_t rows, int64_t step) {
  return i < rows ? (int)((rows - i + step - 1) / step) : 0;
}

// Column of element e of vector k of a thread whose rows have `shift`.
template <int W>
__device__ __forceinline__ int shifted(int k, int e, int lane, int lanes, int shift) {
  return (k * lanes + lane) * W + e - shift;
}
// Bytes of vector k that a row has (from the vector's start: one that holds the
// row's start is read from there, in the same aligned 16 bytes, so in the same
// allocation; of one that holds its end only the row's are read).
template <int W>
__device__ __forceinline__ int vector_bytes(int k, int cols, int lane, int lanes, int shift, int size) {
  const int left = cols - shifted<W>(k, 0, lane, lanes, shift);
  return (left < 0 ? 0 : left < W ? left : W) * size;
}
// Starts the copies of a row's vectors into a thread's slots, `PITCH` bytes apart;
// what a vector past the row's end does not have of it becomes zero.  Slots of
// vectors that have nothing of it are zero from the start.
template <int W, int NV, int PITCH, class T>
__device__ __forceinline__ void stream_row(unsigned char *slot, const T *vector, int lanes, const int (&bytes)[NV]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (bytes[k]) copy_async_part<W * sizeof(T)>(slot + k * PITCH, vector + k * lanes * W, bytes[k]);
}
template <int W, int NV, int PITCH, class T>
__device__ __forceinline__ void clear_row(unsigned char *slot, const int (&bytes)[NV]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (!bytes[k]) {
#pragma unroll
      for (int q = 0; q < W * (int)sizeof(T); q += 8) *reinterpret_cast<uint2 *>(slot + k * PITCH + q) = make_uint2(0, 0);
    }
}
// Bit e: whether element e of vector k is in the row.
template <int W>
__device__ __forceinline__ unsigned inside(int k, int cols, int lane, int lanes, int shift) {
  unsigned m = 0;
#pragma unroll
  for (int e = 0; e < W; ++e) {
    const int c = shifted<W>(k, e, lane, lanes, shift);
    if (c >= 0 && c < cols) m |= 1u << e;
  }
  return m;
}
// What of its vectors a thread has in a row: bit k of `whole`, all of vector k.
// `edges`: whether a lane of the warp has one that is there in part (the row's
// start or end); `front`: this one has the start, `shift` elements of another row
// before it.
struct Held {
  unsigned whole;
  bool edges, front;
};
template <int W, int NV>
__device__ __forceinline__ Held held(int cols, int lane, int lanes, int shift) {
  Held h{0, false, lane == 0 && shift > 0};
  bool part = false;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const unsigned in = inside<W>(k, cols, lane, lanes, shift);
    if (in == (1u << W) - 1) h.whole |= 1u << k;
    else part |= in != 0;
  }
  h.edges = __any_sync(0xffffffffu, part);
  return h;
}
// A vector out of a thread's slot as pairs.  What of another row is before this
// one's start is made zero first, so that sums need no tests.
template <int W, class T>
__device__ __forceinline__ void take_pairs(const unsigned char *slot, F2 (&v)[W / 2]) {
  float f[W];
  take_vec<W, T>(slot, f);
#pragma unroll
  for (int e = 0; e < W / 2; ++e) v[e] = {f[2 * e], f[2 * e + 1]};
}
template <class T>
__device__ __forceinline__ void clear_front(unsigned char *slot, int shift) {
#pragma unroll 1
  for (int e = 0; e < shift; ++e) reinterpret_cast<T *>(slot)[e] = from_f32<T>(0.0f);
}
// Weight or bias of a thread's columns; `rest` without one and past the row's ends.
template <int W, int NV>
__device__ __forceinline__ void stream_weight(const void *p, int type, int cols, int lane, int lanes, int shift, float rest,
                                              float (&v)[NV][W]) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    if (p && shift == 0 && (uintptr_t)p % 16 == 0 && shifted<W>(k, W, lane, lanes, 0) <= cols) {
      load_kept<W>(p, type, shifted<W>(k, 0, lane, lanes, 0), v[k]);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int c = shifted<W>(k, e, lane, lanes, shift);
        v[k][e] = p && c >= 0 && c < cols ? load_as_f32(p, type, c) : rest;
      }
    }
  }
}
// A row's vectors to memory: whole ones at once, the others element by element.
template <int W, int NV, class T>
__device__ __forceinline__ void stream_store(T *vector, const Held &have, int cols, int lane, int lanes, int shift,
                                             const F2 (&v)[NV][W / 2]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (have.whole >> k & 1) {
      float f[W];
#pragma unroll
      for (int e = 0; e < W / 2; ++e) f[2 * e] = v[k][e].x, f[2 * e + 1] = v[k][e].y;
      store_vec<W>(vector + k * lanes * W, f);
    }
  if (have.edges) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (!(have.whole >> k & 1)) {
        const unsigned in = inside<W>(k, cols, lane, lanes, shift);
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (in >> e & 1) vector[k * lanes * W + e] = from_f32<T>(e & 1 ? v[k][e / 2].y : v[k][e / 2].x);
      }
  }
}

// Rows of views that start equally far into a vector, all of them or a period
// of w rows: where an element lies modulo w.
inline bool same_shift(const void *p, const Rows &r, int p_size, const void *q, const Rows &t, int q_size, int64_t rows, int w) {
  const uint64_t uw = (uint64_t)w;
  return ((uintptr_t)p / p_size - (uintptr_t)q / q_size) % uw == 0 &&
         (rows < 2 || ((uint64_t)(r.s1 - t.s1) % uw == 0 && (rows <= r.n1 && rows <= t.n1)) ||
          ((uint64_t)r.s1 % uw == 0 && (uint64_t)t.s1 % uw == 0 && (rows <= r.n1 || (uint64_t)r.s0 % uw == 0) &&
           (rows <= t.n1 || (uint64_t)t.s0 % uw == 0)));
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

// Lanes of a row: as few as hold it at `most` elements each (`spare` of them
// for a start within a vector), which leaves a thread several loads in flight;
// more, down to one vector each, where that leaves the GPU unfilled (a few rows:
// latency counts).
inline int row_lanes(int64_t rows, int64_t cols, int w, int most, int spare) {
  int lanes = 1;
  cols += spare;
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

// Blocks of streamed rows: a row each, at most `most`, and where they come
// around again a stride of rows that is a multiple of w.
inline int stream_grid(int64_t rows, int64_t groups, int most, int w) {
  const int64_t blocks = (rows + groups - 1) / groups;
  if (blocks <= most) return (int)blocks;
  while (most * groups % w != 0) --most;
  return most;
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
