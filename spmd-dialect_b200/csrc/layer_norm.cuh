// layer_norm.cuh -- what the two directions of the layer norm share.
//
// A row is taken by `lanes` threads (a power of two in a block, or the threads of
// up to twelve blocks, a cluster), each with NV vectors of W elements; W is what 16
// bytes of the wider type hold.  Two layouts:
// - Vectors: thread t has the aligned vectors t, t + lanes, ... that cover the
//   row, whose last dimension is contiguous.  The row may start `shift` elements
//   into its first vector (odd lengths, odd addresses), an input's elsewhere than
//   the output's (Source).
// - Any strides and addresses: single elements t, t + lanes, ...
// A block that goes through rows with vectors does so with a stride of rows that
// is a multiple of W, so that a thread's rows all have one shift, and its
// columns, with their weights and sums in registers, are the same in all of them.
// Columns are 32-bit numbers: a cluster holds at most some fifty thousand, longer
// rows are cut into runs.
#pragma once

#include <cooperative_groups.h>

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

// Two such sums at once; `sh` as above, of pairs.  The first exchange gives either
// half of the lanes one of the two to go on with.
__device__ __forceinline__ float add_lanes(float v, int from) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o <= from) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int MAXT>
__device__ __forceinline__ F2 row_sum2(F2 v, int lanes, F2 *sh) {
  const int lane = threadIdx.x & 31;
  if (lanes < 32) {
    if (lanes == 1) return v;
    const int half = lanes >> 1;
    const bool upper = lane & half;
    float s = (upper ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, half);
    for (int o = half >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float t = __shfl_xor_sync(0xffffffffu, s, half);
    return upper ? F2{t, s} : F2{s, t};
  }
  const bool upper = lane & 16;
  float s = (upper ? v.y : v.x) + __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
  s = add_lanes(s, 8);
  if (lanes == 32) return {__shfl_sync(0xffffffffu, s, 0), __shfl_sync(0xffffffffu, s, 16)};
  const int warp = threadIdx.x >> 5, warps = lanes >> 5;
  if ((lane & 15) == 0) (upper ? sh[warp].y : sh[warp].x) = s;
  __syncthreads();
  const float4 *two = reinterpret_cast<const float4 *>(sh + (warp & ~(warps - 1)));
  F2 t{0.0f, 0.0f};
  if (warps == MAXT / 32) {
#pragma unroll
    for (int q = 0; q < MAXT / 64; ++q) {
      const float4 f = two[q];
      t = add2(t, add2({f.x, f.y}, {f.z, f.w}));
    }
  } else {
    for (int q = 0; q < warps / 2; ++q) {
      const float4 f = two[q];
      t = add2(t, add2({f.x, f.y}, {f.z, f.w}));
    }
  }
  return t;
}

// Four sums at once, for two rows; `sh` holds four floats per warp.
struct F4 {
  F2 a, b;
};
template <int MAXT>
__device__ __forceinline__ F4 row_sum4(F4 v, int lanes, float4 *sh) {
  const int lane = threadIdx.x & 31;
  const unsigned all = 0xffffffffu;
  if (lanes < 4) {
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      v.a = add2(v.a, {__shfl_xor_sync(all, v.a.x, o), __shfl_xor_sync(all, v.a.y, o)});
      v.b = add2(v.b, {__shfl_xor_sync(all, v.b.x, o), __shfl_xor_sync(all, v.b.y, o)});
    }
    return v;
  }
  auto halves = [&](int half, int quarter) {
    const bool second = lane & half, odd = lane & quarter;
    const F2 keep = second ? v.b : v.a, give = second ? v.a : v.b;
    const F2 two = add2(keep, {__shfl_xor_sync(all, give.x, half), __shfl_xor_sync(all, give.y, half)});
    return (odd ? two.y : two.x) + __shfl_xor_sync(all, odd ? two.x : two.y, quarter);
  };
  auto spread = [&](float s, int base, int half, int quarter) {
    return F4{{__shfl_sync(all, s, base), __shfl_sync(all, s, base | quarter)},
              {__shfl_sync(all, s, base | half), __shfl_sync(all, s, base | half | quarter)}};
  };
  if (lanes < 32) {
    float s = halves(lanes >> 1, lanes >> 2);
    for (int o = lanes >> 3; o > 0; o >>= 1) s += __shfl_xor_sync(all, s, o);
    return spread(s, lane & ~(lanes - 1), lanes >> 1, lanes >> 2);
  }
  const float s = add_lanes(halves(16, 8), 4);
  if (lanes == 32) return spread(s, 0, 16, 8);
  const int warp = threadIdx.x >> 5, warps = lanes >> 5;
  if ((lane & 7) == 0) reinterpret_cast<float *>(sh + warp)[lane >> 3] = s;
  __syncthreads();
  const float4 *row = sh + (warp & ~(warps - 1));
  F4 t{{0.0f, 0.0f}, {0.0f, 0.0f}};
  auto add = [&](int q) {
    const float4 f = row[q];
    t.a = add2(t.a, {f.x, f.y});
    t.b = add2(t.b, {f.z, f.w});
  };
  if (warps == MAXT / 32) {
#pragma unroll
    for (int q = 0; q < MAXT / 32; ++q) add(q);
  } else {
    for (int q = 0; q < warps; ++q) add(q);
  }
  return t;
}

// Sums over a cluster's blocks: every warp puts its own into each block's shared
// memory, where `sh` has an entry for each warp of the cluster.  Two uses in turn of
// two of them need no other barrier.
//
// Twelve blocks at most: the more, the longer a row waits for all of them, and the
// fewer clusters fit the groups of SMs that hold them.  Against the two passes
// below, us: the gradient of 4096 x 40001 f32 554 to 748, bf16 305 to 464, of 4096 x
// 49152 579 to 656 and 314 to 416; the forward pass of 49152 is 370 to some 410 in
// f32 and level in bf16 (243 to some 235).  Sixteen blocks are behind on both: 2048 x
// 65536 bf16 335 forward and 407 backward, two passes 145 and 274 (of 8192 rows).
constexpr int kSpread = 12;
__device__ __forceinline__ float *in_block(float *p, int rank) {
  return cooperative_groups::this_cluster().map_shared_rank(p, rank);
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Four values of a warp into its entry of every block's `sh`.
__device__ __forceinline__ void cluster_share(F4 s, int blocks, int entry, float4 *sh) {
  const int lane = threadIdx.x & 31, which = lane >> 3;
  const float mine = which < 2 ? (which ? s.a.y : s.a.x) : which == 2 ? s.b.x : s.b.y;
#pragma unroll
  for (int o = 0; o < kSpread; o += 8)
    if (const int r = o + (lane & 7); r < blocks) *in_block(reinterpret_cast<float *>(sh + entry) + which, r) = mine;
}
template <int MAXT>
__device__ __forceinline__ F4 cluster_sum4(F4 v, int blocks, int entry, float4 *sh) {
  cluster_share(row_sum4<MAXT>(v, 32, nullptr), blocks, entry, sh);
  cluster_arrive();
  cluster_wait();
  F4 t{{0.0f, 0.0f}, {0.0f, 0.0f}};
  for (int q = threadIdx.x & 31; q < blocks * (MAXT / 32); q += 32) {
    const float4 f = sh[q];
    t.a = add2(t.a, {f.x, f.y});
    t.b = add2(t.b, {f.z, f.w});
  }
  return row_sum4<MAXT>(t, 32, nullptr);
}

// Column of element e of vector k of a thread (relative to a run's first, where a
// row is cut).
template <int W, bool VEC>
__device__ __forceinline__ int column(int k, int e, int lane, int lanes, int shift) {
  return VEC ? (k * lanes + lane) * W + e - shift : (k * W + e) * lanes + lane;
}
// The elements of a row of any stride that a thread has of columns c < high; `rest`
// elsewhere.  `p` is column 0's address.
template <int W, int NV, class T>
__device__ __forceinline__ void load_row(const T *p, int64_t stride, int high, int lane, int lanes, float rest, float (&v)[NV][W]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, false>(k, e, lane, lanes, 0);
      v[k][e] = c < high ? to_f32(p[c * stride]) : rest;
    }
}
template <int W, int NV, class T>
__device__ __forceinline__ void store_row(T *p, int64_t stride, int high, int lane, int lanes, const float (&v)[NV][W]) {
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, false>(k, e, lane, lanes, 0);
      if (c < high) p[c * stride] = from_f32<T>(v[k][e]);
    }
}
// A vector of weight or bias that a thread has of columns low <= c < high, `rest`
// elsewhere and without one.  Column 0 is element `first`.
template <int W, bool VEC>
__device__ __forceinline__ void load_weight(const void *p, int type, int64_t first, int low, int high, int k, int lane, int lanes,
                                            int shift, float rest, float (&v)[W]) {
#pragma unroll
  for (int e = 0; e < W; ++e) v[e] = rest;
  if (!p) return;
  const int j = column<W, VEC>(k, 0, lane, lanes, shift);
  if (VEC && j >= low && j + W <= high && ((first + j) & 3) == 0 && (uintptr_t)p % 16 == 0) {
    load_kept<W>(p, type, first + j, v);
    return;
  }
  auto each = [&](auto *q) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, VEC>(k, e, lane, lanes, shift);
      if (c >= low && c < high) v[e] = to_f32(q[first + c]);
    }
  };
  if (type == kF32) each(static_cast<const float *>(p));
  else if (type == kF16) each(static_cast<const __half *>(p));
  else each(static_cast<const __nv_bfloat16 *>(p));
}

// ---- streamed rows ------------------------------------------------------------------
// A view as a block goes through its rows: `step` elements from one to the next,
// or (WRAPS), where the rows are not at one stride, each row's own offset.
struct RowWalk {
  Rows r;
  int64_t step;
};
inline RowWalk row_walk(const Rows &r, int64_t step) { return {r, step * r.s1}; }
template <bool WRAPS, class T>
__device__ __forceinline__ T *next_row(T *row, T *view, const RowWalk &w, int64_t i) {
  if constexpr (WRAPS) return view + row_offset(w.r, i);
  else return row + w.step;
}
// Rows i, i + step, ... below `rows`.
__device__ __forceinline__ int row_count(int64_t i, int64_t rows, int64_t step) {
  return i < rows ? (int)((rows - i + step - 1) / step) : 0;
}

template <int W>
__device__ __forceinline__ int shifted(int k, int e, int lane, int lanes, int shift) {
  return column<W, true>(k, e, lane, lanes, shift);
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
// Which elements of its vectors a thread has in a row; `full`: whether the warp's
// vectors are all whole; `front`: this thread has the row's start, with `shift`
// elements of another row before it.
template <int W, int NV>
struct Held {
  unsigned in[NV];
  bool full, front;
};
template <int W, int NV>
__device__ __forceinline__ Held<W, NV> held(int cols, int lane, int lanes, int shift) {
  Held<W, NV> h;
  bool whole = true;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    h.in[k] = inside<W>(k, cols, lane, lanes, shift);
    whole &= h.in[k] == (1u << W) - 1;
  }
  h.full = __all_sync(0xffffffffu, whole);
  h.front = lane == 0 && shift > 0 && shift < W;
  return h;
}
// Elements `off` to off + W of two vectors side by side.
template <int W, class T>
__device__ __forceinline__ void take_across(const unsigned char *slot, int off, float (&f)[W]) {
  constexpr int N = W * sizeof(T) / 4;
  unsigned w[2 * N];
#pragma unroll
  for (int q = 0; q < 2 * N; q += N) {
    if constexpr (N == 4) {
      const uint4 u = *reinterpret_cast<const uint4 *>(slot + q * 4);
      w[q] = u.x, w[q + 1] = u.y, w[q + 2] = u.z, w[q + 3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2 *>(slot + q * 4);
      w[q] = u.x, w[q + 1] = u.y;
    }
  }
  const int words = off * (int)sizeof(T) / 4;
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1)
#pragma unroll
    for (int q = 0; q < 2 * N - o; ++q) w[q] = words & o ? w[q + o] : w[q];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const float2 p = unpack(__funnelshift_r(w[q], w[q + 1], 16 * (off & 1)), T{});
      f[2 * q] = p.x, f[2 * q + 1] = p.y;
    }
  } else {
#pragma unroll
    for (int q = 0; q < N; ++q) f[q] = __uint_as_float(w[q]);
  }
}

// An input's vectors on their way through shared memory: the copies of a row's
// vectors go to a thread's slots, kPitch bytes apart.  Vectors are laid out by where
// the output's rows start.  APART: an input's rows may start elsewhere within a
// vector.  Then a thread copies the aligned vector that holds its first element and
// takes its own out of that and the next thread's, `off` elements on; the last
// thread of a warp (or of a narrower row) copies that next vector too, into a slot
// of its own.  Rows have eight lanes at least there.
template <int W, int NV, int THREADS, bool APART, class T>
struct Source {
  static constexpr int kVec = W * sizeof(T), kPitch = (APART ? THREADS / 8 * 9 : THREADS) * kVec, kBytes = NV * kPitch;
  unsigned char *slot;
  int start;  // the first copy's column
  int off, front, lanes;  // front: elements before the row's start in the thread's first vector
  int left[NV], after[APART ? NV : 1];
  bool full, last;

  // Elements of the vector at column c to copy.  One that holds the row's start is
  // read from its own, in the same aligned 16 bytes, so in the same allocation; of one
  // that holds the row's end only the row's are read.
  static __device__ __forceinline__ int to_copy(int c, int cols) { return c <= -W || c >= cols ? 0 : cols - c < W ? cols - c : W; }

  // `row`: column 0; `area`: kBytes for each of `stages`.
  __device__ __forceinline__ void place(const T *row, int cols, int lane, int row_lanes, int shift, const Held<W, NV> &have,
                                        unsigned char *area, int stages, int stage_bytes) {
    const int t = threadIdx.x, width = row_lanes < 32 ? row_lanes : 32;
    lanes = row_lanes;
    off = 0;
    if constexpr (APART) {
      off = (int)((uintptr_t)row / sizeof(T) % W) - shift;
      off += off < 0 ? W : 0;
    }
    start = lane * W - shift - off;
    front = have.front ? shift : 0;
    slot = area + (APART ? t + t / width : t) * kVec;
    full = have.full;
    bool whole = true;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      left[k] = to_copy(start + k * lanes * W, cols);
      whole &= left[k] == W;
    }
    if constexpr (APART) {
      full = __all_sync(0xffffffffu, whole);
      last = (t & (width - 1)) == width - 1;
#pragma unroll
      for (int k = 0; k < NV; ++k) after[k] = last ? to_copy(start + k * lanes * W + W, cols) : 0;
    }
    // Slots of vectors that have nothing of the row are zero from the start.
    for (int s = 0; s < stages; ++s)
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (!left[k]) clear(slot + s * stage_bytes + k * kPitch);
        if constexpr (APART)
          if (last && !after[k]) clear(slot + s * stage_bytes + k * kPitch + kVec);
      }
  }
  static __device__ __forceinline__ void clear(unsigned char *p) {
#pragma unroll
    for (int q = 0; q < kVec; q += 8) *reinterpret_cast<uint2 *>(p + q) = make_uint2(0, 0);
  }
  // The copies of a row into the stage `at` bytes on; what a vector past the row's end
  // does not have of it becomes zero.  `from`: the row's column `start`.
  __device__ __forceinline__ void fetch(int at, const T *from) const {
    if (full) {
#pragma unroll
      for (int k = 0; k < NV; ++k) copy_async<kVec>(slot + at + k * kPitch, from + k * lanes * W);
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (left[k]) copy_async_part<kVec>(slot + at + k * kPitch, from + k * lanes * W, left[k] * (int)sizeof(T));
    }
    if constexpr (APART) {
      if (last) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (after[k]) copy_async_part<kVec>(slot + at + k * kPitch + kVec, from + k * lanes * W + W, after[k] * (int)sizeof(T));
      }
    }
  }
  // Once a stage is there.  What of another row is before this one's start becomes
  // zero, so that sums need no tests (APART: as it is taken).
  __device__ __forceinline__ void arrived(int at) const {
    if constexpr (APART) {
      __syncwarp();  // the next thread's copies are there too
    } else if (!full && front) {
#pragma unroll 1
      for (int e = 0; e < front; ++e) reinterpret_cast<T *>(slot + at)[e] = from_f32<T>(0.0f);
    }
  }
  // Before a stage is filled again.
  static __device__ __forceinline__ void emptied() {
    if constexpr (APART) __syncwarp();
  }
  // Vector k of a stage, as pairs.
  __device__ __forceinline__ void take(int at, int k, F2 (&v)[W / 2]) const {
    float f[W];
    if constexpr (APART) {
      take_across<W, T>(slot + at + k * kPitch, off, f);
      if (k == 0 && front) {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (e < front) f[e] = 0.0f;
      }
    } else {
      take_vec<W, T>(slot + at + k * kPitch, f);
    }
#pragma unroll
    for (int e = 0; e < W / 2; ++e) v[e] = {f[2 * e], f[2 * e + 1]};
  }
};
// A row's vectors to memory: whole ones at once, the others element by element.
template <int W, int NV, class T>
__device__ __forceinline__ void stream_store(T *vector, const Held<W, NV> &have, int lanes, const F2 (&v)[NV][W / 2]) {
  auto put = [&](int k) {
    float f[W];
#pragma unroll
    for (int e = 0; e < W / 2; ++e) f[2 * e] = v[k][e].x, f[2 * e + 1] = v[k][e].y;
    store_vec<W>(vector + k * lanes * W, f);
  };
  if (have.full) {
#pragma unroll
    for (int k = 0; k < NV; ++k) put(k);
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (have.in[k] == (1u << W) - 1) {
        put(k);
      } else if (have.in[k]) {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (have.in[k] >> e & 1) vector[k * lanes * W + e] = from_f32<T>(e & 1 ? v[k][e / 2].y : v[k][e / 2].x);
      }
    }
  }
}
// v - mean inside the row (zero elsewhere, as it was), and the squares' sum.
template <int W, int NV>
__device__ __forceinline__ F2 deviations(F2 (&v)[NV][W / 2], float mean, const Held<W, NV> &have) {
  F2 t{0.0f, 0.0f};
  if (have.full) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        v[k][e] = add2(v[k][e], both(-mean));
        t = fma2(v[k][e], v[k][e], t);
      }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const float off = have.in[k] ? -mean : 0.0f;
      const bool part = have.in[k] && have.in[k] != (1u << W) - 1;
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        v[k][e] = add2(v[k][e], both(off));
        if (part) {
          if (!(have.in[k] >> (2 * e) & 1)) v[k][e].x = 0.0f;
          if (!(have.in[k] >> (2 * e + 1) & 1)) v[k][e].y = 0.0f;
        }
        t = fma2(v[k][e], v[k][e], t);
      }
    }
  }
  return t;
}

// ---- rows longer than a cluster holds ---------------------------------------------------
// They are cut into runs of kRun columns (of the row's vectors).  Two passes over
// as many rows as L2 holds: each run's share of its rows' sums into the workspace,
// with no barrier between rows, then the rest of the work.  Block (run, part) takes every
// parts-th of the rows `first` to `last`, streamed, its columns' weights in
// registers.
constexpr int kCutMost = 16;                // elements of a run in a thread
constexpr int kRun = kThreads * kCutMost;
constexpr int kCutWarps = kThreads / 32;
constexpr int kCutRows = 64;                // rows of a block at most

struct Cut {
  int64_t first, last, runs;
  int parts;
};

// Runs at the most: a start within a vector may need one more.
inline int64_t most_runs(int64_t cols) { return (cols + 7 + kRun - 1) / kRun; }
// Rows of a batch at `bytes` read per column: 88 MB, of the L2's 126 (72 MB: the
// gradient of 1024 x 131072 bf16 297 us, so 273; 56 MB: 5 % slower still).
inline int64_t batch_rows(int64_t rows, int64_t cols, int bytes) {
  if (rows <= 8 || rows * cols * bytes <= (int64_t)100 << 20) return rows;
  const int64_t fit = ((int64_t)88 << 20) / bytes / cols, batch = fit < 8 ? 8 : fit / 8 * 8;
  return batch < rows ? batch : rows;
}
// Parts of a batch that give about `blocks` blocks.  A block's rows have one
// start within a vector: where starts come around after `period` rows, parts are a
// multiple of it, or one row each.
inline int cut_parts(int64_t batch, int64_t runs, int blocks, int period) {
  int64_t p = blocks / runs, least = (batch + kCutRows - 1) / kCutRows;
  if (p < least) p = least;
  if (period > 1) p = (p + period - 1) / period * period;
  p = p < batch ? p : batch;
  return (int)(p < 1 ? 1 : p);
}
// Rows after which starts within a vector come around.
inline int row_period(const Rows &r, int64_t rows, int w) {
  return rows < 2 || ((uint64_t)r.s1 % w == 0 && (rows <= r.n1 || (uint64_t)r.s0 % w == 0)) ? 1 : w;
}

// A block's place in its cut: rows i, i + parts, ..., `rows` of them, and column 0
// relative to its first vector.
struct CutPlace {
  int64_t run, i;
  int rows;
};
__device__ __forceinline__ CutPlace cut_place(const Cut &cut) {
  const int64_t run = blockIdx.x % cut.runs, i = cut.first + blockIdx.x / cut.runs;
  return {run, i, row_count(i, cut.last, cut.parts)};
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

// Rows whose starts within a vector of w come around after w of them, or sooner.
inline bool steady(const Rows &r, int64_t rows, int w) {
  return r.sc == 1 && (rows <= r.n1 || ((uint64_t)r.s0 % w == 0 && ((uint64_t)r.s1 % w == 0 || r.n1 % w == 0)));
}

inline int device_sms() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? num_sms(dev) : 148;
}
// Shared memory past 48 KB, with a kernel's own arrays of up to 20 KB, has to be
// asked for.
template <class Kernel>
cudaError_t allow_shared(Kernel kernel, int bytes) {
  return bytes <= 28 * 1024 ? cudaSuccess : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
// A call's kernels after its first may start while the one before ends: they
// begin the copies of their inputs, which no kernel of the call writes (dx or y in an
// input's place: other rows of it), and wait for the one before with them on their way.
// Every block waits, so that the last kernel's end is the call's.
template <class... P, class... A>
cudaError_t launch(bool first, void (*kernel)(P...), unsigned grid, unsigned threads, size_t bytes, cudaStream_t s, A... args) {
  if (!first) return launch_pdl(kernel, grid, threads, bytes, s, args...);
  kernel<<<grid, threads, bytes, s>>>(args...);
  return cudaGetLastError();
}
// Blocks of kThreads that hold a row at 16 elements a thread.
inline int spread_blocks(int64_t cols) { return (int)((cols + kThreads * 16 - 1) / (kThreads * 16)); }
// Clusters of `blocks` blocks that run at once.
template <class Kernel>
cudaError_t resident_clusters(Kernel kernel, int blocks, int threads, int bytes, int *clusters) {
  if (blocks > 8)
    if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg);
}
template <class... P, class... A>
cudaError_t launch_clusters(void (*kernel)(P...), int clusters, int blocks, int threads, int bytes, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(clusters * blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
inline unsigned grid_for(int64_t items) { return (unsigned)(items < INT32_MAX ? items : INT32_MAX); }

// Rows whose every vector of w elements is aligned to its size.
inline bool vec_rows(const void *p, const Rows &r, int64_t rows, int size, int w) {
  const uint64_t unit = (uint64_t)w * size;
  return r.sc == 1 && (uintptr_t)p % unit == 0 &&
         (rows < 2 || ((uint64_t)r.s1 * size % unit == 0 && (rows <= r.n1 || (uint64_t)r.s0 * size % unit == 0)));
}

// Lanes of a row: as few as hold it at `most` elements each (with `spare` more
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
// around again a stride of rows that is a multiple of w.  Where fewer than w are
// resident at once (a part of a GPU), w of them take turns.
inline int stream_grid(int64_t rows, int64_t groups, int most, int w) {
  if (most < w) most = w;
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
