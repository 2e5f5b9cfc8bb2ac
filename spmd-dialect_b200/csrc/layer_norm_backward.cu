// layer_norm_backward.cu -- gradients of the layer norm.
//
// With xh = (x - mean) rstd, a = dy w, c1 = sum a / N, c2 = sum a xh / N
//   dx = rstd (a - c1 - xh c2),  dw = sum over rows of dy xh,  db = sum over rows of dy.
// Sums are held in f32; dx, dw and db are rounded once to their type.  Bound by
// memory: x and dy are read once, dx is written.  The sums over rows have a
// fixed order: a block adds up its rows in registers and writes one partial
// row, a second kernel adds up the partial rows.
#include "layer_norm.cuh"

namespace spmdb200 {

namespace {

constexpr int kMost = 16;        // elements of a row in a thread: two sums are held for each too
constexpr int kWideLanes = 512;  // threads of a block for rows past kThreads * kMost columns
constexpr int kMaxParts = 444;   // three blocks per SM
constexpr int kColWidth = 32, kColDepth = 32;
constexpr int64_t kHeld = (int64_t)kWideLanes * kMost;  // columns that a block holds

// What the kernels are given.
template <class TX, class TY>
struct Back {
  const TY *dy;
  Rows gr;
  const TX *x;
  Rows xr;
  const float *mean, *rstd;
  const void *w;
  int wtype;
  TX *dx;  // may be null
  Rows dr;
  float *part;  // column sums, or null
  int64_t rows, cols;
};

// At the end of a block: its groups' column sums, added up in order, into partial
// row blockIdx.x.  col(k, e) is a thread's column (groups may differ in theirs,
// by their shifts); `sums` holds a row for each group.
template <int W, int NV, class Column>
__device__ __forceinline__ void reduce_columns(const float (&sw)[NV][W], const float (&sb)[NV][W], int lanes, int cols,
                                               float *sums, float *part, Column col) {
  const int groups = blockDim.x / lanes;
  float *mine = sums + (int)(threadIdx.x / lanes) * cols;
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int c = col(k, e);
        if (c >= 0 && c < cols) mine[c] = which ? sb[k][e] : sw[k][e];
      }
    __syncthreads();
    for (int j = threadIdx.x; j < cols; j += blockDim.x) {
      float s = 0.0f;
#pragma unroll 8
      for (int q = 0; q < groups; ++q) s += sums[q * cols + j];
      part[(2 * (int64_t)blockIdx.x + which) * cols + j] = s;
    }
  }
}

// Rows that a block's lanes hold, any strides: a block goes through rows with
// stride and keeps the column sums of its rows in registers.
template <class TX, class TY, int W, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT) ln_backward(const __grid_constant__ Back<TX, TY> p, int lanes) {
  extern __shared__ __align__(16) float sums[];
  __shared__ __align__(16) F2 sh[2][32];
  const int lane = threadIdx.x & (lanes - 1), groups = blockDim.x / lanes, group = threadIdx.x / lanes;
  const int cols = (int)p.cols;
  const float inv_n = 1.0f / (float)cols;
  float w[NV][W], sw[NV][W], sb[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<W, false>(p.w, p.wtype, 0, cols, k, lane, lanes, 1.0f, w[k]);
#pragma unroll
    for (int e = 0; e < W; ++e) sw[k][e] = sb[k][e] = 0.0f;
  }
  int turn = 0;
  for (int64_t r = (int64_t)blockIdx.x * groups; r < p.rows; r += (int64_t)gridDim.x * groups, turn ^= 1) {
    const int64_t i = r + group;
    const int n = i < p.rows ? cols : 0;
    const float mean = n ? p.mean[i] : 0.0f, rstd = n ? p.rstd[i] : 0.0f;
    float g[NV][W], x[NV][W];
    load_row<W, NV, false>(p.dy + (n ? row_offset(p.gr, i) : 0), p.gr.sc, n, lane, lanes, 0.0f, g);
    load_row<W, NV, false>(p.x + (n ? row_offset(p.xr, i) : 0), p.xr.sc, n, lane, lanes, mean, x);
    F2 s{0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float xh = (x[k][e] - mean) * rstd, a = g[k][e] * w[k][e];
        sw[k][e] = fmaf(g[k][e], xh, sw[k][e]);
        sb[k][e] += g[k][e];
        s.x += a;
        s.y = fmaf(a, xh, s.y);
        g[k][e] = a;
        x[k][e] = xh;
      }
    if (!p.dx) continue;
    s = row_sum2(s, lanes, sh[turn]);
    const float c1 = s.x * inv_n, c2 = s.y * inv_n;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) g[k][e] = (g[k][e] - c1 - x[k][e] * c2) * rstd;
    if (n) store_row<W, NV, false>(p.dx + row_offset(p.dr, i), p.dr.sc, n, lane, lanes, g);
  }
  if (p.part)
    reduce_columns<W, NV>(sw, sb, lanes, cols, sums, p.part, [&](int k, int e) { return column<W, false>(k, e, lane, lanes); });
}

// Streamed rows (layer_norm.cuh): x and dy of the next rows are on their way
// while one is computed, its mean and rstd with them.
constexpr int kStages = 3;

template <class TX, class TY, int W, int NV, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > kThreads ? 1 : NV * W > 8 ? 2 : 3)
ln_backward_stream(const __grid_constant__ Back<TX, TY> p, const __grid_constant__ RowWalk gr, const __grid_constant__ RowWalk xr,
                   const __grid_constant__ RowWalk dr, int lanes) {
  constexpr int kXBytes = W * sizeof(TX), kGBytes = W * sizeof(TY), kStage = NV * MAXT * (kXBytes + kGBytes);
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) F2 sh[2][32];
  __shared__ float2 stats[kStages][MAXT];  // a group's row, or a warp's where the group is wider
  const int lane = threadIdx.x & (lanes - 1), groups = MAXT / lanes, group = threadIdx.x / lanes;
  const int cols = (int)p.cols, slot = lanes <= 32 ? group : threadIdx.x >> 5;
  const bool first = (threadIdx.x & (lanes <= 32 ? lanes - 1 : 31)) == 0;  // copies the statistics for its group or warp
  const float inv_n = 1.0f / (float)cols;
  const int64_t step = (int64_t)gridDim.x * groups, i = (int64_t)blockIdx.x * groups + group;
  const int mine = row_count(i, p.rows, step), turns = row_count(i - group, p.rows, step);
  const TX *x_from = p.x + (mine ? row_offset(xr.r, i) : 0);
  const int shift = (int)((uintptr_t)x_from / sizeof(TX) % W);
  const int64_t start = lane * W - shift;  // of the thread's first vector in a row
  const TY *g_from = p.dy + (mine ? row_offset(gr.r, i) : 0) + start;
  TX *to = p.dx + (mine && p.dx ? row_offset(dr.r, i) : 0) + start;
  x_from += start;
  const Held have = held<W, NV>(cols, lane, lanes, shift);
  int x_bytes[NV], g_bytes[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    x_bytes[k] = vector_bytes<W>(k, cols, lane, lanes, shift, sizeof(TX));
    g_bytes[k] = vector_bytes<W>(k, cols, lane, lanes, shift, sizeof(TY));
  }
  unsigned char *const x_slots = smem + threadIdx.x * kXBytes, *const g_slots = smem + NV * MAXT * kXBytes + threadIdx.x * kGBytes;
#pragma unroll
  for (int q = 0; q < kStages; ++q) {
    clear_row<W, NV, MAXT * kXBytes, TX>(x_slots + q * kStage, x_bytes);
    clear_row<W, NV, MAXT * kGBytes, TY>(g_slots + q * kStage, g_bytes);
  }
  int stage_in = 0, stage = 0, fetched = 0;
  auto fetch = [&] {
    if (fetched < mine) {
      stream_row<W, NV, MAXT * kXBytes>(x_slots + stage_in * kStage, x_from, lanes, x_bytes);
      stream_row<W, NV, MAXT * kGBytes>(g_slots + stage_in * kStage, g_from, lanes, g_bytes);
      if (first) {
        copy_async<4>(&stats[stage_in][slot].x, p.mean + (i + fetched * step));
        copy_async<4>(&stats[stage_in][slot].y, p.rstd + (i + fetched * step));
      }
    }
    copy_commit();  // empty past the last row, so that the count of groups stays
    ++fetched;
    x_from = next_row(x_from, p.x + start, xr, i + fetched * step);
    g_from = next_row(g_from, p.dy + start, gr, i + fetched * step);
    stage_in = stage_in + 1 == kStages ? 0 : stage_in + 1;
  };
#pragma unroll
  for (int q = 0; q < kStages - 1; ++q) fetch();
  float w[NV][W];
  F2 sw[NV][W / 2], sb[NV][W / 2];
  stream_weight<W, NV>(p.w, p.wtype, cols, lane, lanes, shift, 1.0f, w);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W / 2; ++e) sw[k][e] = sb[k][e] = {0.0f, 0.0f};
  for (int turn = 0; turn < turns; ++turn) {
    fetch();
    copy_wait<kStages - 1>();
    __syncwarp();  // the first lane's copies are there too
    const bool live = turn < mine;
    const float2 stat = stats[stage][slot];
    F2 s1{0.0f, 0.0f}, s2{0.0f, 0.0f}, g[NV][W / 2], x[NV][W / 2];
    if (live) {
      // An element outside the row has g = 0 and a finite x, and adds nothing to any sum.
      unsigned char *const xs = x_slots + stage * kStage, *const gs = g_slots + stage * kStage;
      if (have.front) {
        clear_front<TX>(xs, shift);
        clear_front<TY>(gs, shift);
      }
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        take_pairs<W, TX>(xs + k * (MAXT * kXBytes), x[k]);
        take_pairs<W, TY>(gs + k * (MAXT * kGBytes), g[k]);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) {
          x[k][e] = mul2(add2(x[k][e], both(-stat.x)), both(stat.y));
          sw[k][e] = fma2(g[k][e], x[k][e], sw[k][e]);
          sb[k][e] = add2(g[k][e], sb[k][e]);
          g[k][e] = mul2(g[k][e], {w[k][2 * e], w[k][2 * e + 1]});
          s1 = add2(s1, g[k][e]);
          s2 = fma2(g[k][e], x[k][e], s2);
        }
      }
    }
    __syncwarp();  // every lane has its statistics: the slot may be filled again
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (!p.dx) continue;
    const F2 c = mul2(row_sum2({s1.x + s1.y, s2.x + s2.y}, lanes, sh[turn & 1]), both(-inv_n));
    if (live) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < W / 2; ++e) g[k][e] = mul2(fma2(x[k][e], both(c.y), add2(g[k][e], both(c.x))), both(stat.y));
      stream_store<W, NV>(to, have, cols, lane, lanes, shift, g);
    }
    to = next_row(to, p.dx + start, dr, i + (turn + 1) * step);
  }
  copy_wait<0>();
  if (p.part) {
    float tw[NV][W], tb[NV][W];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        tw[k][e] = e & 1 ? sw[k][e / 2].y : sw[k][e / 2].x;
        tb[k][e] = e & 1 ? sb[k][e / 2].y : sb[k][e / 2].x;
      }
    reduce_columns<W, NV>(tw, tb, lanes, cols, reinterpret_cast<float *>(smem), p.part,
                          [&](int k, int e) { return shifted<W>(k, e, lane, lanes, shift); });
  }
}

// Longer rows, first pass: the two sums of each run of kRun columns of a row.
constexpr int kRun = kThreads * kMost;

template <class TX, class TY, int W, bool VEC>
__global__ void __launch_bounds__(kThreads) ln_row_sums(const __grid_constant__ Back<TX, TY> p, float2 *run_sums, int64_t runs) {
  constexpr int NV = kMost / W;
  __shared__ float sh[2][2][32];
  int turn = 0;
  for (int64_t item = blockIdx.x; item < p.rows * runs; item += gridDim.x, turn ^= 1) {
    const int64_t i = item / runs, first = (item - i * runs) * kRun;
    const int n = p.cols - first < kRun ? (int)(p.cols - first) : kRun;
    const float mean = p.mean[i], rstd = p.rstd[i];
    float g[NV][W], x[NV][W];
    load_row<W, NV, VEC>(p.dy + row_offset(p.gr, i) + first * p.gr.sc, p.gr.sc, n, threadIdx.x, kThreads, 0.0f, g);
    load_row<W, NV, VEC>(p.x + row_offset(p.xr, i) + first * p.xr.sc, p.xr.sc, n, threadIdx.x, kThreads, mean, x);
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float w[W];
      load_weight<W, VEC>(p.w, p.wtype, first, n, k, threadIdx.x, kThreads, 1.0f, w);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float a = g[k][e] * w[e];
        s1 += a;
        s2 = fmaf(a, (x[k][e] - mean) * rstd, s2);
      }
    }
    s1 = row_sum(s1, kThreads, sh[turn][0]);
    s2 = row_sum(s2, kThreads, sh[turn][1]);
    if (threadIdx.x == 0) run_sums[item] = make_float2(s1, s2);
  }
}

// Second pass: block (run, part) takes kRun columns of the part's rows, writes
// dx and keeps the column sums.  x and dy come from L2 where they fit there.
template <class TX, class TY, int W, bool VEC>
__global__ void __launch_bounds__(kThreads)
ln_row_grads(const __grid_constant__ Back<TX, TY> p, const float2 *run_sums, int64_t runs, int parts) {
  constexpr int NV = kMost / W;
  const int64_t run = blockIdx.x % runs, part = blockIdx.x / runs, first = run * kRun;
  const int n = p.cols - first < kRun ? (int)(p.cols - first) : kRun;
  const float inv_n = 1.0f / (float)p.cols;
  float w[NV][W], sw[NV][W], sb[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<W, VEC>(p.w, p.wtype, first, n, k, threadIdx.x, kThreads, 1.0f, w[k]);
#pragma unroll
    for (int e = 0; e < W; ++e) sw[k][e] = sb[k][e] = 0.0f;
  }
  for (int64_t i = part; i < p.rows; i += parts) {
    const float mean = p.mean[i], rstd = p.rstd[i];
    float g[NV][W], x[NV][W];
    load_row<W, NV, VEC>(p.dy + row_offset(p.gr, i) + first * p.gr.sc, p.gr.sc, n, threadIdx.x, kThreads, 0.0f, g);
    load_row<W, NV, VEC>(p.x + row_offset(p.xr, i) + first * p.xr.sc, p.xr.sc, n, threadIdx.x, kThreads, mean, x);
    float c1 = 0.0f, c2 = 0.0f;
    if (p.dx) {  // every warp adds up the row's runs for itself, in one order
      for (int64_t q = threadIdx.x & 31; q < runs; q += 32) {
        const float2 s = run_sums[i * runs + q];
        c1 += s.x;
        c2 += s.y;
      }
      c1 = warp_sum_f32(c1) * inv_n;
      c2 = warp_sum_f32(c2) * inv_n;
    }
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float xh = (x[k][e] - mean) * rstd;
        sw[k][e] = fmaf(g[k][e], xh, sw[k][e]);
        sb[k][e] += g[k][e];
        g[k][e] = (g[k][e] * w[k][e] - c1 - xh * c2) * rstd;
      }
    if (p.dx) store_row<W, NV, VEC>(p.dx + row_offset(p.dr, i) + first * p.dr.sc, p.dr.sc, n, threadIdx.x, kThreads, g);
  }
  if (!p.part) return;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, VEC>(k, e, threadIdx.x, kThreads);
      if (c < n) {
        p.part[2 * part * p.cols + first + c] = sw[k][e];
        p.part[(2 * part + 1) * p.cols + first + c] = sb[k][e];
      }
    }
}

// dw and db from the partial rows (part p: dw at row 2p, db at row 2p + 1).
__global__ void __launch_bounds__(kColWidth *kColDepth)
ln_finish(const float *__restrict__ part, int parts, int64_t cols, void *dw, void *db, int type) {
  __shared__ float sh[2][kColDepth][kColWidth];
  const int tx = threadIdx.x & (kColWidth - 1), ty = threadIdx.x / kColWidth;
  const int64_t j = (int64_t)blockIdx.x * kColWidth + tx;
  float sw = 0.0f, sb = 0.0f;
  if (j < cols)
#pragma unroll 4
    for (int p = ty; p < parts; p += kColDepth) {
      sw += part[(2 * (int64_t)p) * cols + j];
      sb += part[(2 * (int64_t)p + 1) * cols + j];
    }
  sh[0][ty][tx] = sw;
  sh[1][ty][tx] = sb;
  __syncthreads();
  if (ty < 2 && j < cols) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kColDepth; ++k) s += sh[ty][k][tx];
    void *out = ty == 0 ? dw : db;
    if (out) store_from_f32(out, type, j, s);
  }
}

// ---- launches ---------------------------------------------------------------------
// Partial rows of the column sums for rows that a block holds, and for longer
// ones: there, few parts of few rows each, so that blocks fill the GPU.
int held_parts(int64_t rows, int groups) {
  const int64_t p = (rows + groups - 1) / groups;
  return (int)(p < 1 ? 1 : p < kMaxParts ? p : kMaxParts);
}
int64_t long_runs(int64_t cols) { return (cols + kRun - 1) / kRun; }
int long_parts(int64_t rows, int64_t cols) {
  const int64_t most = (4 * kMaxParts + long_runs(cols) - 1) / long_runs(cols);
  const int64_t p = rows < most ? rows : most;
  return (int)(p < 1 ? 1 : p);
}
size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

template <class TX, class TY, int NV, int MAXT>
cudaError_t backward_rows(const Back<TX, TY> &b, int lanes, int *parts, cudaStream_t s) {
  *parts = held_parts(b.rows, MAXT / lanes);
  ln_backward<TX, TY, kWidth<TX, TY>, NV, MAXT><<<*parts, MAXT, b.part ? MAXT / lanes * b.cols * sizeof(float) : 0, s>>>(b, lanes);
  return cudaGetLastError();
}

template <class TX, class TY, int NV, int MAXT>
cudaError_t stream_rows(const Back<TX, TY> &b, int lanes, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, staged = kStages * NV * MAXT * W * (int)(sizeof(TX) + sizeof(TY));
  const int sums = b.part ? (int)(MAXT / lanes * b.cols * sizeof(float)) : 0, bytes = staged > sums ? staged : sums;
  auto kernel = ln_backward_stream<TX, TY, W, NV, MAXT>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  const int64_t groups = MAXT / lanes;
  const int most = (MAXT > kThreads ? 1 : NV * W > 8 ? 2 : 3) * device_sms();
  *parts = stream_grid(b.rows, groups, most < kMaxParts ? most : kMaxParts, W);
  const int64_t step = *parts * groups;
  kernel<<<*parts, MAXT, bytes, s>>>(b, row_walk(b.gr, b.rows, step), row_walk(b.xr, b.rows, step), row_walk(b.dr, b.rows, step), lanes);
  return cudaGetLastError();
}

template <class TX, class TY, bool VEC>
cudaError_t backward_long(const Back<TX, TY> &b, void *ws, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>;
  const int64_t runs = long_runs(b.cols);
  *parts = long_parts(b.rows, b.cols);
  float2 *run_sums = reinterpret_cast<float2 *>(static_cast<char *>(ws) + round16((size_t)*parts * 2 * b.cols * sizeof(float)));
  if (b.dx) {
    ln_row_sums<TX, TY, W, VEC><<<grid_for(b.rows * runs), kThreads, 0, s>>>(b, run_sums, runs);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  ln_row_grads<TX, TY, W, VEC><<<grid_for(runs * *parts), kThreads, 0, s>>>(b, run_sums, runs, *parts);
  return cudaGetLastError();
}

template <class TX, class TY>
cudaError_t backward_of(const Back<TX, TY> &b, void *ws, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kMost / W;
  const bool even = vec_rows(b.x, b.xr, b.rows, sizeof(TX), W) && vec_rows(b.dy, b.gr, b.rows, sizeof(TY), W) &&
                    (!b.dx || vec_rows(b.dx, b.dr, b.rows, sizeof(TX), W));
  const int spare = even ? 0 : W - 1;
  if (b.cols > kHeld - spare)
    return even && vec_weight(b.w) ? backward_long<TX, TY, true>(b, ws, parts, s) : backward_long<TX, TY, false>(b, ws, parts, s);
  const bool wide = b.cols + spare > kThreads * kMost;
  const int lanes = wide ? kWideLanes : row_lanes(b.rows, b.cols, W, kMost, spare), nv = row_vectors(b.cols + spare, lanes, W);
  if (b.xr.sc == 1 && b.gr.sc == 1 && (!b.dx || b.dr.sc == 1) &&
      same_shift(b.x, b.xr, sizeof(TX), b.dy, b.gr, sizeof(TY), b.rows, W) &&
      (!b.dx || same_shift(b.x, b.xr, sizeof(TX), b.dx, b.dr, sizeof(TX), b.rows, W))) {
    if (wide) return stream_rows<TX, TY, NV, kWideLanes>(b, lanes, parts, s);
    if (nv == 1) return stream_rows<TX, TY, 1, kThreads>(b, lanes, parts, s);
    if (nv < NV) return stream_rows<TX, TY, 2, kThreads>(b, lanes, parts, s);
    return stream_rows<TX, TY, NV, kThreads>(b, lanes, parts, s);
  }
  if (wide) return backward_rows<TX, TY, NV, kWideLanes>(b, lanes, parts, s);
  if (nv == 1) return backward_rows<TX, TY, 1, kThreads>(b, lanes, parts, s);
  if (nv < NV) return backward_rows<TX, TY, 2, kThreads>(b, lanes, parts, s);
  return backward_rows<TX, TY, NV, kThreads>(b, lanes, parts, s);
}

template <class TX, class TY>
cudaError_t backward(const LayerNormProblem &p, cudaStream_t s) {
  const Back<TX, TY> b{static_cast<const TY *>(p.y), p.yr, static_cast<const TX *>(p.x), p.xr, p.mean, p.rstd, p.w, p.wtype,
                       static_cast<TX *>(p.dx), p.dr, p.dw || p.db ? static_cast<float *>(p.ws) : nullptr, p.rows, p.cols};
  int parts = 0;
  if (p.rows > 0) {
    if (cudaError_t e = backward_of<TX, TY>(b, p.ws, &parts, s)) return e;
  }
  if (!b.part) return cudaSuccess;
  const int64_t tiles = (p.cols + kColWidth - 1) / kColWidth;
  ln_finish<<<grid_for(tiles), kColWidth * kColDepth, 0, s>>>(b.part, parts, p.cols, p.dw, p.db, p.dwtype);
  return cudaGetLastError();
}

}  // namespace

size_t layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
  // Rows a few columns short of what a block holds may take either way, as their addresses have it.
  const size_t held = cols <= kHeld ? (size_t)held_parts(rows, 1) * 2 * (size_t)cols * sizeof(float) : 0;
  if (cols <= kHeld - 7) return held;
  const size_t cut = round16((size_t)long_parts(rows, cols) * 2 * (size_t)cols * sizeof(float)) +
                     (size_t)rows * (size_t)long_runs(cols) * sizeof(float2);
  return held > cut ? held : cut;
}

cudaError_t launch_layer_norm_backward(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return backward<decltype(tx), decltype(ty)>(p, s); });
}

}  // namespace spmdb200
