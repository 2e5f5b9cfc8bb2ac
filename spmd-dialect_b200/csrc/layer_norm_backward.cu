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
  pdl_trigger();
  const int lane = threadIdx.x & (lanes - 1), groups = blockDim.x / lanes, group = threadIdx.x / lanes;
  const int cols = (int)p.cols;
  const float inv_n = 1.0f / (float)cols;
  float w[NV][W], sw[NV][W], sb[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    load_weight<W, false>(p.w, p.wtype, 0, 0, cols, k, lane, lanes, 0, 1.0f, w[k]);
#pragma unroll
    for (int e = 0; e < W; ++e) sw[k][e] = sb[k][e] = 0.0f;
  }
  int turn = 0;
  for (int64_t r = (int64_t)blockIdx.x * groups; r < p.rows; r += (int64_t)gridDim.x * groups, turn ^= 1) {
    const int64_t i = r + group;
    const int n = i < p.rows ? cols : 0;
    const float mean = n ? p.mean[i] : 0.0f, rstd = n ? p.rstd[i] : 0.0f;
    float g[NV][W], x[NV][W];
    load_row<W, NV>(p.dy + (n ? row_offset(p.gr, i) : 0), p.gr.sc, n, lane, lanes, 0.0f, g);
    load_row<W, NV>(p.x + (n ? row_offset(p.xr, i) : 0), p.xr.sc, n, lane, lanes, mean, x);
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
    s = row_sum2<MAXT>(s, lanes, sh[turn]);
    const float c1 = s.x * inv_n, c2 = s.y * inv_n;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) g[k][e] = (g[k][e] - c1 - x[k][e] * c2) * rstd;
    if (n) store_row<W, NV>(p.dx + row_offset(p.dr, i), p.dr.sc, n, lane, lanes, g);
  }
  if (p.part)
    reduce_columns<W, NV>(sw, sb, lanes, cols, sums, p.part, [&](int k, int e) { return column<W, false>(k, e, lane, lanes, 0); });
}

// Streamed rows (layer_norm.cuh): x and dy of the next rows are on their way
// while R are computed, their mean and rstd with them.  The row's sums come first,
// then, with x and dy read from shared memory once more, dx and the column sums:
// holding them in registers over the reduction would leave no room for a second
// row, whose instructions fill the reduction's waits.  SPREAD: a row is held by the
// `lanes` threads of a cluster's blocks.
constexpr int kStages = 3;
template <class TX, class TY>
constexpr int kRowsAtOnce = sizeof(TX) + sizeof(TY) <= 6 ? 2 : 1;  // as two blocks' stages fit an SM

template <class TX, class TY, int W, int NV, int MAXT, int R, int STAGES, bool WRAPS, bool APART, bool SPREAD>
__global__ void __launch_bounds__(MAXT, MAXT > kThreads ? 1 : NV * W > 8 ? 2 : 3)
ln_backward_stream(const __grid_constant__ Back<TX, TY> p, const __grid_constant__ RowWalk gr, const __grid_constant__ RowWalk xr,
                   const __grid_constant__ RowWalk dr, int lanes) {
  using InX = Source<W, NV, MAXT, APART, TX>;
  using InG = Source<W, NV, MAXT, APART, TY>;
  constexpr int kRow = InX::kBytes + InG::kBytes, kStage = R * kRow;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) float4 sh[2][SPREAD ? kSpread * MAXT / 32 : 32];
  constexpr int kSlots = SPREAD || MAXT > kThreads ? MAXT / 32 : APART ? MAXT / 8 : MAXT;
  __shared__ float2 stats[STAGES * R][kSlots];  // a group's row, or a warp's where the group is wider
  const int blocks = SPREAD ? lanes / MAXT : 1, rank = SPREAD ? blockIdx.x % blocks : 0, team = blockIdx.x / blocks;
  const int lane = SPREAD ? rank * MAXT + threadIdx.x : threadIdx.x & (lanes - 1);
  const int groups = SPREAD ? 1 : MAXT / lanes, group = SPREAD ? 0 : threadIdx.x / lanes;
  const int cols = (int)p.cols, slot = lanes <= 32 ? group : threadIdx.x >> 5;
  pdl_trigger();
  if constexpr (SPREAD) cluster_arrive();
  const bool first = (threadIdx.x & (lanes <= 32 ? lanes - 1 : 31)) == 0;  // copies the statistics for its group or warp
  const float inv_n = 1.0f / (float)cols;
  const int64_t step = (int64_t)(gridDim.x / blocks) * groups, i = (int64_t)team * groups + group;
  const int mine = row_count(i, p.rows, step), turns = row_count(i - group, p.rows, step);
  const TX *x_from = p.x + (mine ? row_offset(xr.r, i) : 0);
  const TY *g_from = p.dy + (mine ? row_offset(gr.r, i) : 0);
  TX *to = p.dx + (mine && p.dx ? row_offset(dr.r, i) : 0);
  const int shift = (int)((uintptr_t)(APART && p.dx ? to : x_from) / sizeof(TX) % W);
  const Held<W, NV> have = held<W, NV>(cols, lane, lanes, shift);
  InX in_x;
  InG in_g;
  in_x.place(x_from, cols, lane, lanes, shift, have, smem, STAGES * R, kRow);
  in_g.place(g_from, cols, lane, lanes, shift, have, smem + InX::kBytes, STAGES * R, kRow);
  const int64_t start = lane * W - shift;  // of the thread's first vector in a row
  x_from += in_x.start;
  g_from += in_g.start;
  to += start;
  int stage_in = 0, stage = 0, fetched = 0;
  const float *mean_in = p.mean + i, *rstd_in = p.rstd + i;
  auto fetch = [&] {
    InX::emptied();
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (fetched < mine) {
        in_x.fetch(stage_in * kStage + q * kRow, x_from);
        in_g.fetch(stage_in * kStage + q * kRow, g_from);
        if (first) {
          copy_async<4>(&stats[stage_in * R + q][slot].x, mean_in);
          copy_async<4>(&stats[stage_in * R + q][slot].y, rstd_in);
        }
      }
      ++fetched;
      mean_in += step, rstd_in += step;
      x_from = next_row<WRAPS>(x_from, p.x + in_x.start, xr, i + fetched * step);
      g_from = next_row<WRAPS>(g_from, p.dy + in_g.start, gr, i + fetched * step);
    }
    copy_commit();  // empty past the last row, so that the count of groups stays
    stage_in = stage_in + 1 == STAGES ? 0 : stage_in + 1;
  };
#pragma unroll
  for (int q = 0; q < STAGES - 1; ++q) fetch();
  float w[NV][W];
  F2 sw[NV][W / 2], sb[NV][W / 2];
#pragma unroll
  for (int k = 0; k < NV; ++k) load_weight<W, true>(p.w, p.wtype, 0, 0, cols, k, lane, lanes, shift, 1.0f, w[k]);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W / 2; ++e) sw[k][e] = sb[k][e] = {0.0f, 0.0f};
  if constexpr (SPREAD) cluster_wait();  // the others have begun
  for (int turn = 0; turn < turns; turn += R) {
    fetch();
    copy_wait<STAGES - 1>();
    __syncwarp();  // the first lane's copies are there too
    float2 stat[R];
    F2 c[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      // An element outside the row has g = 0 and x = 0: it adds nothing to any sum, as rstd multiplies a, which is
      // zero there, and not mean, which may take it past f32.  The sums of a row past the last are not used.
      const bool live = turn + q < mine;
      const int here = stage * kStage + q * kRow;
      stat[q] = live ? stats[stage * R + q][slot] : make_float2(0.0f, 0.0f);
      in_x.arrived(here);
      in_g.arrived(here);
      F2 s1{0.0f, 0.0f}, s2{0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        F2 x[W / 2], g[W / 2];
        in_x.take(here, k, x);
        in_g.take(here, k, g);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) {
          const F2 a = mul2(g[e], {w[k][2 * e], w[k][2 * e + 1]});
          s1 = add2(s1, a);
          s2 = fma2(mul2(a, both(stat[q].y)), add2(x[e], both(-stat[q].x)), s2);
        }
      }
      c[q] = {s1.x + s1.y, s2.x + s2.y};
    }
    __syncwarp();  // every lane has its statistics: the slot may be filled again
    if constexpr (SPREAD) {
      const F4 t = cluster_sum4<MAXT>({c[0], c[R - 1]}, blocks, lane >> 5, sh[(turn / R) & 1]);
      c[0] = t.a, c[R - 1] = R == 2 ? t.b : t.a;
    } else if constexpr (R == 2) {
      const F4 t = row_sum4<MAXT>({c[0], c[1]}, lanes, sh[(turn / R) & 1]);
      c[0] = t.a, c[1] = t.b;
    } else {
      c[0] = row_sum2<MAXT>(c[0], lanes, reinterpret_cast<F2 *>(sh[turn & 1]));
    }
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (turn + q < mine) {
        const F2 c1 = both(-c[q].x * inv_n), c2 = both(-c[q].y * inv_n);
        const int here = stage * kStage + q * kRow;
        F2 g[NV][W / 2];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          F2 x[W / 2];
          in_x.take(here, k, x);
          in_g.take(here, k, g[k]);
#pragma unroll
          for (int e = 0; e < W / 2; ++e) {
            const F2 xh = mul2(add2(x[e], both(-stat[q].x)), both(stat[q].y));
            sw[k][e] = fma2(g[k][e], xh, sw[k][e]);
            sb[k][e] = add2(g[k][e], sb[k][e]);
            g[k][e] = mul2(fma2(xh, c2, fma2(g[k][e], {w[k][2 * e], w[k][2 * e + 1]}, c1)), both(stat[q].y));
          }
        }
        if (p.dx) stream_store<W, NV>(to, have, lanes, g);
      }
      to = next_row<WRAPS>(to, p.dx + start, dr, i + (turn + q + 1) * step);
    }
    stage = stage + 1 == STAGES ? 0 : stage + 1;
  }
  copy_wait<0>();
  if constexpr (SPREAD) {  // a column is one thread's
    if (!p.part) return;
    float *const part_w = p.part + 2 * (int64_t)team * cols, *const part_b = part_w + cols;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const int c = shifted<W>(k, e, lane, lanes, shift);
        if (c >= 0 && c < cols) {
          part_w[c] = e & 1 ? sw[k][e / 2].y : sw[k][e / 2].x;
          part_b[c] = e & 1 ? sb[k][e / 2].y : sb[k][e / 2].x;
        }
      }
  } else if (p.part) {
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

// Longer rows (layer_norm.cuh), first pass: each run's share of a row's two sums.
template <class TX, class TY, int W, bool WRAPS, bool APART>
__global__ void __launch_bounds__(kThreads, sizeof(TX) + sizeof(TY) == 4 ? 4 : 2)
ln_shares(const __grid_constant__ Back<TX, TY> p, const __grid_constant__ RowWalk gr, const __grid_constant__ RowWalk xr,
          const __grid_constant__ Cut cut, float2 *shares) {
  constexpr int NV = kCutMost / W;
  using InX = Source<W, NV, kThreads, false, TX>;  // there is no output: as x has it
  using InG = Source<W, NV, kThreads, APART, TY>;
  constexpr int kStage = InX::kBytes + InG::kBytes;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float2 stats[kCutRows], warps[kCutRows][kCutWarps];
  const CutPlace at = cut_place(cut);
  pdl_trigger();
  if (at.rows == 0) return pdl_wait();
  const int lane = threadIdx.x;
  for (int r = lane; r < at.rows; r += kThreads) stats[r] = make_float2(-p.mean[at.i + (int64_t)r * cut.parts], p.rstd[at.i + (int64_t)r * cut.parts]);
  const TX *x_from = p.x + row_offset(xr.r, at.i);
  const int64_t first = at.run * kRun;
  const int begin = (int)((uintptr_t)x_from / sizeof(TX) % W);
  const int low = at.run == 0 ? 0 : -begin, high = p.cols - first < kRun - begin ? (int)(p.cols - first) : kRun - begin;
  const int shift = at.run == 0 ? begin : 0, n = high - low;
  const TY *g_from = p.dy + row_offset(gr.r, at.i);
  const Held<W, NV> have = held<W, NV>(n, lane, kThreads, shift);
  InX in_x;
  InG in_g;
  in_x.place(x_from + first + low, n, lane, kThreads, shift, have, smem, kStages, kStage);
  in_g.place(g_from + first + low, n, lane, kThreads, shift, have, smem + InX::kBytes, kStages, kStage);
  x_from += first + low + in_x.start;
  g_from += first + low + in_g.start;
  int stage_in = 0, stage = 0, fetched = 0;
  auto fetch = [&] {
    InG::emptied();
    if (fetched < at.rows) {
      in_x.fetch(stage_in, x_from);
      in_g.fetch(stage_in, g_from);
    }
    copy_commit();
    ++fetched;
    x_from = next_row<WRAPS>(x_from, p.x + first + low + in_x.start, xr, at.i + (int64_t)fetched * cut.parts);
    g_from = next_row<WRAPS>(g_from, p.dy + first + low + in_g.start, gr, at.i + (int64_t)fetched * cut.parts);
    stage_in = stage_in == (kStages - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kStages - 1; ++q) fetch();
  float w[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k) load_weight<W, true>(p.w, p.wtype, first + low, 0, n, k, lane, kThreads, shift, 1.0f, w[k]);
  __syncthreads();
  for (int turn = 0; turn < at.rows; ++turn) {
    fetch();
    copy_wait<kStages - 1>();
    const float2 stat = stats[turn];
    in_x.arrived(stage);
    in_g.arrived(stage);
    F2 s1{0.0f, 0.0f}, s2{0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      F2 x[W / 2], g[W / 2];
      in_x.take(stage, k, x);
      in_g.take(stage, k, g);
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        const F2 a = mul2(g[e], {w[k][2 * e], w[k][2 * e + 1]});
        s1 = add2(s1, a);
        s2 = fma2(mul2(a, both(stat.y)), add2(x[e], both(stat.x)), s2);
      }
    }
    stage = stage == (kStages - 1) * kStage ? 0 : stage + kStage;
    const F2 s = row_sum2<kThreads>({s1.x + s1.y, s2.x + s2.y}, 32, nullptr);
    if ((lane & 31) == 0) warps[turn][lane >> 5] = make_float2(s.x, s.y);
  }
  copy_wait<0>();
  __syncthreads();
  pdl_wait();  // the shares of the batch before have been read
  if (lane < at.rows) {
    float2 s = warps[lane][0];
#pragma unroll
    for (int k = 1; k < kCutWarps; ++k) s = make_float2(s.x + warps[lane][k].x, s.y + warps[lane][k].y);
    shares[(at.i - cut.first + (int64_t)lane * cut.parts) * cut.runs + at.run] = s;
  }
}

// Second pass: dx and the column sums, which go on from what the batches before
// left in the part's partial row.
template <class TX, class TY, int W, bool WRAPS, bool APART>
__global__ void __launch_bounds__(kThreads, 2)
ln_grads(const __grid_constant__ Back<TX, TY> p, const __grid_constant__ RowWalk gr, const __grid_constant__ RowWalk xr,
         const __grid_constant__ RowWalk dr, const __grid_constant__ Cut cut, const float2 *shares) {
  constexpr int NV = kCutMost / W;
  using InX = Source<W, NV, kThreads, APART, TX>;
  using InG = Source<W, NV, kThreads, APART, TY>;
  constexpr int kStage = InX::kBytes + InG::kBytes;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float4 stats[kCutRows];  // -mean, rstd, -c1, -c2
  const CutPlace at = cut_place(cut);
  pdl_trigger();
  if (at.rows == 0) return pdl_wait();
  const int lane = threadIdx.x;
  const float inv_n = 1.0f / (float)p.cols;
  const TX *x_from = p.x + row_offset(xr.r, at.i);
  TX *to = p.dx + (p.dx ? row_offset(dr.r, at.i) : 0);
  const int64_t first = at.run * kRun, part = blockIdx.x / cut.runs;
  const int begin = (int)((uintptr_t)(APART && p.dx ? to : x_from) / sizeof(TX) % W);
  const int low = at.run == 0 ? 0 : -begin, high = p.cols - first < kRun - begin ? (int)(p.cols - first) : kRun - begin;
  const int shift = at.run == 0 ? begin : 0, n = high - low;
  const TY *g_from = p.dy + row_offset(gr.r, at.i);
  const int64_t start = first + low + lane * W - shift;
  const Held<W, NV> have = held<W, NV>(n, lane, kThreads, shift);
  InX in_x;
  InG in_g;
  in_x.place(x_from + first + low, n, lane, kThreads, shift, have, smem, kStages, kStage);
  in_g.place(g_from + first + low, n, lane, kThreads, shift, have, smem + InX::kBytes, kStages, kStage);
  x_from += first + low + in_x.start;
  g_from += first + low + in_g.start;
  to += start;
  int stage_in = 0, stage = 0, fetched = 0;
  auto fetch = [&] {
    InG::emptied();
    if (fetched < at.rows) {
      in_x.fetch(stage_in, x_from);
      in_g.fetch(stage_in, g_from);
    }
    copy_commit();
    ++fetched;
    x_from = next_row<WRAPS>(x_from, p.x + first + low + in_x.start, xr, at.i + (int64_t)fetched * cut.parts);
    g_from = next_row<WRAPS>(g_from, p.dy + first + low + in_g.start, gr, at.i + (int64_t)fetched * cut.parts);
    stage_in = stage_in == (kStages - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kStages - 1; ++q) fetch();
  float *const part_w = p.part + 2 * part * p.cols + first + low, *const part_b = part_w + p.cols;
  float w[NV][W];
  F2 sw[NV][W / 2], sb[NV][W / 2];
#pragma unroll
  for (int k = 0; k < NV; ++k) load_weight<W, true>(p.w, p.wtype, first + low, 0, n, k, lane, kThreads, shift, 1.0f, w[k]);
  pdl_wait();  // the shares are there, and the partial row
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    float tw[W], tb[W];
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = shifted<W>(k, e, lane, kThreads, shift);
      const bool goes_on = p.part && cut.first > 0 && c >= 0 && c < n;
      tw[e] = goes_on ? part_w[c] : 0.0f;
      tb[e] = goes_on ? part_b[c] : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < W / 2; ++e) sw[k][e] = {tw[2 * e], tw[2 * e + 1]}, sb[k][e] = {tb[2 * e], tb[2 * e + 1]};
  }
  for (int r = lane >> 5; r < at.rows; r += kCutWarps) {  // a warp a row, in one order
    const int64_t i = at.i + (int64_t)r * cut.parts;
    float c1 = 0.0f, c2 = 0.0f;
    if (p.dx)
      for (int64_t q = lane & 31; q < cut.runs; q += 32) {
        const float2 s = shares[(i - cut.first) * cut.runs + q];
        c1 += s.x;
        c2 += s.y;
      }
    c1 = warp_sum_f32(c1);
    c2 = warp_sum_f32(c2);
    if ((lane & 31) == 0) stats[r] = make_float4(-p.mean[i], p.rstd[i], -c1 * inv_n, -c2 * inv_n);
  }
  __syncthreads();
  for (int turn = 0; turn < at.rows; ++turn) {
    fetch();
    copy_wait<kStages - 1>();
    const float4 stat = stats[turn];
    in_x.arrived(stage);
    in_g.arrived(stage);
    F2 g[NV][W / 2];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      F2 x[W / 2];
      in_x.take(stage, k, x);
      in_g.take(stage, k, g[k]);
#pragma unroll
      for (int e = 0; e < W / 2; ++e) {
        const F2 xh = mul2(add2(x[e], both(stat.x)), both(stat.y));
        sw[k][e] = fma2(g[k][e], xh, sw[k][e]);
        sb[k][e] = add2(g[k][e], sb[k][e]);
        g[k][e] = mul2(fma2(xh, both(stat.w), fma2(g[k][e], {w[k][2 * e], w[k][2 * e + 1]}, both(stat.z))), both(stat.y));
      }
    }
    stage = stage == (kStages - 1) * kStage ? 0 : stage + kStage;
    if (p.dx) stream_store<W, NV>(to, have, kThreads, g);
    to = next_row<WRAPS>(to, p.dx + start, dr, at.i + (int64_t)(turn + 1) * cut.parts);
  }
  copy_wait<0>();
  if (!p.part) return;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = shifted<W>(k, e, lane, kThreads, shift);
      if (c >= 0 && c < n) {
        part_w[c] = e & 1 ? sw[k][e / 2].y : sw[k][e / 2].x;
        part_b[c] = e & 1 ? sb[k][e / 2].y : sb[k][e / 2].x;
      }
    }
}

// Longer rows of any strides, the same two passes with single elements and one
// share a block.
template <class TX, class TY, int W>
__global__ void __launch_bounds__(kThreads, 2) ln_strided_shares(const __grid_constant__ Back<TX, TY> p, const __grid_constant__ Cut cut, float2 *shares) {
  constexpr int NV = kCutMost / W;
  __shared__ __align__(16) F2 sh[2][32];
  const CutPlace at = cut_place(cut);
  pdl_trigger();
  pdl_wait();
  const int64_t first = at.run * kRun;
  const int n = p.cols - first < kRun ? (p.cols > first ? (int)(p.cols - first) : 0) : kRun;
  for (int turn = 0; turn < at.rows; ++turn) {
    const int64_t i = at.i + (int64_t)turn * cut.parts;
    const float mean = p.mean[i], rstd = p.rstd[i];
    float g[NV][W], x[NV][W];
    load_row<W, NV>(p.dy + row_offset(p.gr, i) + first * p.gr.sc, p.gr.sc, n, threadIdx.x, kThreads, 0.0f, g);
    load_row<W, NV>(p.x + row_offset(p.xr, i) + first * p.xr.sc, p.xr.sc, n, threadIdx.x, kThreads, mean, x);
    F2 s{0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float w[W];
      load_weight<W, false>(p.w, p.wtype, first, 0, n, k, threadIdx.x, kThreads, 0, 1.0f, w);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float a = g[k][e] * w[e];
        s.x += a;
        s.y = fmaf(a, (x[k][e] - mean) * rstd, s.y);
      }
    }
    s = row_sum2<kThreads>(s, kThreads, sh[turn & 1]);
    if (threadIdx.x == 0) shares[(i - cut.first) * cut.runs + at.run] = make_float2(s.x, s.y);
  }
}

template <class TX, class TY, int W>
__global__ void __launch_bounds__(kThreads, 2) ln_strided_grads(const __grid_constant__ Back<TX, TY> p, const __grid_constant__ Cut cut, const float2 *shares) {
  constexpr int NV = kCutMost / W;
  const CutPlace at = cut_place(cut);
  pdl_trigger();
  pdl_wait();
  if (at.rows == 0) return;
  const int64_t first = at.run * kRun, part = blockIdx.x / cut.runs;
  const int n = p.cols - first < kRun ? (p.cols > first ? (int)(p.cols - first) : 0) : kRun;
  const float inv_n = 1.0f / (float)p.cols;
  float *const part_w = p.part + 2 * part * p.cols + first, *const part_b = part_w + p.cols;
  float sw[NV][W], sb[NV][W];
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, false>(k, e, threadIdx.x, kThreads, 0);
      const bool goes_on = p.part && cut.first > 0 && c < n;
      sw[k][e] = goes_on ? part_w[c] : 0.0f;
      sb[k][e] = goes_on ? part_b[c] : 0.0f;
    }
  for (int turn = 0; turn < at.rows; ++turn) {
    const int64_t i = at.i + (int64_t)turn * cut.parts;
    const float mean = p.mean[i], rstd = p.rstd[i];
    float c1 = 0.0f, c2 = 0.0f;
    if (p.dx) {  // every warp adds up the row's shares for itself, in one order
      for (int64_t q = threadIdx.x & 31; q < cut.runs; q += 32) {
        const float2 s = shares[(i - cut.first) * cut.runs + q];
        c1 += s.x;
        c2 += s.y;
      }
      c1 = warp_sum_f32(c1) * inv_n;
      c2 = warp_sum_f32(c2) * inv_n;
    }
    float g[NV][W], x[NV][W];
    load_row<W, NV>(p.dy + row_offset(p.gr, i) + first * p.gr.sc, p.gr.sc, n, threadIdx.x, kThreads, 0.0f, g);
    load_row<W, NV>(p.x + row_offset(p.xr, i) + first * p.xr.sc, p.xr.sc, n, threadIdx.x, kThreads, mean, x);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float w[W];
      load_weight<W, false>(p.w, p.wtype, first, 0, n, k, threadIdx.x, kThreads, 0, 1.0f, w);
#pragma unroll
      for (int e = 0; e < W; ++e) {
        const float xh = (x[k][e] - mean) * rstd;
        sw[k][e] = fmaf(g[k][e], xh, sw[k][e]);
        sb[k][e] += g[k][e];
        g[k][e] = (g[k][e] * w[e] - c1 - xh * c2) * rstd;
      }
    }
    if (p.dx) store_row<W, NV>(p.dx + row_offset(p.dr, i) + first * p.dr.sc, p.dr.sc, n, threadIdx.x, kThreads, g);
  }
  if (!p.part) return;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int c = column<W, false>(k, e, threadIdx.x, kThreads, 0);
      if (c < n) {
        part_w[c] = sw[k][e];
        part_b[c] = sb[k][e];
      }
    }
}

// dw and db from the partial rows (part p: dw at row 2p, db at row 2p + 1): `depth`
// threads a column, each of them every depth-th part.  It may start while the kernel
// before still writes `part`, which therefore is no read-only memory.
__global__ void __launch_bounds__(1024)
ln_finish(const float *part, int parts, int64_t cols, int depth, void *dw, void *db, int type) {
  __shared__ float sh[2][1024];
  pdl_wait();
  const int width = blockDim.x / depth, tx = threadIdx.x % width, ty = threadIdx.x / width;
  const int64_t j = (int64_t)blockIdx.x * width + tx;
  float sw = 0.0f, sb = 0.0f;
  if (j < cols)
#pragma unroll 4
    for (int p = ty; p < parts; p += depth) {
      sw += part[(2 * (int64_t)p) * cols + j];
      sb += part[(2 * (int64_t)p + 1) * cols + j];
    }
  if (depth > 1) {
    sh[0][threadIdx.x] = sw;
    sh[1][threadIdx.x] = sb;
    __syncthreads();
    if (ty > 0) return;
    for (int k = 1; k < depth; ++k) {
      sw += sh[0][k * width + tx];
      sb += sh[1][k * width + tx];
    }
  }
  if (j >= cols || ty > 0) return;
  if (dw) store_from_f32(dw, type, j, sw);
  if (db) store_from_f32(db, type, j, sb);
}

// ---- launches ---------------------------------------------------------------------
// Partial rows of the column sums for rows that a block holds.
int held_parts(int64_t rows, int groups) {
  const int64_t p = (rows + groups - 1) / groups;
  return (int)(p < 1 ? 1 : p < kMaxParts ? p : kMaxParts);
}
// Blocks of the two passes over longer rows.
constexpr int kShareBlocks = 592, kGradBlocks = 296;
size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

template <class TX, class TY, int NV, int MAXT>
cudaError_t backward_rows(const Back<TX, TY> &b, int lanes, int *parts, cudaStream_t s) {
  *parts = held_parts(b.rows, MAXT / lanes);
  ln_backward<TX, TY, kWidth<TX, TY>, NV, MAXT><<<*parts, MAXT, b.part ? MAXT / lanes * b.cols * sizeof(float) : 0, s>>>(b, lanes);
  return cudaGetLastError();
}

template <class TX, class TY>
bool wraps(const Back<TX, TY> &b) {
  return b.rows > b.xr.n1 || b.rows > b.gr.n1 || (b.dx && b.rows > b.dr.n1);
}

template <class TX, class TY, int NV, int MAXT, bool WRAPS, bool APART>
cudaError_t stream_rows_as(const Back<TX, TY> &b, int lanes, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, R = kRowsAtOnce<TX, TY>, stages = R == 2 ? 2 : kStages;
  constexpr int staged = stages * R * (Source<W, NV, MAXT, APART, TX>::kBytes + Source<W, NV, MAXT, APART, TY>::kBytes);
  const int sums = b.part ? (int)(MAXT / lanes * b.cols * sizeof(float)) : 0, bytes = staged > sums ? staged : sums;
  auto kernel = ln_backward_stream<TX, TY, W, NV, MAXT, R, stages, WRAPS, APART, false>;
  if (cudaError_t e = allow_shared(kernel, bytes)) return e;
  const int64_t groups = MAXT / lanes;
  const int most = (MAXT > kThreads ? 1 : NV * W > 8 ? 2 : 3) * device_sms();
  *parts = stream_grid(b.rows, groups, most < kMaxParts ? most : kMaxParts, W);
  const int64_t step = *parts * groups;
  kernel<<<*parts, MAXT, bytes, s>>>(b, row_walk(b.gr, step), row_walk(b.xr, step), row_walk(b.dr, step), lanes);
  return cudaGetLastError();
}

template <class TX, class TY, int NV, int MAXT, bool APART>
cudaError_t stream_rows(const Back<TX, TY> &b, int lanes, int *parts, cudaStream_t s) {
  if (APART || wraps(b)) return stream_rows_as<TX, TY, NV, MAXT, true, APART>(b, lanes, parts, s);
  return stream_rows_as<TX, TY, NV, MAXT, APART, APART>(b, lanes, parts, s);
}
template <class TX, class TY, bool APART>
cudaError_t backward_streamed(const Back<TX, TY> &b, int spare, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kMost / W;
  if (b.cols + spare > kThreads * kMost) return stream_rows<TX, TY, NV, kWideLanes, APART>(b, kWideLanes, parts, s);
  int lanes = row_lanes(b.rows, b.cols, W, kMost, spare);
  if (APART && lanes < 8) lanes = 8;
  const int nv = row_vectors(b.cols + spare, lanes, W);
  if (nv == 1) return stream_rows<TX, TY, 1, kThreads, APART>(b, lanes, parts, s);
  if (nv < NV) return stream_rows<TX, TY, 2, kThreads, APART>(b, lanes, parts, s);
  return stream_rows<TX, TY, NV, kThreads, APART>(b, lanes, parts, s);
}

// Rows of a cluster's blocks: a column's sums stay one thread's.
template <class TX, class TY, bool WRAPS, bool APART>
cudaError_t backward_spread(const Back<TX, TY> &b, int blocks, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kMost / W, R = kRowsAtOnce<TX, TY>, stages = R == 2 ? 2 : kStages;
  constexpr int bytes = stages * R * (Source<W, NV, kThreads, APART, TX>::kBytes + Source<W, NV, kThreads, APART, TY>::kBytes);
  auto kernel = ln_backward_stream<TX, TY, W, NV, kThreads, R, stages, WRAPS, APART, true>;
  if (cudaError_t e = allow_shared(kernel, bytes)) return e;
  int most = 0;
  if (cudaError_t e = resident_clusters(kernel, blocks, kThreads, bytes, &most)) return e;
  *parts = stream_grid(b.rows, 1, most < kGradBlocks / blocks ? most : kGradBlocks / blocks, APART ? W : row_period(b.xr, b.rows, W));
  return launch_clusters(kernel, *parts, blocks, kThreads, bytes, s, b, row_walk(b.gr, *parts), row_walk(b.xr, *parts),
                         row_walk(b.dr, *parts), blocks * kThreads);
}

// Two passes over each batch of longer rows: shares(first, cut, grid), where dx is
// wanted, and grads(first, cut, grid).
template <class Shares, class Grads>
cudaError_t batches(int64_t rows, int64_t batch, int64_t runs, int parts1, int parts2, bool dx, Shares shares, Grads grads) {
  for (int64_t row = 0; row < rows; row += batch) {
    const int64_t last = row + batch < rows ? row + batch : rows;
    if (dx) {
      if (cudaError_t e = shares(row == 0, Cut{row, last, runs, parts1}, grid_for(runs * parts1))) return e;
    }
    if (cudaError_t e = grads(row == 0 && !dx, Cut{row, last, runs, parts2}, grid_for(runs * parts2))) return e;
  }
  return cudaSuccess;
}
template <class TX, class TY>
float2 *shares_room(const Back<TX, TY> &b, void *ws, int parts) {
  return reinterpret_cast<float2 *>(static_cast<char *>(ws) + round16((size_t)parts * 2 * b.cols * sizeof(float)));
}

template <class TX, class TY, bool WRAPS, bool APART>
cudaError_t backward_cut(const Back<TX, TY> &b, void *ws, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kCutMost / W, g_bytes = Source<W, NV, kThreads, APART, TY>::kBytes;
  constexpr int bytes1 = kStages * (Source<W, NV, kThreads, false, TX>::kBytes + g_bytes);
  constexpr int bytes2 = kStages * (Source<W, NV, kThreads, APART, TX>::kBytes + g_bytes);
  auto first = ln_shares<TX, TY, W, WRAPS, APART>;
  auto second = ln_grads<TX, TY, W, WRAPS, APART>;
  if (cudaError_t e = allow_shared(first, bytes1)) return e;
  if (cudaError_t e = allow_shared(second, bytes2)) return e;
  const int64_t runs = most_runs(b.cols), batch = batch_rows(b.rows, b.cols, sizeof(TX) + sizeof(TY));
  int period = row_period(b.xr, b.rows, W);
  if (APART && (row_period(b.gr, b.rows, W) > 1 || (b.dx && row_period(b.dr, b.rows, W) > 1))) period = W;
  const int parts1 = cut_parts(batch, runs, kShareBlocks, period), parts2 = *parts = cut_parts(batch, runs, kGradBlocks, period);
  float2 *shares = shares_room(b, ws, parts2);
  return batches(
      b.rows, batch, runs, parts1, parts2, b.dx,
      [&](bool at_first, const Cut &cut, unsigned grid) {
        return launch(at_first, first, grid, kThreads, bytes1, s, b, row_walk(b.gr, parts1), row_walk(b.xr, parts1), cut, shares);
      },
      [&](bool at_first, const Cut &cut, unsigned grid) {
        return launch(at_first, second, grid, kThreads, bytes2, s, b, row_walk(b.gr, parts2), row_walk(b.xr, parts2),
                      row_walk(b.dr, parts2), cut, shares);
      });
}

template <class TX, class TY>
cudaError_t backward_cut_strided(const Back<TX, TY> &b, void *ws, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>;
  const int64_t runs = most_runs(b.cols), batch = batch_rows(b.rows, b.cols, sizeof(TX) + sizeof(TY));
  const int parts1 = cut_parts(batch, runs, kShareBlocks, 1), parts2 = *parts = cut_parts(batch, runs, kGradBlocks, 1);
  float2 *shares = shares_room(b, ws, parts2);
  return batches(
      b.rows, batch, runs, parts1, parts2, b.dx,
      [&](bool first, const Cut &cut, unsigned grid) {
        return launch(first, ln_strided_shares<TX, TY, W>, grid, kThreads, 0, s, b, cut, shares);
      },
      [&](bool first, const Cut &cut, unsigned grid) {
        return launch(first, ln_strided_grads<TX, TY, W>, grid, kThreads, 0, s, b, cut, shares);
      });
}

template <class TX, class TY>
cudaError_t backward_of(const Back<TX, TY> &b, void *ws, int *parts, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kMost / W;
  if (steady(b.xr, b.rows, W) && steady(b.gr, b.rows, W) && (!b.dx || steady(b.dr, b.rows, W))) {
    const bool same = same_shift(b.x, b.xr, sizeof(TX), b.dy, b.gr, sizeof(TY), b.rows, W) &&
                      (!b.dx || same_shift(b.x, b.xr, sizeof(TX), b.dx, b.dr, sizeof(TX), b.rows, W));
    const bool whole = b.dx ? vec_rows(b.dx, b.dr, b.rows, sizeof(TX), W) : vec_rows(b.x, b.xr, b.rows, sizeof(TX), W);
    const int spare = whole ? 0 : W - 1;
    if (b.cols + spare <= kHeld) return same ? backward_streamed<TX, TY, false>(b, spare, parts, s) : backward_streamed<TX, TY, true>(b, spare, parts, s);
    if (b.cols + spare <= kSpread * kThreads * kMost) {
      const int blocks = spread_blocks(b.cols + spare);
      if (!same) return backward_spread<TX, TY, true, true>(b, blocks, parts, s);
      return wraps(b) ? backward_spread<TX, TY, true, false>(b, blocks, parts, s) : backward_spread<TX, TY, false, false>(b, blocks, parts, s);
    }
    if (!same) return backward_cut<TX, TY, true, true>(b, ws, parts, s);
    return wraps(b) ? backward_cut<TX, TY, true, false>(b, ws, parts, s) : backward_cut<TX, TY, false, false>(b, ws, parts, s);
  }
  if (b.cols > kHeld) return backward_cut_strided(b, ws, parts, s);
  if (b.cols > kThreads * kMost) return backward_rows<TX, TY, NV, kWideLanes>(b, kWideLanes, parts, s);
  const int lanes = row_lanes(b.rows, b.cols, W, kMost, 0), nv = row_vectors(b.cols, lanes, W);
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
  // Eight parts or so a thread, up to 32 threads a column in blocks of 1024.
  int depth = 1;
  while (depth < 32 && depth * 8 < parts) depth *= 2;
  const int threads = depth < 32 ? 256 : 1024, width = threads / depth;
  return launch(p.rows == 0, ln_finish, grid_for((p.cols + width - 1) / width), threads, 0, s, b.part, parts, p.cols, depth, p.dw,
                p.db, p.dwtype);
}

}  // namespace

size_t layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
  // Rows a few columns short of what a block holds may take either way, as their addresses have it.
  const size_t whole = cols <= kHeld ? (size_t)held_parts(rows, 1) * 2 * (size_t)cols * sizeof(float) : 0;
  if (cols <= kHeld - 7) return whole;
  // The fewest bytes an element leave the most rows to a batch; parts grow with rows and the period.
  const int64_t runs = most_runs(cols), batch = batch_rows(rows, cols, 4);
  const size_t cut = round16((size_t)cut_parts(batch, runs, kGradBlocks, 8) * 2 * (size_t)cols * sizeof(float)) +
                     (size_t)batch * (size_t)runs * sizeof(float2);
  const int64_t teams = cols <= kSpread * kThreads * kMost ? kGradBlocks / spread_blocks(cols) : 0;
  const size_t spread = (size_t)(rows < teams ? rows : teams) * 2 * (size_t)cols * sizeof(float), most = whole > cut ? whole : cut;
  return most > spread ? most : spread;
}

cudaError_t launch_layer_norm_backward(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return backward<decltype(tx), decltype(ty)>(p, s); });
}

}  // namespace spmdb200
