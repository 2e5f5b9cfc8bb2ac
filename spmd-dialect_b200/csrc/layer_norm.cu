// layer_norm.cu -- layer norm over the last dimension of a rank 1-3 view.
//
//   mean = sum x / N,  var = sum (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  y = xh w + b
// Sums are held in f32; x, w and b are widened exactly, y is rounded once to
// its type.  A few operations an element: bound by memory.  A row's elements
// stay on the SM, so that the variance is taken around the mean from the same
// read.
#include <cooperative_groups.h>

#include "layer_norm.cuh"

namespace cg = cooperative_groups;

namespace spmdb200 {

namespace {

constexpr int kMost = 32;          // elements of a row in a thread of a block of kThreads
constexpr int kWideLanes = 1024;   // longer rows: blocks of so many threads,
constexpr int kWideMost = 16;      // with so many elements each (64 registers a thread)
constexpr int kCluster = 8;        // still longer ones: blocks that share a row
constexpr int64_t kHeld = (int64_t)kThreads * kMost, kWideHeld = (int64_t)kWideLanes * kWideMost;

template <bool CLUSTER>
__device__ __forceinline__ float whole_sum(float v, int lanes, float *sh, float *mine) {
  v = row_sum(v, lanes, sh);
  if constexpr (CLUSTER) {
    cg::cluster_group cluster = cg::this_cluster();
    if (threadIdx.x == 0) *mine = v;
    cluster.sync();
    const int lane = threadIdx.x & 31;
    v = warp_sum_f32(lane < (int)cluster.num_blocks() ? *cluster.map_shared_rank(mine, lane) : 0.0f);
  }
  return v;
}

// Streamed rows (layer_norm.cuh): weight and bias are loaded once a thread.  A
// group of lanes takes R rows at a time, one or two: the two reductions of a row
// are a long chain of waits, and a second row fills them.
constexpr int kStages = 3;
constexpr int kStreamMost = 16;  // elements of a row in a thread

template <class TX, class TY, int W, int NV, int R, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT > kThreads ? 1 : NV * W * R > 8 ? 2 : 3)
ln_forward_stream(const TX *x, const __grid_constant__ RowWalk xr, TY *y, const __grid_constant__ RowWalk yr, const void *w,
                  const void *b, int wtype, int64_t rows, int cols, float eps, float *mean_out, float *rstd_out, int lanes) {
  constexpr int kBytes = W * sizeof(TX), kPitch = MAXT * kBytes, kStage = R * NV * kPitch;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(16) F2 sh[2][32];
  const int lane = threadIdx.x & (lanes - 1), groups = MAXT / lanes, group = threadIdx.x / lanes;
  const float inv_n = 1.0f / (float)cols;
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t i = (int64_t)blockIdx.x * groups + group;
  const int mine = row_count(i, rows, step), turns = row_count(i - group, rows, step);
  const TX *from = x + (mine ? row_offset(xr.r, i) : 0);
  const int shift = (int)((uintptr_t)from / sizeof(TX) % W);
  TY *to = y + (mine ? row_offset(yr.r, i) : 0) + lane * W - shift;
  from += lane * W - shift;
  const Held have = held<W, NV>(cols, lane, lanes, shift);
  int bytes[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) bytes[k] = vector_bytes<W>(k, cols, lane, lanes, shift, sizeof(TX));
  unsigned char *const slots = smem + threadIdx.x * kBytes;
#pragma unroll
  for (int q = 0; q < kStages * R; ++q) clear_row<W, NV, kPitch, TX>(slots + q * (NV * kPitch), bytes);
  int stage_in = 0, stage = 0, fetched = 0;  // stages as offsets
  auto fetch = [&] {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (fetched < mine) stream_row<W, NV, kPitch>(slots + stage_in + q * (NV * kPitch), from, lanes, bytes);
      ++fetched;
      from = next_row(from, x + lane * W - shift, xr, i + fetched * step);
    }
    copy_commit();  // empty past the last row, so that the count of groups stays
    stage_in = stage_in == (kStages - 1) * kStage ? 0 : stage_in + kStage;
  };
#pragma unroll
  for (int q = 0; q < kStages - 1; ++q) fetch();
  float wv[NV][W], bv[NV][W];
  stream_weight<W, NV>(w, wtype, cols, lane, lanes, shift, 1.0f, wv);
  stream_weight<W, NV>(b, wtype, cols, lane, lanes, shift, 0.0f, bv);
  // R sums of a row each, as a pair.
  auto sums = [&](const F2 (&t)[R], F2 *space) {
    if constexpr (R == 2) return row_sum2({t[0].x + t[0].y, t[1].x + t[1].y}, lanes, space);
    else return both(row_sum(t[0].x + t[0].y, lanes, &space->x));
  };
  for (int turn = 0; turn < turns; turn += R) {
    fetch();
    copy_wait<kStages - 1>();
    F2 v[R][NV][W / 2], t[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      unsigned char *const slot = slots + stage + q * (NV * kPitch);
      if (have.front) clear_front<TX>(slot, shift);
      t[q] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        take_pairs<W, TX>(slot + k * kPitch, v[q][k]);
#pragma unroll
        for (int e = 0; e < W / 2; ++e) t[q] = add2(t[q], v[q][k][e]);
      }
    }
    stage = stage == (kStages - 1) * kStage ? 0 : stage + kStage;
    const F2 mean2 = mul2(sums(t, sh[0]), both(inv_n));
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const float mean = q ? mean2.y : mean2.x;
      t[q] = {0.0f, 0.0f};
      if (have.edges) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const unsigned in = inside<W>(k, cols, lane, lanes, shift);
#pragma unroll
          for (int e = 0; e < W / 2; ++e) {  // elements outside the row stay zero
            v[q][k][e] = add2(v[q][k][e], {in >> (2 * e) & 1 ? -mean : 0.0f, in >> (2 * e + 1) & 1 ? -mean : 0.0f});
            t[q] = fma2(v[q][k][e], v[q][k][e], t[q]);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const F2 off = both(have.whole >> k & 1 ? -mean : 0.0f);
#pragma unroll
          for (int e = 0; e < W / 2; ++e) {
            v[q][k][e] = add2(v[q][k][e], off);
            t[q] = fma2(v[q][k][e], v[q][k][e], t[q]);
          }
        }
      }
    }
    const F2 var2 = mul2(sums(t, sh[1]), both(inv_n));
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const float rstd = 1.0f / sqrtf((q ? var2.y : var2.x) + eps);
      if (turn + q < mine) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
          for (int e = 0; e < W / 2; ++e)
            v[q][k][e] = fma2(mul2(v[q][k][e], both(rstd)), {wv[k][2 * e], wv[k][2 * e + 1]}, {bv[k][2 * e], bv[k][2 * e + 1]});
        stream_store<W, NV>(to, have, cols, lane, lanes, shift, v[q]);
        if (lane == 0) {
          if (mean_out) mean_out[i + (turn + q) * step] = q ? mean2.y : mean2.x;
          if (rstd_out) rstd_out[i + (turn + q) * step] = rstd;
        }
      }
      to = next_row(to, y + lane * W - shift, yr, i + (turn + q + 1) * step);
    }
  }
  copy_wait<0>();
}

template <class TX, class TY, int W, int NV, bool VEC, int MAXT, bool CLUSTER>
__global__ void __launch_bounds__(MAXT, MAXT == kThreads ? 3 : 1)
ln_forward(const TX *x, Rows xr, TY *y, Rows yr, const void *w, const void *b, int wtype, int64_t rows, int64_t all_cols,
           float eps, float *mean_out, float *rstd_out, int lanes) {
  __shared__ float sh[2][32];
  __shared__ float mine[2];
  const int lane = threadIdx.x & (lanes - 1);
  const float inv_n = 1.0f / (float)all_cols;
  int64_t first = 0, i = (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes,
          step = (int64_t)gridDim.x * (blockDim.x / lanes);
  int cols = (int)all_cols;
  if constexpr (CLUSTER) {  // each block of a cluster has an equal run of the row's columns
    first = (int64_t)cg::this_cluster().block_rank() * (lanes * NV * W);
    const int64_t left = all_cols - first;
    cols = left < 0 ? 0 : left < lanes * NV * W ? (int)left : lanes * NV * W;
    i = blockIdx.x / cg::this_cluster().num_blocks(), step = gridDim.x / cg::this_cluster().num_blocks();
  }
  // Rows past the last take part in the barriers, with no columns.
  for (int64_t block_row = CLUSTER ? i : i - threadIdx.x / lanes; block_row < rows; block_row += step, i += step) {
    const int n = i < rows ? cols : 0;
    float v[NV][W], s = 0.0f;
    load_row<W, NV, VEC>(x + (n ? row_offset(xr, i) + first * xr.sc : 0), xr.sc, n, lane, lanes, 0.0f, v);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < W; ++e) s += v[k][e];
    const float mean = whole_sum<CLUSTER>(s, lanes, sh[0], &mine[0]) * inv_n;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const bool whole = VEC && column<W, VEC>(k, W - 1, lane, lanes) < n;
#pragma unroll
      for (int e = 0; e < W; ++e) {
        v[k][e] -= mean;
        if (whole || column<W, VEC>(k, e, lane, lanes) < n) s = fmaf(v[k][e], v[k][e], s);
      }
    }
    const float rstd = 1.0f / sqrtf(whole_sum<CLUSTER>(s, lanes, sh[1], &mine[1]) * inv_n + eps);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float wv[W], bv[W];
      load_weight<W, VEC>(w, wtype, first, n, k, lane, lanes, 1.0f, wv);
      load_weight<W, VEC>(b, wtype, first, n, k, lane, lanes, 0.0f, bv);
#pragma unroll
      for (int e = 0; e < W; ++e) v[k][e] = fmaf(v[k][e] * rstd, wv[e], bv[e]);
    }
    store_row<W, NV, VEC>(y + (n ? row_offset(yr, i) + first * yr.sc : 0), yr.sc, n, lane, lanes, v);
    if (lane == 0 && n && first == 0) {
      if (mean_out) mean_out[i] = mean;
      if (rstd_out) rstd_out[i] = rstd;
    }
    if constexpr (CLUSTER) cg::this_cluster().sync();  // the others have read `mine`
  }
}

// Rows longer than a cluster holds: the same cluster reads them twice, the
// second time from L2.  A thread's elements are taken kWideMost at a time; two
// sets' count, mean and sum of squares around it join into those of both.
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(Moments a, Moments b) {
  const float n = a.n + b.n;
  if (n == 0.0f) return a;
  const float d = b.mean - a.mean, share = b.n / n;
  return {n, fmaf(d, share, a.mean), a.m2 + b.m2 + d * d * a.n * share};
}
template <class TX, class TY, int W, bool VEC>
__global__ void __launch_bounds__(kWideLanes)
ln_forward_long(const TX *x, Rows xr, TY *y, Rows yr, const void *w, const void *b, int wtype, int64_t rows, int64_t cols,
                float eps, float *mean_out, float *rstd_out) {
  constexpr int NV = kWideMost / W;
  __shared__ Moments sh[kWideLanes / 32], mine;
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31;
  const int64_t runs = (cols + kWideHeld - 1) / kWideHeld;
  for (int64_t i = blockIdx.x / kCluster; i < rows; i += gridDim.x / kCluster) {
    const TX *px = x + row_offset(xr, i);
    Moments m{0.0f, 0.0f, 0.0f};
    float v[NV][W];
    for (int64_t r = cluster.block_rank(); r < runs; r += kCluster) {
      const int64_t first = r * kWideHeld;
      const int n = cols - first < kWideHeld ? (int)(cols - first) : (int)kWideHeld;
      load_row<W, NV, VEC>(px + first * xr.sc, xr.sc, n, threadIdx.x, kWideLanes, 0.0f, v);
      Moments t{0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e) {
          t.mean += v[k][e];
          t.n += column<W, VEC>(k, e, threadIdx.x, kWideLanes) < n ? 1.0f : 0.0f;
        }
      t.mean /= fmaxf(t.n, 1.0f);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (column<W, VEC>(k, e, threadIdx.x, kWideLanes) < n) t.m2 = fmaf(v[k][e] - t.mean, v[k][e] - t.mean, t.m2);
      m = join(m, t);
    }
    auto over_warp = [](Moments a) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        a = join(a, {__shfl_xor_sync(0xffffffffu, a.n, o), __shfl_xor_sync(0xffffffffu, a.mean, o),
                     __shfl_xor_sync(0xffffffffu, a.m2, o)});
      return a;
    };
    m = over_warp(m);
    if (lane == 0) sh[threadIdx.x >> 5] = m;
    __syncthreads();
    m = over_warp(sh[lane]);
    if (threadIdx.x == 0) mine = m;
    cluster.sync();
    m = over_warp(lane < kCluster ? *cluster.map_shared_rank(&mine, lane) : Moments{0.0f, 0.0f, 0.0f});
    // Lanes join in orders of their own: the first one's result is the row's.
    const float mean = __shfl_sync(0xffffffffu, m.mean, 0);
    const float rstd = 1.0f / sqrtf(__shfl_sync(0xffffffffu, m.m2, 0) / (float)cols + eps);
    TY *py = y + row_offset(yr, i);
    for (int64_t r = cluster.block_rank(); r < runs; r += kCluster) {
      const int64_t first = r * kWideHeld;
      const int n = cols - first < kWideHeld ? (int)(cols - first) : (int)kWideHeld;
      load_row<W, NV, VEC>(px + first * xr.sc, xr.sc, n, threadIdx.x, kWideLanes, 0.0f, v);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        float wv[W], bv[W];
        load_weight<W, VEC>(w, wtype, first, n, k, threadIdx.x, kWideLanes, 1.0f, wv);
        load_weight<W, VEC>(b, wtype, first, n, k, threadIdx.x, kWideLanes, 0.0f, bv);
#pragma unroll
        for (int e = 0; e < W; ++e) v[k][e] = fmaf((v[k][e] - mean) * rstd, wv[e], bv[e]);
      }
      store_row<W, NV, VEC>(py + first * yr.sc, yr.sc, n, threadIdx.x, kWideLanes, v);
    }
    if (threadIdx.x == 0 && cluster.block_rank() == 0) {
      if (mean_out) mean_out[i] = mean;
      if (rstd_out) rstd_out[i] = rstd;
    }
    cluster.sync();  // the others have read `mine`, and sh may be written again
  }
}

// ---- launches ---------------------------------------------------------------------
struct Launch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  Launch(int64_t blocks, int threads, int cluster, cudaStream_t s) {
    cfg.gridDim = dim3(grid_for(blocks < ((int64_t)1 << 30) ? blocks : (int64_t)1 << 30));  // a multiple of the cluster
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
  }
};

template <class TX, class TY, int NV, bool VEC, int MAXT, bool CLUSTER>
cudaError_t forward_rows(const LayerNormProblem &p, int lanes, int cluster, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>;
  const int threads = CLUSTER || lanes > kThreads ? lanes : kThreads;
  const int64_t per_block = threads / lanes;
  const Launch l(CLUSTER ? (p.rows < (1 << 24) ? p.rows : (1 << 24)) * cluster : (p.rows + per_block - 1) / per_block, threads, cluster, s);
  return cudaLaunchKernelEx(&l.cfg, ln_forward<TX, TY, W, NV, VEC, MAXT, CLUSTER>, static_cast<const TX *>(p.x), p.xr,
                            static_cast<TY *>(p.y), p.yr, p.w, p.b, p.wtype, p.rows, p.cols, p.eps, p.mean, p.rstd, lanes);
}

template <class TX, class TY, int NV, int R, int MAXT>
cudaError_t stream_rows(const LayerNormProblem &p, int lanes, int grid, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, bytes = kStages * R * NV * MAXT * W * (int)sizeof(TX);
  auto kernel = ln_forward_stream<TX, TY, W, NV, R, MAXT>;
  if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  const int64_t step = (int64_t)grid * (MAXT / lanes);
  kernel<<<grid, MAXT, bytes, s>>>(static_cast<const TX *>(p.x), row_walk(p.xr, p.rows, step), static_cast<TY *>(p.y),
                                   row_walk(p.yr, p.rows, step), p.w, p.b, p.wtype, p.rows, (int)p.cols, p.eps, p.mean, p.rstd, lanes);
  return cudaGetLastError();
}

// Streamed rows: as many blocks as are resident, or one for each block of rows
// where those are fewer (then one row at a time).
template <class TX, class TY>
cudaError_t forward_streamed(const LayerNormProblem &p, int spare, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>, NV = kStreamMost / W;
  if (p.cols + spare > kThreads * kStreamMost)
    return stream_rows<TX, TY, NV, 1, 2 * kThreads>(p, 2 * kThreads, stream_grid(p.rows, 1, device_sms(), W), s);
  const int lanes = row_lanes(p.rows, p.cols, W, kStreamMost, spare), groups = kThreads / lanes;
  const int nv = row_vectors(p.cols + spare, lanes, W), most = (nv * W > 8 ? 2 : 3) * device_sms();
  const int grid = stream_grid(p.rows, groups, most, W);
  if (nv == 1) return stream_rows<TX, TY, 1, 1, kThreads>(p, lanes, grid, s);
  if (nv < NV) return stream_rows<TX, TY, 2, 1, kThreads>(p, lanes, grid, s);
  if (p.rows <= (int64_t)most * groups) return stream_rows<TX, TY, NV, 1, kThreads>(p, lanes, grid, s);
  return stream_rows<TX, TY, NV, 2, kThreads>(p, lanes, grid, s);
}

template <class TX, class TY, bool VEC>
cudaError_t forward_of(const LayerNormProblem &p, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>;
  if (p.cols > kWideHeld * kCluster) {
    const Launch l((p.rows < (1 << 24) ? p.rows : (1 << 24)) * kCluster, kWideLanes, kCluster, s);
    return cudaLaunchKernelEx(&l.cfg, ln_forward_long<TX, TY, W, VEC>, static_cast<const TX *>(p.x), p.xr,
                              static_cast<TY *>(p.y), p.yr, p.w, p.b, p.wtype, p.rows, p.cols, p.eps, p.mean, p.rstd);
  }
  if (p.cols > kWideHeld) {
    int cluster = 2;
    while (p.cols > kWideHeld * cluster) cluster *= 2;
    return forward_rows<TX, TY, kWideMost / W, VEC, kWideLanes, true>(p, kWideLanes, cluster, s);
  }
  if (p.cols > kHeld) return forward_rows<TX, TY, kWideMost / W, VEC, kWideLanes, false>(p, kWideLanes, 1, s);
  if constexpr (VEC) {  // what is left of shorter rows: weights at odd addresses
    return forward_rows<TX, TY, kMost / W, true, kThreads, false>(p, kThreads, 1, s);
  }
  const int lanes = row_lanes(p.rows, p.cols, W, kMost, 0);
  switch (row_vectors(p.cols, lanes, W)) {
    case 1: return forward_rows<TX, TY, 1, false, kThreads, false>(p, lanes, 1, s);
    case 2: return forward_rows<TX, TY, 2, false, kThreads, false>(p, lanes, 1, s);
    case 4: return forward_rows<TX, TY, 4, false, kThreads, false>(p, lanes, 1, s);
    default: return forward_rows<TX, TY, kMost / W, false, kThreads, false>(p, lanes, 1, s);
  }
}

template <class TX, class TY>
cudaError_t forward(const LayerNormProblem &p, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>;
  const int spare = vec_rows(p.x, p.xr, p.rows, sizeof(TX), W) ? 0 : W - 1;
  if (p.cols + spare <= 2 * kThreads * kStreamMost && p.xr.sc == 1 && p.yr.sc == 1 &&
      same_shift(p.x, p.xr, sizeof(TX), p.y, p.yr, sizeof(TY), p.rows, W))
    return forward_streamed<TX, TY>(p, spare, s);
  const bool vec = vec_rows(p.x, p.xr, p.rows, sizeof(TX), W) && vec_rows(p.y, p.yr, p.rows, sizeof(TY), W) &&
                   vec_weight(p.w) && vec_weight(p.b);
  return vec ? forward_of<TX, TY, true>(p, s) : forward_of<TX, TY, false>(p, s);
}

}  // namespace

cudaError_t launch_layer_norm(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return forward<decltype(tx), decltype(ty)>(p, s); });
}

}  // namespace spmdb200
