// layer_norm.cu -- layer norm over the last dimension of a rank 1-3 view.
//
//   mean = sum x / N,  var = sum (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  y = xh w + b
// Sums are held in f32; x, w and b are widened exactly, y is rounded once to
// its type.  A few operations an element: bound by memory.  A row's elements
// stay in registers, so that the variance is taken around the mean from the
// same read.
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
  const int lanes = row_lanes(p.rows, p.cols, W, kMost);
  switch (row_vectors(p.cols, lanes, W)) {
    case 1: return forward_rows<TX, TY, 1, VEC, kThreads, false>(p, lanes, 1, s);
    case 2: return forward_rows<TX, TY, 2, VEC, kThreads, false>(p, lanes, 1, s);
    case 4: return forward_rows<TX, TY, 4, VEC, kThreads, false>(p, lanes, 1, s);
    default: return forward_rows<TX, TY, kMost / W, VEC, kThreads, false>(p, lanes, 1, s);
  }
}

template <class TX, class TY>
cudaError_t forward(const LayerNormProblem &p, cudaStream_t s) {
  constexpr int W = kWidth<TX, TY>;
  const bool vec = vec_rows(p.x, p.xr, p.rows, sizeof(TX), W) && vec_rows(p.y, p.yr, p.rows, sizeof(TY), W) &&
                   vec_weight(p.w) && vec_weight(p.b);
  return vec ? forward_of<TX, TY, true>(p, s) : forward_of<TX, TY, false>(p, s);
}

}  // namespace

cudaError_t launch_layer_norm(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return forward<decltype(tx), decltype(ty)>(p, s); });
}

}  // namespace spmdb200
