// layer_norm.cu -- layer norm over the last dimension of a rank 1-3 view, and
// its gradients.
//
//   mean = sum x / N,  var = sum (x - mean)^2 / N,  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd,  y = xh w + b
// and with a = dy w, c1 = sum a / N, c2 = sum a xh / N
//   dx = rstd (a - c1 - xh c2),  dw = sum over rows of dy xh,  db = sum over rows of dy.
// Every sum is held in f32; x, dy, w and b are widened exactly, y and dx are
// rounded once to their type.
#include "dtypes.cuh"
#include "internal.h"

namespace spmdb200 {

namespace {

constexpr int kAnyThreads = 256;
constexpr int kColWidth = 32, kColDepth = 8;

// Sum over the block, in a fixed order; every thread gets it.  `sh` holds 32 floats.
__device__ __forceinline__ float block_sum_f32(float v, float *sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = warp_sum_f32(v);
  __syncthreads();  // the last use of sh is over
  if (lane == 0) sh[warp] = v;
  __syncthreads();
  return warp_sum_f32(lane < warps ? sh[lane] : 0.0f);
}

// One block per row, any strides and any length: the row is read three times
// (mean, variance, output).
template <class TX, class TY>
__global__ void __launch_bounds__(kAnyThreads)
ln_forward_any(const TX *__restrict__ x, Rows xr, TY *y, Rows yr, const void *w, const void *b, int wtype, int64_t rows,
               int64_t cols, float eps, float *mean_out, float *rstd_out) {
  __shared__ float sh[32];
  const float inv_n = 1.0f / (float)cols;
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    const TX *px = x + row_offset(xr, i);
    TY *py = y + row_offset(yr, i);
    float s = 0.0f;
    for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) s += to_f32(px[j * xr.sc]);
    const float mean = block_sum_f32(s, sh) * inv_n;
    s = 0.0f;
    for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
      const float d = to_f32(px[j * xr.sc]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.0f / sqrtf(fmaf(block_sum_f32(s, sh), inv_n, eps));
    for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
      const float xh = (to_f32(px[j * xr.sc]) - mean) * rstd;
      py[j * yr.sc] = from_f32<TY>(fmaf(xh, w ? load_as_f32(w, wtype, j) : 1.0f, b ? load_as_f32(b, wtype, j) : 0.0f));
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[i] = mean;
      if (rstd_out) rstd_out[i] = rstd;
    }
  }
}

// One block per row: c1, c2 and dx.  dx may be dy or x (each element is read
// for the last time by the thread that then writes it).
template <class TX, class TY>
__global__ void __launch_bounds__(kAnyThreads)
ln_dx_any(const TY *dy, Rows gr, const TX *x, Rows xr, const float *mean_in, const float *rstd_in, const void *w,
          int wtype, TX *dx, Rows dr, int64_t rows, int64_t cols) {
  __shared__ float sh[32];
  const float inv_n = 1.0f / (float)cols;
  for (int64_t i = blockIdx.x; i < rows; i += gridDim.x) {
    const TX *px = x + row_offset(xr, i);
    const TY *pg = dy + row_offset(gr, i);
    TX *pd = dx + row_offset(dr, i);
    const float mean = mean_in[i], rstd = rstd_in[i];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
      const float a = to_f32(pg[j * gr.sc]) * (w ? load_as_f32(w, wtype, j) : 1.0f);
      s1 += a;
      s2 = fmaf(a, (to_f32(px[j * xr.sc]) - mean) * rstd, s2);
    }
    const float c1 = block_sum_f32(s1, sh) * inv_n;
    const float c2 = block_sum_f32(s2, sh) * inv_n;
    for (int64_t j = threadIdx.x; j < cols; j += kAnyThreads) {
      const float a = to_f32(pg[j * gr.sc]) * (w ? load_as_f32(w, wtype, j) : 1.0f);
      const float xh = (to_f32(px[j * xr.sc]) - mean) * rstd;
      pd[j * dr.sc] = from_f32<TX>((a - c1 - xh * c2) * rstd);
    }
  }
}

// Partial column sums: block (c, p) adds rows p * kColDepth + k, stepping by
// parts * kColDepth, of 32 columns and writes one partial row pair.
template <class TX, class TY>
__global__ void __launch_bounds__(kColWidth *kColDepth)
ln_columns_any(const TY *dy, Rows gr, const TX *x, Rows xr, const float *mean_in, const float *rstd_in, float *part,
               int parts, int64_t rows, int64_t cols) {
  __shared__ float sh[2][kColDepth][kColWidth];
  const int tx = threadIdx.x & (kColWidth - 1), ty = threadIdx.x / kColWidth;
  const int64_t tiles = (cols + kColWidth - 1) / kColWidth;
  for (int64_t item = blockIdx.x; item < tiles * parts; item += gridDim.x) {
    const int64_t p = item / tiles, j = (item - p * tiles) * kColWidth + tx;
    float sw = 0.0f, sb = 0.0f;
    if (j < cols)
      for (int64_t i = p * kColDepth + ty; i < rows; i += (int64_t)parts * kColDepth) {
        const float g = to_f32(dy[row_offset(gr, i) + j * gr.sc]);
        const float xh = (to_f32(x[row_offset(xr, i) + j * xr.sc]) - mean_in[i]) * rstd_in[i];
        sw = fmaf(g, xh, sw);
        sb += g;
      }
    sh[0][ty][tx] = sw;
    sh[1][ty][tx] = sb;
    __syncthreads();
    if (ty < 2 && j < cols) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kColDepth; ++k) s += sh[ty][k][tx];
      part[(2 * p + ty) * cols + j] = s;
    }
    __syncthreads();
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

// Partial rows of the column sums: at most 296 (two blocks per SM), fewer for
// long rows so that the workspace stays below 20 MB where one part does.
int ln_parts(int64_t rows, int64_t cols) {
  int64_t p = 296 * (int64_t)8192 / cols;
  p = p < 1 ? 1 : p > 296 ? 296 : p;
  return (int)(p < rows ? p : rows < 1 ? 1 : rows);
}

unsigned grid_for(int64_t items) { return (unsigned)(items < (1 << 20) ? items : (1 << 20)); }

template <class TX, class TY>
cudaError_t forward(const LayerNormProblem &p, cudaStream_t s) {
  ln_forward_any<TX, TY><<<grid_for(p.rows), kAnyThreads, 0, s>>>(
      static_cast<const TX *>(p.x), p.xr, static_cast<TY *>(p.y), p.yr, p.w, p.b, p.wtype, p.rows, p.cols, p.eps, p.mean,
      p.rstd);
  return cudaGetLastError();
}

template <class TX, class TY>
cudaError_t backward(const LayerNormProblem &p, cudaStream_t s) {
  const TX *x = static_cast<const TX *>(p.x);
  const TY *dy = static_cast<const TY *>(p.y);
  if (p.dw || p.db) {  // before dx, which may overwrite dy or x
    const int parts = ln_parts(p.rows, p.cols);
    const int64_t tiles = (p.cols + kColWidth - 1) / kColWidth;
    ln_columns_any<TX, TY><<<grid_for(tiles * parts), kColWidth * kColDepth, 0, s>>>(
        dy, p.yr, x, p.xr, p.mean, p.rstd, static_cast<float *>(p.ws), parts, p.rows, p.cols);
    if (cudaError_t e = cudaGetLastError()) return e;
    ln_finish<<<(unsigned)tiles, kColWidth * kColDepth, 0, s>>>(static_cast<const float *>(p.ws), parts, p.cols, p.dw,
                                                                p.db, p.dwtype);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  if (p.dx && p.rows > 0)
    ln_dx_any<TX, TY><<<grid_for(p.rows), kAnyThreads, 0, s>>>(dy, p.yr, x, p.xr, p.mean, p.rstd, p.w, p.wtype,
                                                               static_cast<TX *>(p.dx), p.dr, p.rows, p.cols);
  return cudaGetLastError();
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

size_t layer_norm_workspace_bytes(int64_t rows, int64_t cols) {
  return (size_t)ln_parts(rows, cols) * 2 * (size_t)cols * sizeof(float);
}

cudaError_t launch_layer_norm(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return forward<decltype(tx), decltype(ty)>(p, s); });
}
cudaError_t launch_layer_norm_backward(const LayerNormProblem &p, cudaStream_t s) {
  return by_types(p.xtype, p.ytype, [&](auto tx, auto ty) { return backward<decltype(tx), decltype(ty)>(p, s); });
}

}  // namespace spmdb200
