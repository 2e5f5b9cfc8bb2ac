// adamw.cu -- one AdamW step over a list of tensors in place.
//
//   g' = g * grad_scale;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
// All in f32; p is rounded once to its type (to nearest: a change below half a
// unit of a 16-bit parameter is lost, which is why an f32 parameter with a
// 16-bit copy is offered).
//
// 8-bit states: 256 consecutive elements share one f32 scale.  m is held as
// e4m3(m / s), v as e4m3(sqrt(v) / s), each with s = max(largest magnitude /
// 448, 2^-120).  e4m3 has the same relative step (2^-3) over five decades, and
// the root halves the decades that v needs.  A root above zero keeps at least
// the smallest code: rounded to zero, the next step would divide by eps alone.
// The step itself uses m and v before they are rounded.
#include <cuda_fp8.h>

#include "dtypes.cuh"
#include "internal.h"
#include "tensor_list.cuh"

namespace spmdb200 {

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 2048;  // elements a block takes at a time: 8 warps of one 8-bit state block each
constexpr float kTopCode = 448.0f, kLeastCode = 0x1p-9f, kLeastScale = 0x1p-120f;

struct AdamHyper {
  float beta1, beta2, rest1, rest2;  // 1 - beta, taken in f64
  float eps;
  float lr, step_size, root_scale;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t) (host step and lr)
  double beta1_d, beta2_d;          // for a step number on the device
  int64_t step;
  const float *lr_dev;
  const int64_t *step_dev;
  const float *grad_scale;
};

template <int CAP>
struct AdamTable {
  AdamHyper h;
  int64_t first[CAP + 1];
  void *p[CAP];
  const void *g[CAP];
  void *m[CAP], *v[CAP];
  float *ms[CAP], *vs[CAP];
  void *copy[CAP];
  int64_t n[CAP];
  float decay[CAP];
  uint8_t copy_type[CAP];
  int count;
};
constexpr int kSmallCap = 32, kLargeCap = 384;
static_assert(sizeof(AdamTable<kLargeCap>) <= 32764, "kernel parameters end at 32,764 bytes");

// The step's constants as a block needs them.
struct Now {
  float lr, step_size, root_scale, grad_scale;
};

__device__ __forceinline__ Now constants(const AdamHyper &h, Now *sh) {
  Now c{h.lr, h.step_size, h.root_scale, 1.0f};
  if (h.lr_dev || h.step_dev) {
    if (threadIdx.x == 0) {
      const float lr = h.lr_dev ? *h.lr_dev : h.lr;
      int64_t t = h.step_dev ? *h.step_dev : h.step;
      t = t < 1 ? 1 : t;
      sh->lr = lr;
      sh->step_size = (float)((double)lr / (1.0 - pow(h.beta1_d, (double)t)));
      sh->root_scale = (float)(1.0 / sqrt(1.0 - pow(h.beta2_d, (double)t)));
    }
    __syncthreads();
    c = *sh;
  }
  c.grad_scale = h.grad_scale ? *h.grad_scale : 1.0f;
  return c;
}

__device__ __forceinline__ float updated(float p, float m, float v, const AdamHyper &h, const Now &c, float keep) {
  return fmaf(-c.step_size, m / fmaf(sqrtf(v), c.root_scale, h.eps), p * keep);
}

template <class P, class G, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_32(const __grid_constant__ AdamTable<CAP> t) {
  __shared__ Now sh;
  const AdamHyper &h = t.h;
  const Now c = constants(h, &sh);
  if (!isfinite(c.grad_scale)) return;
  for (int64_t piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    const int k = tensor_of(t.first, t.count, piece);
    const int64_t lo = (piece - t.first[k]) * kPiece;
    const int64_t hi = t.n[k] - lo < kPiece ? t.n[k] : lo + kPiece;
    P *p = static_cast<P *>(t.p[k]);
    const G *g = static_cast<const G *>(t.g[k]);
    float *m = static_cast<float *>(t.m[k]), *v = static_cast<float *>(t.v[k]);
    const float keep = fmaf(-c.lr, t.decay[k], 1.0f);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
      const float gi = to_f32(g[i]) * c.grad_scale;
      const float mi = fmaf(h.beta1, m[i], h.rest1 * gi);
      const float vi = fmaf(h.beta2, v[i], h.rest2 * gi * gi);
      const float pi = updated(to_f32(p[i]), mi, vi, h, c, keep);
      m[i] = mi;
      v[i] = vi;
      p[i] = from_f32<P>(pi);
      if (t.copy[k]) store_from_f32(t.copy[k], t.copy_type[k], i, pi);
    }
  }
}

__device__ __forceinline__ float from_code(uint8_t c) {
  __nv_fp8_e4m3 f;
  f.__x = c;
  return (float)f;
}
__device__ __forceinline__ uint8_t to_code(float v) { return __nv_fp8_e4m3(v).__x; }

// The largest of 32 lanes' non-negative values; NaN above all (its bits are).
__device__ __forceinline__ float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

template <class P, class G, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_8(const __grid_constant__ AdamTable<CAP> t) {
  __shared__ Now sh;
  const AdamHyper &h = t.h;
  const Now c = constants(h, &sh);
  if (!isfinite(c.grad_scale)) return;
  const int lane = threadIdx.x & 31;
  for (int64_t piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    const int k = tensor_of(t.first, t.count, piece);
    const int64_t lo = (piece - t.first[k]) * kPiece + (threadIdx.x >> 5) * kStateBlock;
    if (lo >= t.n[k]) continue;
    const int64_t b = lo / kStateBlock;
    P *p = static_cast<P *>(t.p[k]);
    const G *g = static_cast<const G *>(t.g[k]);
    uint8_t *m = static_cast<uint8_t *>(t.m[k]), *v = static_cast<uint8_t *>(t.v[k]);
    const float keep = fmaf(-c.lr, t.decay[k], 1.0f);
    const float ms = t.ms[k][b], vs = t.vs[k][b];
    float mi[8], ri[8], mtop = 0.0f, rtop = 0.0f;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t i = lo + q * 32 + lane;
      mi[q] = ri[q] = 0.0f;
      if (i < t.n[k]) {
        const float gi = to_f32(g[i]) * c.grad_scale;
        const float r = from_code(v[i]) * vs;
        mi[q] = fmaf(h.beta1, from_code(m[i]) * ms, h.rest1 * gi);
        const float vi = fmaf(h.beta2, r * r, h.rest2 * gi * gi);
        ri[q] = sqrtf(vi);
        const float pi = updated(to_f32(p[i]), mi[q], vi, h, c, keep);
        p[i] = from_f32<P>(pi);
        if (t.copy[k]) store_from_f32(t.copy[k], t.copy_type[k], i, pi);
      }
      mtop = __uint_as_float(max(__float_as_uint(mtop), __float_as_uint(fabsf(mi[q]))));
      rtop = __uint_as_float(max(__float_as_uint(rtop), __float_as_uint(ri[q])));
    }
    const float mscale = warp_top(mtop) / kTopCode, rscale = warp_top(rtop) / kTopCode;
    const float m1 = mscale < kLeastScale ? kLeastScale : mscale, r1 = rscale < kLeastScale ? kLeastScale : rscale;
    __syncwarp();  // every lane has read the old scales
    if (lane == 0) {
      t.ms[k][b] = m1;
      t.vs[k][b] = r1;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int64_t i = lo + q * 32 + lane;
      if (i < t.n[k]) {
        m[i] = to_code(mi[q] / m1);
        const float u = ri[q] / r1;
        v[i] = to_code(u > 0.0f && u < kLeastCode ? kLeastCode : u);
      }
    }
  }
}

template <class P, class G, int CAP>
cudaError_t launch(const AdamTable<CAP> &t, bool bits8, unsigned most, cudaStream_t s) {
  const int64_t pieces = t.first[t.count];
  const unsigned grid = (unsigned)(pieces < (int64_t)most ? pieces : (int64_t)most);
  if (bits8) adamw_8<P, G, CAP><<<grid, kThreads, 0, s>>>(t);
  else adamw_32<P, G, CAP><<<grid, kThreads, 0, s>>>(t);
  return cudaGetLastError();
}

// Launches for the tensors of one type pair, kLargeCap of them at a time.
template <class P, class G>
cudaError_t step_of(const AdamWProblem &p, int pt, int gt, const AdamHyper &h, unsigned most, cudaStream_t s) {
  AdamTable<kLargeCap> t;
  t.h = h;
  t.count = 0;
  t.first[0] = 0;
  for (int k = 0; k <= p.count; ++k) {
    if (t.count == kLargeCap || (k == p.count && t.count > 0)) {
      cudaError_t e;
      if (t.count <= kSmallCap) {  // fewer bytes of parameters to send
        AdamTable<kSmallCap> u;
        u.h = t.h;
        u.count = t.count;
        u.first[t.count] = t.first[t.count];
        for (int i = 0; i < t.count; ++i) {
          u.first[i] = t.first[i];
          u.p[i] = t.p[i], u.g[i] = t.g[i], u.m[i] = t.m[i], u.v[i] = t.v[i], u.ms[i] = t.ms[i], u.vs[i] = t.vs[i];
          u.copy[i] = t.copy[i], u.n[i] = t.n[i], u.decay[i] = t.decay[i], u.copy_type[i] = t.copy_type[i];
        }
        e = launch<P, G, kSmallCap>(u, p.bits8, most, s);
      } else {
        e = launch<P, G, kLargeCap>(t, p.bits8, most, s);
      }
      if (e) return e;
      t.count = 0;
    }
    if (k == p.count) break;
    if (p.sizes[k] == 0 || p.param_types[k] != pt || p.grad_types[k] != gt) continue;
    const int i = t.count++;
    t.first[i + 1] = t.first[i] + (p.sizes[k] + kPiece - 1) / kPiece;
    t.p[i] = p.params[k];
    t.g[i] = p.grads[k];
    t.m[i] = p.m[k];
    t.v[i] = p.v[k];
    t.ms[i] = p.bits8 ? p.m_scales[k] : nullptr;
    t.vs[i] = p.bits8 ? p.v_scales[k] : nullptr;
    t.copy[i] = p.copies ? p.copies[k] : nullptr;
    t.copy_type[i] = (uint8_t)(p.copies ? p.copy_types[k] : 0);
    t.n[i] = p.sizes[k];
    t.decay[i] = (float)p.decay[k];
  }
  return cudaSuccess;
}

template <class P>
cudaError_t step_of_params(const AdamWProblem &p, int pt, const AdamHyper &h, unsigned most, cudaStream_t s) {
  if (cudaError_t e = step_of<P, float>(p, pt, kF32, h, most, s)) return e;
  if (cudaError_t e = step_of<P, __half>(p, pt, kF16, h, most, s)) return e;
  return step_of<P, __nv_bfloat16>(p, pt, kBF16, h, most, s);
}

}  // namespace

cudaError_t launch_adamw(const AdamWProblem &p, cudaStream_t s) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  AdamHyper h{};
  h.beta1 = (float)p.beta1, h.beta2 = (float)p.beta2;
  h.rest1 = (float)(1.0 - p.beta1), h.rest2 = (float)(1.0 - p.beta2);
  h.eps = (float)p.eps;
  h.beta1_d = p.beta1, h.beta2_d = p.beta2;
  h.lr = (float)p.lr;
  h.step = p.step;
  if (!p.step_dev) {
    h.step_size = (float)(p.lr / (1.0 - pow(p.beta1, (double)p.step)));
    h.root_scale = (float)(1.0 / sqrt(1.0 - pow(p.beta2, (double)p.step)));
  }
  h.lr_dev = p.lr_dev;
  h.step_dev = p.step_dev;
  h.grad_scale = p.grad_scale;
  const unsigned most = (unsigned)num_sms(dev) * 8;
  if (cudaError_t e = step_of_params<float>(p, kF32, h, most, s)) return e;
  if (cudaError_t e = step_of_params<__half>(p, kF16, h, most, s)) return e;
  return step_of_params<__nv_bfloat16>(p, kBF16, h, most, s);
}

}  // namespace spmdb200
