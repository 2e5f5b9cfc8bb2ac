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
constexpr int kQuads = kPiece / kThreads / 4;
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
  uint8_t aligned[CAP];  // every address is a multiple of 4 elements (32-bit states) or 8 (8-bit)
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

// One tensor's addresses and constants.
template <class P, class G, class S>
struct Tensor {
  P *p;
  const G *g;
  S *m, *v;
  void *copy;
  int copy_type;
  int64_t n;
  float keep;  // 1 - lr decay
  bool aligned;
};
template <class P, class G, class S, int CAP>
__device__ __forceinline__ Tensor<P, G, S> tensor_at(const AdamTable<CAP> &t, int k, float lr) {
  return {static_cast<P *>(t.p[k]), static_cast<const G *>(t.g[k]), static_cast<S *>(t.m[k]), static_cast<S *>(t.v[k]),
          t.copy[k], t.copy_type[k], t.n[k], fmaf(-lr, t.decay[k], 1.0f), t.aligned[k] != 0};
}

// Every element is read and written once, so the step is bound by memory: 28
// bytes per element with f32 parameters and states, 16-bit gradients and
// copies.  A thread takes quads of four elements (16-byte loads of f32, all of
// a piece's loads before the first use).
template <class P, class G, int CAP>
__global__ void __launch_bounds__(kThreads, 4) adamw_32(const __grid_constant__ AdamTable<CAP> t) {
  __shared__ Now sh;
  const AdamHyper &h = t.h;
  const Now c = constants(h, &sh);
  if (!isfinite(c.grad_scale)) return;
  const int64_t pieces = t.first[t.count];
  int k = tensor_of(t.first, t.count, blockIdx.x);
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    while (piece >= t.first[k + 1]) ++k;
    const Tensor<P, G, float> w = tensor_at<P, G, float>(t, k, c.lr);
    const int64_t lo = (piece - t.first[k]) * kPiece;
    auto one = [&](float &p, float g, float &m, float &v) {
      g *= c.grad_scale;
      m = fmaf(h.beta1, m, h.rest1 * g);
      v = fmaf(h.beta2, v, h.rest2 * g * g);
      p = updated(p, m, v, h, c, w.keep);
    };
    if (w.aligned && lo + kPiece <= w.n) {
      float p[kQuads][4], g[kQuads][4], m[kQuads][4], v[kQuads][4];
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const int64_t i = lo + 4 * (q * kThreads + (int)threadIdx.x);
        load4(w.g + i, g[q]);
        load4(w.m + i, m[q]);
        load4(w.v + i, v[q]);
        load4(w.p + i, p[q]);
      }
#pragma unroll
      for (int q = 0; q < kQuads; ++q) {
        const int64_t i = lo + 4 * (q * kThreads + (int)threadIdx.x);
#pragma unroll
        for (int e = 0; e < 4; ++e) one(p[q][e], g[q][e], m[q][e], v[q][e]);
        store4(w.m + i, m[q]);
        store4(w.v + i, v[q]);
        store4(w.p + i, p[q]);
        if (w.copy) store_vec16<4>(w.copy, w.copy_type, i, p[q]);
      }
    } else {  // a tensor's last piece, and tensors at odd addresses
      const int64_t hi = w.n - lo < kPiece ? w.n : lo + kPiece;
      for (int64_t i = lo + threadIdx.x; i < hi; i += kThreads) {
        float p = to_f32(w.p[i]), m = w.m[i], v = w.v[i];
        one(p, to_f32(w.g[i]), m, v);
        w.m[i] = m;
        w.v[i] = v;
        w.p[i] = from_f32<P>(p);
        if (w.copy) store_from_f32(w.copy, w.copy_type, i, p);
      }
    }
  }
}

__device__ __forceinline__ float from_code(uint8_t c) {
  __nv_fp8_e4m3 f;
  f.__x = c;
  return (float)f;
}
__device__ __forceinline__ uint8_t to_code(float v) { return __nv_fp8_e4m3(v).__x; }

__device__ __forceinline__ float fmaxf_nan(float a, float b) { return a < b ? b : a; }  // a NaN `a` stays

__device__ __forceinline__ void decode8(uint2 q, float v[8]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const unsigned two = ((k & 2) ? q.y : q.x) >> (16 * (k & 1));
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
    v[2 * k] = f.x, v[2 * k + 1] = f.y;
  }
}
__device__ __forceinline__ uint2 encode8(const float v[8]) {
  unsigned w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) w[k] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * k], v[2 * k + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

// A warp takes a state block of 256 elements, eight consecutive ones a lane:
// the block's largest magnitudes are one integer maximum over the warp each
// (bits of non-negative floats order as the floats do, NaN above all).
template <class P, class G, int CAP>
__global__ void __launch_bounds__(kThreads, 4) adamw_8(const __grid_constant__ AdamTable<CAP> t) {
  __shared__ Now sh;
  const AdamHyper &h = t.h;
  const Now c = constants(h, &sh);
  if (!isfinite(c.grad_scale)) return;
  const int lane = threadIdx.x & 31;
  const int64_t pieces = t.first[t.count];
  int k = tensor_of(t.first, t.count, blockIdx.x);
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    while (piece >= t.first[k + 1]) ++k;
    const Tensor<P, G, uint8_t> w = tensor_at<P, G, uint8_t>(t, k, c.lr);
    const int64_t lo = (piece - t.first[k]) * kPiece + (threadIdx.x >> 5) * kStateBlock;
    if (lo >= w.n) continue;
    const int64_t b = lo / kStateBlock;
    const int64_t i0 = lo + 8 * lane;
    const bool whole = w.aligned && lo + kStateBlock <= w.n;  // the same for the whole warp
    const int mine = (int)(w.n - i0 < 8 ? (w.n > i0 ? w.n - i0 : 0) : 8);
    float p[8], g[8], m[8], r[8];
    if (whole) {
      load8(w.g + i0, g);
      decode8(ld_u2(w.m + i0), m);
      decode8(ld_u2(w.v + i0), r);
      load8(w.p + i0, p);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = e < mine;
        p[e] = in ? to_f32(w.p[i0 + e]) : 0.0f;
        g[e] = in ? to_f32(w.g[i0 + e]) : 0.0f;
        m[e] = in ? from_code(w.m[i0 + e]) : 0.0f;
        r[e] = in ? from_code(w.v[i0 + e]) : 0.0f;
      }
    }
    // The scales go into the factors once per block (not their square, which
    // would leave f32's range long before the root does).
    const float ms = t.ms[k][b], vs = t.vs[k][b];
    const float keep1 = h.beta1 * ms, keep2 = h.beta2 * vs;
    unsigned mtop = 0, rtop = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      g[e] *= c.grad_scale;
      m[e] = fmaf(keep1, m[e], h.rest1 * g[e]);
      r[e] = sqrtf(fmaf(keep2 * r[e], vs * r[e], h.rest2 * g[e] * g[e]));
      // The quotient may be off by two units: it is rounded with the parameter.
      p[e] = fmaf(-c.step_size, __fdividef(m[e], fmaf(r[e], c.root_scale, h.eps)), p[e] * w.keep);
      mtop = max(mtop, __float_as_uint(fabsf(m[e])));
      rtop = max(rtop, __float_as_uint(r[e]));
    }
    const float ms1 = fmaxf_nan(__uint_as_float(__reduce_max_sync(0xffffffffu, mtop)) / kTopCode, kLeastScale);
    const float vs1 = fmaxf_nan(__uint_as_float(__reduce_max_sync(0xffffffffu, rtop)) / kTopCode, kLeastScale);
    if (lane == 0) {  // every lane has read the old ones: the maxima came after
      t.ms[k][b] = ms1;
      t.vs[k][b] = vs1;
    }
    const float mi = 1.0f / ms1, ri = 1.0f / vs1;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] *= mi;
      r[e] *= ri;
      r[e] = r[e] > 0.0f && r[e] < kLeastCode ? kLeastCode : r[e];
    }
    if (whole) {
      *reinterpret_cast<uint2 *>(w.m + i0) = encode8(m);
      *reinterpret_cast<uint2 *>(w.v + i0) = encode8(r);
      store8(w.p + i0, p);
      if (w.copy) store_vec16<8>(w.copy, w.copy_type, i0, p);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < mine) {
          w.m[i0 + e] = to_code(m[e]);
          w.v[i0 + e] = to_code(r[e]);
          w.p[i0 + e] = from_f32<P>(p[e]);
          if (w.copy) store_from_f32(w.copy, w.copy_type, i0 + e, p[e]);
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
          u.copy[i] = t.copy[i], u.n[i] = t.n[i], u.decay[i] = t.decay[i], u.copy_type[i] = t.copy_type[i], u.aligned[i] = t.aligned[i];
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
    const unsigned unit = p.bits8 ? 8 : 4;  // elements
    t.aligned[i] = (uintptr_t)t.p[i] % (unit * sizeof(P)) == 0 && (uintptr_t)t.g[i] % (unit * sizeof(G)) == 0 &&
                   ((uintptr_t)t.m[i] | (uintptr_t)t.v[i]) % (p.bits8 ? 8 : 16) == 0 && (uintptr_t)t.copy[i] % (unit * 2) == 0;
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
