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

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPiece = 2048;  // elements a block takes at a time: 8 warps of one 8-bit state block each
constexpr int kMostUnits = 8;  // state blocks a warp takes in a row; at most 32, a lane for each one's scales

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
  uint8_t aligned[CAP];  // p, g and the copy at multiples of 4 elements (32-bit states) or 8 (8-bit), states of 16 bytes
  int count;
};
constexpr int kSmallCap = 32, kLargeCap = 384;
static_assert(sizeof(AdamTable<kLargeCap>) <= 32764, "kernel parameters end at 32,764 bytes");

// The step's constants as a block needs them.  With numbers on the device each block
// works them out before its loads: 1112 us for 2^28 mixed-precision parameters
// where the host's take 1098, 282 for 268 of 2^27 in 8 bits, 1 to 2 us on small lists.
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
// a piece's loads before the first use), a block one piece: 2^28 parameters in
// 1096 us (6.86 TB/s), against 1277 with eight blocks an SM that loop, 1227
// with pieces of twice the size, 1274 of half.
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

// Square root and reciprocal to within 2^-23 of the value.  The root keeps subnormal
// arguments, whose roots are normal; the reciprocal's argument is normal or zero.
__device__ __forceinline__ float sqrt_near(float v) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_near(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Maxima that keep a NaN.
__device__ __forceinline__ float top_of(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float at_least(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Over the warp, of non-negative values: their bits order as they do, NaN above all.
__device__ __forceinline__ float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

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

// The 8-bit step of eight elements a lane, one state block a warp; m and r come
// as decoded codes and leave as the values of new ones, with the block's new
// scales.  A code is the nearest to value / scale: a rounding of 2^-4 that turns on
// the last bit of f32 where the quotient lies half way between two codes, and the
// new m of the next step with it.  So m and v are the formula's in f32, every
// product and sum rounded as it is written, and a quotient near a half way point is
// taken again with an exact root and division; elsewhere the near ones give the
// same code (within 4 units of the last place, against a margin of 8) at half the
// instructions.  Codes below 2^-6, which lie 2^-9 apart whatever their size, are
// not looked at: there a quotient half way may take the other neighbour (one of 5
// million of them; none of 95 million above).  p's change takes the near root and
// reciprocal everywhere, and is off by 2^-22 of itself for it.
struct Scales {
  float m, v;
};
// 0 to 16 << 12 where a value's last 20 bits, those below a code's, are within 8 of
// half way (of a code above the subnormal ones).
__device__ __forceinline__ unsigned half_way(float q) {
  return (__float_as_uint(q) << 12) + ((8u - 0x80000u) << 12);
}
constexpr unsigned kHalfWay = 16u << 12;

__device__ __forceinline__ F2 apart(F2 a, F2 b) { return {__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)}; }

__device__ __forceinline__ Scales step8(float p[8], float g[8], float m[8], float r[8], Scales old, const Now &c,
                                        const AdamHyper &h, float keep) {
  const F2 gs = both(c.grad_scale), ms = both(old.m), vs = both(old.v), b1 = both(h.beta1), b2 = both(h.beta2),
           r1 = both(h.rest1), r2 = both(h.rest2), root = both(c.root_scale), eps = both(h.eps), size = both(-c.step_size),
           kp = both(keep);
  float mtop = 0.0f, vtop = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const F2 ge = mul2({g[e], g[e + 1]}, gs);
    // (The sums are single additions: a packed one is joined with its product into an FMA, which -fmad=false does
    // not keep from happening: a quarter of the blocks' scales came out otherwise.)
    const F2 me = apart(mul2(mul2({m[e], m[e + 1]}, ms), b1), mul2(ge, r1));
    const F2 o = mul2({r[e], r[e + 1]}, vs);
    const F2 v = apart(mul2(mul2(o, o), b2), mul2(mul2(ge, ge), r2));
    const F2 re{sqrt_near(v.x), sqrt_near(v.y)};
    const F2 den = fma2(re, root, eps);
    const F2 pe = fma2(mul2(size, me), {rcp_near(den.x), rcp_near(den.y)}, mul2(kp, {p[e], p[e + 1]}));
    m[e] = me.x, m[e + 1] = me.y;
    r[e] = re.x, r[e + 1] = re.y;
    g[e] = v.x, g[e + 1] = v.y;
    p[e] = pe.x, p[e + 1] = pe.y;
    mtop = top_of(mtop, fabsf(me.x), fabsf(me.y));
    vtop = top_of(vtop, v.x, v.y);
  }
  const Scales now{at_least(warp_top(mtop) * (1.0f / kTopCode), kLeastScale),
                   at_least(sqrtf(warp_top(vtop)) * (1.0f / kTopCode), kLeastScale)};
  const F2 mi = both(rcp_near(now.m)), ri = both(rcp_near(now.v));
  unsigned nearest = 0xffffffffu;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const F2 qm = mul2(mi, {m[e], m[e + 1]}), qr = mul2(ri, {r[e], r[e + 1]});
    nearest = min(nearest, min(min(half_way(qm.x), half_way(qm.y)), min(half_way(qr.x), half_way(qr.y))));
  }
  if (nearest > kHalfWay) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const F2 qm = mul2(mi, {m[e], m[e + 1]}), qr = mul2(ri, {r[e], r[e + 1]});
      m[e] = qm.x, m[e + 1] = qm.y;
      r[e] = qr.x, r[e + 1] = qr.y;
    }
  } else {  // one lane in 4000 or so
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      m[e] = m[e] / now.m;
      r[e] = sqrtf(g[e]) / now.v;
    }
  }
  // With an infinite scale (a square past f32) every code has to stay 0 or NaN, which both decode to NaN: the least
  // code would stand for infinity, and the block would silently stop moving.
  const float least = isinf(now.v) ? 0.0f : kLeastCode;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (g[e] > 0.0f) r[e] = at_least(r[e], least);
  return now;
}

// What a warp has of one state block in shared memory: eight elements a lane of
// p and g in 16-byte chunks, and both states' codes.
template <class P, class G>
struct Stage8 {
  static constexpr int kP = sizeof(P) / 2, kG = sizeof(G) / 2;
  uint4 p[kP][32], g[kG][32], codes[32];  // codes: m in the first half, v in the second
};
constexpr int kStages8 = 2;

template <class T, int N>
__device__ __forceinline__ void fetch_chunks(uint4 (&slot)[N][32], const T *src, int lane) {
#pragma unroll
  for (int q = 0; q < N; ++q) copy_async<16>(&slot[q][lane], reinterpret_cast<const uint4 *>(src) + q);
}
template <class T, int N>
__device__ __forceinline__ void take_chunks(const uint4 (&slot)[N][32], int lane, float v[8]) {
  if constexpr (N == 1) {
    unpack8<T>(slot[0][lane], v);
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 f = *reinterpret_cast<const float4 *>(&slot[q][lane]);
      v[4 * q] = f.x, v[4 * q + 1] = f.y, v[4 * q + 2] = f.z, v[4 * q + 3] = f.w;
    }
  }
}

// A warp takes state blocks of 256 elements, eight consecutive ones a lane: the
// block's largest magnitudes are one integer maximum over the warp each.  2^27
// bf16 parameters take 268 us in a row at 1.62 GHz (1 kW reached) and 303 between other
// work, 5.0 and 4.5 TB/s of 10 bytes an element, bound by instructions (an SM issues in
// 72 % of the cycles): the states' roundings are the formula's, one by one, which
// costs 36 us of it, and 80 registers a thread do not hold eight elements'
// values (84 to 104 bytes spilled and as many read back).  A warp has `units` blocks of a
// tensor in a row, one look-up for all of them, and the next on its way to shared
// memory while one is computed.  Measured before the roundings were exact: a grid
// of all pieces, whose blocks hide each other's first wait, 217 us, three blocks an
// SM that loop 238 (with three stages 245, with four blocks of 64 registers 245).
template <class P, class G, int CAP>
__global__ void __launch_bounds__(kThreads, 3) adamw_8(const __grid_constant__ AdamTable<CAP> t, int units) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ Now sh;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Stage8<P, G> *stages = reinterpret_cast<Stage8<P, G> *>(smem) + warp * kStages8;
  const AdamHyper &h = t.h;
  const Now c = constants(h, &sh);
  if (!isfinite(c.grad_scale)) return;
  const int64_t pieces = t.first[t.count];
  int k = tensor_of(t.first, t.count, blockIdx.x);
  for (int64_t piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    while (piece >= t.first[k + 1]) ++k;
    const Tensor<P, G, uint8_t> w = tensor_at<P, G, uint8_t>(t, k, c.lr);
    const int64_t lo = ((piece - t.first[k]) * kWarps + warp) * units * kStateBlock;
    if (lo >= w.n) continue;
    float *ms = t.ms[k] + lo / kStateBlock, *vs = t.vs[k] + lo / kStateBlock;
    const int64_t left = (w.n - lo) / kStateBlock;
    const int whole = !w.aligned ? 0 : left < units ? (int)left : units;  // the same for the whole warp
    int64_t i = lo + 8 * lane;
    const P *fp = w.p + i;
    const G *fg = w.g + i;
    const uint8_t *fc = (lane < 16 ? w.m : w.v) + lo + 16 * (lane & 15);
    int ahead = 0;  // blocks fetched
    auto fetch = [&] {
      if (ahead < whole) {
        Stage8<P, G> &s = stages[ahead % kStages8];
        fetch_chunks(s.g, fg, lane);
        copy_async<16>(&s.codes[lane], fc);
        fetch_chunks(s.p, fp, lane);
        fp += kStateBlock, fg += kStateBlock, fc += kStateBlock;
        ++ahead;
      }
      copy_commit();  // empty past the last block, so that the count of groups stays
    };
#pragma unroll
    for (int u = 0; u < kStages8 - 1; ++u) fetch();
    // Lane u holds block u's scales from the start: loaded a block ahead only,
    // they were what the warp waited for (305 against 245 us).
    const bool scaled = lane < units && lo + lane * kStateBlock < w.n;
    Scales mine{scaled ? ms[lane] : 0.0f, scaled ? vs[lane] : 0.0f};
    auto scales = [&](int u) { return Scales{__shfl_sync(0xffffffffu, mine.m, u), __shfl_sync(0xffffffffu, mine.v, u)}; };
    int u = 0;
    for (; u < whole; ++u, i += kStateBlock) {
      fetch();
      copy_wait<kStages8 - 1>();
      __syncwarp();  // the other lanes' copies are there too
      const Stage8<P, G> &s = stages[u % kStages8];
      float p[8], g[8], m[8], r[8];
      decode8(reinterpret_cast<const uint2 *>(s.codes)[lane], m);
      decode8(reinterpret_cast<const uint2 *>(s.codes + 16)[lane], r);
      take_chunks<G>(s.g, lane, g);
      take_chunks<P>(s.p, lane, p);
      __syncwarp();  // the stage may be filled again
      const Scales now = step8(p, g, m, r, scales(u), c, h, w.keep);
      if (lane == u) mine = now;
      *reinterpret_cast<uint2 *>(w.m + i) = encode8(m);
      *reinterpret_cast<uint2 *>(w.v + i) = encode8(r);
      store8(w.p + i, p);
      if (w.copy) store_vec16<8>(w.copy, w.copy_type, i, p);
    }
    // A tensor's last block, and tensors at odd addresses.
    for (; u < units && lo + u * kStateBlock < w.n; ++u, i += kStateBlock) {
      const int64_t rest = w.n - i;
      float p[8], g[8], m[8], r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = e < rest ? to_f32(w.p[i + e]) : 0.0f;
        g[e] = e < rest ? to_f32(w.g[i + e]) : 0.0f;
        m[e] = e < rest ? from_code(w.m[i + e]) : 0.0f;
        r[e] = e < rest ? from_code(w.v[i + e]) : 0.0f;
      }
      const Scales now = step8(p, g, m, r, scales(u), c, h, w.keep);
      if (lane == u) mine = now;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < rest) {
          w.m[i + e] = to_code(m[e]);
          w.v[i + e] = to_code(r[e]);
          w.p[i + e] = from_f32<P>(p[e]);
          if (w.copy) store_from_f32(w.copy, w.copy_type, i + e, p[e]);
        }
    }
    if (scaled) {
      ms[lane] = mine.m;
      vs[lane] = mine.v;
    }
  }
  copy_wait<0>();
}

template <class P, class G, int CAP>
cudaError_t launch(AdamTable<CAP> &t, bool bits8, unsigned sms, cudaStream_t s) {
  const int64_t pieces = t.first[t.count];
  if (!bits8) {
    const int64_t most = INT32_MAX;
    adamw_32<P, G, CAP><<<(unsigned)(pieces < most ? pieces : most), kThreads, 0, s>>>(t);
    return cudaGetLastError();
  }
  // As many state blocks in a row per warp as leave every SM 32 pieces, up to
  // kMostUnits (for 2^27 parameters 234 us at 4, 217 at 8, 16 and 32, before the
  // roundings were exact).
  int units = 1;
  while (units < kMostUnits && pieces >= (int64_t)units * 2 * 32 * sms) units *= 2;
  int64_t at = 0;
  for (int i = 0; i < t.count; ++i) {
    t.first[i] = at;
    at += (t.n[i] + units * kPiece - 1) / (units * kPiece);
  }
  t.first[t.count] = at;
  constexpr int bytes = kWarps * kStages8 * (int)sizeof(Stage8<P, G>);
  if (cudaError_t e = cudaFuncSetAttribute(adamw_8<P, G, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return e;
  const int64_t most = INT32_MAX;
  adamw_8<P, G, CAP><<<(unsigned)(at < most ? at : most), kThreads, bytes, s>>>(t, units);
  return cudaGetLastError();
}

// Launches for the tensors of one type pair, kLargeCap of them at a time.
template <class P, class G>
cudaError_t step_of(const AdamWProblem &p, int pt, int gt, const AdamHyper &h, unsigned sms, cudaStream_t s) {
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
        e = launch<P, G, kSmallCap>(u, p.bits8, sms, s);
      } else {
        e = launch<P, G, kLargeCap>(t, p.bits8, sms, s);
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
                   ((uintptr_t)t.m[i] | (uintptr_t)t.v[i]) % 16 == 0 && (uintptr_t)t.copy[i] % (unit * 2) == 0;
    t.n[i] = p.sizes[k];
    t.decay[i] = (float)p.decay[k];
  }
  return cudaSuccess;
}

template <class P>
cudaError_t step_of_params(const AdamWProblem &p, int pt, const AdamHyper &h, unsigned sms, cudaStream_t s) {
  if (cudaError_t e = step_of<P, float>(p, pt, kF32, h, sms, s)) return e;
  if (cudaError_t e = step_of<P, __half>(p, pt, kF16, h, sms, s)) return e;
  return step_of<P, __nv_bfloat16>(p, pt, kBF16, h, sms, s);
}

}  // namespace

cudaError_t launch_adamw(const AdamWProblem &p, cudaStream_t s) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  AdamHyper h{};
  h.beta1 = (float)p.beta1, h.beta2 = (float)p.beta2;
  h.rest1 = (float)(1.0 - p.beta1), h.rest2 = (float)(1.0 - p.beta2);
  h.eps = (float)p.eps;
  // rcp_near takes a subnormal for zero, and zero over zero is NaN where an element has no gradient yet.  A root above
  // zero is 2^-75 at least, beside which any such eps is lost.
  if (p.bits8 && p.eps > 0.0 && h.eps < 0x1p-126f) h.eps = 0x1p-126f;
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
  const unsigned sms = (unsigned)num_sms(dev);
  if (cudaError_t e = step_of_params<float>(p, kF32, h, sms, s)) return e;
  if (cudaError_t e = step_of_params<__half>(p, kF16, h, sms, s)) return e;
  return step_of_params<__nv_bfloat16>(p, kBF16, h, sms, s);
}

}  // namespace spmdb200
