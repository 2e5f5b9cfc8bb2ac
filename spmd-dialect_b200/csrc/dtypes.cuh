// dtypes.cuh -- element types of the training-step entries (f32, f16, bf16) and
// the conversions, block sums and row views their kernels share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace spmdb200 {

// Codes of the header's SPMDB200_F32 / F16 / BF16.
enum DType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// Rows of a rank 1-3 view whose last dimension is the row: row i starts at
// (i / n1) * s0 + (i % n1) * s1 elements; its elements lie sc apart.
struct Rows {
  int64_t n1, s0, s1, sc;
};

#ifdef __CUDACC__

__device__ __forceinline__ int64_t row_offset(const Rows &r, int64_t i) {
  if (i < r.n1) return i * r.s1;  // every row, where the leading dimensions collapse
  const int64_t a = i / r.n1;
  return a * r.s0 + (i - a * r.n1) * r.s1;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ void store_from_f32(void *p, int type, int64_t i, float v) {
  if (type == kF32) static_cast<float *>(p)[i] = v;
  else if (type == kF16) static_cast<__half *>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// ---- vectors of elements, as f32 --------------------------------------------------
// load4 / store4 want the address aligned to four elements, load8 / store8 to
// eight.  Loads skip L1: every use here reads an element once.
__device__ __forceinline__ float2 unpack(unsigned v, __half) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
__device__ __forceinline__ float2 unpack(unsigned v, __nv_bfloat16) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ unsigned pack(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ unsigned pack(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const unsigned *>(&h);
}

__device__ __forceinline__ uint2 ld_u2(const void *p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_u4(const void *p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}
__device__ __forceinline__ void load4(const float *p, float v[4]) {
  const float4 q = ld_f4(p);
  v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
}
template <class T>
__device__ __forceinline__ void load4(const T *p, float v[4]) {
  const uint2 q = ld_u2(p);
  const float2 a = unpack(q.x, T{}), b = unpack(q.y, T{});
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ void store4(float *p, const float v[4]) { st_f4(p, make_float4(v[0], v[1], v[2], v[3])); }
template <class T>
__device__ __forceinline__ void store4(T *p, const float v[4]) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(pack(v[0], v[1], T{}), pack(v[2], v[3], T{}));
}
__device__ __forceinline__ void load8(const float *p, float v[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store8(float *p, const float v[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
               "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
template <class T>
__device__ __forceinline__ void store8(T *p, const float v[8]) {
  *reinterpret_cast<uint4 *>(p) = make_uint4(pack(v[0], v[1], T{}), pack(v[2], v[3], T{}), pack(v[4], v[5], T{}),
                                             pack(v[6], v[7], T{}));
}
template <class T>
__device__ __forceinline__ void unpack8(uint4 q, float v[8]) {
  const float2 a = unpack(q.x, T{}), b = unpack(q.y, T{}), c = unpack(q.z, T{}), d = unpack(q.w, T{});
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}
template <class T>
__device__ __forceinline__ void load8(const T *p, float v[8]) {
  unpack8<T>(ld_u4(p), v);
}
// W elements that a thread has put into shared memory itself.
template <int W, class T>
__device__ __forceinline__ void take_vec(const unsigned char *slot, float *v) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4 *>(slot);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else if constexpr (W == 8) {
    unpack8<T>(*reinterpret_cast<const uint4 *>(slot), v);
  } else {
    const uint2 q = *reinterpret_cast<const uint2 *>(slot);
    const float2 a = unpack(q.x, T{}), b = unpack(q.y, T{});
    v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
  }
}

// ---- asynchronous copies to shared memory -----------------------------------------------
// 32 lanes that copy one address each cost 32 turns: one lane does it for all.
template <int BYTES>
__device__ __forceinline__ void copy_async(void *dst, const void *src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(BYTES) : "memory");
}
// The first `bytes` of a copy come from memory, the rest are zero.
template <int BYTES>
__device__ __forceinline__ void copy_async_part(void *dst, const void *src, int bytes) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Two f32 operations in one instruction, each rounded as the single one.
struct F2 {
  float x, y;
};
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 r, a, b;\n\t"
      "mov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("{\n\t.reg .b64 a, b, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 r, a, b;\n\t"
      "mov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ F2 both(float a) { return {a, a}; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("{\n\t.reg .b64 a, b, c, r;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 r, a, b, c;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

template <int W, class T>
__device__ __forceinline__ void store_vec(T *p, const float *v) {
  if constexpr (W == 8) store8(p, v);
  else store4(p, v);
}
// Of a tensor whose type is known at run time, kept in the caches (weights).
template <int W>
__device__ __forceinline__ void load_kept(const void *p, int type, int64_t i, float *v) {
#pragma unroll
  for (int e = 0; e < W; e += 4) {
    if (type == kF32) {
      const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i + e);
      v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
    } else {
      const uint2 q = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i + e);
      const float2 a = type == kF16 ? unpack(q.x, __half{}) : unpack(q.x, __nv_bfloat16{});
      const float2 b = type == kF16 ? unpack(q.y, __half{}) : unpack(q.y, __nv_bfloat16{});
      v[e] = a.x, v[e + 1] = a.y, v[e + 2] = b.x, v[e + 3] = b.y;
    }
  }
}
// Into a 16-bit tensor whose type is known at run time.
template <int W>
__device__ __forceinline__ void store_vec16(void *p, int type, int64_t i, const float *v) {
  if (type == kF16) store_vec<W>(static_cast<__half *>(p) + i, v);
  else store_vec<W>(static_cast<__nv_bfloat16 *>(p) + i, v);
}

__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

#endif  // __CUDACC__

}  // namespace spmdb200
