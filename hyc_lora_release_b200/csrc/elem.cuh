// Element types of the operators that take bf16, fp16 and fp32 tensors: octets as they travel and as fp32 values.
#pragma once
#include "hyc_common.cuh"
#include <cuda_fp16.h>

namespace hyc {

template <typename T> struct Octet { uint4 v[sizeof(T) / 2]; };

template <typename T>
__device__ __forceinline__ Octet<T> ld_octet(const T* p) {
  Octet<T> o;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) o.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return o;
}
__device__ __forceinline__ float2 half2_bits_to_f32(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t f32_to_half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void octet_to_f32(const Octet<__nv_bfloat16>& o, float (&f)[8]) {
  const uint32_t w[4] = {o.v[0].x, o.v[0].y, o.v[0].z, o.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = bf16lo_to_f32(w[i]); f[2 * i + 1] = bf16hi_to_f32(w[i]); }
}
__device__ __forceinline__ void octet_to_f32(const Octet<__half>& o, float (&f)[8]) {
  const uint32_t w[4] = {o.v[0].x, o.v[0].y, o.v[0].z, o.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = half2_bits_to_f32(w[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
}
__device__ __forceinline__ void octet_to_f32(const Octet<float>& o, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(o.v[i].x); f[4 * i + 1] = __uint_as_float(o.v[i].y);
    f[4 * i + 2] = __uint_as_float(o.v[i].z); f[4 * i + 3] = __uint_as_float(o.v[i].w);
  }
}
// one rounding (to nearest even) per value
__device__ __forceinline__ void st_octet(__nv_bfloat16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2_rn(f[0], f[1]), pack_bf16x2_rn(f[2], f[3]), pack_bf16x2_rn(f[4], f[5]), pack_bf16x2_rn(f[6], f[7]));
}
__device__ __forceinline__ void st_octet(__half* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(f32_to_half2_bits(f[0], f[1]), f32_to_half2_bits(f[2], f[3]), f32_to_half2_bits(f[4], f[5]), f32_to_half2_bits(f[6], f[7]));
}
__device__ __forceinline__ void st_octet(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }

// eight values of a vector whose type is known at run time (HYC_BF16, ...); p on a 16-byte boundary
__device__ __forceinline__ void ld_any8(const void* p, int64_t at, int type, float (&f)[8]) {
  if (type == HYC_F32) octet_to_f32(ld_octet(reinterpret_cast<const float*>(p) + at), f);
  else if (type == HYC_F16) octet_to_f32(ld_octet(reinterpret_cast<const __half*>(p) + at), f);
  else octet_to_f32(ld_octet(reinterpret_cast<const __nv_bfloat16*>(p) + at), f);
}
__device__ __forceinline__ float ld_any(const void* p, int64_t at, int type) {
  if (type == HYC_F32) return reinterpret_cast<const float*>(p)[at];
  if (type == HYC_F16) return __half2float(reinterpret_cast<const __half*>(p)[at]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[at]);
}
__device__ __forceinline__ void st_any(void* p, int64_t at, int type, float v) {
  if (type == HYC_F32) reinterpret_cast<float*>(p)[at] = v;
  else if (type == HYC_F16) reinterpret_cast<__half*>(p)[at] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
}

// ---- pairs of fp32 values in one 64-bit register pair: two operations per instruction
typedef uint64_t f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pair(v, v); }
__device__ __forceinline__ f32x2 add2f(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 mul2f(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 fma2f(f32x2 a, f32x2 b, f32x2 c) { f32x2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

// adjacent values as pairs: 16 bytes of 16-bit elements (N = 4), 16 or 32 of fp32 (N = 2, 4)
__device__ __forceinline__ void bits_to_pairs(const uint4 (&o)[1], f32x2 (&f)[4], __nv_bfloat16) {
  const uint32_t w[4] = {o[0].x, o[0].y, o[0].z, o[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = pair(bf16lo_to_f32(w[i]), bf16hi_to_f32(w[i]));
}
__device__ __forceinline__ void bits_to_pairs(const uint4 (&o)[1], f32x2 (&f)[4], __half) {
  const uint32_t w[4] = {o[0].x, o[0].y, o[0].z, o[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = half2_bits_to_f32(w[i]); f[i] = pair(t.x, t.y); }
}
template <int P>
__device__ __forceinline__ void bits_to_pairs(const uint4 (&o)[P], f32x2 (&f)[2 * P], float) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    f[2 * i] = pair(__uint_as_float(o[i].x), __uint_as_float(o[i].y));
    f[2 * i + 1] = pair(__uint_as_float(o[i].z), __uint_as_float(o[i].w));
  }
}
// one rounding (to nearest even) per value
__device__ __forceinline__ void st_pairs(__nv_bfloat16* p, const f32x2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = unpair(f[i]); w[i] = pack_bf16x2_rn(t.x, t.y); }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void st_pairs(__half* p, const f32x2 (&f)[4]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 t = unpair(f[i]); w[i] = f32_to_half2_bits(t.x, t.y); }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <int N>
__device__ __forceinline__ void st_pairs(float* p, const f32x2 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 a = unpair(f[i]), b = unpair(f[i + 1]);
    *reinterpret_cast<float4*>(p + 2 * i) = make_float4(a.x, a.y, b.x, b.y);
  }
}
// values of a vector whose type is known at run time, from element `at` on (a multiple of 2 N)
template <int N>
__device__ __forceinline__ void ld_any_pairs(const void* p, int64_t at, int type, f32x2 (&f)[N]) {
  if (type == HYC_F32) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + at);
#pragma unroll
    for (int i = 0; i < N; i += 2) { const float4 v = q[i / 2]; f[i] = pair(v.x, v.y); f[i + 1] = pair(v.z, v.w); }
    return;
  }
  const uint2* q = reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + at);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint2 v = q[i / 2];
    if (type == HYC_F16) {
      const float2 a = half2_bits_to_f32(v.x), b = half2_bits_to_f32(v.y);
      f[i] = pair(a.x, a.y); f[i + 1] = pair(b.x, b.y);
    } else {
      f[i] = pair(bf16lo_to_f32(v.x), bf16hi_to_f32(v.x)); f[i + 1] = pair(bf16lo_to_f32(v.y), bf16hi_to_f32(v.y));
    }
  }
}

inline bool elem_type_ok(int t) { return t == HYC_BF16 || t == HYC_F16 || t == HYC_F32; }
inline int elem_bytes(int t) { return t == HYC_F32 ? 4 : 2; }

}  // namespace hyc
