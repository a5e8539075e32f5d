// Element types of the stand-alone operators (f8_*.cu, qk_norm.cu,
// diff_attention*.cu): float32, fp16 and bf16 in memory, float32 in registers.
#pragma once
#include <cuda_bf16.h>

#include "common.cuh"

namespace le {

// Element type ids of the C ABI (LE_DT_*).
enum ElemType : int { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2, DT_E4M3 = 3 };

__host__ __device__ constexpr int elem_size(int dt) { return dt == DT_F32 ? 4 : (dt == DT_E4M3 ? 1 : 2); }

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two values rounded to nearest and packed into one word (lo first).
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_half2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi, __half) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
  lo = f.x;
  hi = f.y;
}
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi, __nv_bfloat16) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}

// Eight consecutive elements as they lie in memory: one 16-byte word for the
// 2-byte types, two for float32.  p is 16-byte aligned.
template <class T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};
template <class T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); i++) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
// load8 of values that are read once (evicted first).
template <class T>
__device__ __forceinline__ Raw8<T> load8_once(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); i++) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <class T>
__device__ __forceinline__ Raw8<T> zero8() {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); i++) r.w[i] = make_uint4(0, 0, 0, 0);
  return r;
}
template <class T>
__device__ __forceinline__ void values8(const Raw8<T>& r, float (&v)[8]) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&r);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) unpack2(u[i], v[2 * i], v[2 * i + 1], T{});
  }
}
// Eight float32 parameters (read-only, 16-byte aligned).
__device__ __forceinline__ void load_f32x8(const float* p, float (&v)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                              pack2<T>(v[6], v[7]));
  }
}

// store8 of values that no kernel reads back soon.
template <class T>
__device__ __forceinline__ void store8_once(T* p, const float (&v)[8]) {
  static_assert(sizeof(T) == 2, "2-byte types");
  __stcs(reinterpret_cast<uint4*>(p), make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                                 pack2<T>(v[6], v[7])));
}

}  // namespace le
