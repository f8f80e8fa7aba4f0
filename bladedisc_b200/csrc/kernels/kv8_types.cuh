// Conversions shared by the kernels of the 8-bit cache: 16-bit floats in and out, eight at a time.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace disc_b200 {

__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, __half) {
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w));
  a = f.x;
  b = f.y;
}
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b, __nv_bfloat16) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float* f, T) {
  unpack2(w.x, f[0], f[1], T());
  unpack2(w.y, f[2], f[3], T());
  unpack2(w.z, f[4], f[5], T());
  unpack2(w.w, f[6], f[7], T());
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* f) {
  unpack8(*reinterpret_cast<const uint4*>(p), f, T());
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* f) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()),
                                            pack2(f[6], f[7], T()));
}
__device__ __forceinline__ __half pack_one(float a, __half) { return __float2half_rn(a); }
__device__ __forceinline__ __nv_bfloat16 pack_one(float a, __nv_bfloat16) { return __float2bfloat16_rn(a); }
__device__ __forceinline__ float level_of(uint32_t w, int byte) {
  return static_cast<float>(static_cast<int8_t>(w >> (8 * byte)));
}

}  // namespace disc_b200
