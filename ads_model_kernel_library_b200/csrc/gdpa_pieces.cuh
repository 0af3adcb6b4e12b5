// Rows of bf16 or fp32 values taken 16 bytes at a time, and the scale of a run of them in 8 bits: what the kernels share that fill
// and read the paged cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace gdpa {

template <class T>
struct Piece;  // 16 bytes of a row
template <>
struct Piece<__nv_bfloat16> {
  static constexpr int kElems = 8;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {  // to nearest even
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // the largest magnitude's bits, in two halves / whole, as long as it goes on; then as bits of fp32
  static __device__ __forceinline__ uint32_t magnitude(uint32_t top, const uint4& u) {
    top = max_u16x2(max_u16x2(top, u.x & 0x7fff7fffu), u.y & 0x7fff7fffu);
    return max_u16x2(max_u16x2(top, u.z & 0x7fff7fffu), u.w & 0x7fff7fffu);
  }
  static __device__ __forceinline__ uint32_t whole(uint32_t top) { return max(top & 0xffffu, top >> 16) << 16; }
};
template <>
struct Piece<float> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ uint32_t magnitude(uint32_t top, const uint4& u) {
    top = max(max(top, u.x & 0x7fffffffu), u.y & 0x7fffffffu);
    return max(max(top, u.z & 0x7fffffffu), u.w & 0x7fffffffu);
  }
  static __device__ __forceinline__ uint32_t whole(uint32_t top) { return top; }
};

__device__ __forceinline__ float2 e4m3x2_values(uint32_t v) {
  const uint32_t h = f16x2_from_e4m3x2(static_cast<uint16_t>(v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// exponent k of the smallest power of two with amax / 2^k <= 448 = 1.75 * 2^8, at least -100; `bits` of a finite fp32 >= 0
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
  const int k = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(k, -100);
}

constexpr uint32_t kInfBits = 0x7f800000u;

}  // namespace gdpa
