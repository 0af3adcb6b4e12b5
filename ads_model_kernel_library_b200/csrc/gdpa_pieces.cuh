// Rows of bf16 or fp32 values taken 16 bytes at a time, the scale of a run of them in 8 bits, and the request that a token belongs to: what the kernels share
// that fill and read the paged cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "gdpa_common.cuh"
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

// The request that has token t: the last of `batch` whose offset is at or before it.  By the whole warp; it ends whatever the offsets say.
__device__ __forceinline__ int request_of(const void* offsets, int off64, int batch, long long t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && load_offset(offsets, at, off64) <= t);
    lo += (below == 0 ? 0 : __popc(below) - 1) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}
// The same for the lane's one of neighbouring tokens, base + lane; those behind `last` need not come out right.
__device__ __forceinline__ int request_of_lane(const void* offsets, int off64, int batch, long long base, long long last) {
  const int lane = threadIdx.x & 31, b0 = request_of(offsets, off64, batch, base);
  int owner = b0;
  for (int b = b0 + 1; b < batch; b += 32) {
    const long long begin = b + lane < batch ? load_offset(offsets, b + lane, off64) : 0x7fffffffffffffffll;
    int count = 0;  // of these 32 that begin at or before the lane's token
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) count += __shfl_sync(0xffffffffu, begin, count + s - 1) <= base + lane ? s : 0;
    count += __shfl_sync(0xffffffffu, begin, count) <= base + lane;
    owner += count;
    if (__shfl_sync(0xffffffffu, begin, 31) > last) break;
  }
  return owner;
}

}  // namespace gdpa
