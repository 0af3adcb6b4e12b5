// A head's RMS norm and its rotation by a position, as a few lanes of a warp do them: what the kernels for training, for prompts and for
// the paged cache share.
//
// For head x [D], weight w, position p (one for each axis) and pair i < R:
//   n = x * rsqrt(mean(x^2) + eps) * w,   angle_i = p[axis of i] * inv_freq[i],
//   (y_a, y_b) = (n_a cos - n_b sin, n_b cos + n_a sin),   (a, b) = (i, i + R) or, interleaved, (2 i, 2 i + 1);   the other values are n.
//
// A lane has two pieces of 16 bytes of a head: those that hold both halves of its pairs, so that nothing but the norm's sum crosses lanes.
// With R a multiple of a piece's E values, lane l < R / E has the pieces l and l + R / E (both styles of pairs lie within these two), the
// other lanes have two neighbouring pieces behind the rotated ones.  A head is L = D / 2E lanes: 8 for 128 values of bf16, so a
// warp-wide load is four heads' 128-byte halves.
//
// Angles: the product of position and frequency is taken in 64 bits and loses its whole turns there, 2 pi in two parts, before it becomes fp32 (a
// position of 10^6 has 10^6 radians: 24 bits would leave an error of 0.03 of a radian); then sincospif.  The 64-bit part is six
// instructions an angle, at half of fp32's rate.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"
#include "gdpa_pieces.cuh"

namespace gdpa {

constexpr unsigned kAllLanes = 0xffffffffu;

template <class T, int D>
struct HeadLanes {
  static constexpr int E = Piece<T>::kElems;
  static constexpr int L = D / (2 * E);  // lanes of a head
  static constexpr int H = 32 / L;       // heads of a warp
  static constexpr int V = 2 * E;        // values of a lane

  int l, sub;    // lane of its head, head of the warp
  int g0, g1;    // its pieces
  bool rotated;  // whether they are

  __device__ __forceinline__ HeadLanes(const RotarySpec& r) {
    const int lane = threadIdx.x & 31, np = r.pairs / E;
    l = lane % L, sub = lane / L;
    rotated = l < np;
    g0 = rotated ? l : 2 * l;  // behind the 2 np rotated pieces: 2 np + 2 (l - np)
    g1 = rotated ? l + np : 2 * l + 1;
  }
  // the sum over a head's lanes
  static __device__ __forceinline__ float sum(float x) {
#pragma unroll
    for (int s = 1; s < L; s <<= 1) x += __shfl_xor_sync(kAllLanes, x, s);
    return x;
  }
  // Where a table of D / 2 values has value e of lane l: the lanes' 16-byte reads are neighbours.
  static __device__ __forceinline__ int slot(int l, int e) { return ((e >> 2) * L + l) * 4 + (e & 3); }
  // ... and where it has pair i's: a lane's values are in the order of its pairs
  static __device__ __forceinline__ int slot_of_pair(const RotarySpec& r, int i) {
    if (!r.interleaved) return slot(i / E, i % E);
    const int g = i / (E / 2), np = r.pairs / E, l = g < np ? g : g - np;
    return slot(l, (g < np ? 0 : E / 2) + i % (E / 2));
  }
  __device__ __forceinline__ void take(const float* table, float (&v)[E]) const {
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const float4 f = *reinterpret_cast<const float4*>(table + (k * L + l) * 4);
      v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
    }
  }
  static __device__ __forceinline__ void unpack(const uint4 (&u)[2], float (&v)[V]) {
    float p[E];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      Piece<T>::unpack(u[k], p);
#pragma unroll
      for (int e = 0; e < E; ++e) v[k * E + e] = p[e];
    }
  }
  // The lane's values turned by its angles; `inverse`: turned back.
  template <bool inverse>
  __device__ __forceinline__ void turn(bool interleaved, const float (&c)[E], const float (&s)[E], float (&v)[V]) const {
    if (!rotated) return;
    if (interleaved) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float a = v[2 * e], b = v[2 * e + 1];
        v[2 * e] = inverse ? a * c[e] + b * s[e] : a * c[e] - b * s[e];
        v[2 * e + 1] = inverse ? b * c[e] - a * s[e] : b * c[e] + a * s[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float a = v[e], b = v[E + e];
        v[e] = inverse ? a * c[e] + b * s[e] : a * c[e] - b * s[e];
        v[E + e] = inverse ? b * c[e] - a * s[e] : b * c[e] + a * s[e];
      }
    }
  }
};

__device__ __forceinline__ float weight_at(const void* w, int is_bf16, int i) {
  if (w == nullptr) return 1.f;
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : static_cast<const float*>(w)[i];
}

// Radians a position, and the axis, of pair i.
__device__ __forceinline__ double frequency_of_pair(const RotarySpec& r, int i) {
  return r.inv_freq_is_fp64 ? static_cast<const double*>(r.inv_freq)[i] : static_cast<double>(static_cast<const float*>(r.inv_freq)[i]);
}
__device__ __forceinline__ int axis_of_pair(const RotarySpec& r, int i) {
  int axis = 0;
#pragma unroll
  for (int k = 0; k + 1 < kMaxAxes; ++k) axis += k + 1 < r.axes && i >= r.ends[k];
  return axis;
}
__device__ __forceinline__ void sin_cos(double frequency, long long position, float& s, float& c) {
  constexpr double kTwoPi = 6.283185307179586232, kTwoPiRest = 2.449293598294706414e-16, kInvPi = 0.31830988618379067154;
  const double angle = static_cast<double>(position) * frequency, turns = rint(angle * (0.5 * kInvPi));
  const double rest = fma(-turns, kTwoPiRest, fma(-turns, kTwoPi, angle));  // in [-pi, pi]
  sincospif(static_cast<float>(rest * kInvPi), &s, &c);
}

// The angles of a token by one warp: a lane has pairs `lane` and `lane + 32`.
template <class T, int D>
struct WarpAngles {
  double frequency[2];
  int axis[2], at[2];
  __device__ __forceinline__ WarpAngles(const RotarySpec& r) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = (threadIdx.x & 31) + 32 * k;
      at[k] = -1, axis[k] = 0, frequency[k] = 0;
      if (i < r.pairs) frequency[k] = frequency_of_pair(r, i), axis[k] = axis_of_pair(r, i), at[k] = HeadLanes<T, D>::slot_of_pair(r, i);
    }
  }
  // into cos[D / 2] and sin[D / 2]; `position` of an axis
  template <class F>
  __device__ __forceinline__ void write(float* cos, float* sin, F position) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (at[k] >= 0) sin_cos(frequency[k], position(axis[k]), sin[at[k]], cos[at[k]]);
    }
  }
};

// Heads of an item and items of a token: a warp takes a whole token, and its angles once, unless there are too few tokens for `warps` warps.
__host__ inline void split_heads(long long tokens, int heads, int a_warp, long long warps, int& per_item, int& chunks) {
  const long long units = (heads + a_warp - 1) / a_warp;
  long long per = tokens * units / warps;
  per = per < 1 ? 1 : per > units ? units : per;
  const long long n = (units + per - 1) / per;
  per = (units + n - 1) / n;
  per_item = static_cast<int>(per) * a_warp;
  chunks = static_cast<int>((units + per - 1) / per);
}

}  // namespace gdpa
