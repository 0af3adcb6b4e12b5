// A head's RMS norm and its rotation by a position, as a few lanes of a warp do them: what the kernels for training, for prompts and for
// the paged cache share.
//
// For head x [D], weight w, position p (one for each axis) and pair i < R:
//   n = x * rsqrt(mean(x^2) + eps) * w,   angle_i = p[axis of i] * inv_freq[i],
//   (y_a, y_b) = (n_a cos - n_b sin, n_b cos + n_a sin),   (a, b) = (i, i + R) or, interleaved, (2 i, 2 i + 1);   the other values are n.
//
// A lane has two pieces of 16 bytes of a head: those that hold both halves of its pairs, so that nothing but the norm's sum crosses lanes.
// With R a multiple of a piece's E values, lane l < R / E has the pieces l and l + R / E (both styles of pairs lie within these two), the
// other lanes have two of those behind them, so that neighbouring lanes have neighbouring pieces.  A head is L = D / 2E lanes: 8 for 128 values of bf16, so a
// warp-wide load is four heads' 128-byte halves.
//
// Angles: the product of position and frequency is taken in 64 bits and loses its whole quarter turns there, pi / 2 in two parts, before it becomes fp32 (a
// position of 10^6 has 10^6 radians: 24 bits would leave an error of 0.03 of a radian).  The 64-bit part is six instructions an angle, at half of fp32's
// rate.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"
#include "gdpa_pieces.cuh"

namespace gdpa {

constexpr unsigned kAllLanes = 0xffffffffu;
constexpr int kMostItemTokens = 8;  // tokens of a warp at a time
static_assert(kMaxAxes * kMostItemTokens <= 32, "a lane has one of their positions");

__device__ __forceinline__ float weight_at(const void* w, int is_bf16, int i) {
  if (w == nullptr) return 1.f;
  return is_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : static_cast<const float*>(w)[i];
}

template <class T, int D>
struct HeadLanes {
  static constexpr int E = Piece<T>::kElems;
  static constexpr int L = D / (2 * E);  // lanes of a head
  static constexpr int H = 32 / L;       // heads of a warp
  static constexpr int C = E / 2;        // pairs of fp32 in a piece: a lane's values are 2 C of them, its angles C

  int l, sub;    // lane of its head, head of the warp
  int g0, g1;    // its pieces
  bool rotated;  // whether they are

  __device__ __forceinline__ HeadLanes(const RotarySpec& r) {
    const int lane = threadIdx.x & 31, np = r.pairs / E;
    l = lane % L, sub = lane / L;
    rotated = l < np;
    g0 = rotated ? l : np + l;  // behind the 2 np rotated pieces, in two halves: 2 np + (l - np)
    g1 = rotated ? l + np : L + l;
  }
  // Which lane of a head has piece g, and whether as its second one.
  static __device__ __forceinline__ int lane_of_piece(const RotarySpec& r, int g, bool& second) {
    const int np = r.pairs / E;
    second = g < 2 * np ? g >= np : g >= np + L;
    return g < np ? g : g < np + L ? g - np : g - L;
  }
  // Where a table of D / 2 values has value e of lane l: the lanes' 16-byte reads are neighbours.
  static __device__ __forceinline__ int slot(int l, int e) { return ((e >> 2) * L + l) * 4 + (e & 3); }
  // ... and where it has pair i's: a lane's values are in the order of its pairs
  static __device__ __forceinline__ int slot_of_pair(const RotarySpec& r, int i) {
    if (!r.interleaved) return slot(i / E, i % E);
    const int g = i / (E / 2), np = r.pairs / E, l = g < np ? g : g - np;
    return slot(l, (g < np ? 0 : E / 2) + i % (E / 2));
  }
  __device__ __forceinline__ void take(const float* table, uint64_t (&v)[C]) const {
#pragma unroll
    for (int k = 0; k < C / 2; ++k) {
      const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(table + (k * L + l) * 4);
      v[2 * k] = f.x, v[2 * k + 1] = f.y;
    }
  }
  // A weight as the lanes take it: table[D] has their first pieces' and, from D / 2 on, their second pieces'.  By one warp.
  __device__ __forceinline__ void write_weight(float* table, const void* weight, int is_bf16) const {
    if (sub != 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      table[slot(l, e)] = weight_at(weight, is_bf16, g0 * E + e);
      table[D / 2 + slot(l, e)] = weight_at(weight, is_bf16, g1 * E + e);
    }
  }
  template <int N>
  __device__ __forceinline__ void times(const float* table, uint64_t (&v)[N][2 * C]) const {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint64_t w[C];
      take(table + p * (D / 2), w);
#pragma unroll
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int k = 0; k < C; ++k) v[n][p * C + k] = mul_f32x2(v[n][p * C + k], w[k]);
      }
    }
  }
  static __device__ __forceinline__ void times(float f, uint64_t (&v)[2 * C]) {
    const uint64_t f2 = pack_f32x2(f, f);
#pragma unroll
    for (int k = 0; k < 2 * C; ++k) v[k] = mul_f32x2(v[k], f2);
  }
  static __device__ __forceinline__ float dot(const uint64_t (&a)[2 * C], const uint64_t (&b)[2 * C]) {  // of a lane's values
    uint64_t s = mul_f32x2(a[0], b[0]);
#pragma unroll
    for (int k = 1; k < 2 * C; ++k) s = fma_f32x2(a[k], b[k], s);
    float lo, hi;
    unpack_f32x2(s, lo, hi);
    return lo + hi;
  }
  static __device__ __forceinline__ void unpack(const uint4 (&u)[2], uint64_t (&v)[2 * C]) {
    float p[E];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      Piece<T>::unpack(u[k], p);
#pragma unroll
      for (int e = 0; e < C; ++e) v[k * C + e] = pack_f32x2(p[2 * e], p[2 * e + 1]);
    }
  }
  static __device__ __forceinline__ uint4 pack(const uint64_t* v) {
    float p[E];
#pragma unroll
    for (int e = 0; e < C; ++e) unpack_f32x2(v[e], p[2 * e], p[2 * e + 1]);
    return Piece<T>::pack(p);
  }
  // The norms of N heads; `weight` as above.  The factor comes before the weight: a head whose squares overflow is zeros, whatever its weight.
  template <int N>
  __device__ __forceinline__ void norm(const RotarySpec& r, const float* weight, uint64_t (&v)[N][2 * C]) const {
    if (!r.norm) return;
    float f[N];
#pragma unroll
    for (int n = 0; n < N; ++n) f[n] = dot(v[n], v[n]);
#pragma unroll
    for (int i = 1; i < L; i <<= 1) {
#pragma unroll
      for (int n = 0; n < N; ++n) f[n] += __shfl_xor_sync(kAllLanes, f[n], i);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) times(rsqrtf(f[n] * (1.f / D) + r.eps), v[n]);
    times(weight, v);
  }
  // The lane's values turned by its angles (not to be called for a lane whose values are not rotated); `back`: the other way.
  template <bool back>
  static __device__ __forceinline__ void turn(bool interleaved, const uint64_t (&c)[C], const uint64_t (&s)[C], uint64_t (&v)[2 * C]) {
    if (interleaved) {
#pragma unroll
      for (int k = 0; k < C; ++k) {
        float cs[2], sn[2];
        unpack_f32x2(c[k], cs[0], cs[1]);
        unpack_f32x2(s[k], sn[0], sn[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float a, b;
          unpack_f32x2(v[2 * k + i], a, b);
          v[2 * k + i] = back ? pack_f32x2(a * cs[i] + b * sn[i], b * cs[i] - a * sn[i]) : pack_f32x2(a * cs[i] - b * sn[i], b * cs[i] + a * sn[i]);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const uint64_t a = v[k], b = v[C + k];
        v[k] = back ? fma_f32x2(a, c[k], mul_f32x2(b, s[k])) : sub_f32x2(mul_f32x2(a, c[k]), mul_f32x2(b, s[k]));
        v[C + k] = back ? sub_f32x2(mul_f32x2(b, c[k]), mul_f32x2(a, s[k])) : fma_f32x2(b, c[k], mul_f32x2(a, s[k]));
      }
    }
  }
};

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
// Less its whole quarter turns (their number is in the low bits of a sum of 1.5 2^52 and itself) an angle is in [-pi / 4, pi / 4], where Taylor's series up to
// x^11 and x^10 are within 2^-33; sine and cosine go through them as a pair of fp32.  With what fp32 rounds they are within 2^-23.  The special-function
// unit's, within 2^-21, moved 390 of 53 million rotated keys' values to another of e4m3's, these 73 (an evaluation in fp32 with library functions 90), for
// 7 of 227 us of that append; where bf16 is written the time is the same.
// An angle of more than 2^51 quarter turns, whose 64 bits do not tell it, counts as a whole number of them.
__device__ __forceinline__ void sin_cos(double frequency, long long position, float& s, float& c) {
  constexpr double kHalfPi = 1.5707963267948966, kHalfPiRest = 6.123233995736766e-17, kQuarters = 0.63661977236758134, kRound = 6755399441055744.0;
  const double angle = static_cast<double>(position) * frequency, sum = fma(angle, kQuarters, kRound), turns = sum - kRound;
  float x = static_cast<float>(fma(-turns, kHalfPiRest, fma(-turns, kHalfPi, angle)));
  if (!(fabsf(x) < 1.f)) x *= 0.f;
  const float x2 = x * x;
  const uint64_t xx = pack_f32x2(x2, x2);
  uint64_t p = pack_f32x2(-1.f / 39916800, -1.f / 3628800);
  p = fma_f32x2(p, xx, pack_f32x2(1.f / 362880, 1.f / 40320));
  p = fma_f32x2(p, xx, pack_f32x2(-1.f / 5040, -1.f / 720));
  p = fma_f32x2(p, xx, pack_f32x2(1.f / 120, 1.f / 24));
  p = fma_f32x2(p, xx, pack_f32x2(-1.f / 6, -1.f / 2));
  float ps, pc;
  unpack_f32x2(p, ps, pc);
  const float sine = fmaf(x * x2, ps, x), cosine = fmaf(x2, pc, 1.f);
  const uint32_t quarter = static_cast<uint32_t>(__double2loint(sum));
  const bool odd = quarter & 1u;
  s = __uint_as_float(__float_as_uint(odd ? cosine : sine) ^ ((quarter & 2u) << 30));
  c = __uint_as_float(__float_as_uint(odd ? sine : cosine) ^ (((quarter + 1) & 2u) << 30));
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
  // into table[D]: cosines, then sines; `position` of an axis
  template <class F>
  __device__ __forceinline__ void write(float* table, F position) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const long long p = position(axis[k]);
      if (at[k] >= 0) sin_cos(frequency[k], p, table[D / 2 + at[k]], table[at[k]]);
    }
  }
  // Tables of an item's tokens, TOKENS at most.  `mine`: lane axis * kMostItemTokens + j has token j's position on the axis.
  template <int TOKENS>
  __device__ __forceinline__ void write_all(float* tables, int tokens, long long mine) const {
    __syncwarp();  // the last item's have been read
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) {
      if (j < tokens) write(tables + j * D, [&](int axis) { return __shfl_sync(kAllLanes, mine, axis * kMostItemTokens + j); });
    }
    __syncwarp();
  }
};

// Where a lane's heads are, from unit to unit of token after token.
template <class T, int D>
struct HeadWalk {
  T* at = nullptr;
  long long unit = 0, step = 0, token = 0;  // to the next unit; to the unit after the next `together`; to the next token, instead of the last such step
  __device__ __forceinline__ void begin(T* x, long long token_stride, long long head_stride, const HeadLanes<T, D>& lanes, long long t0, int u0, int u1,
                                        int together) {
    at = x + t0 * token_stride + (u0 * HeadLanes<T, D>::H + lanes.sub) * head_stride;
    unit = HeadLanes<T, D>::H * head_stride;
    step = together * unit;
    token = token_stride - (u1 - u0 - 1) / together * step;
  }
  __device__ __forceinline__ void next(bool last) { at += last ? token : step; }
  // into the lane's place of a unit's kilobyte of shared memory; zeros where there is no head
  __device__ __forceinline__ void fetch(const HeadLanes<T, D>& lanes, int i, uint4* to, bool there) const {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(to)) + (threadIdx.x & 31) * 16;
    const uint4* const row = reinterpret_cast<const uint4*>(at + i * unit);
    const uint4 *p = row + lanes.g0, *q = row + lanes.g1;
    const int size = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(p), "r"(size) : "memory");
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s + 512), "l"(q), "r"(size) : "memory");
  }
  __device__ __forceinline__ void store(const HeadLanes<T, D>& lanes, int i, const uint64_t (&v)[2 * HeadLanes<T, D>::C]) const {
    uint4* const row = reinterpret_cast<uint4*>(at + i * unit);
    row[lanes.g0] = HeadLanes<T, D>::pack(v);
    row[lanes.g1] = HeadLanes<T, D>::pack(v + HeadLanes<T, D>::C);
  }
};

constexpr int kUnitPieces = 64;  // 16-byte pieces of a unit: a kilobyte, whatever the type and dimension

__device__ __forceinline__ void fetched(const uint4* from, uint4 (&p)[2]) { p[0] = from[threadIdx.x & 31], p[1] = from[32 + (threadIdx.x & 31)]; }
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Some tokens and units: of queries, of keys, or, paired, of both (a token's units are then its queries' and behind them its keys').
struct Item {
  long long token;
  int tokens, u0, u1;
  int first, last;  // tensors
};
// A warp's items, the w-th of every n: what the warps have in hand at a time lies close together.
struct Cursor {
  unsigned w, n;
  int k = -1;  // queries or keys
  unsigned at = 0, end = 0;
  __device__ __forceinline__ Cursor(unsigned warp, unsigned warps) : w(warp), n(warps) {}
  __device__ __forceinline__ bool next(const RotaryArgs& a, Item& it) {
    while (at >= end) {
      if (++k > (a.paired ? 0 : 1)) return false;
      at = w, end = a.items[k];
    }
    it.first = k, it.last = a.paired ? 1 : k;
    it.u0 = 0, it.u1 = a.per[k];
    if (a.chunks[k] == 1) {
      it.token = static_cast<long long>(at) * a.item_tokens;
      it.tokens = static_cast<int>(min(a.t[k].tokens - it.token, static_cast<long long>(a.item_tokens)));
    } else {
      it.token = at / static_cast<unsigned>(a.chunks[k]);
      it.tokens = 1;
      it.u0 = static_cast<int>(at - static_cast<unsigned>(it.token) * a.chunks[k]) * a.per[k];
      it.u1 += it.u0;
    }
    at += n;
    return true;
  }
};
// The units of an item that are tensor k's, [u0, u1) of its own; none: u0 >= u1.
__device__ __forceinline__ void units_of(const RotaryArgs& a, const Item& it, int k, int heads_a_unit, int& u0, int& u1) {
  const int before = k > it.first ? (a.t[0].heads + heads_a_unit - 1) / heads_a_unit : 0;
  u0 = max(it.u0 - before, 0);
  u1 = min(it.u1 - before, (a.t[k].heads + heads_a_unit - 1) / heads_a_unit);
}

// The units of a warp's items, U of a token at a time, fetched ahead of their use: of x, and (N = 2) behind them those of dy.  RING: such groups on
// their way.
template <class T, int D, int N, int U, int RING>
struct Stream {
  using Lanes = HeadLanes<T, D>;
  const RotaryArgs& a;
  const Lanes& lanes;
  uint4* const ring;
  Cursor cursor;
  unsigned slot = 0;
  Item it;
  int k = 0, u = 0, u0 = 0, u1 = 0, left = 0;  // tensor, the unit that is fetched next, of [u0, u1); tokens left of this tensor
  HeadWalk<T, D> walk[N];

  __device__ __forceinline__ Stream(const RotaryArgs& args, const Lanes& l, uint4* r, const Cursor& c) : a(args), lanes(l), ring(r), cursor(c) {
    it.last = -1;
    next_tensor();
#pragma unroll
    for (int i = 0; i + 1 < RING; ++i) fetch();
  }
  __device__ __forceinline__ void next_tensor() {
    while (left == 0) {
      if (++k > it.last) {
        if (!cursor.next(a, it)) return;
        k = it.first;
      }
      units_of(a, it, k, Lanes::H, u0, u1);
      if (u0 >= u1) continue;
      left = it.tokens, u = u0;
      const RotaryTensor& t = a.t[k];
      walk[0].begin(static_cast<T*>(const_cast<void*>(t.x)), t.x_strides[0], t.x_strides[1], lanes, it.token, u0, u1, U);
      if constexpr (N == 2) walk[1].begin(static_cast<T*>(const_cast<void*>(t.dy)), t.dy_strides[0], t.dy_strides[1], lanes, it.token, u0, u1, U);
    }
  }
  __device__ __forceinline__ void fetch() {
    if (left > 0) {
      const int heads = a.t[k].heads;
      const bool last = u + U >= u1;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (N == 1 || i == 1 || a.rotary.norm) {
#pragma unroll
          for (int j = 0; j < U; ++j) {
            if (j == 0 || u + j < u1) walk[i].fetch(lanes, j, ring + ((slot * N + i) * U + j) * kUnitPieces, (u + j) * Lanes::H + lanes.sub < heads);
          }
        }
        walk[i].next(last);
      }
      u = last ? u0 : u + U;
      if (last && --left == 0) next_tensor();
    }
    fetch_commit();
    slot = slot + 1 == RING ? 0 : slot + 1;
  }
};

constexpr int kTogether = 2;  // units of a token at once
constexpr int kTokens = 2;    // tokens of an item

// All of a warp's items.  `weights`: of the tensors, `n_weights` of them, D values each, for the whole CTA; `positions`: the lane's of an item's
// (WarpAngles::write_all), by the whole warp.
template <class T, int D, int RING, class F>
__device__ __forceinline__ void rotate_items(const RotaryArgs& a, uint4* ring, float* tables, float* weights, int n_weights, Cursor cursor, F& positions) {
  using Lanes = HeadLanes<T, D>;
  constexpr int C = Lanes::C, U = kTogether;
  const Lanes lanes(a.rotary);
  Stream<T, D, 1, U, RING> stream(a, lanes, ring, cursor);
  Item it, next;
  bool more = cursor.next(a, next);
  long long next_positions = more ? positions(next) : 0;
  const WarpAngles<T, D> angles(a.rotary);
  const int warp = threadIdx.x >> 5;
  if (warp < n_weights) lanes.write_weight(weights + warp * D, a.t[warp].weight, a.t[warp].weight_is_bf16);
  __syncthreads();
  unsigned slot = 0;
  while (more) {
    it = next;
    const long long its_positions = next_positions;
    if ((more = cursor.next(a, next))) next_positions = positions(next);
    angles.template write_all<kTokens>(tables, it.tokens, its_positions);
    for (int k = it.first; k <= it.last; ++k) {
      const RotaryTensor& t = a.t[k];
      int u0, u1;
      units_of(a, it, k, Lanes::H, u0, u1);
      if (u0 >= u1) continue;
      HeadWalk<T, D> y;
      y.begin(static_cast<T*>(t.y), static_cast<long long>(t.heads) * D, D, lanes, it.token, u0, u1, U);
      const float* const weight = weights + k * D;
      for (int j = 0; j < it.tokens; ++j) {
        uint64_t c[C], s[C];
        if (lanes.rotated) lanes.take(tables + j * D, c), lanes.take(tables + j * D + D / 2, s);
        for (int u = u0; u < u1; u += U) {
          stream.fetch();
          fetch_wait<RING - 1>();
          const uint4* const from = ring + slot * U * kUnitPieces;
          slot = slot + 1 == RING ? 0 : slot + 1;
          auto work = [&](auto together) {
            constexpr int N = decltype(together)::value;
            uint64_t v[N][2 * C];
#pragma unroll
            for (int x = 0; x < N; ++x) {
              uint4 p[2];
              fetched(from + x * kUnitPieces, p);
              Lanes::unpack(p, v[x]);
            }
            lanes.template norm<N>(a.rotary, weight, v);
            if (lanes.rotated) {
#pragma unroll
              for (int x = 0; x < N; ++x) Lanes::template turn<false>(a.rotary.interleaved, c, s, v[x]);
            }
#pragma unroll
            for (int x = 0; x < N; ++x)
              if ((u + x) * Lanes::H + lanes.sub < t.heads) y.store(lanes, x, v[x]);
          };
          if (u + 1 < u1) work(std::integral_constant<int, U>{});
          else work(std::integral_constant<int, 1>{});
          y.next(u + U >= u1);
        }
      }
    }
  }
}

// What is dealt out to about `warps` warps: whole tokens, whose angles are then made once, or, with fewer tokens than warps, parts of some units.
// Of both tensors at once where they have the same positions.
__host__ inline void plan_items(RotaryArgs& a, int head_dim, int is_fp32, long long warps, int item_tokens) {
  const int a_warp = is_fp32 ? 256 / head_dim : 512 / head_dim;
  auto units = [&](int k) { return (a.t[k].heads + a_warp - 1) / a_warp; };
  auto deal = [&](int k, long long tokens, long long n) {
    a.per[k] = a.chunks[k] = 1, a.items[k] = 0;
    if (tokens <= 0 || n <= 0) return;
    long long per = (tokens * n + warps - 1) / warps;  // whole tokens, some to an item, once there are enough for that
    per = per > n ? n : per;
    per = (n + (n + per - 1) / per - 1) / ((n + per - 1) / per);  // as even as it goes
    a.per[k] = static_cast<int>(per);
    a.chunks[k] = static_cast<int>((n + per - 1) / per);
    a.items[k] = static_cast<unsigned>(a.chunks[k] == 1 ? (tokens + item_tokens - 1) / item_tokens : tokens * a.chunks[k]);
  };
  a.item_tokens = item_tokens;
  a.paired = a.t[0].tokens == a.t[1].tokens && a.t[0].positions == a.t[1].positions && a.t[0].position_stride == a.t[1].position_stride &&
             a.t[0].positions_are_int64 == a.t[1].positions_are_int64;
  deal(0, a.t[0].tokens, a.paired ? units(0) + units(1) : units(0));
  deal(1, a.paired ? 0 : a.t[1].tokens, units(1));
}

}  // namespace gdpa
