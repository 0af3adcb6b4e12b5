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
  __device__ __forceinline__ void times(const float* table, uint64_t (&v)[2 * C]) const {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint64_t w[C];
      take(table + p * (D / 2), w);
#pragma unroll
      for (int k = 0; k < C; ++k) v[p * C + k] = mul_f32x2(v[p * C + k], w[k]);
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
  // The lane's values turned by its angles (not to be called for a lane whose values are not rotated); `back`: the other way.
  template <bool back>
  static __device__ __forceinline__ void turn(bool interleaved, const uint64_t (&c)[C], const uint64_t (&s)[C], uint64_t (&v)[2 * C]) {
    constexpr uint64_t kSigns = 0x8000000080000000ull;
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
        const uint64_t a = v[k], b = v[C + k], minus = s[k] ^ kSigns;
        v[k] = fma_f32x2(a, c[k], mul_f32x2(b, back ? s[k] : minus));
        v[C + k] = fma_f32x2(b, c[k], mul_f32x2(a, back ? minus : s[k]));
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
// T is the type of the values that are turned: for bf16 the sine and cosine of the special-function unit, which are within 2^-21 for a reduced angle
// (a bf16 result is rounded to 2^-9 of itself), are a third of the instructions.
template <class T>
__device__ __forceinline__ void sin_cos(double frequency, long long position, float& s, float& c) {
  constexpr double kTwoPi = 6.283185307179586232, kTwoPiRest = 2.449293598294706414e-16, kInvPi = 0.31830988618379067154;
  const double angle = static_cast<double>(position) * frequency, turns = rint(angle * (0.5 * kInvPi));
  const double rest = fma(-turns, kTwoPiRest, fma(-turns, kTwoPi, angle));  // in [-pi, pi]
  if constexpr (sizeof(T) == 2) __sincosf(static_cast<float>(rest), &s, &c);
  else sincospif(static_cast<float>(rest * kInvPi), &s, &c);
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
      if (at[k] >= 0) sin_cos<T>(frequency[k], position(axis[k]), table[D / 2 + at[k]], table[at[k]]);
    }
  }
};

// Where a lane's heads are, from unit to unit of token after token.
template <class T, int D>
struct HeadWalk {
  T* at = nullptr;
  long long unit = 0, token = 0;  // steps to the next unit; to the next token, from its last unit
  __device__ __forceinline__ void begin(T* x, long long token_stride, long long head_stride, const HeadLanes<T, D>& lanes, long long t0, int u0, int u1) {
    at = x + t0 * token_stride + (u0 * HeadLanes<T, D>::H + lanes.sub) * head_stride;
    unit = HeadLanes<T, D>::H * head_stride;
    token = token_stride - (u1 - u0 - 1) * unit;
  }
  __device__ __forceinline__ void next(bool last) { at += last ? token : unit; }
  // into the lane's place of a unit's kilobyte of shared memory; zeros where there is no head
  __device__ __forceinline__ void fetch(const HeadLanes<T, D>& lanes, uint4* to, bool there) const {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(to)) + (threadIdx.x & 31) * 16;
    const uint4 *p = reinterpret_cast<const uint4*>(at) + lanes.g0, *q = reinterpret_cast<const uint4*>(at) + lanes.g1;
    const int size = there ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(p), "r"(size) : "memory");
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s + 512), "l"(q), "r"(size) : "memory");
  }
  __device__ __forceinline__ void store(const HeadLanes<T, D>& lanes, const uint64_t (&v)[2 * HeadLanes<T, D>::C]) const {
    reinterpret_cast<uint4*>(at)[lanes.g0] = HeadLanes<T, D>::pack(v);
    reinterpret_cast<uint4*>(at)[lanes.g1] = HeadLanes<T, D>::pack(v + HeadLanes<T, D>::C);
  }
};

constexpr int kUnitPieces = 64;  // 16-byte pieces of a unit: a kilobyte, whatever the type and dimension

__device__ __forceinline__ void fetched(const uint4* from, uint4 (&p)[2]) { p[0] = from[threadIdx.x & 31], p[1] = from[32 + (threadIdx.x & 31)]; }
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A unit's heads, normed and turned.
template <class T, int D>
__device__ __forceinline__ void rotate_unit(const RotarySpec& r, const HeadLanes<T, D>& lanes, const float* weight, const uint64_t (&c)[HeadLanes<T, D>::C],
                                            const uint64_t (&s)[HeadLanes<T, D>::C], uint64_t (&v)[2 * HeadLanes<T, D>::C]) {
  using Lanes = HeadLanes<T, D>;
  float f = 1;
  if (r.norm) {
    f = rsqrtf(Lanes::sum(Lanes::dot(v, v)) * (1.f / D) + r.eps);
    lanes.times(weight, v);
  }
  if (lanes.rotated) Lanes::template turn<false>(r.interleaved, c, s, v);
  if (r.norm) Lanes::times(f, v);
}

// Some tokens and units: of queries, of keys, or, paired, of both (a token's units are then its queries' and behind them its keys').
struct Item {
  long long token;
  int tokens, u0, u1;
  int first, last;  // tensors
};
__device__ __forceinline__ Item item_at(const RotaryArgs& a, unsigned i) {
  Item it;
  const int k = i >= a.items[0];
  if (k) i -= a.items[0];
  const unsigned group = a.chunks[k] == 1 ? i : i / static_cast<unsigned>(a.chunks[k]);
  it.token = static_cast<long long>(group) * a.item_tokens[k];
  it.tokens = static_cast<int>(min(static_cast<long long>(a.item_tokens[k]), a.t[k].tokens - it.token));
  it.u0 = static_cast<int>(i - group * static_cast<unsigned>(a.chunks[k])) * a.per[k];
  it.u1 = it.u0 + a.per[k];
  it.first = k, it.last = a.paired ? 1 : k;
  return it;
}
// The units of an item that are tensor k's, [u0, u1) of its own; none: u0 >= u1.
__device__ __forceinline__ void units_of(const RotaryArgs& a, const Item& it, int k, int heads_a_unit, int& u0, int& u1) {
  const int before = k > it.first ? (a.t[0].heads + heads_a_unit - 1) / heads_a_unit : 0;
  u0 = max(it.u0 - before, 0);
  u1 = min(it.u1 - before, (a.t[k].heads + heads_a_unit - 1) / heads_a_unit);
}

// The units of a warp's items, one after the other, fetched ahead of their use: of x, and (N = 2) behind it of dy.
template <class T, int D, int N, int RING>
struct Stream {
  using Lanes = HeadLanes<T, D>;
  const RotaryArgs& a;
  const Lanes& lanes;
  uint4* const ring;
  const unsigned items, step;
  unsigned item, slot = 0;
  Item it;
  int k = 0, u = 0, u0 = 0, u1 = 0, left = 0;  // tensor, the unit that is fetched next, of [u0, u1); units left of this tensor
  HeadWalk<T, D> walk[N];

  __device__ __forceinline__ Stream(const RotaryArgs& args, const Lanes& l, uint4* r, unsigned first, unsigned s)
      : a(args), lanes(l), ring(r), items(args.items[0] + args.items[1]), step(s), item(first) {
    if (item < items) it = item_at(a, item), k = it.first - 1, next_tensor();
#pragma unroll
    for (int i = 0; i + 1 < RING; ++i) fetch();
  }
  __device__ __forceinline__ void next_tensor() {
    while (left == 0) {
      if (++k > it.last) {
        item += step;
        if (item >= items) return;
        it = item_at(a, item), k = it.first;
      }
      units_of(a, it, k, Lanes::H, u0, u1);
      if (u0 >= u1) continue;
      left = it.tokens * (u1 - u0), u = u0;
      const RotaryTensor& t = a.t[k];
      walk[0].begin(static_cast<T*>(const_cast<void*>(t.x)), t.x_strides[0], t.x_strides[1], lanes, it.token, u0, u1);
      if constexpr (N == 2) walk[1].begin(static_cast<T*>(const_cast<void*>(t.dy)), t.dy_strides[0], t.dy_strides[1], lanes, it.token, u0, u1);
    }
  }
  __device__ __forceinline__ void fetch() {
    if (left > 0) {
      const bool there = u * Lanes::H + lanes.sub < a.t[k].heads, last = u + 1 == u1;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (N == 1 || i == 1 || a.rotary.norm) walk[i].fetch(lanes, ring + (slot * N + i) * kUnitPieces, there);
        walk[i].next(last);
      }
      u = last ? u0 : u + 1;
      if (--left == 0) next_tensor();
    }
    fetch_commit();
    slot = slot + 1 == RING ? 0 : slot + 1;
  }
};

// All of a warp's items: first, first + step, ...  `weights`: of the tensors, `n_weights` of them, D values each, for the whole CTA; `position`: of a
// tensor's token on an axis, after the whole warp's `look` at the token.
template <class T, int D, int RING, class F, class G>
__device__ __forceinline__ void rotate_items(const RotaryArgs& a, uint4* ring, float* tables, float* weights, int n_weights, unsigned first, unsigned step, F position, G look) {
  using Lanes = HeadLanes<T, D>;
  constexpr int C = Lanes::C;
  const Lanes lanes(a.rotary);
  Stream<T, D, 1, RING> stream(a, lanes, ring, first, step);
  const WarpAngles<T, D> angles(a.rotary);
  const int warp = threadIdx.x >> 5;
  if (warp < n_weights) lanes.write_weight(weights + warp * D, a.t[warp].weight, a.t[warp].weight_is_bf16);
  __syncthreads();
  const unsigned n = a.items[0] + a.items[1];
  unsigned slot = 0;
  for (unsigned i = first; i < n; i += step) {
    const Item it = item_at(a, i);
    __syncwarp();  // the last item's angles have been read
    for (int j = 0; j < it.tokens; ++j) {
      look(it.token + j);
      angles.write(tables + j * D, [&](int axis) { return position(it.first, axis, it.token + j); });
    }
    __syncwarp();
    for (int k = it.first; k <= it.last; ++k) {
      const RotaryTensor& t = a.t[k];
      int u0, u1;
      units_of(a, it, k, Lanes::H, u0, u1);
      if (u0 >= u1) continue;
      HeadWalk<T, D> y;
      y.begin(static_cast<T*>(t.y), static_cast<long long>(t.heads) * D, D, lanes, it.token, u0, u1);
      for (int j = 0; j < it.tokens; ++j) {
        uint64_t c[C], s[C];
        if (lanes.rotated) lanes.take(tables + j * D, c), lanes.take(tables + j * D + D / 2, s);
        for (int u = u0; u < u1; ++u) {
          stream.fetch();
          fetch_wait<RING - 1>();
          uint4 p[2];
          fetched(ring + slot * kUnitPieces, p);
          slot = slot + 1 == RING ? 0 : slot + 1;
          uint64_t v[2 * C];
          Lanes::unpack(p, v);
          rotate_unit<T, D>(a.rotary, lanes, weights + k * D, c, s, v);
          if (u * Lanes::H + lanes.sub < t.heads) y.store(lanes, v);
          y.next(u + 1 == u1);
        }
      }
    }
  }
}

// How `tokens` tokens of `units` units each are dealt out to about `warps` warps: some tokens to an item, eight at most, or, with too few tokens for that,
// some units of one.  A token's angles are made once for each of its items.
constexpr int kItemTokens = 8;
struct Split {
  int tokens;  // of an item
  int per;     // units of an item
  int chunks;  // items of a token
  long long items;
};
__host__ inline Split split_tokens(long long tokens, long long units, long long warps) {
  Split s{1, 1, 1, 0};
  if (tokens <= 0 || units <= 0) return s;
  const long long n = tokens / warps;
  s.tokens = static_cast<int>(n < 1 ? 1 : n > kItemTokens ? kItemTokens : n);
  long long per = (tokens * units + warps - 1) / warps;
  per = per > units ? units : per;
  s.chunks = static_cast<int>((units + per - 1) / per);
  s.per = static_cast<int>((units + s.chunks - 1) / s.chunks);
  s.chunks = static_cast<int>((units + s.per - 1) / s.per);
  s.items = (tokens + s.tokens - 1) / s.tokens * s.chunks;
  return s;
}

// Items for about `warps` warps: of both tensors at once where they have the same positions.
__host__ inline void plan_items(RotaryArgs& a, int head_dim, int is_fp32, long long warps) {
  const int a_warp = is_fp32 ? 256 / head_dim : 512 / head_dim;
  auto units = [&](int k) { return (a.t[k].heads + a_warp - 1) / a_warp; };
  auto take = [&](int k, const Split& s) { a.item_tokens[k] = s.tokens, a.per[k] = s.per, a.chunks[k] = s.chunks, a.items[k] = static_cast<unsigned>(s.items); };
  a.paired = a.t[0].tokens == a.t[1].tokens && a.t[0].positions == a.t[1].positions && a.t[0].position_stride == a.t[1].position_stride &&
             a.t[0].positions_are_int64 == a.t[1].positions_are_int64;
  if (a.paired) {
    take(0, split_tokens(a.t[0].tokens, units(0) + units(1), warps));
    take(1, Split{1, 1, 1, 0});
  } else {
    for (int k = 0; k < 2; ++k) take(k, split_tokens(a.t[k].tokens, units(k), warps));
  }
}

}  // namespace gdpa
