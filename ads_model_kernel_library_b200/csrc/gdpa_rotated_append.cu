// A serving step's queries, keys and values between the projection and the attention: queries and keys are normed and rotated
// (gdpa_rotary.cuh), keys and values quantised into their slots of the paged cache as gdpa_cache.cu does it (the same runs, scales and
// rules), queries written for the attention.
//
// What bounds it: HBM for prompts (a query value is 2 bytes in and 2 out, a key or value 2 and 1), latency for single tokens.  Rotated keys stay in
// fp32 registers between the maximum of a run and its conversion: they are rounded once, to e4m3.
//
// A few tokens of each request are one launch: the first CTAs have keys and values, the others queries.  Prompts are two: queries as in
// gdpa_rotary.cu, then keys and values, a CTA to a block's run, whose loads overlap the end of the first.  In one kernel, each kind of work has the registers of all.
//
// Keys and values: a CTA looks at a window of 32 tokens for the runs that begin there, and each run is taken according to its length: by
// a head's lanes (one or two tokens), by a warp with a head's lanes to a row, or by a CTA, so that a prompt among single tokens does not keep a few lanes busy for
// long (255 single tokens and a prompt of 512: 118 us with one way for all of a window's runs, 21 so).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_rotary.cuh"

namespace gdpa {

namespace {

// position of the request's token with index 0 of the call
__device__ __forceinline__ long long origin_of(const RotatedAppendArgs& a, int owner) {
  return a.batch == 0 ? 0 : load_offset(a.seq_lens, owner, a.lens64) - load_offset(a.q_off, owner + 1, a.off64);
}
__device__ __forceinline__ long long given_position(const RotatedAppendArgs& a, int axis, long long token) {
  const RotaryTensor& q = a.queries.t[0];
  const long long i = axis * q.position_stride + token;
  return q.positions_are_int64 ? static_cast<const long long*>(q.positions)[i] : static_cast<const int*>(q.positions)[i];
}

// The largest of `top` and a row's magnitudes; a NaN is none, nor, if they are to be finite, an infinity.
template <int N>
__device__ __forceinline__ float largest(float top, const uint64_t (&v)[N], bool finite) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    float lo, hi;
    unpack_f32x2(v[e], lo, hi);
    if (finite) {
      lo = fabsf(lo) < INFINITY ? lo : 0.f;
      hi = fabsf(hi) < INFINITY ? hi : 0.f;
    }
    top = max3_abs(top, lo, hi);
  }
  return top;
}

// A row's values times `inv`, in 8 bits.
template <class T, int D>
__device__ __forceinline__ void store_row(const HeadLanes<T, D>& lanes, uint8_t* row, uint64_t (&v)[2 * HeadLanes<T, D>::C], float inv) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E, C = Lanes::C;
  Lanes::times(inv, v);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    uint32_t q[E / 4];
#pragma unroll
    for (int e = 0; e < E / 4; ++e) {
      float f[4];
      unpack_f32x2(v[k * C + 2 * e], f[0], f[1]);
      unpack_f32x2(v[k * C + 2 * e + 1], f[2], f[3]);
      q[e] = pack_e4m3x4(f[0], f[1], f[2], f[3]);
    }
    uint8_t* const at = row + (k == 0 ? lanes.g0 : lanes.g1) * E;
    if constexpr (E == 8) *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
    else *reinterpret_cast<uint32_t*>(at) = q[0];
  }
}

// A run's scale from its largest finite magnitude, and, where it has grown, the rows before the run rescaled: r0, r0 + step, ... of them by these lanes.
template <class T, int D>
__device__ __forceinline__ float scale_of_run(const HeadLanes<T, D>& lanes, float top, float old, uint8_t* block, long long row_stride, int o, int r0, int step) {
  using Lanes = HeadLanes<T, D>;
  const float fresh = __uint_as_float(static_cast<uint32_t>(scale_exponent(__float_as_uint(top)) + 127) << 23);
  const float scale = old > fresh ? old : fresh;
  if (o > 0 && scale != old) {
    const float ratio = old / scale;
    constexpr int P = D / 16;  // 16-byte pieces of a row, over the lanes of a head
    constexpr int K = (P + Lanes::L - 1) / Lanes::L, AT_ONCE = 4;
    for (int r = r0; r < o; r += AT_ONCE * step) {
      uint4 held[AT_ONCE][K];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (r + i * step < o && k * Lanes::L + lanes.l < P)
            held[i][k] = reinterpret_cast<const uint4*>(block + (r + i * step) * row_stride)[k * Lanes::L + lanes.l];
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (r + i * step >= o || k * Lanes::L + lanes.l >= P) continue;
          uint32_t q[4] = {held[i][k].x, held[i][k].y, held[i][k].z, held[i][k].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 lo = e4m3x2_values(q[j] & 0xffffu), hi = e4m3x2_values(q[j] >> 16);
            q[j] = pack_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
          }
          reinterpret_cast<uint4*>(block + (r + i * step) * row_stride)[k * Lanes::L + lanes.l] = make_uint4(q[0], q[1], q[2], q[3]);
        }
      }
    }
  }
  return scale;
}

// One run of one head, keys (KEY) or values, by the lanes that have its rows r0, r0 + step, ...; the first stays in registers, further ones are read
// and made again.  `angles(row, c, s)` gives a lane its angles; `top_of` makes a maximum over all the run's lanes.
// Lanes without a run have len 0; every lane of a warp comes along.  `first`: whether this lane writes the scale.
template <class T, int D, bool KEY, class Angles, class Top>
__device__ __forceinline__ void store_run(const RotatedAppendArgs& a, const HeadLanes<T, D>& lanes, const float* s_weight, int r0, int step, int h,
                                          long long t0, long long blk, int o, int len, bool first, Angles angles, Top top_of) {
  using Lanes = HeadLanes<T, D>;
  constexpr int C = Lanes::C;
  const CacheAppendArgs& ca = a.cache;
  const long long row_stride = KEY ? ca.key_strides[0] : ca.value_strides[0];
  const T* const x = static_cast<const T*>(KEY ? ca.key : ca.value) + t0 * row_stride + h * (KEY ? ca.key_strides[1] : ca.value_strides[1]);
  float* const scale_at = (KEY ? ca.k_scales : ca.v_scales) + blk * ca.heads + h;
  const long long* const cs = KEY ? ca.k_cache_strides : ca.v_cache_strides;
  uint8_t* const out = (KEY ? ca.k_cache : ca.v_cache) + blk * cs[0] + h * cs[2];
  auto values = [&](int r, uint64_t (&v)[1][2 * C]) {
    uint4 p[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (r < len) {
      const uint4* const at = reinterpret_cast<const uint4*>(x + r * row_stride);
      p[0] = __ldg(at + lanes.g0), p[1] = __ldg(at + lanes.g1);
    }
    Lanes::unpack(p, v[0]);
    if constexpr (KEY) {
      lanes.template norm<1>(a.queries.rotary, s_weight, v);
      if (lanes.rotated) {
        uint64_t c[C], s[C];
        angles(r < len ? r : 0, c, s);
        Lanes::template turn<false>(a.queries.rotary.interleaved, c, s, v[0]);
      }
    }
  };
  const float old = o > 0 && len > 0 ? *scale_at : 0.f;
  uint64_t held[1][2 * C];
  values(r0, held);
  float top = 0, scale = 0, inv = 0;
  // Three passes over the rows: their maximum; if it is infinite (rare), that of the others; their conversion.
  for (int pass = 0;;) {
    if (pass < 2) top = largest(top, held[0], pass == 1);
    else if (r0 < len) store_row<T, D>(lanes, out + (o + r0) * cs[1], held[0], inv);
    for (int r = r0 + step; __any_sync(kAllLanes, r < len); r += step) {
      uint64_t w[1][2 * C];
      values(r, w);
      if (r >= len) continue;
      if (pass < 2) top = largest(top, w[0], pass == 1);
      else store_row<T, D>(lanes, out + (o + r) * cs[1], w[0], inv);
    }
    if (pass == 2) break;
    top = top_of(top);
    if (pass == 0 && __any_sync(kAllLanes, top == INFINITY)) {
      pass = 1, top = 0;
      continue;
    }
    pass = 2;
    scale = scale_of_run<T, D>(lanes, top, old, out, cs[1], len > 0 ? o : 0, r0, step);
    inv = 1.f / scale;
  }
  if (first && len > 0 && scale != old) *scale_at = scale;
}

// Where a window of 32 tokens has its runs, as every warp of a CTA sees it.
struct Window {
  const RotatedAppendArgs& a;
  long long base, slot;  // its first token; the lane's slot, or -1
  unsigned leaders;      // lanes whose token begins a run
  int len;               // the lane's run, as far as the slots go on, at most to the end of the block; 0: it leads none

  __device__ __forceinline__ long long slot_of(long long t) const {
    const CacheAppendArgs& ca = a.cache;
    if (t < 0 || t >= ca.tokens) return -1;
    const long long s = ca.slot_mapping[t];
    return s >= 0 && s < (ca.num_blocks << ca.block_shift) ? s : -1;
  }
  __device__ __forceinline__ Window(const RotatedAppendArgs& args, long long first) : a(args), base(first) {
    const int lane = threadIdx.x & 31, S = 1 << a.cache.block_shift;
    slot = slot_of(base + lane);
    long long before = __shfl_up_sync(kAllLanes, slot, 1);
    if (lane == 0) before = slot_of(base - 1);
    leaders = __ballot_sync(kAllLanes, slot >= 0 && ((slot & (S - 1)) == 0 || before != slot - 1));
    const unsigned ends = (leaders | __ballot_sync(kAllLanes, slot < 0)) & ~((2u << lane) - 1);  // behind the lane
    len = (leaders >> lane & 1u) == 0 ? 0 : ends != 0 ? __ffs(ends) - 1 - lane : 32 - lane;
    // the last run may go on behind the window
    if (leaders == 0) return;
    const int last = 31 - __clz(leaders);
    int its = __shfl_sync(kAllLanes, len, last);
    if (last + its < 32) return;
    const long long s0 = __shfl_sync(kAllLanes, slot, last);
    const int o = static_cast<int>(s0 & (S - 1));
    for (bool more = true; more;) {
      const int i = its + lane;
      const unsigned stops = __ballot_sync(kAllLanes, !(o + i < S && slot_of(base + last + i) == s0 + i));
      its += stops ? __ffs(stops) - 1 : 32;
      more = stops == 0;
    }
    if (lane == last) len = its;
  }
  // position of the first token of the run that the lane leads, less its index
  __device__ __forceinline__ long long origin() const {
    if (a.queries.t[0].positions != nullptr) return 0;
    return origin_of(a, request_of_lane(a.q_off, a.off64, a.batch, base, base + 31));
  }
};

// What the lanes make angles from by themselves, for a whole CTA: frequency and axis of the pairs, in a lane's order.
template <int D>
struct PairTable {
  double frequency[D / 2];
  int axis[D / 2];
};
template <class T, int D>
__device__ __forceinline__ void write_pairs(const RotarySpec& r, PairTable<D>& table) {
  for (int i = threadIdx.x; i < r.pairs; i += blockDim.x) {
    const int at = HeadLanes<T, D>::slot_of_pair(r, i);
    table.frequency[at] = frequency_of_pair(r, i), table.axis[at] = axis_of_pair(r, i);
  }
}

// The maximum of W warps' numbers.  Two places for each, in turn: the next maximum is written while this one may still be read.
template <int W>
__device__ __forceinline__ float top_of_cta(float top, float* tops, unsigned& turn) {
  float* const s = tops + (turn++ & 1u) * W;
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = top;
  __syncthreads();
  top = s[0];
#pragma unroll
  for (int i = 1; i < W; ++i) top = fmaxf(top, s[i]);
  return top;
}

// Some of a window's runs, dealt out: a head's lanes to each run and head; a warp to each, its heads' lanes to a row each; or a CTA to each, by its warps' lanes.
// This is taker `me` of `takers` (warps, or CTAs); `tops`: two words for each warp, of a CTA's maximum.
enum Taker { kHeadLanes, kWarp, kCta };
template <class T, int D, Taker TAKER, int W>
__device__ __forceinline__ void deal(const Window& window, unsigned leaders, long long origin, const HeadLanes<T, D>& lanes, const float* s_weight, const PairTable<D>& pairs,
                                     int me, int takers, float* tops) {
  using Lanes = HeadLanes<T, D>;
  constexpr bool SINGLE = TAKER == kHeadLanes;
  constexpr int C = Lanes::C, a_warp = SINGLE ? Lanes::H : 1, step = SINGLE ? 1 : TAKER == kWarp ? Lanes::H : W * Lanes::H;
  const int warp = threadIdx.x >> 5;
  unsigned turn = 0;
  if (leaders == 0) return;
  const RotatedAppendArgs& a = window.a;
  const CacheAppendArgs& ca = a.cache;
  const bool given = a.queries.t[0].positions != nullptr;
  const int tasks = __popc(leaders) * ca.heads, rounds = (tasks + a_warp - 1) / a_warp;
  for (int i = me; i < 2 * rounds; i += takers) {
    const bool is_key = i < rounds;
    const int task = (is_key ? i : i - rounds) * a_warp + (SINGLE ? lanes.sub : 0);
    const bool there = task < tasks;
    const int at = there ? __fns(leaders, 0, task / ca.heads + 1) : 0, h = there ? task % ca.heads : 0;
    const long long s0 = __shfl_sync(kAllLanes, window.slot, at), run_origin = __shfl_sync(kAllLanes, origin, at), t0 = window.base + at;
    const int run_len = __shfl_sync(kAllLanes, window.len, at), len = there ? run_len : 0;
    const long long blk = there ? s0 >> ca.block_shift : 0;
    const int o = there ? static_cast<int>(s0 & ((1 << ca.block_shift) - 1)) : 0, r0 = SINGLE ? 0 : TAKER == kWarp ? lanes.sub : warp * Lanes::H + lanes.sub;
    auto top_of = [&](float top) {
      if constexpr (SINGLE) {
#pragma unroll
        for (int s = 1; s < Lanes::L; s <<= 1) top = fmaxf(top, __shfl_xor_sync(kAllLanes, top, s));
      } else {
        top = __uint_as_float(__reduce_max_sync(kAllLanes, __float_as_uint(top)));
        if constexpr (TAKER == kCta) top = top_of_cta<W>(top, tops, turn);
      }
      return top;
    };
    const bool first = lanes.l == 0 && (SINGLE || r0 == 0);
    if (is_key) {
      store_run<T, D, true>(a, lanes, s_weight, r0, step, h, t0, blk, o, len, first, [&](int r, uint64_t (&c)[C], uint64_t (&s)[C]) {
#pragma unroll
        for (int e = 0; e < C; ++e) {
          float sn[2], cs[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int pair = Lanes::slot(lanes.l, 2 * e + j);
            sin_cos(pairs.frequency[pair], given ? given_position(a, pairs.axis[pair], t0 + r) : run_origin + t0 + r, sn[j], cs[j]);
          }
          c[e] = pack_f32x2(cs[0], cs[1]), s[e] = pack_f32x2(sn[0], sn[1]);
        }
      }, top_of);
    } else {
      store_run<T, D, false>(a, lanes, s_weight, r0, step, h, t0, blk, o, len, first, [](int, uint64_t (&)[C], uint64_t (&)[C]) {}, top_of);
    }
  }
}

// The lane's position of an item's of the queries.  Items come in the order of their tokens, so the next request is this one or, mostly, one of the next 32: what
// is needed of those comes in one trip to memory.
struct QueryPositions {
  const RotatedAppendArgs& a;
  int owner = -1;                       // request at hand
  long long origin = 0, begin = 0, end = -1;  // position of token 0 by it, its first token and the one behind its last
  __device__ __forceinline__ void find(long long t) {
    if (a.batch == 0) {
      end = 0x7fffffffffffffffll;
      return;
    }
    const int lane = threadIdx.x & 31;
    if (owner < 0) owner = request_of(a.q_off, a.off64, a.batch, t);
    for (bool searched = false;; searched = true) {
      const int next = min(owner + 1 + lane, a.batch);
      const long long ends = load_offset(a.q_off, next, a.off64), len = load_offset(a.seq_lens, min(owner + lane, a.batch - 1), a.lens64);
      const unsigned behind = __ballot_sync(kAllLanes, owner + 1 + lane < a.batch && ends <= t);
      if (behind == kAllLanes && !searched) {
        owner = request_of(a.q_off, a.off64, a.batch, t);
        continue;
      }
      const int count = behind == kAllLanes ? 0 : __ffs(~behind) - 1;  // all of them after a search: offsets that are none
      end = __shfl_sync(kAllLanes, ends, count);
      origin = __shfl_sync(kAllLanes, len, count) - end;
      owner += count;
      begin = count > 0 ? __shfl_sync(kAllLanes, ends, count - 1) : load_offset(a.q_off, owner, a.off64);
      return;
    }
  }
  __device__ __forceinline__ long long operator()(const Item& it) {
    const int lane = threadIdx.x & 31, axis = lane / kMostItemTokens, j = lane % kMostItemTokens;
    if (a.queries.t[0].positions != nullptr) return axis < a.queries.rotary.axes && j < it.tokens ? given_position(a, axis, it.token + j) : 0;
    long long p = 0;
    for (int i = 0; i < it.tokens; ++i) {
      const long long t = it.token + i;
      if (!(t >= begin && t < end)) find(t);
      if (j == i) p = origin + t;  // on every axis
    }
    return p;
  }
};

// ------------------------------------------------------------------------------------------ a few tokens of each request: one launch

constexpr int kWarps = 4, kQueryRing = 3;  // groups of units of a warp on their way
constexpr int kQueryBytes = kWarps * kQueryRing * kTogether * kUnitPieces * 16;

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32, 4) gdpa_rotated_step_kernel(const __grid_constant__ RotatedAppendArgs a) {
  extern __shared__ uint4 s_ring[];
  __shared__ float4 s_tables[kWarps][kTokens][D / 4];
  __shared__ float4 s_weight4[D / 4];
  __shared__ PairTable<D> s_pairs;
  __shared__ float s_top[2 * kWarps];
  float* const s_weight = reinterpret_cast<float*>(s_weight4);
  const int warp = threadIdx.x >> 5, kv_ctas = a.kv_windows * a.kv_parts;
  if (static_cast<int>(blockIdx.x) >= kv_ctas) {
    QueryPositions positions{a};
    rotate_items<T, D, kQueryRing>(a.queries, s_ring + warp * kQueryRing * kTogether * kUnitPieces, reinterpret_cast<float*>(s_tables[warp]), s_weight, 1,
                                   Cursor((blockIdx.x - kv_ctas) * kWarps + warp, (gridDim.x - kv_ctas) * kWarps), positions);
    return;
  }
  const HeadLanes<T, D> lanes(a.queries.rotary);
  const int part = blockIdx.x / a.kv_windows;
  const Window window(a, static_cast<long long>(blockIdx.x - part * a.kv_windows) * 32);
  if (window.leaders == 0) return;
  if (warp == 0) lanes.write_weight(s_weight, a.queries.t[1].weight, a.queries.t[1].weight_is_bf16);
  write_pairs<T, D>(a.queries.rotary, s_pairs);
  __syncthreads();
  const long long origin = window.origin();
  const unsigned longer = __ballot_sync(kAllLanes, window.len > 2), longest = __ballot_sync(kAllLanes, window.len > kWarps * HeadLanes<T, D>::H);
  deal<T, D, kCta, kWarps>(window, longest, origin, lanes, s_weight, s_pairs, part, a.kv_parts, s_top);
  deal<T, D, kWarp, kWarps>(window, longer & ~longest, origin, lanes, s_weight, s_pairs, part * kWarps + warp, a.kv_parts * kWarps, s_top);
  deal<T, D, kHeadLanes, kWarps>(window, window.leaders & ~longer, origin, lanes, s_weight, s_pairs, part * kWarps + warp, a.kv_parts * kWarps, s_top);
}

// ------------------------------------------------------------------------------------------ prompts: queries, then keys and values

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32, 4) gdpa_rotated_queries_kernel(const __grid_constant__ RotatedAppendArgs a) {
  extern __shared__ uint4 s_ring[];
  __shared__ float4 s_tables[kWarps][kTokens][D / 4];
  __shared__ float4 s_weight[D / 4];
  const int warp = threadIdx.x >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // keys and values may begin when there is room: neither reads what the other writes
  QueryPositions positions{a};
  rotate_items<T, D, kQueryRing>(a.queries, s_ring + warp * kQueryRing * kTogether * kUnitPieces, reinterpret_cast<float*>(s_tables[warp]),
                                 reinterpret_cast<float*>(s_weight), 1, Cursor(blockIdx.x * kWarps + warp, gridDim.x * kWarps), positions);
}

// Warps of an SM: a lane that holds 64 values needs 168 registers, one that holds 32 or 16 has enough in 128 (prompts of 512 to 4096 tokens in blocks of 16: 283
// us with 12 warps, 262 with 16; blocks of 64 with 32 values a lane and 16 warps: 240, with 64 and 12: 225).
__host__ __device__ constexpr int runs_ctas(int W, int values) { return (values >= 64 ? 12 : 16) / W; }

// W warps on one run of one head after the other, keys, then values; the next head is on its way while one is worked on.  HOLD rows of a lane, so that a
// whole block is held.
template <class T, int D, int W, int HOLD>
__global__ void __launch_bounds__(W * 32, runs_ctas(W, HOLD * 2 * HeadLanes<T, D>::E)) gdpa_rotated_runs_kernel(const __grid_constant__ RotatedAppendArgs a) {
  using Lanes = HeadLanes<T, D>;
  constexpr int C = Lanes::C, step = W * Lanes::H;
  extern __shared__ uint4 s_dynamic[];  // [warp][HOLD] units; angles of a block's rows, [row][D]
  __shared__ float4 s_weight4[D / 4];
  __shared__ PairTable<D> s_pairs;
  __shared__ float s_top[2 * W];
  float* const s_weight = reinterpret_cast<float*>(s_weight4);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint4* const ring = s_dynamic + warp * HOLD * kUnitPieces;
  float* const tables = reinterpret_cast<float*>(s_dynamic + W * HOLD * kUnitPieces);
  const Lanes lanes(a.queries.rotary);
  const CacheAppendArgs& ca = a.cache;
  const int part = blockIdx.x / a.kv_windows;
  const Window window(a, static_cast<long long>(blockIdx.x - part * a.kv_windows) * 32);
  if (window.leaders != 0) {
    if (warp == 0) lanes.write_weight(s_weight, a.queries.t[1].weight, a.queries.t[1].weight_is_bf16);
    const long long origin = window.origin();
    unsigned mine = window.leaders;  // runs that are taken by the whole CTA, one after the other: long ones, and a few short ones
    if (__popc(mine) > 2) {
      mine = __ballot_sync(kAllLanes, window.len > step);
      write_pairs<T, D>(a.queries.rotary, s_pairs);
      __syncthreads();
      deal<T, D, kWarp, W>(window, window.leaders & ~mine, origin, lanes, s_weight, s_pairs, part * W + warp, a.kv_parts * W, s_top);
    }
    const bool given = a.queries.t[0].positions != nullptr;
    unsigned turn = 0;
    auto top_of = [&](float top) {
      return top_of_cta<W>(__uint_as_float(__reduce_max_sync(kAllLanes, __float_as_uint(top))), s_top, turn);
    };
    const int r0 = warp * Lanes::H + lanes.sub, S = 1 << ca.block_shift;
    for (unsigned left = mine; left != 0; left &= left - 1) {
      const int at = __ffs(left) - 1;
      const long long s0 = __shfl_sync(kAllLanes, window.slot, at), t0 = window.base + at, blk = s0 >> ca.block_shift;
      const int len = __shfl_sync(kAllLanes, window.len, at), o = static_cast<int>(s0 & (S - 1));
      auto fetch = [&](int head2) {
        const bool key = head2 < ca.heads;
        const long long* const xs = key ? ca.key_strides : ca.value_strides;
        HeadWalk<T, D> walk;
        walk.at = static_cast<T*>(const_cast<void*>(key ? ca.key : ca.value)) + (t0 + r0) * xs[0] + (key ? head2 : head2 - ca.heads) * xs[1];
        walk.unit = step * xs[0];
#pragma unroll
        for (int i = 0; i < HOLD; ++i) walk.fetch(lanes, i, ring + i * kUnitPieces, r0 + i * step < len);
        fetch_commit();
      };
      if (part < 2 * ca.heads) fetch(part);
      if (part < ca.heads) {  // this CTA has keys of the run: its angles
        const long long run_origin = __shfl_sync(kAllLanes, origin, at);
        __syncthreads();      // the last run's have been read
        const WarpAngles<T, D> angles(a.queries.rotary);
        for (int r = warp; r < len; r += W)
          angles.write(tables + r * D, [&](int axis) { return given ? given_position(a, axis, t0 + r) : run_origin + t0 + r; });
        __syncthreads();
      }
      for (int head2 = part; head2 < 2 * ca.heads; head2 += a.kv_parts) {
        const bool key = head2 < ca.heads;
        const int h = key ? head2 : head2 - ca.heads;
        float* const scale_at = (key ? ca.k_scales : ca.v_scales) + blk * ca.heads + h;
        const float old = o > 0 ? *scale_at : 0.f;
        fetch_wait<0>();
        uint64_t v[HOLD][2 * C];
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
          uint4 p[2];
          fetched(ring + i * kUnitPieces, p);
          Lanes::unpack(p, v[i]);
        }
        if (head2 + a.kv_parts < 2 * ca.heads) fetch(head2 + a.kv_parts);
        if (key) {
          lanes.template norm<HOLD>(a.queries.rotary, s_weight, v);
          if (lanes.rotated) {
#pragma unroll
            for (int i = 0; i < HOLD; ++i) {
              uint64_t c[C], s[C];
              const float* const table = tables + min(r0 + i * step, S - 1) * D;
              lanes.take(table, c), lanes.take(table + D / 2, s);
              Lanes::template turn<false>(a.queries.rotary.interleaved, c, s, v[i]);
            }
          }
        }
        float top = 0;
#pragma unroll
        for (int i = 0; i < HOLD; ++i)
          if (r0 + i * step < len) top = largest(top, v[i], false);
        top = top_of(top);
        if (top == INFINITY) {  // rare; the same for all warps
          top = 0;
#pragma unroll
          for (int i = 0; i < HOLD; ++i)
            if (r0 + i * step < len) top = largest(top, v[i], true);
          top = top_of(top);
        }
        const long long* const cs = key ? ca.k_cache_strides : ca.v_cache_strides;
        uint8_t* const block = (key ? ca.k_cache : ca.v_cache) + blk * cs[0] + h * cs[2];
        const float scale = scale_of_run<T, D>(lanes, top, old, block, cs[1], o, r0, step), inv = 1.f / scale;
        uint8_t* const row = block + (o + r0) * cs[1];
#pragma unroll
        for (int i = 0; i < HOLD; ++i)
          if (r0 + i * step < len) store_row<T, D>(lanes, row + i * step * cs[1], v[i], inv);
        if (threadIdx.x == 0 && scale != old) *scale_at = scale;
      }
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // this kernel ends after the queries': what follows on the stream waits for both
}

}  // namespace

int launch_rotated_append(RotatedAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  if (a.cache.tokens == 0) return 0;
  const long long windows = (a.cache.tokens + 31) / 32, resident = 4ll * sm_count;
  const int heads_a_warp = (is_fp32 ? 256 : 512) / head_dim;
  // CTAs for a window, of `warps` warps: until `wanted` of them are there, at most one warp for each run and head of single tokens
  auto parts = [&](long long wanted, int warps) -> long long {
    if (a.cache.num_blocks == 0) return 0;
    const long long most = (32ll * 2 * a.cache.heads / heads_a_warp + warps - 1) / warps, n = (wanted + windows - 1) / windows;
    return n > most ? most : n;
  };
  auto query_ctas = [&]() {
    const long long n = (static_cast<long long>(a.queries.items[0]) + kWarps - 1) / kWarps;
    return n < resident ? n : resident;
  };
  auto by_type = [&](auto body) -> int {
    using D64 = std::integral_constant<int, 64>;
    using D128 = std::integral_constant<int, 128>;
    if (is_fp32) return head_dim == 128 ? body(float{}, D128{}) : body(float{}, D64{});
    return head_dim == 128 ? body(__nv_bfloat16{}, D128{}) : body(__nv_bfloat16{}, D64{});
  };
  a.kv_windows = static_cast<int>(windows);
  // One launch for a few tokens of each request; keys and values then have a third of the CTAs that are resident.  bf16, 16 and 4 heads of 128 values, one
  // launch against two, us: 256 requests with 16 tokens 26 and 36, with 32 tokens 42 and 44; 1024 with 32 126 and 103; 64 with 64 39 and 26; one with
  // 8 tokens 11 and 11, with 4096 38 and 26.  How the tokens are spread over the requests is not known here.
  if (a.cache.tokens < 24ll * a.batch) {
    a.kv_parts = static_cast<int>(parts(resident / 3, kWarps));
    plan_items(a.queries, head_dim, is_fp32, (resident - (resident / 3)) * kWarps, kTokens);
    const long long grid = windows * a.kv_parts + query_ctas();
    if (grid > 0x7fffffffll) return -GDPA_ERR_LAUNCH_;
    return by_type([&](auto type, auto dim) -> int {
      gdpa_rotated_step_kernel<decltype(type), decltype(dim)::value><<<static_cast<unsigned>(grid), kWarps * 32, kQueryBytes, stream>>>(a);
      return cudaGetLastError() == cudaSuccess ? 1 : -GDPA_ERR_LAUNCH_;
    });
  }
  plan_items(a.queries, head_dim, is_fp32, resident * kWarps, kTokens);
  const int rc = by_type([&](auto type, auto dim) -> int {
    gdpa_rotated_queries_kernel<decltype(type), decltype(dim)::value><<<static_cast<unsigned>(query_ctas()), kWarps * 32, kQueryBytes, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? 1 : -GDPA_ERR_LAUNCH_;
  });
  if (rc < 0 || a.cache.num_blocks == 0) return rc;
  auto launch = [&](auto type, auto dim, auto warps, auto hold) -> int {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value, W = decltype(warps)::value, HOLD = decltype(hold)::value;
    a.kv_parts = static_cast<int>(parts(2ll * runs_ctas(W, HOLD * 2 * HeadLanes<T, D>::E) * sm_count, W));
    const long long grid = windows * a.kv_parts;
    if (grid > 0x7fffffffll) return -GDPA_ERR_LAUNCH_;
    auto kernel = gdpa_rotated_runs_kernel<T, D, W, HOLD>;
    // A block of fewer rows than the lanes hold takes less; what the kernel may have at most, which other host threads' calls set too, stays the same.
    constexpr int kRing = W * HOLD * kUnitPieces * 16, kTables = W * HOLD * HeadLanes<T, D>::H * D * static_cast<int>(sizeof(float));
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing + kTables) != cudaSuccess) return -GDPA_ERR_LAUNCH_;
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(static_cast<unsigned>(grid));
    c.blockDim = dim3(W * 32);
    c.dynamicSmemBytes = kRing + (D << a.cache.block_shift) * static_cast<int>(sizeof(float));
    c.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, static_cast<const RotatedAppendArgs&>(a)) == cudaSuccess ? 2 : -GDPA_ERR_LAUNCH_;
  };
  // Warps so that a lane holds 64 values of a block at most: a head of 64 tokens and 128 values takes four, one of 128 tokens eight.
  return by_type([&](auto type, auto dim) -> int {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value, V = 2 * HeadLanes<T, D>::E;
    using W4 = std::integral_constant<int, 4>;
    using W8 = std::integral_constant<int, 8>;
    const int values = D << a.cache.block_shift;
    if constexpr (D == 128) {
      if (values == 16384) return launch(type, dim, W8{}, std::integral_constant<int, 64 / V>{});
    }
    if (values == 8192) return launch(type, dim, W4{}, std::integral_constant<int, 64 / V>{});
    if (values == 4096) return launch(type, dim, W4{}, std::integral_constant<int, 32 / V>{});
    return launch(type, dim, W4{}, std::integral_constant<int, 16 / V>{});
  });
}

}  // namespace gdpa
