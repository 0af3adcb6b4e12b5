// A serving step's queries, keys and values between the projection and the attention: queries and keys are normed and rotated
// (gdpa_rotary.cuh), keys and values quantised into their slots of the paged cache as gdpa_cache.cu does it (the same runs, scales and
// rules), queries written for the attention.  One launch: the first CTAs have keys and values, the others queries.
//
// What bounds it: HBM for prompts (a query value is 2 bytes in and 2 out, a key or value 2 and 1), latency for single tokens.  Rotated keys stay in
// fp32 registers between the maximum of a run and its conversion: they are rounded once, to e4m3.
//
// Keys and values: a CTA looks at a window of 32 tokens for the runs that begin there.  Three ways to share the work, by the window's
// number of runs: all warps on one (run, head), the run's angles in shared memory for all its heads (prompts); a warp to each (run, head), a
// head's lanes to a row (drafts); a head's lanes to each (run, head) (single tokens).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_rotary.cuh"

namespace gdpa {

namespace {

// The request that has token t, by the whole warp: the last one that begins at or before it.
__device__ __forceinline__ int owner_of(const RotatedAppendArgs& a, long long t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = a.batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(kAllLanes, at < hi && load_offset(a.q_off, at, a.off64) <= t);
    lo += (below == 0 ? 0 : __popc(below) - 1) * step;
    hi = min(hi, lo + step);
  }
  return lo;
}
// position of the request's token with index 0 of the call
__device__ __forceinline__ long long origin_of(const RotatedAppendArgs& a, int owner) {
  return a.batch == 0 ? 0 : load_offset(a.seq_lens, owner, a.lens64) - load_offset(a.q_off, owner + 1, a.off64);
}
__device__ __forceinline__ long long given_position(const RotatedAppendArgs& a, int axis, long long token) {
  const long long i = axis * a.position_stride + token;
  return a.positions_are_int64 ? static_cast<const long long*>(a.positions)[i] : static_cast<const int*>(a.positions)[i];
}

// One run of one head, keys (KEY) or values, by the lanes that hold its rows r0, r0 + step, ...; the first HOLD of them stay in registers, further
// ones are made again.  `angles(row, c, s)` gives a lane its angles; `top_of` makes a maximum over all the run's lanes.  Lanes without a
// run have len 0; every lane of a warp comes along.  `first`: whether this lane writes the scale.
template <class T, int D, int HOLD, bool KEY, class Angles, class Top>
__device__ __forceinline__ void store_run(const RotatedAppendArgs& a, const HeadLanes<T, D>& lanes, const float* s_weight, int r0, int step, int h,
                                          long long t0, long long blk, int o, int len, bool first, Angles angles, Top top_of) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E, V = Lanes::V;
  const CacheAppendArgs& ca = a.cache;
  const long long row_stride = KEY ? ca.key_strides[0] : ca.value_strides[0];
  const T* const x = static_cast<const T*>(KEY ? ca.key : ca.value) + t0 * row_stride + h * (KEY ? ca.key_strides[1] : ca.value_strides[1]);
  float* const scale_at = (KEY ? ca.k_scales : ca.v_scales) + blk * ca.heads + h;
  const long long* const cs = KEY ? ca.k_cache_strides : ca.v_cache_strides;
  uint8_t* const out = (KEY ? ca.k_cache : ca.v_cache) + blk * cs[0] + h * cs[2];
  auto load = [&](int r, uint4 (&u)[2]) {
    u[0] = u[1] = make_uint4(0, 0, 0, 0);
    if (r < len) {
      const uint4* const p = reinterpret_cast<const uint4*>(x + r * row_stride);
      u[0] = __ldg(p + lanes.g0), u[1] = __ldg(p + lanes.g1);
    }
  };
  auto values = [&](int r, const uint4 (&u)[2], float (&v)[V]) {
    Lanes::unpack(u, v);
    if constexpr (KEY) {
      if (a.rotary.norm) {
        float ss = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) ss += v[e] * v[e];
        const float f = rsqrtf(Lanes::sum(ss) * (1.f / D) + a.rotary.eps);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = v[e] * f;
        float w[E];
        lanes.take(s_weight, w);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= w[e];
        lanes.take(s_weight + D / 2, w);
#pragma unroll
        for (int e = 0; e < E; ++e) v[E + e] *= w[e];
      }
      if (r < len && lanes.rotated) {
        float c[E], s[E];
        angles(r, c, s);
        lanes.template turn<false>(a.rotary.interleaved, c, s, v);
      }
    }
  };
  const float old = o > 0 && len > 0 ? *scale_at : 0.f;
  float v[HOLD][V];
  uint32_t top = 0;
  {
    uint4 u[HOLD][2];
#pragma unroll
    for (int i = 0; i < HOLD; ++i) load(r0 + i * step, u[i]);
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      values(r0 + i * step, u[i], v[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(v[i][e]) & 0x7fffffffu);
    }
  }
  auto further = [&](auto body) {  // the rows that are not held
    for (int r = r0 + HOLD * step; __any_sync(kAllLanes, r < len); r += step) {
      uint4 u[2];
      float w[V];
      load(r, u);
      values(r, u, w);
      if (r < len) body(r, w);
    }
  };
  further([&](int, const float (&w)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) top = max(top, __float_as_uint(w[e]) & 0x7fffffffu);
  });
  top = top_of(top);
  if (__any_sync(kAllLanes, top >= kInfBits)) {
    // rare: an infinity or NaN.  The maximum over the others.
    top = 0;
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t m = __float_as_uint(v[i][e]) & 0x7fffffffu;
        top = max(top, m < kInfBits ? m : 0u);
      }
    }
    further([&](int, const float (&w)[V]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const uint32_t m = __float_as_uint(w[e]) & 0x7fffffffu;
        top = max(top, m < kInfBits ? m : 0u);
      }
    });
    top = top_of(top);
  }
  const float fresh = __uint_as_float(static_cast<uint32_t>(scale_exponent(top) + 127) << 23);
  const float scale = old > fresh ? old : fresh;
  if (o > 0 && len > 0 && scale != old) {
    // the rows before the run, rescaled
    const float ratio = old / scale;
    constexpr int P = D / 16;  // 16-byte pieces of a row, over the lanes of a head
    for (int r = r0; r < o; r += step) {
#pragma unroll
      for (int k = 0; k < (P + Lanes::L - 1) / Lanes::L; ++k) {
        if (k * Lanes::L + lanes.l >= P) continue;
        uint4* const p = reinterpret_cast<uint4*>(out + r * cs[1]) + k * Lanes::L + lanes.l;
        const uint4 held = *p;
        uint32_t q[4] = {held.x, held.y, held.z, held.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 lo = e4m3x2_values(q[i] & 0xffffu), hi = e4m3x2_values(q[i] >> 16);
          q[i] = pack_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
        }
        *p = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
  }
  const float inv = 1.f / scale;
  auto store = [&](int r, const float (&w)[V]) {
    uint8_t* const p = out + (o + r) * cs[1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t q[E / 4];
#pragma unroll
      for (int e = 0; e < E / 4; ++e)
        q[e] = pack_e4m3x4(w[k * E + 4 * e] * inv, w[k * E + 4 * e + 1] * inv, w[k * E + 4 * e + 2] * inv, w[k * E + 4 * e + 3] * inv);
      uint8_t* const at = p + (k == 0 ? lanes.g0 : lanes.g1) * E;
      if constexpr (E == 8) *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<uint32_t*>(at) = q[0];
    }
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (r0 + i * step < len) store(r0 + i * step, v[i]);
  further(store);
  if (first && len > 0 && scale != old) *scale_at = scale;
}

// Queries of a warp: a stretch of (token, heads) items, so that neighbouring tokens find their request at once.
template <class T, int D>
__device__ __forceinline__ void rotate_queries(const RotatedAppendArgs& a, const HeadLanes<T, D>& lanes, const float* s_weight, float* s_cos, float* s_sin,
                                               long long first) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E, V = Lanes::V, U = 2;
  const WarpAngles<T, D> angles(a.rotary);
  const long long items = a.cache.tokens * a.chunks, last = min(first + a.items_per_warp, items);
  long long token = -1, origin = 0, begin = 0, end = -1;  // of the request that is at hand: its first token and the one behind its last
  float c[E], s[E];
  for (long long i = first; i < last; ++i) {
    const long long t = a.chunks == 1 ? i : i / a.chunks;
    const int head0 = static_cast<int>(i - t * a.chunks) * a.per_item, head1 = min(head0 + a.per_item, a.heads);
    const T* const x = static_cast<const T*>(a.query) + t * a.query_strides[0];
    T* const y = static_cast<T*>(a.query_out) + t * a.heads * D;
    uint4 u[U][2];
    auto load = [&](int h0) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int head = h0 + k * Lanes::H + lanes.sub;
        u[k][0] = u[k][1] = make_uint4(0, 0, 0, 0);
        if (head < head1) {
          const uint4* const p = reinterpret_cast<const uint4*>(x + head * a.query_strides[1]);
          u[k][0] = __ldg(p + lanes.g0), u[k][1] = __ldg(p + lanes.g1);
        }
      }
    };
    load(head0);
    if (t != token) {
      token = t;
      if (a.positions == nullptr && !(t >= begin && t < end)) {
        const int owner = owner_of(a, t);
        origin = origin_of(a, owner);
        begin = a.batch == 0 ? 0 : load_offset(a.q_off, owner, a.off64);
        end = a.batch == 0 ? 0x7fffffffffffffffll : load_offset(a.q_off, owner + 1, a.off64);
      }
      __syncwarp();
      angles.write(s_cos, s_sin, [&](int axis) { return a.positions != nullptr ? given_position(a, axis, t) : origin + t; });
      __syncwarp();
      if (lanes.rotated) lanes.take(s_cos, c), lanes.take(s_sin, s);
    }
    for (int h0 = head0;;) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int head = h0 + k * Lanes::H + lanes.sub;
        float v[V];
        Lanes::unpack(u[k], v);
        if (a.rotary.norm) {
          float ss = 0;
#pragma unroll
          for (int e = 0; e < V; ++e) ss += v[e] * v[e];
          const float r = rsqrtf(Lanes::sum(ss) * (1.f / D) + a.rotary.eps);
          float w[E];
          lanes.take(s_weight, w);
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = v[e] * r * w[e];
          lanes.take(s_weight + D / 2, w);
#pragma unroll
          for (int e = 0; e < E; ++e) v[E + e] = v[E + e] * r * w[e];
        }
        lanes.template turn<false>(a.rotary.interleaved, c, s, v);
        if (head < head1) {
          uint4* const p = reinterpret_cast<uint4*>(y + static_cast<long long>(head) * D);
          p[lanes.g0] = Piece<T>::pack(v);
          p[lanes.g1] = Piece<T>::pack(v + E);
        }
      }
      h0 += U * Lanes::H;
      if (h0 >= head1) break;
      load(h0);
    }
  }
}

// W warps of a CTA; HOLD rows of a lane when all of them are on one run, so that a whole block is held.
template <class T, int D, int W, int HOLD>
__global__ void __launch_bounds__(W * 32) gdpa_rotated_append_kernel(const __grid_constant__ RotatedAppendArgs a) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E;
  extern __shared__ float4 s_table[];  // angles: a block's rows, [row][2][D / 2]
  __shared__ float4 s_weight4[D / 4];  // the weight, as the lanes take it: their first pieces' and their second ones'
  __shared__ double s_frequency[D / 2];    // of the pairs, in a lane's order
  __shared__ int s_axis[D / 2];
  __shared__ uint32_t s_top[2][W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Lanes lanes(a.rotary);
  float* const s_weight = reinterpret_cast<float*>(s_weight4);
  float* const table = reinterpret_cast<float*>(s_table);
  const int kv_ctas = a.kv_windows * a.kv_parts;
  const bool queries = static_cast<int>(blockIdx.x) >= kv_ctas;
  if (warp == 0 && lane < Lanes::L) {
    const void* const weight = queries ? a.query_weight : a.key_weight;
    const int bf16 = queries ? a.query_weight_is_bf16 : a.key_weight_is_bf16;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s_weight[Lanes::slot(lane, e)] = weight_at(weight, bf16, lanes.g0 * E + e);
      s_weight[D / 2 + Lanes::slot(lane, e)] = weight_at(weight, bf16, lanes.g1 * E + e);
    }
  }
  if (!queries) {
    for (int i = threadIdx.x; i < a.rotary.pairs; i += W * 32) {
      const int at = Lanes::slot_of_pair(a.rotary, i);
      s_frequency[at] = frequency_of_pair(a.rotary, i), s_axis[at] = axis_of_pair(a.rotary, i);
    }
  }
  __syncthreads();
  if (queries) {
    const long long first = (static_cast<long long>(blockIdx.x - kv_ctas) * W + warp) * a.items_per_warp;
    rotate_queries<T, D>(a, lanes, s_weight, table + warp * D, table + warp * D + D / 2, first);
    return;
  }
  const CacheAppendArgs& ca = a.cache;
  const int S = 1 << ca.block_shift;
  const int part = blockIdx.x / a.kv_windows;
  const long long base = static_cast<long long>(blockIdx.x - part * a.kv_windows) * 32;
  const long long slots = ca.num_blocks << ca.block_shift;
  auto slot_of = [&](long long t) -> long long {
    if (t < 0 || t >= ca.tokens) return -1;
    const long long s = ca.slot_mapping[t];
    return s >= 0 && s < slots ? s : -1;
  };
  const long long slot = slot_of(base + lane);
  long long before = __shfl_up_sync(kAllLanes, slot, 1);
  if (lane == 0) before = slot_of(base - 1);
  const bool leads = slot >= 0 && ((slot & (S - 1)) == 0 || before != slot - 1);
  const unsigned leaders = __ballot_sync(kAllLanes, leads);
  const int runs = __popc(leaders);
  if (runs == 0) return;
  // position of the first token of the run that this lane leads, less its index
  long long origin = 0;
  if (a.positions == nullptr) {
    // the requests of the 32 tokens: the first one's, and whose beginnings follow
    const int b0 = owner_of(a, base);
    int owner = b0;
    for (int b = b0 + 1; b < a.batch; b += 32) {
      const long long begin = b + lane < a.batch ? load_offset(a.q_off, b + lane, a.off64) : 0x7fffffffffffffffll;
      int count = 0;  // of these 32 that begin at or before the lane's token
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) count += __shfl_sync(kAllLanes, begin, count + s - 1) <= base + lane ? s : 0;
      count += __shfl_sync(kAllLanes, begin, count) <= base + lane;
      owner += count;
      if (__shfl_sync(kAllLanes, begin, 31) > base + 31) break;
    }
    origin = origin_of(a, owner);
  }
  // tokens of the run that begins with token base + at: as far as the slots go on, at most to the end of the block
  auto length_of = [&](int at, long long s0) -> int {
    const int o = static_cast<int>(s0 & (S - 1));
    int len = 0;
    for (bool more = true; more;) {
      const int i = len + lane;
      const long long near = __shfl_sync(kAllLanes, slot, (at + i) & 31);
      const bool goes_on = o + i < S && (at + i < 32 ? near : slot_of(base + at + i)) == s0 + i;
      const unsigned stops = __ballot_sync(kAllLanes, !goes_on);
      len += stops ? __ffs(stops) - 1 : 32;
      more = stops == 0;
    }
    return len;
  };
  // a lane's angles, made by itself
  auto own_angles = [&](long long t, long long run_origin, float (&c)[E], float (&s)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = Lanes::slot(lanes.l, e);
      sin_cos(s_frequency[at], a.positions != nullptr ? given_position(a, s_axis[at], t) : run_origin + t, s[e], c[e]);
    }
  };
  if (runs <= 2) {
    unsigned turn = 0;
    for (unsigned left = leaders; left != 0; left &= left - 1) {
      const int at = __ffs(left) - 1;
      const long long s0 = __shfl_sync(kAllLanes, slot, at), run_origin = __shfl_sync(kAllLanes, origin, at), t0 = base + at;
      const int len = length_of(at, s0);
      auto top_of = [&](uint32_t top) {
        top = __reduce_max_sync(kAllLanes, top);
        uint32_t* const s = s_top[turn++ & 1u];  // two in turn: the next maximum is written while this one may still be read
        if (lane == 0) s[warp] = top;
        __syncthreads();
        top = s[0];
#pragma unroll
        for (int i = 1; i < W; ++i) top = max(top, s[i]);
        return top;
      };
      const long long blk = s0 >> ca.block_shift;
      const int o = static_cast<int>(s0 & (S - 1)), r0 = warp * Lanes::H + lanes.sub;
      if (part < ca.heads) {  // this CTA has keys of the run: its angles
        __syncthreads();      // the last run's have been read
        const WarpAngles<T, D> angles(a.rotary);
        for (int r = warp; r < len; r += W) {
          const long long t = t0 + r;
          angles.write(table + r * D, table + r * D + D / 2,
                       [&](int axis) { return a.positions != nullptr ? given_position(a, axis, t) : run_origin + t; });
        }
        __syncthreads();
      }
      for (int head2 = part; head2 < 2 * ca.heads; head2 += a.kv_parts) {
        if (head2 < ca.heads) {
          store_run<T, D, HOLD, true>(a, lanes, s_weight, r0, W * Lanes::H, head2, t0, blk, o, len, threadIdx.x == 0,
                                      [&](int r, float (&c)[E], float (&s)[E]) {
            lanes.take(table + r * D, c);
            lanes.take(table + r * D + D / 2, s);
          }, top_of);
        } else {
          store_run<T, D, HOLD, false>(a, lanes, s_weight, r0, W * Lanes::H, head2 - ca.heads, t0, blk, o, len, threadIdx.x == 0,
                                       [](int, float (&)[E], float (&)[E]) {}, top_of);
        }
      }
    }
    return;
  }
  const bool single = runs > 16;  // two tokens a run at most, on average: a head's lanes to a run, else a warp
  const int a_warp = single ? Lanes::H : 1, tasks = runs * ca.heads;
  const int rounds = (tasks + a_warp - 1) / a_warp;
  for (int i = part * W + warp; i < 2 * rounds; i += a.kv_parts * W) {
    const bool is_key = i < rounds;
    const int task = (is_key ? i : i - rounds) * a_warp + (single ? lanes.sub : 0);
    const bool there = task < tasks;
    const int at = there ? __fns(leaders, 0, task / ca.heads + 1) : 0;
    const int h = there ? task % ca.heads : 0;
    const long long s0 = __shfl_sync(kAllLanes, slot, at), run_origin = __shfl_sync(kAllLanes, origin, at), t0 = base + at;
    int len = 0;
    if (single) {
      // up to four runs: each by the whole warp
#pragma unroll
      for (int k = 0; k < Lanes::H; ++k) {
        const int l = length_of(__shfl_sync(kAllLanes, at, k * Lanes::L), __shfl_sync(kAllLanes, s0, k * Lanes::L));
        if (lanes.sub == k) len = l;
      }
    } else {
      len = length_of(at, s0);
    }
    if (!there) len = 0;
    const long long blk = there ? s0 >> ca.block_shift : 0;
    const int o = there ? static_cast<int>(s0 & (S - 1)) : 0;
    const int r0 = single ? 0 : lanes.sub, step = single ? 1 : Lanes::H;
    auto top_of = [&](uint32_t top) {
      if (!single) return __reduce_max_sync(kAllLanes, top);
#pragma unroll
      for (int s = 1; s < Lanes::L; s <<= 1) top = max(top, __shfl_xor_sync(kAllLanes, top, s));
      return top;
    };
    const bool first = lanes.l == 0 && (single || lanes.sub == 0);
    if (is_key) {
      store_run<T, D, 2, true>(a, lanes, s_weight, r0, step, h, t0, blk, o, len, first,
                               [&](int r, float (&c)[E], float (&s)[E]) { own_angles(t0 + r, run_origin, c, s); }, top_of);
    } else {
      store_run<T, D, 2, false>(a, lanes, s_weight, r0, step, h, t0, blk, o, len, first, [](int, float (&)[E], float (&)[E]) {}, top_of);
    }
  }
}

}  // namespace

int launch_rotated_append(RotatedAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  if (a.cache.tokens == 0) return 0;
  auto launch = [&](auto type, auto dim, auto warps) -> int {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value, W = decltype(warps)::value;
    using Lanes = HeadLanes<T, D>;
    const int S = 1 << a.cache.block_shift;
    // keys and values: as many CTAs for a window as make a few waves, at most one warp for each run and head of single tokens
    const long long windows = (a.cache.tokens + 31) / 32, wanted = (96ll / W) * sm_count;
    const long long most = (32ll * 2 * a.cache.heads / Lanes::H + W) / W;
    long long parts = a.cache.num_blocks > 0 ? (wanted + windows - 1) / windows : 0;
    parts = parts > most ? most : parts;
    a.kv_windows = static_cast<int>(windows);
    a.kv_parts = static_cast<int>(parts);
    split_heads(a.cache.tokens, a.heads, Lanes::H, 16ll * sm_count, a.per_item, a.chunks);
    const long long items = a.cache.tokens * a.chunks, at_once = 48ll * sm_count;
    a.items_per_warp = (items + at_once - 1) / at_once;
    const long long query_ctas = (items + a.items_per_warp * W - 1) / (a.items_per_warp * W);
    const long long grid = windows * parts + query_ctas;
    if (grid > 0x7fffffffll) return GDPA_ERR_LAUNCH_;
    auto kernel_for = [&](auto hold) -> int {
      auto kernel = gdpa_rotated_append_kernel<T, D, W, decltype(hold)::value>;
      const int rows = S > W ? S : W;
      const int smem = rows * D * static_cast<int>(sizeof(float));
      if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return GDPA_ERR_LAUNCH_;
      kernel<<<static_cast<unsigned>(grid), W * 32, smem, stream>>>(a);
      return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
    };
    const int hold = S / (W * Lanes::H);
    if constexpr (64 / (4 * Lanes::H) >= 4) {  // blocks of 64 and 128 (with twice the warps)
      if (hold > 2) {
        using All = std::integral_constant<int, 64 / (4 * Lanes::H)>;
        return kernel_for(All{});
      }
    }
    return kernel_for(std::integral_constant<int, 2>{});
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  auto by_warps = [&](auto type, auto dim) -> int {
    if (a.cache.block_shift == 7) return launch(type, dim, std::integral_constant<int, 8>{});
    return launch(type, dim, std::integral_constant<int, 4>{});
  };
  if (is_fp32) return head_dim == 128 ? by_warps(float{}, D128{}) : by_warps(float{}, D64{});
  return head_dim == 128 ? by_warps(__nv_bfloat16{}, D128{}) : by_warps(__nv_bfloat16{}, D64{});
}

}  // namespace gdpa
