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
  const RotaryTensor& q = a.queries.t[0];
  const long long i = axis * q.position_stride + token;
  return q.positions_are_int64 ? static_cast<const long long*>(q.positions)[i] : static_cast<const int*>(q.positions)[i];
}

// One run of one head, keys (KEY) or values, by the lanes that hold its rows r0, r0 + step, ...; the first HOLD of them come as they are in `u` and
// stay in registers, further ones (ALL: there are none) are read and made again.  `angles(row, c, s)` gives a lane its angles; `top_of` makes a maximum over all the
// run's lanes.  Lanes without a run have len 0; every lane of a warp comes along.  `first`: whether this lane writes the scale.
template <class T, int D, int HOLD, bool ALL, bool KEY, class Angles, class Top>
__device__ __forceinline__ void store_run(const RotatedAppendArgs& a, const HeadLanes<T, D>& lanes, const float* s_weight, const uint4 (&u)[HOLD][2], int r0, int step,
                                          int h, long long t0, long long blk, int o, int len, bool first, Angles angles, Top top_of) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E, C = Lanes::C;
  const CacheAppendArgs& ca = a.cache;
  const RotarySpec& spec = a.queries.rotary;
  const long long row_stride = KEY ? ca.key_strides[0] : ca.value_strides[0];
  const T* const x = static_cast<const T*>(KEY ? ca.key : ca.value) + t0 * row_stride + h * (KEY ? ca.key_strides[1] : ca.value_strides[1]);
  float* const scale_at = (KEY ? ca.k_scales : ca.v_scales) + blk * ca.heads + h;
  const long long* const cs = KEY ? ca.k_cache_strides : ca.v_cache_strides;
  uint8_t* const out = (KEY ? ca.k_cache : ca.v_cache) + blk * cs[0] + h * cs[2];
  auto values = [&](int r, const uint4 (&p)[2], uint64_t (&v)[2 * C]) {
    Lanes::unpack(p, v);
    if constexpr (KEY) {
      uint64_t c[C], s[C];
      if (lanes.rotated) angles(r < len ? r : 0, c, s);
      rotate_unit<T, D>(spec, lanes, s_weight, c, s, v);
    }
  };
  auto largest = [](uint32_t top, const uint64_t (&v)[2 * C], bool finite) {
#pragma unroll
    for (int e = 0; e < 2 * C; ++e) {
      float lo, hi;
      unpack_f32x2(v[e], lo, hi);
      const uint32_t p = __float_as_uint(lo) & 0x7fffffffu, q = __float_as_uint(hi) & 0x7fffffffu;
      top = max(top, finite && p >= kInfBits ? 0u : p);
      top = max(top, finite && q >= kInfBits ? 0u : q);
    }
    return top;
  };
  const float old = o > 0 && len > 0 ? *scale_at : 0.f;
  uint64_t v[HOLD][2 * C];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < HOLD; ++i) values(r0 + i * step, u[i], v[i]);
  float scale = 0, inv = 0;
  auto store = [&](int r, const uint64_t (&given)[2 * C]) {
    uint8_t* const p = out + (o + r) * cs[1];
    uint64_t w[2 * C];
#pragma unroll
    for (int e = 0; e < 2 * C; ++e) w[e] = given[e];
    Lanes::times(inv, w);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t q[E / 4];
#pragma unroll
      for (int e = 0; e < E / 4; ++e) {
        float f[4];
        unpack_f32x2(w[k * C + 2 * e], f[0], f[1]);
        unpack_f32x2(w[k * C + 2 * e + 1], f[2], f[3]);
        q[e] = pack_e4m3x4(f[0], f[1], f[2], f[3]);
      }
      uint8_t* const at = p + (k == 0 ? lanes.g0 : lanes.g1) * E;
      if constexpr (E == 8) *reinterpret_cast<uint2*>(at) = make_uint2(q[0], q[1]);
      else *reinterpret_cast<uint32_t*>(at) = q[0];
    }
  };
  // Three passes over the rows: their maximum; if it is none, an infinity or NaN among them (rare), that of the others; their conversion.
  for (int pass = 0;;) {
#pragma unroll
    for (int i = 0; i < HOLD; ++i) {
      if (pass < 2) top = largest(top, v[i], pass == 1);
      else if (r0 + i * step < len) store(r0 + i * step, v[i]);
    }
    if constexpr (!ALL) {
      for (int r = r0 + HOLD * step; __any_sync(kAllLanes, r < len); r += step) {
        uint4 p[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (r < len) {
          const uint4* const at = reinterpret_cast<const uint4*>(x + r * row_stride);
          p[0] = __ldg(at + lanes.g0), p[1] = __ldg(at + lanes.g1);
        }
        uint64_t w[2 * C];
        values(r, p, w);
        if (r >= len) continue;
        if (pass < 2) top = largest(top, w, pass == 1);
        else store(r, w);
      }
    }
    if (pass == 2) break;
    top = top_of(top);
    if (pass == 0 && __any_sync(kAllLanes, top >= kInfBits)) {
      pass = 1, top = 0;
      continue;
    }
    pass = 2;
    const float fresh = __uint_as_float(static_cast<uint32_t>(scale_exponent(top) + 127) << 23);
    scale = old > fresh ? old : fresh;
    inv = 1.f / scale;
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
  }
  if (first && len > 0 && scale != old) *scale_at = scale;
}

// A warp's share of a CTA's shared memory: its ring of units; and of its tables, which for keys and values are those of a block's rows.
template <int HOLD>
constexpr int kRing = 2 * HOLD > 6 ? 2 * HOLD : 6;

// W warps of a CTA; HOLD rows of a lane when all of them are on one run, so that a whole block is held.
template <class T, int D, int W, int HOLD>
__global__ void __launch_bounds__(W * 32, 16 / W) gdpa_rotated_append_kernel(const __grid_constant__ RotatedAppendArgs a) {
  using Lanes = HeadLanes<T, D>;
  constexpr int C = Lanes::C, RING = kRing<HOLD>;
  extern __shared__ uint4 s_dynamic[];
  __shared__ float4 s_weight4[D / 4];
  __shared__ double s_frequency[D / 2];  // of the pairs, in a lane's order
  __shared__ int s_axis[D / 2];
  __shared__ uint32_t s_top[2][W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* const s_weight = reinterpret_cast<float*>(s_weight4);
  uint4* const ring = s_dynamic + warp * RING * kUnitPieces;
  float* const tables = reinterpret_cast<float*>(s_dynamic + W * RING * kUnitPieces);
  const bool given = a.queries.t[0].positions != nullptr;
  const int kv_ctas = a.kv_windows * a.kv_parts;
  if (static_cast<int>(blockIdx.x) >= kv_ctas) {
    long long origin = 0, begin = 0, end = -1;  // of the request at hand: its first token and the one behind its last
    rotate_items<T, D, RING>(a.queries, ring, tables + warp * kItemTokens * D, s_weight, 1, (blockIdx.x - kv_ctas) * W + warp, (gridDim.x - kv_ctas) * W,
                             [&](int, int axis, long long t) -> long long {
      return given ? given_position(a, axis, t) : origin + t;
    }, [&](long long t) {
      if (given || (t >= begin && t < end)) return;
      const int owner = owner_of(a, t);
      origin = origin_of(a, owner);
      begin = a.batch == 0 ? 0 : load_offset(a.q_off, owner, a.off64);
      end = a.batch == 0 ? 0x7fffffffffffffffll : load_offset(a.q_off, owner + 1, a.off64);
    });
    return;
  }
  const Lanes lanes(a.queries.rotary);
  if (warp == 0) lanes.write_weight(s_weight, a.queries.t[1].weight, a.queries.t[1].weight_is_bf16);
  for (int i = threadIdx.x; i < a.queries.rotary.pairs; i += W * 32) {
    const int at = Lanes::slot_of_pair(a.queries.rotary, i);
    s_frequency[at] = frequency_of_pair(a.queries.rotary, i), s_axis[at] = axis_of_pair(a.queries.rotary, i);
  }
  __syncthreads();
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
  auto origin_of_run = [&]() -> long long {
    if (given) return 0;
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
    return origin_of(a, owner);
  };
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
  auto none = [](int, uint64_t (&)[C], uint64_t (&)[C]) {};
  if (runs <= 2) {
    // all warps on one run of one head after the other; the next ones are on their way
    constexpr int AHEAD = RING / HOLD;
    unsigned turn = 0;
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
    long long origin = 0;
    bool found = false;
    for (unsigned left = leaders; left != 0; left &= left - 1) {
      const int at = __ffs(left) - 1;
      const long long s0 = __shfl_sync(kAllLanes, slot, at), t0 = base + at, blk = s0 >> ca.block_shift;
      const int len = length_of(at, s0), o = static_cast<int>(s0 & (S - 1)), r0 = warp * Lanes::H + lanes.sub;
      constexpr int step = W * Lanes::H;
      int ahead = part, ahead_slot = 0;
      auto fetch = [&]() {
        if (ahead < 2 * ca.heads) {
          const bool key = ahead < ca.heads;
          const int h = key ? ahead : ahead - ca.heads;
          const long long* const xs = key ? ca.key_strides : ca.value_strides;
          HeadWalk<T, D> walk;
          walk.at = static_cast<T*>(const_cast<void*>(key ? ca.key : ca.value)) + (t0 + r0) * xs[0] + h * xs[1];
          walk.unit = step * xs[0];
#pragma unroll
          for (int i = 0; i < HOLD; ++i) {
            walk.fetch(lanes, ring + (ahead_slot * HOLD + i) * kUnitPieces, r0 + i * step < len);
            walk.next(false);
          }
          ahead += a.kv_parts;
        }
        fetch_commit();
        ahead_slot = ahead_slot + 1 == AHEAD ? 0 : ahead_slot + 1;
      };
#pragma unroll
      for (int i = 0; i + 1 < AHEAD; ++i) fetch();
      if (!found) origin = origin_of_run(), found = true;
      if (part < ca.heads) {  // this CTA has keys of the run: its angles
        const long long run_origin = __shfl_sync(kAllLanes, origin, at);
        __syncthreads();      // the last run's have been read
        const WarpAngles<T, D> angles(a.queries.rotary);
        for (int r = warp; r < len; r += W)
          angles.write(tables + r * D, [&](int axis) { return given ? given_position(a, axis, t0 + r) : run_origin + t0 + r; });
        __syncthreads();
      }
      int at_slot = 0;
      for (int head2 = part; head2 < 2 * ca.heads; head2 += a.kv_parts) {
        fetch();
        fetch_wait<AHEAD - 1>();
        uint4 u[HOLD][2];
#pragma unroll
        for (int i = 0; i < HOLD; ++i) fetched(ring + (at_slot * HOLD + i) * kUnitPieces, u[i]);
        at_slot = at_slot + 1 == AHEAD ? 0 : at_slot + 1;
        if (head2 < ca.heads) {
          store_run<T, D, HOLD, true, true>(a, lanes, s_weight, u, r0, step, head2, t0, blk, o, len, threadIdx.x == 0, [&](int r, uint64_t (&c)[C], uint64_t (&s)[C]) {
            lanes.take(tables + r * D, c);
            lanes.take(tables + r * D + D / 2, s);
          }, top_of);
        } else {
          store_run<T, D, HOLD, true, false>(a, lanes, s_weight, u, r0, step, head2 - ca.heads, t0, blk, o, len, threadIdx.x == 0, none, top_of);
        }
      }
    }
    return;
  }
  const long long origin = origin_of_run();
  // a lane's angles, made by itself
  auto own_angles = [&](long long t, long long run_origin, uint64_t (&c)[C], uint64_t (&s)[C]) {
#pragma unroll
    for (int e = 0; e < C; ++e) {
      float sn[2], cs[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = Lanes::slot(lanes.l, 2 * e + i);
        sin_cos<T>(s_frequency[at], given ? given_position(a, s_axis[at], t) : run_origin + t, sn[i], cs[i]);
      }
      c[e] = pack_f32x2(cs[0], cs[1]), s[e] = pack_f32x2(sn[0], sn[1]);
    }
  };
  // a warp to each run and head, its heads' lanes to a row each; or, with two tokens a run at most on average, a head's lanes to each run and head
  auto deal = [&](auto lanes_of_a_head) {
    constexpr bool single = decltype(lanes_of_a_head)::value;
    constexpr int a_warp = single ? Lanes::H : 1, HELD = 1, step = single ? 1 : Lanes::H;
    const int tasks = runs * ca.heads, rounds = (tasks + a_warp - 1) / a_warp;
    for (int i = part * W + warp; i < 2 * rounds; i += a.kv_parts * W) {
      const bool is_key = i < rounds;
      const int task = (is_key ? i : i - rounds) * a_warp + (single ? lanes.sub : 0);
      const bool there = task < tasks;
      const int at = there ? __fns(leaders, 0, task / ca.heads + 1) : 0, h = there ? task % ca.heads : 0;
      const long long s0 = __shfl_sync(kAllLanes, slot, at), run_origin = __shfl_sync(kAllLanes, origin, at), t0 = base + at;
      int len = 0;
      if constexpr (single) {
#pragma unroll
        for (int k = 0; k < Lanes::H; ++k) {  // each by the whole warp
          const int l = length_of(__shfl_sync(kAllLanes, at, k * Lanes::L), __shfl_sync(kAllLanes, s0, k * Lanes::L));
          if (lanes.sub == k) len = l;
        }
      } else {
        len = length_of(at, s0);
      }
      if (!there) len = 0;
      const long long blk = there ? s0 >> ca.block_shift : 0;
      const int o = there ? static_cast<int>(s0 & (S - 1)) : 0, r0 = single ? 0 : lanes.sub;
      auto top_of = [&](uint32_t top) {
        if (!single) return __reduce_max_sync(kAllLanes, top);
#pragma unroll
        for (int s = 1; s < Lanes::L; s <<= 1) top = max(top, __shfl_xor_sync(kAllLanes, top, s));
        return top;
      };
      const bool first = lanes.l == 0 && (single || lanes.sub == 0);
      const long long* const xs = is_key ? ca.key_strides : ca.value_strides;
      const T* const x = static_cast<const T*>(is_key ? ca.key : ca.value) + t0 * xs[0] + h * xs[1];
      uint4 u[HELD][2];
#pragma unroll
      for (int k = 0; k < HELD; ++k) {
        u[k][0] = u[k][1] = make_uint4(0, 0, 0, 0);
        if (r0 + k * step < len) {
          const uint4* const p = reinterpret_cast<const uint4*>(x + (r0 + k * step) * xs[0]);
          u[k][0] = __ldg(p + lanes.g0), u[k][1] = __ldg(p + lanes.g1);
        }
      }
      if (is_key) {
        store_run<T, D, HELD, false, true>(a, lanes, s_weight, u, r0, step, h, t0, blk, o, len, first,
                                    [&](int r, uint64_t (&c)[C], uint64_t (&s)[C]) { own_angles(t0 + r, run_origin, c, s); }, top_of);
      } else {
        store_run<T, D, HELD, false, false>(a, lanes, s_weight, u, r0, step, h, t0, blk, o, len, first, none, top_of);
      }
    }
  };
  if (runs > 16) deal(std::true_type{});
  else deal(std::false_type{});
}

}  // namespace

int launch_rotated_append(RotatedAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  if (a.cache.tokens == 0) return 0;
  auto launch = [&](auto type, auto dim, auto warps, auto hold) -> int {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value, W = decltype(warps)::value, HOLD = decltype(hold)::value;
    using Lanes = HeadLanes<T, D>;
    const int S = 1 << a.cache.block_shift;
    // keys and values: as many CTAs for a window as make two waves, at most one warp for each run and head of single tokens
    const long long windows = (a.cache.tokens + 31) / 32, wanted = (32ll / W) * sm_count;
    const long long most = (32ll * 2 * a.cache.heads / Lanes::H + W - 1) / W;
    long long parts = a.cache.num_blocks > 0 ? (wanted + windows - 1) / windows : 0;
    parts = parts > most ? most : parts;
    a.kv_windows = static_cast<int>(windows);
    a.kv_parts = static_cast<int>(parts);
    plan_items(a.queries, head_dim, is_fp32, 10ll * sm_count);
    long long query_ctas = (static_cast<long long>(a.queries.items[0]) + W - 1) / W;
    if (query_ctas > (16ll / W) * sm_count) query_ctas = (16ll / W) * sm_count;
    const long long grid = windows * parts + query_ctas;
    if (grid > 0x7fffffffll) return GDPA_ERR_LAUNCH_;
    auto kernel = gdpa_rotated_append_kernel<T, D, W, HOLD>;
    const int rows = S > W * kItemTokens ? S : W * kItemTokens;
    const int smem = W * kRing<HOLD> * kUnitPieces * 16 + rows * D * static_cast<int>(sizeof(float));
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return GDPA_ERR_LAUNCH_;
    kernel<<<static_cast<unsigned>(grid), W * 32, smem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
  };
  // Warps so that a lane holds 32 values of a block at most: those of one head of 64 tokens and 128 values take eight.
  auto by_block = [&](auto type, auto dim) -> int {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value, H = HeadLanes<T, D>::H;
    using W4 = std::integral_constant<int, 4>;
    using W8 = std::integral_constant<int, 8>;
    using W16 = std::integral_constant<int, 16>;
    using Most = std::integral_constant<int, 128 * 128 / (16 * HeadLanes<T, 128>::H * 128)>;  // 2 (bf16), 4 (fp32)
    using Half = std::integral_constant<int, Most::value / 2>;
    const int values = D << a.cache.block_shift;
    if constexpr (D == 128) {
      if (values == 128 * 128) return launch(type, dim, W16{}, Most{});
    }
    if (values == 128 * 64) return launch(type, dim, W8{}, std::integral_constant<int, 128 * 64 / (8 * H * D)>{});
    if (values == 128 * 32) return launch(type, dim, W4{}, std::integral_constant<int, 128 * 32 / (4 * H * D)>{});
    return launch(type, dim, W4{}, Half{});
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (is_fp32) return head_dim == 128 ? by_block(float{}, D128{}) : by_block(float{}, D64{});
  return head_dim == 128 ? by_block(__nv_bfloat16{}, D128{}) : by_block(__nv_bfloat16{}, D64{});
}

}  // namespace gdpa
