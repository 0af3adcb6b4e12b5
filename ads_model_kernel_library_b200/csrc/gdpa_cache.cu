// What fills a paged key / value cache of 8-bit values: the block tables and slot maps of a batch of requests, built from their
// lengths, and the quantiser that writes new keys and values into their slots.
//
// A cache is [blocks, block_size, heads, head_dim] e4m3 with one fp32 scale per (block, head); slot = block * block_size + row.  The
// table of a request holds the blocks of its tokens in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"

namespace gdpa {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// ------------------------------------------------------------------------------------------ block tables, slot maps
//
// Request b has c cached and n new tokens: blocks [ceil(c / S), ceil((c + n) / S)) of its table are taken from the top of the stack of
// free blocks, in the order of the requests; token i goes to row (c + i) % S of block (c + i) / S.  Every CTA scans the
// lengths for itself (4 bytes a request from L2: cheaper than a second launch, and nothing waits for another CTA) and then
// writes its share of the tokens; the thread that has the first token of a new block also writes that block into the table.
//
// Latency is all of it: three trips to memory one after the other (lengths, free blocks, slots) between a launch and its end.  PER is the
// number of requests a thread has in one round, in registers; the small form (64 requests: 4.9 -> 4.0 us) has neither the
// unrolled code nor the threads of the large one.  Alone: 64 requests with a token each 4.0 us, 512 new ones (1.2 M tokens) 11.4, 8192 9.2.
__device__ __forceinline__ int clamp_len(const void* p, int b, int flags) {
  return static_cast<int>(clamp_ll(load_offset(p, b, flags), 0, 0x3fffff00));  // two of them and a block fit in an int
}

// Where there are more tokens than slots: the new blocks that begin with a token without one, by one CTA.  For itself and at the kernel's end: not
// what a caller should do, and a call within the rounds cost the usual case 1.3 us.  A thread has a stretch of requests, and the sums before it.
__device__ __noinline__ void blocks_without_slots(const BlockTableArgs& a, long long have) {
  const int S = 1 << a.block_shift;
  const int per = (a.batch + blockDim.x - 1) / blockDim.x;
  const int b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
  long long tok = 0, blk = 0;
  for (int b = 0; b < b1; ++b) {
    const int cached = clamp_len(a.cached_lens, b, a.lens_are_int64), n = clamp_len(a.new_lens, b, a.lens_are_int64);
    const int held = min((cached + S - 1) >> a.block_shift, a.table_width), after = min((cached + n + S - 1) >> a.block_shift, a.table_width);
    if (b >= b0) {
      for (int j = held; j < after; ++j) {
        const long long at = have - 1 - (blk + (j - held));
        if (tok + ((static_cast<long long>(j) << a.block_shift) - cached) >= a.total_new)
          a.block_tables[static_cast<long long>(b) * a.table_stride + j] = at >= 0 ? a.free_blocks[at] : -1;
      }
    }
    tok += n;
    blk += after - held;
  }
}

template <int kTableThreads, int PER>
__global__ void __launch_bounds__(kTableThreads) gdpa_block_tables_kernel(const __grid_constant__ BlockTableArgs a) {
  constexpr int kWarps = kTableThreads / 32;
  // of the round's requests: new tokens and blocks before them (from the start of the round), cached tokens
  extern __shared__ unsigned s_tokens[];
  constexpr int round = kTableThreads * PER;
  unsigned* const s_blocks = s_tokens + round;
  int* const s_cached = reinterpret_cast<int*>(s_blocks + round);
  __shared__ unsigned long long s_warp[kWarps];
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  const int S = 1 << a.block_shift;
  const long long have = clamp_ll(*a.num_free, 0, a.free_capacity);
  long long tok0 = 0, blk0 = 0;  // before this round's requests
  for (int b0 = 0; b0 < a.batch; b0 += round) {
    const int nb = min(round, a.batch - b0);
    // A warp has 32 * per neighbouring requests, 32 at a time over its lanes: new tokens in the high half of the sums, new
    // blocks in the low one.
    int cached[PER];
    unsigned long long mine[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = (wp * PER + i) * 32 + lane;
      cached[i] = 0, mine[i] = 0;
      if (at < nb) {
        cached[i] = clamp_len(a.cached_lens, b0 + at, a.lens_are_int64);
        mine[i] = clamp_len(a.new_lens, b0 + at, a.lens_are_int64);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int n = static_cast<int>(mine[i]);
      const int held = min((cached[i] + S - 1) >> a.block_shift, a.table_width);
      const int after = min((cached[i] + n + S - 1) >> a.block_shift, a.table_width);
      const unsigned long long m = (static_cast<unsigned long long>(n) << 32) | static_cast<unsigned>(after - held);
      unsigned long long incl = m;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const unsigned long long o = __shfl_up_sync(kFull, incl, s);
        if (lane >= s) incl += o;
      }
      mine[i] = sum + incl - m;  // before this request, in the warp
      sum += __shfl_sync(kFull, incl, 31);
    }
    if (lane == 0) s_warp[wp] = sum;
    __syncthreads();
    unsigned long long warps = lane < kWarps ? s_warp[lane] : 0ull;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const unsigned long long o = __shfl_up_sync(kFull, warps, s);
      if (lane >= s) warps += o;
    }
    const unsigned long long all = __shfl_sync(kFull, warps, 31), before = __shfl_sync(kFull, warps, (wp + 31) & 31);
    const unsigned n_tok = static_cast<unsigned>(all >> 32);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int at = (wp * PER + i) * 32 + lane;
      const unsigned long long run = mine[i] + (wp > 0 ? before : 0ull);
      s_cached[at] = cached[i];
      s_tokens[at] = static_cast<unsigned>(run >> 32);
      s_blocks[at] = static_cast<unsigned>(run);
    }
    __syncthreads();
    for (int i = blockIdx.x * kTableThreads + t; i < nb; i += gridDim.x * kTableThreads) {
      const unsigned end = i + 1 < nb ? s_tokens[i + 1] : n_tok;
      a.query_offset[b0 + i] = static_cast<int>(tok0 + s_tokens[i]);
      a.seq_lens[b0 + i] = static_cast<int>(min(static_cast<long long>(s_cached[i]) + (end - s_tokens[i]), 0x7fffffffll));
    }
    // tokens that have a slot to write: all, if total_new is what the lengths add up to, which bounds the walk whatever they say
    const unsigned n_walk = static_cast<unsigned>(clamp_ll(a.total_new - tok0, 0, n_tok));
    // A warp takes 128 tokens at a time, four of each lane's at once.  The last request that begins at or before a token has it (one
    // without tokens begins where the next does): looked for among all requests by the whole warp for the first and the last
    // of the 128, between these two by each lane.
    auto owner_by_warp = [&](unsigned k) -> int {
      int lo = 0, hi = nb;
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        lo += (__popc(__ballot_sync(kFull, at < hi && s_tokens[at] <= k)) - 1) * step;
        hi = min(hi, lo + step);
      }
      return lo;
    };
    for (unsigned k0 = (blockIdx.x * kWarps + wp) * 128u; k0 < n_walk; k0 += gridDim.x * kWarps * 128u) {
      const int from = owner_by_warp(k0), to = owner_by_warp(min(k0 + 127u, n_walk - 1)) + 1;
      int owner[4], blk[4];
      long long p[4];
      bool begins[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned k = min(k0 + 32u * i + lane, n_walk - 1);
        int lo = from, hi = to;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_tokens[mid] <= k) lo = mid;
          else hi = mid;
        }
        owner[i] = lo;
        p[i] = static_cast<long long>(s_cached[lo]) + (k - s_tokens[lo]);
        const long long j = p[i] >> a.block_shift;
        const int held = min((s_cached[lo] + S - 1) >> a.block_shift, a.table_width);
        blk[i] = -1;
        begins[i] = false;
        if (j < held) {
          blk[i] = a.block_tables[static_cast<long long>(b0 + lo) * a.table_stride + j];
        } else if (j < a.table_width) {
          const long long at = have - 1 - (blk0 + s_blocks[lo] + (j - held));
          if (at >= 0) blk[i] = a.free_blocks[at];
          begins[i] = (p[i] & (S - 1)) == 0;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned k = k0 + 32u * i + lane;
        if (k >= n_walk) continue;
        if (begins[i]) a.block_tables[static_cast<long long>(b0 + owner[i]) * a.table_stride + (p[i] >> a.block_shift)] = blk[i];
        a.slots[tok0 + k] = blk[i] < 0 ? -1ll : (static_cast<long long>(blk[i]) << a.block_shift) + (p[i] & (S - 1));
      }
    }
    tok0 += n_tok;
    blk0 += static_cast<unsigned>(all);
    __syncthreads();
  }
  for (long long k = tok0 + blockIdx.x * kTableThreads + t; k < a.total_new; k += static_cast<long long>(gridDim.x) * kTableThreads) a.slots[k] = -1;
  if (blockIdx.x == 0 && t == 0) {
    a.query_offset[a.batch] = static_cast<int>(min(tok0, 0x7fffffffll));
    *a.num_free_after = static_cast<int>(clamp_ll(have - blk0, -0x7fffffff, 0x7fffffff));
  }
  if (blockIdx.x == 0 && tok0 > a.total_new) blocks_without_slots(a, have);
}

// ------------------------------------------------------------------------------------------ new keys and values
//
// A run is a stretch of new tokens with consecutive slots of one block; its first row is o.  For every run and head, keys and values each:
//   fresh = the smallest power of two with amax / fresh <= 448 (finite values only), at least 2^-100;
//   scale = fresh if o = 0 (the block is new), else max(the block's scale, fresh);
//   rows below o become e4m3(value * old scale / scale) if the scale has grown, the run's rows are e4m3(x / scale).
// Powers of two: the division is exact, and a value that is rescaled keeps its three mantissa bits (down to e4m3's subnormals), so
// that a block filled token by token holds what it would hold if filled at once.
//
// What bounds it: HBM with long runs (2 or 4 bytes in, one out per value), latency with single tokens.  So with long runs four warps share a
// (run, head, key or value) and hold it in registers between the maximum and the conversion: one pass over the values, 16 KB and more
// in flight per CTA.  With short ones a warp has one to itself, and nothing waits for another.  The 32 tokens of a window find
// their runs with a vote; a window's triples are dealt out to gridDim.y CTAs.  Measured: 128 histories of 512 to 4096 tokens, 8 heads of 128
// values, 318 us (5.8 TB/s; a warp to a run 577), one token for 256 requests 4.1, 300 ragged runs of fp32 7.0.
constexpr int kAppendWarps = 4;

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

// W warps (1 or kAppendWarps) quantise one run of one head; `w` is this warp's number among them.  `top_of` makes a maximum over the
// lanes of all W warps of the fp32 bits it is given.  The first HOLD pieces of a lane stay in registers, further ones are read again.
template <class T, int D, int W, int HOLD, class F>
__device__ __forceinline__ void quantise_run(const CacheAppendArgs& a, int w, bool is_value, int h, long long t0, long long blk, int o, int len,
                                             F top_of) {
  constexpr int E = Piece<T>::kElems;
  constexpr int kLanesPerRow = D / E;       // lanes that hold one row
  constexpr int kRows = 32 / kLanesPerRow;  // rows of one warp-wide load
  constexpr int kStep = W * kRows;
  const int lane = threadIdx.x & 31;
  const long long row_stride = is_value ? a.value_strides[0] : a.key_strides[0];
  const int r0 = w * kRows + lane / kLanesPerRow, e0 = (lane % kLanesPerRow) * E;
  const T* const x = static_cast<const T*>(is_value ? a.value : a.key) + t0 * row_stride + h * (is_value ? a.value_strides[1] : a.key_strides[1]) + e0;
  float* const scale_at = (is_value ? a.v_scales : a.k_scales) + blk * a.heads + h;
  const long long* const cs = is_value ? a.v_cache_strides : a.k_cache_strides;
  uint8_t* const out = (is_value ? a.v_cache : a.k_cache) + blk * cs[0] + h * cs[2];
  auto piece = [&](int r) { return __ldg(reinterpret_cast<const uint4*>(x + r * row_stride)); };
  const float old = o > 0 ? *scale_at : 0.f;
  uint4 u[HOLD];
#pragma unroll
  for (int i = 0; i < HOLD; ++i) u[i] = r0 + i * kStep < len ? piece(r0 + i * kStep) : make_uint4(0, 0, 0, 0);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < HOLD; ++i) top = Piece<T>::magnitude(top, u[i]);
  for (int r = r0 + HOLD * kStep; r < len; r += kStep) top = Piece<T>::magnitude(top, piece(r));
  top = top_of(Piece<T>::whole(top));
  if (top >= kInfBits) {
    // rare: an infinity or NaN.  The maximum over the others.
    top = 0;
    for (int r = r0; r < len; r += kStep) {
      float v[E];
      Piece<T>::unpack(piece(r), v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
        top = max(top, m < kInfBits ? m : 0u);
      }
    }
    top = top_of(top);
  }
  const float fresh = __uint_as_float(static_cast<uint32_t>(scale_exponent(top) + 127) << 23);
  const float scale = old > fresh ? old : fresh;
  if (o > 0 && scale != old) {
    // the rows before the run, rescaled
    const float ratio = old / scale;
    constexpr int kCacheLanes = D / 16;
    for (int r = w * (32 / kCacheLanes) + lane / kCacheLanes; r < o; r += W * (32 / kCacheLanes)) {
      uint4* const p = reinterpret_cast<uint4*>(out + r * cs[1] + (lane % kCacheLanes) * 16);
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
  const float inv = 1.f / scale;
  uint8_t* const first = out + o * cs[1] + e0;
  auto store = [&](int r, const uint4& from) {
    float v[E];
    Piece<T>::unpack(from, v);
    uint32_t q[E / 4];
#pragma unroll
    for (int e = 0; e < E / 4; ++e) q[e] = pack_e4m3x4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv, v[4 * e + 3] * inv);
    uint8_t* const p = first + r * cs[1];
    if constexpr (E == 8) *reinterpret_cast<uint2*>(p) = make_uint2(q[0], q[1]);
    else *reinterpret_cast<uint32_t*>(p) = q[0];
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (r0 + i * kStep < len) store(r0 + i * kStep, u[i]);
  for (int r = r0 + HOLD * kStep; r < len; r += kStep) store(r, piece(r));
  if (w == 0 && lane == 0 && scale != old) *scale_at = scale;
}

// HOLD: pieces of a lane that a whole block of one head takes with kAppendWarps warps, 16 at most.
template <class T, int D, int HOLD>
__global__ void __launch_bounds__(kAppendWarps * 32) gdpa_cache_append_kernel(const CacheAppendArgs a) {
  __shared__ uint32_t s_top[2][kAppendWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int S = 1 << a.block_shift;
  const long long base = static_cast<long long>(blockIdx.x) * 32;
  const long long slots = a.num_blocks << a.block_shift;
  auto slot_of = [&](long long t) -> long long {
    if (t < 0 || t >= a.tokens) return -1;
    const long long s = a.slot_mapping[t];
    return s >= 0 && s < slots ? s : -1;
  };
  const long long slot = slot_of(base + lane);
  long long before = __shfl_up_sync(kFull, slot, 1);
  if (lane == 0) before = slot_of(base - 1);
  const bool leads = slot >= 0 && ((slot & (S - 1)) == 0 || before != slot - 1);
  const unsigned leaders = __ballot_sync(kFull, leads);
  // the run that begins with token base + at
  struct Run {
    long long s0;
    int len;
  };
  auto run_at = [&](int at) -> Run {
    Run r{__shfl_sync(kFull, slot, at), 0};
    const int o = static_cast<int>(r.s0 & (S - 1));
    // as far as the slots go on, at most to the end of the block
    for (bool more = true; more;) {
      const int i = r.len + lane;
      const long long near = __shfl_sync(kFull, slot, (at + i) & 31);
      const bool goes_on = o + i < S && (at + i < 32 ? near : slot_of(base + at + i)) == r.s0 + i;
      const unsigned stops = __ballot_sync(kFull, !goes_on);
      r.len += stops ? __ffs(stops) - 1 : 32;
      more = stops == 0;
    }
    return r;
  };
  // Runs of 16 tokens and more on average: all warps on one.  (300 requests with runs of some ten tokens that way: 8.5 -> 11.0 us.)
  if (__popc(leaders) <= 2) {
    unsigned turn = 0;
    for (unsigned left = leaders; left != 0; left &= left - 1) {
      const int at = __ffs(left) - 1;
      const Run r = run_at(at);
      for (int head2 = blockIdx.y; head2 < 2 * a.heads; head2 += gridDim.y) {
        const bool is_value = head2 >= a.heads;
        quantise_run<T, D, kAppendWarps, HOLD>(a, warp, is_value, is_value ? head2 - a.heads : head2, base + at, r.s0 >> a.block_shift,
                                               static_cast<int>(r.s0 & (S - 1)), r.len, [&](uint32_t top) {
          top = __reduce_max_sync(kFull, top);
          uint32_t* const s = s_top[turn++ & 1u];  // two in turn: the next maximum is written while this one may still be read
          if (lane == 0) s[warp] = top;
          __syncthreads();
          return max(max(s[0], s[1]), max(s[2], s[3]));
        });
      }
    }
  } else {
    const int tasks = __popc(leaders) * 2 * a.heads;
    for (int task = blockIdx.y * kAppendWarps + warp; task < tasks; task += gridDim.y * kAppendWarps) {
      const int head2 = task % (2 * a.heads);
      const int at = __fns(leaders, 0, task / (2 * a.heads) + 1);  // lane of the run's first token
      const Run r = run_at(at);
      const bool is_value = head2 >= a.heads;
      quantise_run<T, D, 1, 4>(a, 0, is_value, is_value ? head2 - a.heads : head2, base + at, r.s0 >> a.block_shift,
                               static_cast<int>(r.s0 & (S - 1)), r.len, [&](uint32_t top) { return __reduce_max_sync(kFull, top); });
    }
  }
}

}  // namespace

int launch_block_tables(const BlockTableArgs& a, int sm_count, cudaStream_t stream) {
  auto launch = [&](auto kernel, int threads, int per) -> int {
    const int smem = threads * per * 3 * static_cast<int>(sizeof(int));
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return GDPA_ERR_LAUNCH_;
    long long grid = (a.total_new + 4 * threads - 1) / (4 * threads);
    const long long most = 2ll * sm_count;
    grid = grid < 1 ? 1 : grid > most ? most : grid;
    kernel<<<static_cast<unsigned>(grid), threads, smem, stream>>>(a);
    return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
  };
  if (a.batch <= 256) return launch(gdpa_block_tables_kernel<256, 1>, 256, 1);
  if (a.batch <= 1024) return launch(gdpa_block_tables_kernel<1024, 1>, 1024, 1);
  return launch(gdpa_block_tables_kernel<1024, 8>, 1024, 8);
}

int launch_cache_append(const CacheAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  if (a.tokens == 0) return 0;
  const long long windows = (a.tokens + 31) / 32;
  // CTAs for a window: enough for a few waves of them, at most one warp for each triple of a window of single tokens
  const long long wanted = 24ll * sm_count, most = (32ll * 2 * a.heads + kAppendWarps - 1) / kAppendWarps;
  long long y = (wanted + windows - 1) / windows;
  y = y > most ? most : y < 1 ? 1 : y;
  const dim3 grid(static_cast<unsigned>(windows), static_cast<unsigned>(y));
  const int pieces = (head_dim * (is_fp32 ? 4 : 2) << a.block_shift) / (kAppendWarps * 32 * 16);
  auto launch = [&](auto type, auto dim) {
    using T = decltype(type);
    constexpr int D = decltype(dim)::value;
    if (pieces <= 4) gdpa_cache_append_kernel<T, D, 4><<<grid, kAppendWarps * 32, 0, stream>>>(a);
    else if (pieces <= 8) gdpa_cache_append_kernel<T, D, 8><<<grid, kAppendWarps * 32, 0, stream>>>(a);
    else gdpa_cache_append_kernel<T, D, 16><<<grid, kAppendWarps * 32, 0, stream>>>(a);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (is_fp32) head_dim == 128 ? launch(float{}, D128{}) : launch(float{}, D64{});
  else head_dim == 128 ? launch(__nv_bfloat16{}, D128{}) : launch(__nv_bfloat16{}, D64{});
  return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

}  // namespace gdpa
