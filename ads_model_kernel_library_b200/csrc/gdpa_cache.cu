// What fills a paged key / value cache of 8-bit values: the block tables and slot maps of a batch of requests, built from their
// lengths, and the quantiser that writes new keys and values into their slots.
//
// A cache is [blocks, block_size, heads, head_dim] e4m3 with one fp32 scale per (block, head); slot = block * block_size + row.  The
// table of a request holds the blocks of its tokens in order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

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
constexpr int kTableThreads = 1024;
constexpr int kTableMostPer = 8;  // requests per thread in one round: 8192 requests with 96 KB of shared memory

struct RequestScan {
  unsigned tokens, blocks;  // before this request, from the start of the round
  int cached;
};

__device__ __forceinline__ int clamp_len(const void* p, int b, int flags) {
  return static_cast<int>(clamp_ll(load_offset(p, b, flags), 0, 0x3fffffff));
}

__global__ void __launch_bounds__(kTableThreads) gdpa_block_tables_kernel(const BlockTableArgs a) {
  extern __shared__ RequestScan s_req[];
  __shared__ unsigned long long s_warp[32];
  const int t = threadIdx.x, lane = t & 31, wp = t >> 5;
  const int S = 1 << a.block_shift;
  const long long have = clamp_ll(*a.num_free, 0, a.free_capacity);
  long long tok0 = 0, blk0 = 0;  // before this round's requests
  for (int b0 = 0; b0 < a.batch; b0 += kTableThreads * a.per) {
    const int nb = min(kTableThreads * a.per, a.batch - b0);
    const int first = t * a.per;
    int cached[kTableMostPer];
    unsigned long long mine[kTableMostPer], sum = 0;  // new tokens in the high half, new blocks in the low one
#pragma unroll
    for (int i = 0; i < kTableMostPer; ++i) {
      cached[i] = 0, mine[i] = 0;
      if (i < a.per && first + i < nb) {
        const int b = b0 + first + i;
        const int c = clamp_len(a.cached_lens, b, a.lens_are_int64), n = clamp_len(a.new_lens, b, a.lens_are_int64);
        const int held = min((c + S - 1) >> a.block_shift, a.table_width);
        const int after = static_cast<int>(min((static_cast<long long>(c) + n + S - 1) >> a.block_shift, static_cast<long long>(a.table_width)));
        cached[i] = c;
        mine[i] = (static_cast<unsigned long long>(n) << 32) | static_cast<unsigned>(after - held);
        if (blockIdx.x == 0) a.seq_lens[b] = static_cast<int>(min(static_cast<long long>(c) + n, 0x7fffffffll));
      }
    }
#pragma unroll
    for (int i = 0; i < kTableMostPer; ++i) sum += mine[i];
    unsigned long long incl = sum;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const unsigned long long o = __shfl_up_sync(kFull, incl, s);
      if (lane >= s) incl += o;
    }
    if (lane == 31) s_warp[wp] = incl;
    __syncthreads();
    if (wp == 0) {
      unsigned long long w = s_warp[lane];
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const unsigned long long o = __shfl_up_sync(kFull, w, s);
        if (lane >= s) w += o;
      }
      s_warp[lane] = w;
    }
    __syncthreads();
    unsigned long long run = incl - sum + (wp > 0 ? s_warp[wp - 1] : 0ull);
    const unsigned long long all = s_warp[31];
#pragma unroll
    for (int i = 0; i < kTableMostPer; ++i) {
      if (i < a.per && first + i < nb) {
        s_req[first + i] = RequestScan{static_cast<unsigned>(run >> 32), static_cast<unsigned>(run), cached[i]};
        if (blockIdx.x == 0) a.query_offset[b0 + first + i] = static_cast<int>(tok0 + static_cast<long long>(run >> 32));
      }
      run += mine[i];
    }
    __syncthreads();
    const unsigned n_tok = static_cast<unsigned>(all >> 32);
    for (unsigned k = blockIdx.x * kTableThreads + t; k < n_tok; k += gridDim.x * kTableThreads) {
      int lo = 0, hi = nb;  // the last request that begins at or before token k has it: those without tokens begin where the next one does
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_req[mid].tokens <= k) lo = mid;
        else hi = mid;
      }
      const RequestScan r = s_req[lo];
      const long long p = static_cast<long long>(r.cached) + (k - r.tokens);
      const long long j = p >> a.block_shift;
      const int held = min((r.cached + S - 1) >> a.block_shift, a.table_width);
      int* const row = a.block_tables + static_cast<long long>(b0 + lo) * a.table_stride;
      int blk = -1;
      if (j < held) {
        blk = row[j];
      } else if (j < a.table_width) {
        const long long at = have - 1 - (blk0 + r.blocks + (j - held));
        if (at >= 0) blk = a.free_blocks[at];
        if ((p & (S - 1)) == 0) row[j] = blk;
      }
      if (tok0 + k < a.total_new)
        a.slots[tok0 + k] = blk < 0 ? -1ll : (static_cast<long long>(blk) << a.block_shift) + (p & (S - 1));
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
// One warp has a run and a head: it needs no barrier, and a whole block of one head is 16 to 32 KB, enough in flight for
// a warp.  The 32 tokens of a window find their runs with a vote; a window's (run, head, key or value) triples are dealt
// out to the warps of gridDim.y CTAs, many of them when there are few tokens (a step of generation), one when there are many.
constexpr int kAppendWarps = 8;

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
};
template <>
struct Piece<float> {
  static constexpr int kElems = 4;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
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

template <class T, int D>
__global__ void __launch_bounds__(kAppendWarps * 32) gdpa_cache_append_kernel(const CacheAppendArgs a) {
  constexpr int E = Piece<T>::kElems;
  constexpr int kLanesPerRow = D / E;              // lanes that hold one row
  constexpr int kRows = 32 / kLanesPerRow;         // rows of one warp-wide load
  constexpr int kUnroll = 8;
  const int lane = threadIdx.x & 31;
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
  const int tasks = __popc(leaders) * 2 * a.heads;
  for (int task = blockIdx.y * kAppendWarps + (threadIdx.x >> 5); task < tasks; task += gridDim.y * kAppendWarps) {
    const int head2 = task % (2 * a.heads);
    const int at = __fns(leaders, 0, task / (2 * a.heads) + 1);  // lane of the run's first token
    const bool is_value = head2 >= a.heads;
    const int h = is_value ? head2 - a.heads : head2;
    const long long s0 = __shfl_sync(kFull, slot, at), t0 = base + at;
    const int o = static_cast<int>(s0 & (S - 1));
    const long long blk = s0 >> a.block_shift;
    // length: as far as the slots go on, at most to the end of the block
    int len = 0;
    for (bool more = true; more;) {
      const int i = len + lane;
      const bool goes_on = o + i < S && slot_of(t0 + i) == s0 + i;
      const unsigned stops = __ballot_sync(kFull, !goes_on);
      len += stops ? __ffs(stops) - 1 : 32;
      more = stops == 0;
    }
    const T* const x = static_cast<const T*>(is_value ? a.value : a.key) + t0 * (is_value ? a.value_strides[0] : a.key_strides[0]) +
                       h * (is_value ? a.value_strides[1] : a.key_strides[1]);
    const long long row_stride = is_value ? a.value_strides[0] : a.key_strides[0];
    float* const scale_at = (is_value ? a.v_scales : a.k_scales) + blk * a.heads + h;
    const long long* const cs = is_value ? a.v_cache_strides : a.k_cache_strides;
    uint8_t* const out = (is_value ? a.v_cache : a.k_cache) + blk * cs[0] + h * cs[2];
    const int r0 = lane / kLanesPerRow, e0 = (lane % kLanesPerRow) * E;
    const float old = o > 0 ? *scale_at : 0.f;
    // the largest magnitude as bits of fp32: they order like the values
    uint32_t top = 0;
    for (int r = r0; r < len; r += kRows * kUnroll) {
      uint4 u[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        u[i] = r + i * kRows < len ? *reinterpret_cast<const uint4*>(x + (r + i * kRows) * row_stride + e0) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        float v[E];
        Piece<T>::unpack(u[i], v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t m = __float_as_uint(v[e]) & 0x7fffffffu;
          top = max(top, m < 0x7f800000u ? m : 0u);
        }
      }
    }
    top = __reduce_max_sync(kFull, top);
    const float fresh = __uint_as_float(static_cast<uint32_t>(scale_exponent(top) + 127) << 23);
    const float scale = old > fresh ? old : fresh;
    if (o > 0 && scale != old) {
      // the rows before the run, rescaled
      const float ratio = old / scale;
      constexpr int kCacheLanes = D / 16;
      for (int r = lane / kCacheLanes; r < o; r += 32 / kCacheLanes) {
        uint4* const p = reinterpret_cast<uint4*>(out + r * cs[1] + (lane % kCacheLanes) * 16);
        uint4 u = *p;
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 lo = e4m3x2_values(w[i] & 0xffffu), hi = e4m3x2_values(w[i] >> 16);
          w[i] = pack_e4m3x4(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    const float inv = 1.f / scale;
    for (int r = r0; r < len; r += kRows * kUnroll) {
      uint4 u[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i)
        if (r + i * kRows < len) u[i] = *reinterpret_cast<const uint4*>(x + (r + i * kRows) * row_stride + e0);
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        if (r + i * kRows >= len) break;
        float v[E];
        Piece<T>::unpack(u[i], v);
        uint32_t w[E / 4];
#pragma unroll
        for (int e = 0; e < E / 4; ++e) w[e] = pack_e4m3x4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv, v[4 * e + 3] * inv);
        uint8_t* const p = out + (o + r + i * kRows) * cs[1] + e0;
        if constexpr (E == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t*>(p) = w[0];
      }
    }
    if (lane == 0 && scale != old) *scale_at = scale;
  }
}

}  // namespace

int launch_block_tables(const BlockTableArgs& args, int sm_count, cudaStream_t stream) {
  BlockTableArgs a = args;
  a.per = a.batch > kTableThreads * kTableMostPer ? kTableMostPer : (a.batch + kTableThreads - 1) / kTableThreads;
  if (a.per < 1) a.per = 1;
  const size_t smem = static_cast<size_t>(kTableThreads) * a.per * sizeof(RequestScan);
  if (smem > 48 * 1024) {
    if (cudaFuncSetAttribute(gdpa_block_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess)
      return GDPA_ERR_LAUNCH_;
  }
  long long grid = (a.total_new + kTableThreads - 1) / kTableThreads;
  grid = grid < 1 ? 1 : grid > sm_count ? sm_count : grid;
  gdpa_block_tables_kernel<<<static_cast<unsigned>(grid), kTableThreads, smem, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

int launch_cache_append(const CacheAppendArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  if (a.tokens == 0) return 0;
  const long long windows = (a.tokens + 31) / 32;
  // CTAs for a window: enough for two dozen warps on every SM, at most one warp for each triple of a window of single tokens
  const long long wanted = 24ll * sm_count / kAppendWarps, most = (32ll * 2 * a.heads + kAppendWarps - 1) / kAppendWarps;
  long long y = (wanted + windows - 1) / windows;
  y = y > most ? most : y < 1 ? 1 : y;
  const dim3 grid(static_cast<unsigned>(windows), static_cast<unsigned>(y));
  auto launch = [&](auto kernel) { kernel<<<grid, kAppendWarps * 32, 0, stream>>>(a); };
  if (is_fp32) head_dim == 128 ? launch(gdpa_cache_append_kernel<float, 128>) : launch(gdpa_cache_append_kernel<float, 64>);
  else head_dim == 128 ? launch(gdpa_cache_append_kernel<__nv_bfloat16, 128>) : launch(gdpa_cache_append_kernel<__nv_bfloat16, 64>);
  return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

}  // namespace gdpa
