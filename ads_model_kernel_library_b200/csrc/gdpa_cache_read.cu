// What a paged cache of 8-bit values holds, read back as packed keys and values: token i of request b is its cached token first[b] + i.
//
// value = e4m3 * scale, in fp32, rounded once (a power of two times e4m3 is a bf16 number: then nothing is rounded).  A token
// without a block (one beyond the table, an entry outside the cache) and a row that no request has are zeros.
//
// HBM-bound: a byte in, two or four out.  A warp takes some neighbouring tokens, 32 at most; its lanes find their requests and blocks, then the warp walks
// over the tokens' rows, keys, then values, 16 bytes of the output a lane, several pieces asked for before the first is written.  300 000 tokens of 8 heads of 128
// values to bf16, 1.84 GB: 317 us cold, 5.8 TB/s (a plain copy 6.5); 1500 tokens of one request 6 us, three trips to memory in a row.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"
#include "gdpa_pieces.cuh"

namespace gdpa {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kReadWarps = 4;

template <class T, int D>
__global__ void __launch_bounds__(kReadWarps * 32) gdpa_cache_read_kernel(const __grid_constant__ CacheReadArgs a) {
  constexpr int E = Piece<T>::kElems;  // values of a lane at a time: 16 bytes of the output
  constexpr int P = D / E;             // pieces of a head
  constexpr int U = 8;                 // pieces of a lane that are asked for at once
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long base = (static_cast<long long>(blockIdx.x) * kReadWarps + warp) * a.warp_tokens;
  if (base >= a.total) return;
  const int tokens = static_cast<int>(min(static_cast<long long>(a.warp_tokens), a.total - base));
  // where the lane's token is: its block (-1: nowhere) and row
  const int owner = request_of_lane(a.offsets, a.off64, a.batch, base, base + tokens - 1);
  int block = -1, row = 0;
  if (a.batch > 0 && lane < tokens) {
    const long long begin = load_offset(a.offsets, owner, a.off64), end = load_offset(a.offsets, owner + 1, a.off64);
    const long long first = a.first != nullptr ? load_offset(a.first, owner, a.first64) : 0, p = first + (base + lane - begin);
    if (base + lane >= begin && base + lane < end && first < (1ll << 31) && p >= 0 && (p >> a.block_shift) < a.table_width) {
      block = a.block_tables[owner * a.table_stride + (p >> a.block_shift)];
      row = static_cast<int>(p & ((1 << a.block_shift) - 1));
      if (block < 0 || block >= a.num_blocks) block = -1;
    }
  }
  // Pieces of a token's row over the lanes: `wide` rounds of 32 of one token, or several tokens in a round.
  const int pieces = a.heads * P;
  const int in_round = pieces < 32 ? 32 / pieces : 1, wide = (pieces + 31) / 32;
  const int my_token = pieces < 32 ? lane / pieces : 0, my_piece = pieces < 32 ? lane - my_token * pieces : lane;
  const int rounds = (tokens + in_round - 1) / in_round * wide;
#pragma unroll 1
  for (int kv = 0; kv < 2; ++kv) {
    const uint8_t* const cache = kv == 0 ? a.k_cache : a.v_cache;
    const long long* const cs = kv == 0 ? a.k_cache_strides : a.v_cache_strides;
    const float* const scales = kv == 0 ? a.k_scales : a.v_scales;
    T* const out = static_cast<T*>(kv == 0 ? a.key : a.value) + base * a.heads * D;
    int token = 0, part = 0;  // of the next round
#pragma unroll 1
    for (int i0 = 0; i0 < rounds; i0 += U) {
      uint32_t u[U][E / 4];
      float scale[U];
      int to[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int t = token + my_token, piece = my_piece + part * 32, h = piece / P;
        const int blk = __shfl_sync(kFull, block, t & 31), r = __shfl_sync(kFull, row, t & 31);
        const bool there = t < tokens && piece < pieces && my_token < in_round;
        to[k] = there ? t * pieces + piece : -1;
        scale[k] = 0;
#pragma unroll
        for (int j = 0; j < E / 4; ++j) u[k][j] = 0;
        if (there && blk >= 0) {
          const uint8_t* const p = cache + blk * cs[0] + r * cs[1] + h * cs[2] + piece % P * E;
          scale[k] = __ldg(scales + static_cast<long long>(blk) * a.heads + h);
          if constexpr (E == 8) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
            u[k][0] = x.x, u[k][1] = x.y;
          } else {
            u[k][0] = __ldg(reinterpret_cast<const uint32_t*>(p));
          }
        }
        if (++part == wide) part = 0, token += in_round;
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        float v[E];
#pragma unroll
        for (int j = 0; j < E / 4; ++j) {
          const float2 x = e4m3x2_values(u[k][j] & 0xffffu), y = e4m3x2_values(u[k][j] >> 16);
          v[4 * j] = x.x * scale[k], v[4 * j + 1] = x.y * scale[k], v[4 * j + 2] = y.x * scale[k], v[4 * j + 3] = y.y * scale[k];
        }
        if (to[k] >= 0) reinterpret_cast<uint4*>(out)[to[k]] = Piece<T>::pack(v);
      }
    }
  }
}

}  // namespace

int launch_cache_read(CacheReadArgs& a, int head_dim, int out_is_fp32, int sm_count, cudaStream_t stream) {
  if (a.total == 0) return 0;
  // Tokens of a warp: few where that makes more warps run at once.
  const long long per = a.total / (16ll * sm_count);
  a.warp_tokens = per >= 32 ? 32 : per < 1 ? 1 : static_cast<int>(per);
  const long long grid = (a.total + kReadWarps * a.warp_tokens - 1) / (kReadWarps * a.warp_tokens);
  if (grid > 0x7fffffffll) return GDPA_ERR_LAUNCH_;
  auto launch = [&](auto type, auto dim) {
    gdpa_cache_read_kernel<decltype(type), decltype(dim)::value><<<static_cast<unsigned>(grid), kReadWarps * 32, 0, stream>>>(a);
  };
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (out_is_fp32) head_dim == 128 ? launch(float{}, D128{}) : launch(float{}, D64{});
  else head_dim == 128 ? launch(__nv_bfloat16{}, D128{}) : launch(__nv_bfloat16{}, D64{});
  return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

}  // namespace gdpa
