// Norms of queries and keys for each head and their rotation by position, in one pass, with the gradient.  The arithmetic is in
// gdpa_rotary.cuh.
//
// Gradient, for y = R n, n = x r w, r = rsqrt(mean(x^2) + eps), all of a head:
//   dn = R^T dy,   dw = sum over tokens and heads of dn x r,   g = dn w,   dx = r (g - x r^2 mean(g x)).
// R is a rotation, so its transpose turns back by the same angles; x is read again and r made anew: nothing is kept by the forward.
//
// Both are bound by HBM (forward: each value read and written once; backward: x and dy read, dx written), small calls by latency.  A
// warp takes the heads of a token, four heads of 128 bf16 values at a time, so that a token's angles are made once.  Units come through shared memory, fetched ahead by the
// lanes that use them, so that no barrier stands between; a few tokens to a warp, then the next ones far behind, keep what all warps have in hand close together in memory.
// bf16, 128 values, cold: 16 and 4 heads of 67 000 tokens 115 us, 690 MB, 6.0 TB/s (a plain copy 6.5); 8 and 8 heads of 300 000 tokens 398 us forward (6.2), 600
// to 633 backward (5.8 to 6.1), of it 5 to 6 the joining of the weights' gradients; 64 tokens of 32 and 4 heads 5.4 us.  The rotation alone, 8 and 8 heads of 300 000 tokens: 436
// us forward (5.6), 387 backward (6.3; x is not read).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_rotary.cuh"

namespace gdpa {

namespace {

constexpr int kWarps = 4;
constexpr int kFwdCtas = 4;  // resident on an SM
constexpr int kBwdCtas = 3;
constexpr int kFwdRing = 3;  // groups of units of a warp on their way
constexpr int kBwdRing = 4;
constexpr int kBwdTokens = 6;  // of an item

// The lane's position of an item's.
__device__ __forceinline__ long long position_of(const RotaryArgs& a, const Item& it) {
  const RotaryTensor& t = a.t[it.first];
  const int lane = threadIdx.x & 31, axis = lane / kMostItemTokens, j = lane % kMostItemTokens;
  if (axis >= a.rotary.axes || j >= it.tokens || a.rotary.pairs == 0) return 0;
  const long long i = axis * t.position_stride + it.token + j;
  return t.positions_are_int64 ? static_cast<const long long*>(t.positions)[i] : static_cast<const int*>(t.positions)[i];
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32, kFwdCtas) gdpa_rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ uint4 s_ring[];  // [warp][kFwdRing][kTogether] units
  __shared__ float4 s_tables[kWarps][kTokens][D / 4];
  __shared__ float4 s_weight[2][D / 4];
  const int warp = threadIdx.x >> 5;
  auto positions = [&](const Item& it) { return position_of(a, it); };
  rotate_items<T, D, kFwdRing>(a, s_ring + warp * kFwdRing * kTogether * kUnitPieces, reinterpret_cast<float*>(s_tables[warp]), reinterpret_cast<float*>(s_weight), 2,
                               Cursor(blockIdx.x * kWarps + warp, gridDim.x * kWarps), positions);
}

// dx, and the sums of dn x r of this CTA's items.  The sums are made twice over: a lane's over an item's heads in registers, then, in shared memory,
// over its items.  One sum over all of a lane's heads would carry an error of 2^-24 sqrt(heads / 2), which long batches see.
template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32, kBwdCtas) gdpa_rotary_bwd_kernel(const __grid_constant__ RotaryArgs a) {
  using Lanes = HeadLanes<T, D>;
  constexpr int C = Lanes::C, E = Lanes::E;
  extern __shared__ uint4 s_ring[];  // [warp][kBwdRing][x, dy] units; then, for the weights' gradients, sums [warp][2][2 C][32]
  __shared__ float4 s_tables[kWarps][kBwdTokens][D / 4];
  __shared__ float4 s_weight[2][D / 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lanes lanes(a.rotary);
  Cursor cursor(blockIdx.x * kWarps + warp, gridDim.x * kWarps);
  uint4* const ring = s_ring + warp * kBwdRing * 2 * kUnitPieces;
  Stream<T, D, 2, 1, kBwdRing> stream(a, lanes, ring, cursor);
  Item it, next;
  bool more = cursor.next(a, next);
  long long next_position = more ? position_of(a, next) : 0;
  const WarpAngles<T, D> angles(a.rotary);
  float* const tables = reinterpret_cast<float*>(s_tables[warp]);
  uint64_t* const all_sums = reinterpret_cast<uint64_t*>(s_ring + kWarps * kBwdRing * 2 * kUnitPieces);
  uint64_t* const sums = all_sums + warp * 2 * 2 * C * 32 + lane;
  if (warp < 2) lanes.write_weight(reinterpret_cast<float*>(s_weight[warp]), a.t[warp].weight, a.t[warp].weight_is_bf16);
  if (a.partial != nullptr) {
    for (int e = 0; e < 2 * 2 * C; ++e) sums[e * 32] = 0;
  }
  __syncthreads();
  unsigned slot = 0;
  while (more) {
    it = next;
    const long long its_position = next_position;
    if ((more = cursor.next(a, next))) next_position = position_of(a, next);
    angles.template write_all<kBwdTokens>(tables, it.tokens, its_position);
    for (int k = it.first; k <= it.last; ++k) {
      const RotaryTensor& t = a.t[k];
      int u0, u1;
      units_of(a, it, k, Lanes::H, u0, u1);
      if (u0 >= u1) continue;
      HeadWalk<T, D> dx;
      dx.begin(static_cast<T*>(t.y), static_cast<long long>(t.heads) * D, D, lanes, it.token, u0, u1, 1);
      const float* const weight = reinterpret_cast<const float*>(s_weight[k]);
      uint64_t part[2 * C];
#pragma unroll
      for (int e = 0; e < 2 * C; ++e) part[e] = 0;
      for (int j = 0; j < it.tokens; ++j) {
        uint64_t c[C], s[C];
        if (lanes.rotated) lanes.take(tables + j * D, c), lanes.take(tables + j * D + D / 2, s);
        for (int u = u0; u < u1; ++u) {
          stream.fetch();
          fetch_wait<kBwdRing - 1>();
          const uint4* const from = ring + slot * 2 * kUnitPieces;
          slot = slot + 1 == kBwdRing ? 0 : slot + 1;
          uint4 p[2];
          fetched(from + kUnitPieces, p);
          uint64_t g[2 * C];
          Lanes::unpack(p, g);
          if (lanes.rotated) Lanes::template turn<true>(a.rotary.interleaved, c, s, g);
          const bool there = u * Lanes::H + lanes.sub < t.heads;
          if (a.rotary.norm) {
            uint64_t v[2 * C], weighed[1][2 * C];
            uint64_t(&gw)[2 * C] = weighed[0];
            fetched(from, p);
            Lanes::unpack(p, v);
#pragma unroll
            for (int e = 0; e < 2 * C; ++e) gw[e] = g[e];
            lanes.times(weight, weighed);
            float sums_of[2] = {Lanes::dot(v, v), Lanes::dot(gw, v)};
#pragma unroll
            for (int l = 1; l < Lanes::L; l <<= 1) {
#pragma unroll
              for (int x = 0; x < 2; ++x) sums_of[x] += __shfl_xor_sync(kAllLanes, sums_of[x], l);
            }
            const float r = rsqrtf(sums_of[0] * (1.f / D) + a.rotary.eps), m = sums_of[1] * (1.f / D) * r * r;
            Lanes::times(r, v);  // the normed head, without its weight
            const uint64_t r2 = pack_f32x2(r, r), m2 = pack_f32x2(-m, -m);
#pragma unroll
            for (int e = 0; e < 2 * C; ++e) {
              if (there) part[e] = fma_f32x2(g[e], v[e], part[e]);
              g[e] = fma_f32x2(gw[e], r2, mul_f32x2(v[e], m2));  // r gw - x r m
            }
          }
          if (there) dx.store(lanes, 0, g);
          dx.next(u + 1 == u1);
        }
      }
      if (t.dweight != nullptr) {
#pragma unroll
        for (int e = 0; e < 2 * C; ++e) sums[(k * 2 * C + e) * 32] = add_f32x2(sums[(k * 2 * C + e) * 32], part[e]);
      }
    }
  }
  if (a.partial != nullptr) {
    // value i of a head: piece, and the lanes that have it in each of the warp's heads
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
      const int k = i / D, g = i % D / E, e = i % E;
      bool second;
      const int l = Lanes::lane_of_piece(a.rotary, g, second);
      float x = 0;
      for (int w = 0; w < kWarps; ++w) {
        for (int h = 0; h < Lanes::H; ++h)
          x += reinterpret_cast<const float*>(all_sums)[2 * (((w * 2 + k) * 2 * C + second * C + e / 2) * 32 + h * Lanes::L + l) + e % 2];
      }
      a.partial[static_cast<long long>(blockIdx.x) * 2 * D + i] = x;
    }
  }
}

// The CTAs' sums together, in their order: 32 columns for each CTA, 32 warps over the rows.
__global__ void __launch_bounds__(1024) gdpa_rotary_join_kernel(const float* __restrict__ partial, int rows, int dim, RotaryArgs a) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, column = blockIdx.x * 32 + lane;
  float x = 0;
  for (int r = warp; r < rows; r += 32) x += partial[static_cast<long long>(r) * 2 * dim + column];
  s[warp][lane] = x;
  __syncthreads();
  if (warp != 0) return;
  x = 0;
#pragma unroll
  for (int k = 0; k < 32; ++k) x += s[k][lane];
  const int which = column / dim, e = column % dim;
  const RotaryTensor& t = a.t[which];
  if (t.dweight == nullptr) return;
  if (t.weight_is_bf16) static_cast<__nv_bfloat16*>(t.dweight)[e] = __float2bfloat16_rn(x);
  else static_cast<float*>(t.dweight)[e] = x;
}

template <class F>
int by_type(int head_dim, int is_fp32, F launch) {
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (is_fp32) head_dim == 128 ? launch(float{}, D128{}) : launch(float{}, D64{});
  else head_dim == 128 ? launch(__nv_bfloat16{}, D128{}) : launch(__nv_bfloat16{}, D64{});
  return cudaGetLastError() == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

unsigned ctas(const RotaryArgs& a, long long most) {
  const long long grid = (static_cast<long long>(a.items[0]) + a.items[1] + kWarps - 1) / kWarps;
  return static_cast<unsigned>(grid < most ? grid : most);
}

}  // namespace

int rotary_bwd_ctas(int sm_count) { return kBwdCtas * sm_count; }

int launch_rotary(RotaryArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  plan_items(a, head_dim, is_fp32, static_cast<long long>(kFwdCtas) * kWarps * sm_count, kTokens);
  const unsigned grid = ctas(a, static_cast<long long>(kFwdCtas) * sm_count);
  if (grid == 0) return 0;
  return by_type(head_dim, is_fp32, [&](auto type, auto dim) {
    gdpa_rotary_kernel<decltype(type), decltype(dim)::value><<<grid, kWarps * 32, kWarps * kFwdRing * kTogether * kUnitPieces * 16, stream>>>(a);
  });
}

int launch_rotary_bwd(RotaryArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  plan_items(a, head_dim, is_fp32, static_cast<long long>(kBwdCtas) * kWarps * sm_count, kBwdTokens);
  const unsigned grid = ctas(a, rotary_bwd_ctas(sm_count));
  if (grid > 0) {
    // The ring and, for the weights' gradients, a lane's sums of both tensors.  What a kernel may have at most is its own state, which other host threads'
    // calls set too: always the most that it ever takes.
    const int rc = by_type(head_dim, is_fp32, [&](auto type, auto dim) {
      using T = decltype(type);
      constexpr int D = decltype(dim)::value, kRing = kWarps * kBwdRing * 2 * kUnitPieces * 16, kSums = kWarps * 2 * 2 * HeadLanes<T, D>::C * 32 * sizeof(uint64_t);
      auto kernel = gdpa_rotary_bwd_kernel<T, D>;
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing + kSums) != cudaSuccess) return;  // the launch then fails, and says so
      kernel<<<grid, kWarps * 32, kRing + (a.partial != nullptr ? kSums : 0), stream>>>(a);
    });
    if (rc != 0) return -rc;
  }
  if (a.partial == nullptr) return grid > 0;
  gdpa_rotary_join_kernel<<<2 * head_dim / 32, 1024, 0, stream>>>(a.partial, static_cast<int>(grid), head_dim, a);
  return cudaGetLastError() == cudaSuccess ? (grid > 0) + 1 : -GDPA_ERR_LAUNCH_;
}

}  // namespace gdpa
