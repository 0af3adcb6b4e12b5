// Norms of queries and keys for each head and their rotation by position, in one pass, with the gradient.  The arithmetic is in
// gdpa_rotary.cuh.
//
// Gradient, for y = R n, n = x r w, r = rsqrt(mean(x^2) + eps), all of a head:
//   dn = R^T dy,   dw = sum over tokens and heads of dn x r,   g = dn w,   dx = r (g - x r^2 mean(g x)).
// R is a rotation, so its transpose turns back by the same angles; x is read again and r made anew: nothing is kept by the forward.
//
// Both are bound by HBM (forward: each value read and written once; backward: x and dy read, dx written), small calls by latency.  A
// warp takes the heads of a token, four heads of 128 bf16 values at a time, so that a token's angles are made once.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_rotary.cuh"

namespace gdpa {

namespace {

constexpr int kWarps = 4;
constexpr int kFwdCtas = 12;  // of an SM, at most
constexpr int kBwdCtas = 4;

// Item `i` of queries (0) or keys (1).
struct Item {
  int which, head0, head1;
  long long token;
};
__device__ __forceinline__ Item item_at(const RotaryArgs& a, unsigned i, unsigned query_items) {
  Item it;
  it.which = i >= query_items;
  const RotaryTensor& t = a.t[it.which];
  if (it.which) i -= query_items;
  const unsigned token = t.chunks == 1 ? i : i / static_cast<unsigned>(t.chunks);
  it.token = token;
  it.head0 = static_cast<int>(i - token * static_cast<unsigned>(t.chunks)) * t.per_item;
  it.head1 = min(it.head0 + t.per_item, t.heads);
  return it;
}

__device__ __forceinline__ long long position_at(const RotaryTensor& t, int axis, long long token) {
  const long long i = axis * t.position_stride + token;
  return t.positions_are_int64 ? static_cast<const long long*>(t.positions)[i] : static_cast<const int*>(t.positions)[i];
}

template <class T, int D>
__device__ __forceinline__ void take_weight(const HeadLanes<T, D>& h, const RotaryTensor& t, float (&w)[HeadLanes<T, D>::V]) {
  constexpr int E = HeadLanes<T, D>::E;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = weight_at(t.weight, t.weight_is_bf16, h.g0 * E + e);
    w[E + e] = weight_at(t.weight, t.weight_is_bf16, h.g1 * E + e);
  }
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) gdpa_rotary_kernel(const __grid_constant__ RotaryArgs a) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E, V = Lanes::V, U = 2;  // U warp-wide heads at once
  __shared__ float4 s_angles[kWarps][2][D / 8];
  const int warp = threadIdx.x >> 5;
  const Lanes lanes(a.rotary);
  const WarpAngles<T, D> angles(a.rotary);
  float* const s_cos = reinterpret_cast<float*>(s_angles[warp][0]);
  float* const s_sin = reinterpret_cast<float*>(s_angles[warp][1]);
  const unsigned nq = static_cast<unsigned>(a.t[0].tokens * a.t[0].chunks), n = nq + static_cast<unsigned>(a.t[1].tokens * a.t[1].chunks);
  int held = -1;  // whose weight this is
  float w[V];
  for (unsigned i = blockIdx.x * kWarps + warp; i < n; i += gridDim.x * kWarps) {
    const Item it = item_at(a, i, nq);
    const RotaryTensor& t = a.t[it.which];
    const T* const x = static_cast<const T*>(t.x) + it.token * t.x_strides[0];
    T* const y = static_cast<T*>(t.y) + it.token * t.heads * D;
    uint4 u[U][2];
    auto load = [&](int head0) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int head = head0 + k * Lanes::H + lanes.sub;
        u[k][0] = u[k][1] = make_uint4(0, 0, 0, 0);
        if (head < it.head1) {
          const T* const p = x + head * t.x_strides[1];
          u[k][0] = __ldg(reinterpret_cast<const uint4*>(p) + lanes.g0);
          u[k][1] = __ldg(reinterpret_cast<const uint4*>(p) + lanes.g1);
        }
      }
    };
    load(it.head0);
    if (held != it.which) {
      held = it.which;
      take_weight<T, D>(lanes, t, w);
    }
    __syncwarp();  // the last item's angles have been read
    angles.write(s_cos, s_sin, [&](int axis) { return position_at(t, axis, it.token); });
    __syncwarp();
    float c[E], s[E];
    if (lanes.rotated) lanes.take(s_cos, c), lanes.take(s_sin, s);
    for (int head0 = it.head0;;) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int head = head0 + k * Lanes::H + lanes.sub;
        float v[V];
        Lanes::unpack(u[k], v);
        if (a.rotary.norm) {
          float ss = 0;
#pragma unroll
          for (int e = 0; e < V; ++e) ss += v[e] * v[e];
          const float r = rsqrtf(Lanes::sum(ss) * (1.f / D) + a.rotary.eps);
#pragma unroll
          for (int e = 0; e < V; ++e) v[e] = v[e] * r * w[e];
        }
        lanes.template turn<false>(a.rotary.interleaved, c, s, v);
        if (head < it.head1) {
          uint4* const p = reinterpret_cast<uint4*>(y + static_cast<long long>(head) * D);
          p[lanes.g0] = Piece<T>::pack(v);
          p[lanes.g1] = Piece<T>::pack(v + E);
        }
      }
      head0 += U * Lanes::H;
      if (head0 >= it.head1) break;
      load(head0);
    }
  }
}

// dx, and the sums of dn x r of this CTA's items.  The sums are made twice over: a lane's over a few heads first, then those.  One sum over all of a
// lane's heads would carry an error of 2^-24 sqrt(heads / 2), which long batches see.
template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32, kBwdCtas) gdpa_rotary_bwd_kernel(const __grid_constant__ RotaryArgs a) {
  using Lanes = HeadLanes<T, D>;
  constexpr int E = Lanes::E, V = Lanes::V;
  __shared__ float4 s_angles[kWarps][2][D / 8];
  __shared__ float s_dw[kWarps][2][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Lanes lanes(a.rotary);
  const WarpAngles<T, D> angles(a.rotary);
  float* const s_cos = reinterpret_cast<float*>(s_angles[warp][0]);
  float* const s_sin = reinterpret_cast<float*>(s_angles[warp][1]);
  const unsigned nq = static_cast<unsigned>(a.t[0].tokens * a.t[0].chunks), n = nq + static_cast<unsigned>(a.t[1].tokens * a.t[1].chunks);
  int held = -1, few = 0;
  float w[V], sum[V], part[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = part[e] = 0;
  if (a.partial != nullptr) {
    for (int i = lane; i < 2 * D; i += 32) s_dw[warp][i / D][i % D] = 0;
    __syncwarp();
  }
  auto flush = [&]() {  // a warp's sums of one tensor
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float x = sum[e] + part[e];
#pragma unroll
      for (int s = Lanes::L; s < 32; s <<= 1) x += __shfl_xor_sync(kAllLanes, x, s);
      if (lanes.sub == 0) s_dw[warp][held][(e < E ? lanes.g0 : lanes.g1) * E + e % E] = x;
      sum[e] = part[e] = 0;
    }
  };
  for (unsigned i = blockIdx.x * kWarps + warp; i < n; i += gridDim.x * kWarps) {
    const Item it = item_at(a, i, nq);
    const RotaryTensor& t = a.t[it.which];
    const T* const x = static_cast<const T*>(t.x) + it.token * t.x_strides[0];
    const T* const dy = static_cast<const T*>(t.dy) + it.token * t.dy_strides[0];
    T* const dx = static_cast<T*>(t.y) + it.token * t.heads * D;
    uint4 ux[2], ug[2];
    auto load = [&](int head0) {
      const int head = head0 + lanes.sub;
      ux[0] = ux[1] = ug[0] = ug[1] = make_uint4(0, 0, 0, 0);
      if (head < it.head1) {
        const T* const p = dy + head * t.dy_strides[1];
        ug[0] = __ldg(reinterpret_cast<const uint4*>(p) + lanes.g0);
        ug[1] = __ldg(reinterpret_cast<const uint4*>(p) + lanes.g1);
        if (a.rotary.norm) {
          const T* const q = x + head * t.x_strides[1];
          ux[0] = __ldg(reinterpret_cast<const uint4*>(q) + lanes.g0);
          ux[1] = __ldg(reinterpret_cast<const uint4*>(q) + lanes.g1);
        }
      }
    };
    load(it.head0);
    if (held != it.which) {
      if (held >= 0 && a.partial != nullptr) flush();
      held = it.which;
      take_weight<T, D>(lanes, t, w);
    }
    __syncwarp();
    angles.write(s_cos, s_sin, [&](int axis) { return position_at(t, axis, it.token); });
    __syncwarp();
    float c[E], s[E];
    if (lanes.rotated) lanes.take(s_cos, c), lanes.take(s_sin, s);
    for (int head0 = it.head0;;) {
      const int head = head0 + lanes.sub;
      float v[V], g[V];
      Lanes::unpack(ux, v);
      Lanes::unpack(ug, g);
      head0 += Lanes::H;
      if (head0 < it.head1) load(head0);
      lanes.template turn<true>(a.rotary.interleaved, c, s, g);
      if (a.rotary.norm) {
        float ss = 0, gx = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) ss += v[e] * v[e], gx += g[e] * w[e] * v[e];
        const float r = rsqrtf(Lanes::sum(ss) * (1.f / D) + a.rotary.eps);
        const float m = Lanes::sum(gx) * (1.f / D) * r * r;
        if (head < it.head1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            part[e] += g[e] * (v[e] * r);
            g[e] = r * (g[e] * w[e] - v[e] * m);
          }
        }
        if (++few == 16) {
          few = 0;
#pragma unroll
          for (int e = 0; e < V; ++e) sum[e] += part[e], part[e] = 0;
        }
      }
      if (head < it.head1) {
        uint4* const p = reinterpret_cast<uint4*>(dx + static_cast<long long>(head) * D);
        p[lanes.g0] = Piece<T>::pack(g);
        p[lanes.g1] = Piece<T>::pack(g + E);
      }
      if (head0 >= it.head1) break;
    }
  }
  if (a.partial != nullptr) {
    if (held >= 0) flush();
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
      float x = 0;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) x += s_dw[k][i / D][i % D];
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

// Items for about `warps` warps, and CTAs for them, `most` at most.
unsigned plan(RotaryArgs& a, int head_dim, int is_fp32, long long warps, long long most) {
  const int a_warp = is_fp32 ? 256 / head_dim : 512 / head_dim;
  long long items = 0;
  for (RotaryTensor& t : a.t) {
    split_heads(t.tokens, t.heads, a_warp, warps, t.per_item, t.chunks);
    items += t.tokens * t.chunks;
  }
  const long long grid = (items + kWarps - 1) / kWarps;
  return static_cast<unsigned>(grid < most ? grid : most);
}

}  // namespace

int rotary_bwd_ctas(int sm_count) { return kBwdCtas * sm_count; }

int launch_rotary(RotaryArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  const unsigned grid = plan(a, head_dim, is_fp32, 16ll * sm_count, static_cast<long long>(kFwdCtas) * sm_count);
  if (grid == 0) return 0;
  return by_type(head_dim, is_fp32, [&](auto type, auto dim) {
    gdpa_rotary_kernel<decltype(type), decltype(dim)::value><<<grid, kWarps * 32, 0, stream>>>(a);
  });
}

int launch_rotary_bwd(RotaryArgs& a, int head_dim, int is_fp32, int sm_count, cudaStream_t stream) {
  const unsigned grid = plan(a, head_dim, is_fp32, 16ll * sm_count, rotary_bwd_ctas(sm_count));
  if (grid > 0) {
    const int rc = by_type(head_dim, is_fp32, [&](auto type, auto dim) {
      gdpa_rotary_bwd_kernel<decltype(type), decltype(dim)::value><<<grid, kWarps * 32, 0, stream>>>(a);
    });
    if (rc != 0) return -rc;
  }
  if (a.partial == nullptr) return grid > 0;
  gdpa_rotary_join_kernel<<<2 * head_dim / 32, 1024, 0, stream>>>(a.partial, static_cast<int>(grid), head_dim, a);
  return cudaGetLastError() == cudaSuccess ? (grid > 0) + 1 : -GDPA_ERR_LAUNCH_;
}

}  // namespace gdpa
