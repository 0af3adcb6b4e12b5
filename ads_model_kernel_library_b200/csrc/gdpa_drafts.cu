// Drafted tokens: their verification against the target's probabilities, and the way of the refused ones out of the paged cache.
//
// Verification of a request's drafts x_1 .. x_n, drawn from distributions q_j (or, without them, from nowhere: q_j is one at x_j), against the
// target's p_j, j = 1 .. n + 1, with uniform numbers u_j and u:
//   draft j is accepted if u_j q_j(x_j) < p_j(x_j) and all before it are;  a = number of accepted ones;
//   the next token is drawn from max(p_{a+1} - q_{a+1}, 0) if a < n, from p_{n+1} else: the first index i whose partial sum up to i
//   exceeds u times the sum (and that has a share of its own).  Where nothing is left of a difference, p itself is drawn from.
// An accepted or drawn token is then distributed as p.  A share that is not a positive finite number counts as zero; without any share the
// token is -1.
//
// Sums are in 64 bits: a vocabulary's partial sums in fp32 would be off by more than most tokens' shares, and what comes out is a whole
// number.  A request needs two rows at most, one pass over them: a cluster of CTAs sums stretches of 256 or 1024 tokens, and the stretch in which the
// sum passes its mark is looked at again (it is in the L2 cache).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"

namespace cg = cooperative_groups;

namespace gdpa {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCtas = 4;          // resident on an SM
constexpr int kMostVocab = 1 << 20;
constexpr int kMostStretches = kMostVocab / 1024;  // of a vocabulary
constexpr int kMaxCluster = 8;

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// positive finite numbers, as they are; anything else is 0
__device__ __forceinline__ float share(float x) { return __float_as_uint(x) < 0x7f800000u ? x : 0.f; }

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(kFull, x, s);
  return x;
}

// What is drawn from: p, less q or less the token `without`.
template <class T>
struct Left {
  const T* p;
  const T* q;  // or null
  int without;  // or -1
  __device__ __forceinline__ double operator()(int i) const {
    const float pv = share(as_float(p[i])), qv = q != nullptr ? fmaxf(as_float(q[i]), 0.f) : 0.f;
    return i != without && pv > qv ? static_cast<double>(pv) - static_cast<double>(qv) : 0;
  }
  // The sum of 32 U tokens from i0 on, by a warp; WHOLE: they are all there.  Some of them are on their way while others are added.
  template <int U, bool WHOLE>
  __device__ __forceinline__ double sum(int i0, int vocab) const {
    constexpr int B = 8;
    double sums[2] = {0, 0};
    const int lane = threadIdx.x & 31;
    const T* const pp = p + i0 + lane;
    auto load = [&](const T* from, int u0, T (&x)[B]) {
#pragma unroll
      for (int u = 0; u < B; ++u) x[u] = WHOLE || i0 + lane + (u0 + u) * 32 < vocab ? from[(u0 + u) * 32] : static_cast<T>(0.f);
    };
    T a[2][B];
    load(pp, 0, a[0]);
    if (q != nullptr) {
      const T* const qq = q + i0 + lane;
      T b[2][B];
      load(qq, 0, b[0]);
#pragma unroll
      for (int u0 = 0; u0 < U; u0 += B) {
        const int now = u0 / B & 1;
        if (u0 + B < U) load(pp, u0 + B, a[now ^ 1]), load(qq, u0 + B, b[now ^ 1]);
#pragma unroll
        for (int u = 0; u < B; ++u) {
          const float qv = fmaxf(as_float(b[now][u]), 0.f), larger = fmaxf(share(as_float(a[now][u])), qv);
          sums[u & 1] += static_cast<double>(larger) - static_cast<double>(qv);
        }
      }
    } else {
#pragma unroll
      for (int u0 = 0; u0 < U; u0 += B) {
        const int now = u0 / B & 1;
        if (u0 + B < U) load(pp, u0 + B, a[now ^ 1]);
#pragma unroll
        for (int u = 0; u < B; ++u) sums[u & 1] += static_cast<double>(share(as_float(a[now][u])));
      }
    }
    double s = sums[0] + sums[1];
    // the token that was refused, if it is one of the lane's
    const int at = without - i0 - lane;
    if (without >= 0 && at >= 0 && at < 32 * U && at % 32 == 0) s = sum_without(i0, U, vocab);
    return warp_sum(s);
  }
  __device__ __noinline__ double sum_without(int i0, int U, int vocab) const {
    double s = 0;
    for (int u = 0; u < U; ++u) {
      const int i = i0 + (threadIdx.x & 31) + u * 32;
      if (i < vocab) s += (*this)(i);
    }
    return s;
  }
};

// U * 32 tokens are a stretch.
template <class T, int U>
__global__ void __launch_bounds__(kVerifyThreads, kVerifyCtas) gdpa_verify_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int kStretch = 32 * U;
  __shared__ double s_sum[kMostStretches];  // of a stretch; then up to its end
  __shared__ double s_total;                // of this CTA, for the cluster
  __shared__ double s_share[32 * (U + 1)];
  __shared__ int s_accepted, s_stretch;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row0 = clamp_ll(load_offset(a.row_offsets, b, a.off64), 0, a.rows), row1 = clamp_ll(load_offset(a.row_offsets, b + 1, a.off64), row0, a.rows);
  const long long d0 = clamp_ll(load_offset(a.draft_offsets, b, a.off64), 0, a.drafts),
                  d1 = clamp_ll(load_offset(a.draft_offsets, b + 1, a.off64), d0, a.drafts);
  const int n = static_cast<int>(clamp_ll(min(d1 - d0, row1 - row0 - 1), 0, a.max_drafts));
  const T* const target = static_cast<const T*>(a.target);
  const T* const draft = static_cast<const T*>(a.draft);
  auto token_of = [&](long long d) -> long long {
    return a.tokens64 ? static_cast<const long long*>(a.tokens)[d] : static_cast<const int*>(a.tokens)[d];
  };
  const long long out_row = static_cast<long long>(b) * (a.max_drafts + 1);
  auto put = [&](int j, long long token) {
    if (a.tokens64) static_cast<long long*>(a.out_tokens)[out_row + j] = token;
    else static_cast<int*>(a.out_tokens)[out_row + j] = static_cast<int>(token);
  };
  // accepted drafts, by every CTA for itself
  if (warp == 0) {
    int accepted = n;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane;
      bool refused = false;
      if (j < n) {
        const long long x = token_of(d0 + j);
        refused = true;
        if (x >= 0 && x < a.vocab) {
          const double p = as_float(target[(row0 + j) * a.target_stride + x]);
          const double q = draft != nullptr ? static_cast<double>(as_float(draft[(d0 + j) * a.draft_stride + x])) : 1.0;
          refused = !(static_cast<double>(a.accept[d0 + j]) * q < p);
        }
      }
      const unsigned those = __ballot_sync(kFull, refused);
      if (those != 0) {
        accepted = j0 + __ffs(those) - 1;
        break;
      }
    }
    if (lane == 0) s_accepted = accepted;
  }
  __syncthreads();
  const int accepted = s_accepted;
  const bool there = row1 > row0;  // the same for the whole cluster
  if (rank == 0) {
    for (int j = threadIdx.x; j <= a.max_drafts; j += kVerifyThreads)
      if (j != accepted || !there) put(j, j < accepted ? token_of(d0 + j) : -1);
    if (threadIdx.x == 0) a.accepted[b] = accepted, a.refused[b] = n - accepted;
  }
  if (!there) return;
  Left<T> left{target + (row0 + accepted) * a.target_stride, nullptr, -1};
  if (accepted < n) {
    if (draft != nullptr) left.q = draft + (d0 + accepted) * a.draft_stride;
    else left.without = static_cast<int>(clamp_ll(token_of(d0 + accepted), -1, a.vocab));
  }
  // this CTA's stretches
  const int stretches = (a.vocab + kStretch - 1) / kStretch;
  const int k0 = static_cast<int>(static_cast<long long>(stretches) * rank / ranks);
  const int mine = static_cast<int>(static_cast<long long>(stretches) * (rank + 1) / ranks) - k0;
  double total, base, mark;
  int owner;
  for (;;) {
    for (int k = warp; k < mine; k += kVerifyWarps) {
      const int i0 = (k0 + k) * kStretch;
      const double s = i0 + kStretch <= a.vocab ? left.template sum<U, true>(i0, a.vocab) : left.template sum<U, false>(i0, a.vocab);
      if (lane == 0) s_sum[k] = s;
    }
    __syncthreads();
    if (warp == 0) {
      double before = 0;
      for (int k = 0; k < mine; k += 32) {
        double up_to = k + lane < mine ? s_sum[k + lane] : 0;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const double o = __shfl_up_sync(kFull, up_to, s);
          if (lane >= s) up_to += o;
        }
        if (k + lane < mine) s_sum[k + lane] = before + up_to;
        before += __shfl_sync(kFull, up_to, 31);
      }
      if (lane == 0) s_total = before;
    }
    cluster.sync();
    // The CTA in whose stretches the sum passes its mark: the first whose end lies above it.  If rounding, or a number that is not below one, has left
    // none: the last with a share.
    total = 0;
    for (int r = 0; r < ranks; ++r) total += *cluster.map_shared_rank(&s_total, r);
    mark = static_cast<double>(a.sample[b]) * total;
    double end = 0;
    base = 0, owner = -1;
    bool above = false;
    for (int r = 0; r < ranks && !above; ++r) {
      const double of_r = *cluster.map_shared_rank(&s_total, r);
      if (of_r > 0) owner = r, base = end;
      end += of_r;
      above = of_r > 0 && end > mark;
    }
    cluster.sync();  // before a CTA ends or writes its sum again
    if (total > 0) break;
    if (left.q == nullptr && left.without < 0) break;
    left.q = nullptr, left.without = -1;
  }
  if (owner < 0) {  // nothing to draw from
    if (rank == 0 && threadIdx.x == 0) put(accepted, -1);
    return;
  }
  if (rank != owner) return;
  // the stretch, in the same way
  if (warp == 0) {
    int found = -1, last = 0;
    for (int k = 0; k < mine && found < 0; k += 32) {
      const double from = k + lane > 0 && k + lane < mine ? s_sum[k + lane - 1] : 0, to = k + lane < mine ? s_sum[k + lane] : 0;
      const bool some = k + lane < mine && to > from;
      const unsigned with = __ballot_sync(kFull, some), those = __ballot_sync(kFull, some && base + to > mark);
      if (with != 0) last = k + 31 - __clz(with);
      if (those != 0) found = k + __ffs(those) - 1;
    }
    if (lane == 0) s_stretch = found >= 0 ? found : last;
  }
  __syncthreads();
  const int k = s_stretch;
  for (int i = threadIdx.x; i < kStretch; i += kVerifyThreads) {
    const int at = (k0 + k) * kStretch + i;
    s_share[i / U * (U + 1) + i % U] = at < a.vocab ? left(at) : 0;
  }
  __syncthreads();
  if (warp != 0) return;
  // U tokens of the stretch for each lane, then one
  double sum = 0;
#pragma unroll
  for (int i = 0; i < U; ++i) sum += s_share[lane * (U + 1) + i];
  double up_to = sum;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const double o = __shfl_up_sync(kFull, up_to, s);
    if (lane >= s) up_to += o;
  }
  const double at_start = base + (k > 0 ? s_sum[k - 1] : 0);
  unsigned with = __ballot_sync(kFull, sum > 0), those = __ballot_sync(kFull, sum > 0 && at_start + up_to > mark);
  const int row = those != 0 ? __ffs(those) - 1 : with != 0 ? 31 - __clz(with) : 0;
  const double at_row = at_start + __shfl_sync(kFull, up_to - sum, row);
  const double mine_here = lane < U ? s_share[row * (U + 1) + lane] : 0;
  up_to = mine_here;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const double o = __shfl_up_sync(kFull, up_to, s);
    if (lane >= s) up_to += o;
  }
  with = __ballot_sync(kFull, mine_here > 0), those = __ballot_sync(kFull, mine_here > 0 && at_row + up_to > mark);
  const int column = those != 0 ? __ffs(those) - 1 : with != 0 ? 31 - __clz(with) : 0;
  if (lane == 0) put(accepted, (k0 + k) * kStretch + row * U + column);
}

// ------------------------------------------------------------------------------------------ tokens that leave the cache
//
// The last dropped[b] tokens of each request leave; the blocks that none of its tokens needs any more go onto the stack of free blocks, in
// the order of the requests and of their tables (entries that are no block, -1, do not).  Tables are left as they are: what lies behind a
// request's length is not looked at.
//
// Latency is all of it.  A warp has four requests, up to 128 entries of each, all asked for at once and kept in registers until it is known how many go
// before them.  Up to 256 requests, a cluster of CTAs adds that up in shared memory.  More of them: one kernel counts, another, whose loads the end
// of the first overlaps, adds up the counts of the CTAs before its own; 4096 requests with 64 entries each 48 us in one cluster, 9 so.
constexpr int kDropWarps = 8, kDropRequests = 4;

enum DropWay { kDropCluster, kDropCount, kDropStore };

template <DropWay WAY>
__global__ void __launch_bounds__(kDropWarps * 32) gdpa_drop_kernel(const __grid_constant__ DropArgs a) {
  __shared__ int s_count[kDropWarps];
  __shared__ int s_total;
  __shared__ long long s_before[kDropWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int S = 1 << a.block_shift;
  const int b0 = (blockIdx.x * kDropWarps + warp) * kDropRequests;
  // the warp's requests, and those of their entries that may go
  int keep = 0, held = 0;
  if (lane < kDropRequests && b0 + lane < a.batch) {
    const long long len = clamp_ll(load_offset(a.seq_lens, b0 + lane, a.lens64), 0, 0x7fffff00);
    const long long after = len - clamp_ll(load_offset(a.dropped, b0 + lane, a.dropped64), 0, len);
    if (WAY != kDropCount) a.seq_lens_after[b0 + lane] = static_cast<int>(after);
    keep = static_cast<int>(min((after + S - 1) >> a.block_shift, static_cast<long long>(a.table_width)));
    held = static_cast<int>(min((len + S - 1) >> a.block_shift, static_cast<long long>(a.table_width)));
  }
  int entry[kDropRequests][4];
#pragma unroll
  for (int i = 0; i < kDropRequests; ++i) {
    const int from = __shfl_sync(kFull, keep, i), to = __shfl_sync(kFull, held, i);
    const int* const row = a.block_tables + static_cast<long long>(b0 + i) * a.table_stride;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = from + 32 * u + lane;
      entry[i][u] = j < to ? row[j] : -1;
    }
  }
  // all of them in order: body(the lane's entry or -1, votes of the lanes that have one)
  auto walk = [&](auto body) {
#pragma unroll
    for (int i = 0; i < kDropRequests; ++i) {
      const int from = __shfl_sync(kFull, keep, i), to = __shfl_sync(kFull, held, i);
#pragma unroll
      for (int u = 0; u < 4; ++u) body(entry[i][u], __ballot_sync(kFull, entry[i][u] >= 0));
      // a request with more
      const int* const row = a.block_tables + static_cast<long long>(b0 + i) * a.table_stride;
      for (int j = from + 128 + lane; j - lane < to; j += 32) {
        const int e = j < to ? row[j] : -1;
        body(e, __ballot_sync(kFull, e >= 0));
      }
    }
  };
  if (WAY != kDropStore) {
    long long count = 0;
    walk([&](int, unsigned those) { count += __popc(those); });
    if (lane == 0) s_count[warp] = static_cast<int>(min(count, 0x0fffffffll));  // more than a stack that holds them once has places
    __syncthreads();
    if (threadIdx.x == 0) {
      int total = 0;
      for (int w = 0; w < kDropWarps; ++w) {
        const int n = s_count[w];
        s_count[w] = total;
        total += n;
      }
      s_total = total;
    }
    __syncthreads();
  }
  if (WAY == kDropCount) {
    int* const counts = a.counts + blockIdx.x * (kDropWarps + 1);
    if (threadIdx.x < kDropWarps) counts[1 + threadIdx.x] = s_count[threadIdx.x];
    if (threadIdx.x == 0) counts[0] = s_total;
    return;
  }
  const long long have = clamp_ll(*a.num_free, 0, a.free_capacity);
  long long place = have, total = 0;
  if (WAY == kDropCluster) {
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    cluster.sync();
    const int of_rank = lane < ranks ? *cluster.map_shared_rank(&s_total, lane) : 0;
    for (int r = 0; r < ranks; ++r) {
      const int n = __shfl_sync(kFull, of_rank, r);
      if (r == rank) place += total;
      total += n;
    }
    place += s_count[warp];
    cluster.sync();  // before a CTA ends
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // for the counts
    long long before = 0;
    for (int c = threadIdx.x; c < static_cast<int>(gridDim.x); c += kDropWarps * 32) {
      const int n = a.counts[c * (kDropWarps + 1)];
      total += n;
      before += c < static_cast<int>(blockIdx.x) ? n : 0;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) total += __shfl_xor_sync(kFull, total, s), before += __shfl_xor_sync(kFull, before, s);
    __shared__ long long s_all[kDropWarps];
    if (lane == 0) s_before[warp] = before, s_all[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kDropWarps; ++w) place += s_before[w], total += s_all[w];
    place += a.counts[blockIdx.x * (kDropWarps + 1) + 1 + warp];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.num_free_after = static_cast<int>(clamp_ll(have + total, 0, a.free_capacity));
  walk([&](int entry_here, unsigned those) {
    const long long at = place + __popc(those & ((1u << lane) - 1));
    if (entry_here >= 0 && at < a.free_capacity) a.free_blocks[at] = entry_here;
    place += __popc(those);
  });
}

// `ranks`: CTAs of a cluster; 0: none, and the kernel before it on the stream may still run.
template <class K, class A>
int launch_cluster(K kernel, const A& args, unsigned grid, unsigned threads, unsigned ranks, cudaStream_t stream) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.stream = stream;
  cudaLaunchAttribute at[1];
  if (ranks > 0) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  } else {
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
  }
  c.attrs = at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args) == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

}  // namespace

int verify_most_vocab() { return kMostVocab; }

int launch_verify(const VerifyArgs& a, int is_bf16, int sm_count, cudaStream_t stream) {
  // CTAs of a request: as many as are resident at once with all requests', and as long as each has a few hundred tokens for each warp
  unsigned ranks = 1;
  while (ranks < kMaxCluster && 2ll * a.batch * ranks <= static_cast<long long>(kVerifyCtas) * sm_count && a.vocab > static_cast<int>(ranks) * kVerifyThreads * 8)
    ranks *= 2;
  const unsigned grid = static_cast<unsigned>(a.batch) * ranks;
  auto launch = [&](auto type) {
    using T = decltype(type);
    // stretches of 256 tokens where long ones would leave warps without one
    if (a.vocab < static_cast<int>(ranks) * kVerifyWarps * 1024) return launch_cluster(gdpa_verify_kernel<T, 8>, a, grid, kVerifyThreads, ranks, stream);
    return launch_cluster(gdpa_verify_kernel<T, 32>, a, grid, kVerifyThreads, ranks, stream);
  };
  return is_bf16 ? launch(__nv_bfloat16{}) : launch(float{});
}

namespace {
unsigned drop_ctas(long long batch) { return static_cast<unsigned>((batch + kDropWarps * kDropRequests - 1) / (kDropWarps * kDropRequests)); }
}  // namespace

long long drop_workspace_ints(long long batch) {
  const unsigned ctas = drop_ctas(batch);
  return ctas <= kMaxCluster ? 0 : static_cast<long long>(ctas) * (kDropWarps + 1);
}

int launch_drop(const DropArgs& a, cudaStream_t stream) {
  const unsigned ctas = a.batch > 0 ? drop_ctas(a.batch) : 1;
  if (ctas <= kMaxCluster) return launch_cluster(gdpa_drop_kernel<kDropCluster>, a, ctas, kDropWarps * 32, ctas, stream);
  gdpa_drop_kernel<kDropCount><<<ctas, kDropWarps * 32, 0, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return GDPA_ERR_LAUNCH_;
  return launch_cluster(gdpa_drop_kernel<kDropStore>, a, ctas, kDropWarps * 32, 0, stream);
}

}  // namespace gdpa
