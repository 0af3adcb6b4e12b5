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
// number.  A request needs two rows at most, one pass over them: a cluster of CTAs sums stretches of 1024 tokens, and the stretch in which the
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
constexpr int kVerifyThreads = 512, kVerifyWarps = kVerifyThreads / 32;
constexpr int kStretch = 1024;          // tokens of a stretch
constexpr int kMostStretches = 1024;    // of a vocabulary
constexpr int kMaxCluster = 8;

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

__device__ __forceinline__ double share(double x) { return x > 0 && x <= 1.7976931348623157e308 ? x : 0; }

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(kFull, x, s);
  return x;
}

// What is drawn from: p, less q or less the token `without`.
template <class T>
struct Left {
  const T* p;
  const T* q;       // or null
  long long without;  // or -1
  __device__ __forceinline__ double at(float pv, float qv, int i) const {
    double x = pv;
    if (q != nullptr) x -= fmax(static_cast<double>(qv), 0.0);
    return i == without ? 0 : share(x);
  }
  __device__ __forceinline__ double operator()(int i) const { return at(as_float(p[i]), q != nullptr ? as_float(q[i]) : 0.f, i); }
};

template <class T>
__global__ void __launch_bounds__(kVerifyThreads) gdpa_verify_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ double s_sum[kMostStretches];  // of a stretch; then up to its end
  __shared__ double s_total;                // of this CTA, for the cluster
  __shared__ double s_share[32 * 33];
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
    else left.without = token_of(d0 + accepted);
  }
  // this CTA's stretches
  const int stretches = (a.vocab + kStretch - 1) / kStretch;
  const int k0 = static_cast<int>(static_cast<long long>(stretches) * rank / ranks);
  const int mine = static_cast<int>(static_cast<long long>(stretches) * (rank + 1) / ranks) - k0;
  double total, base, mark;
  int owner;
  for (;;) {
    for (int k = warp; k < mine; k += kVerifyWarps) {
      double sum[2] = {0, 0};
      const int i0 = (k0 + k) * kStretch + lane;
#pragma unroll
      for (int u0 = 0; u0 < kStretch / 32; u0 += 8) {
        float p[8], q[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = i0 + (u0 + u) * 32;
          p[u] = i < a.vocab ? as_float(left.p[i]) : 0.f;
          q[u] = left.q != nullptr && i < a.vocab ? as_float(left.q[i]) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) sum[u & 1] += left.at(p[u], q[u], i0 + (u0 + u) * 32);
      }
      const double s = warp_sum(sum[0] + sum[1]);
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
    s_share[i / 32 * 33 + i % 32] = at < a.vocab ? left(at) : 0;
  }
  __syncthreads();
  if (warp != 0) return;
  // 32 tokens of the stretch for each lane, then one
  double sum = 0;
  for (int i = 0; i < 32; ++i) sum += s_share[lane * 33 + i];
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
  const double mine_here = s_share[row * 33 + lane];
  up_to = mine_here;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const double o = __shfl_up_sync(kFull, up_to, s);
    if (lane >= s) up_to += o;
  }
  with = __ballot_sync(kFull, mine_here > 0), those = __ballot_sync(kFull, mine_here > 0 && at_row + up_to > mark);
  const int column = those != 0 ? __ffs(those) - 1 : with != 0 ? 31 - __clz(with) : 0;
  if (lane == 0) put(accepted, (k0 + k) * kStretch + row * 32 + column);
}

// ------------------------------------------------------------------------------------------ tokens that leave the cache
//
// The last dropped[b] tokens of each request leave; the blocks that none of its tokens needs any more go onto the stack of free blocks, in
// the order of the requests and of their tables (entries that are no block, -1, do not).  Tables are left as they are: what lies behind a
// request's length is not looked at.
//
// Latency is all of it.  A warp has eight requests, whose entries it walks over 128 at a time: once to count them, once, when a
// cluster of CTAs has added up what comes before, to put them on the stack.
constexpr int kDropWarps = 32, kDropRequests = 8;

__global__ void __launch_bounds__(kDropWarps * 32) gdpa_drop_kernel(const __grid_constant__ DropArgs a) {
  __shared__ long long s_count[kDropWarps];
  __shared__ long long s_total;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int S = 1 << a.block_shift;
  const long long have = clamp_ll(*a.num_free, 0, a.free_capacity);
  // this warp's requests
  const int groups = (a.batch + kDropRequests - 1) / kDropRequests, all = ranks * kDropWarps, me = rank * kDropWarps + warp;
  const int g0 = static_cast<int>(static_cast<long long>(groups) * me / all), g1 = static_cast<int>(static_cast<long long>(groups) * (me + 1) / all);
  // all entries of the warp's requests, in order: body(lane has one, the entry, votes of the lanes that have one)
  auto walk = [&](bool write_lens, auto body) {
    for (int g = g0; g < g1; ++g) {
      const int b = g * kDropRequests + lane;
      int keep = 0, count = 0;
      if (lane < kDropRequests && b < a.batch) {
        const long long len = clamp_ll(load_offset(a.seq_lens, b, a.lens64), 0, 0x7fffff00);
        const long long after = len - clamp_ll(load_offset(a.dropped, b, a.dropped64), 0, len);
        if (write_lens) a.seq_lens_after[b] = static_cast<int>(after);
        keep = static_cast<int>(min((after + S - 1) >> a.block_shift, static_cast<long long>(a.table_width)));
        count = static_cast<int>(min((len + S - 1) >> a.block_shift, static_cast<long long>(a.table_width))) - keep;
      }
      long long up_to = count;
#pragma unroll
      for (int s = 1; s < kDropRequests; s <<= 1) {
        const long long o = __shfl_up_sync(kFull, up_to, s);
        if (lane >= s) up_to += o;
      }
      const long long entries = __shfl_sync(kFull, up_to, kDropRequests - 1), before = up_to - count;
      for (long long e0 = 0; e0 < entries; e0 += 128) {
        int entry[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const long long e = e0 + 32 * u + lane;
          int owner = 0;  // requests whose entries all lie before this one
#pragma unroll
          for (int s = kDropRequests / 2; s > 0; s >>= 1) owner += __shfl_sync(kFull, up_to, owner + s - 1) <= e ? s : 0;
          const long long j = __shfl_sync(kFull, keep, owner) + e - __shfl_sync(kFull, before, owner);
          entry[u] = e < entries ? a.block_tables[static_cast<long long>(g * kDropRequests + owner) * a.table_stride + j] : -1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) body(entry[u], __ballot_sync(kFull, entry[u] >= 0));
      }
    }
  };
  long long count = 0;
  walk(true, [&](int, unsigned those) { count += __popc(those); });
  if (lane == 0) s_count[warp] = count;
  __syncthreads();
  long long place = have, cta = 0;
  for (int w = 0; w < kDropWarps; ++w) {
    if (w < warp) place += s_count[w];
    cta += s_count[w];
  }
  if (threadIdx.x == 0) s_total = cta;
  cluster.sync();
  long long total = 0;
  for (int r = 0; r < ranks; ++r) {
    if (r == rank) place += total;
    total += *cluster.map_shared_rank(&s_total, r);
  }
  cluster.sync();  // before a CTA ends
  if (rank == 0 && threadIdx.x == 0) *a.num_free_after = static_cast<int>(clamp_ll(have + total, 0, a.free_capacity));
  walk(false, [&](int entry, unsigned those) {
    const long long at = place + __popc(those & ((1u << lane) - 1));
    if (entry >= 0 && at < a.free_capacity) a.free_blocks[at] = entry;
    place += __popc(those);
  });
}

template <class K, class A>
int launch_cluster(K kernel, const A& args, unsigned grid, unsigned threads, unsigned ranks, cudaStream_t stream) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ranks, at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args) == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

}  // namespace

int verify_most_vocab() { return kMostStretches * kStretch; }

int launch_verify(const VerifyArgs& a, int is_bf16, int sm_count, cudaStream_t stream) {
  // CTAs of a request: until there are a few for each SM, and as long as each has several stretches
  unsigned ranks = 1;
  while (ranks < kMaxCluster && static_cast<long long>(a.batch) * ranks < 8ll * sm_count && a.vocab >= static_cast<int>(ranks) * 2 * 2 * kStretch) ranks *= 2;
  const unsigned grid = static_cast<unsigned>(a.batch) * ranks;
  return is_bf16 ? launch_cluster(gdpa_verify_kernel<__nv_bfloat16>, a, grid, kVerifyThreads, ranks, stream)
                 : launch_cluster(gdpa_verify_kernel<float>, a, grid, kVerifyThreads, ranks, stream);
}

int launch_drop(const DropArgs& a, cudaStream_t stream) {
  const unsigned ranks = a.batch > kDropWarps * kDropRequests ? kMaxCluster : 1;
  return launch_cluster(gdpa_drop_kernel, a, ranks, kDropWarps * 32, ranks, stream);
}

}  // namespace gdpa
