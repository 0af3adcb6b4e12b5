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
// number.  A request needs two rows at most, one pass over them: stretches of half a kilobyte or two are added up, and the one in which the sum
// passes its mark is looked at again (it is in the L2 cache).
//
// Few requests: one launch, a cluster of CTAs to each, and latency is all of it.  Many: three kernels, whose beginnings overlap the ends of those before
// them: who is accepted; the stretches' sums, dealt out over the whole GPU (a CTA to a request leaves SMs with one row to add up and SMs with four);
// the token.  256 requests of 131071 bf16 tokens, 116 MB, cold: 55 us in one kernel, 43 in three, 28 of them for the sums
// (4.1 TB/s; half of their time waits for memory, half goes to instructions: rows staged through shared memory, with more on its way, took 33).  Calls in a row: 47
// and 39.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"
#include "sm100_ptx.cuh"

namespace cg = cooperative_groups;

namespace gdpa {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kVerifyThreads = 256, kVerifyWarps = kVerifyThreads / 32;
constexpr int kVerifyCtas = 3, kSumCtas = 4;  // resident on an SM
constexpr int kMostVocab = 1 << 20;
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
  const T* q;   // or null
  int without;  // or -1
  __device__ __forceinline__ double of(float pv, float qv) const {
    const float least = share(qv);
    return static_cast<double>(fmaxf(share(pv), least)) - static_cast<double>(least);
  }
  __device__ __forceinline__ double operator()(int i) const {
    return i == without ? 0 : of(as_float(p[i]), q != nullptr ? as_float(q[i]) : 0.f);
  }
};

// The sum of n tokens from t on, those that are there.  (By value: an address would put the rows into memory.)
template <class T>
__device__ __noinline__ double sum_of_some(const T* p, const T* q, int without, int t, int n, int vocab) {
  const Left<T> left{p, q, without};
  double s = 0;
#pragma unroll 4
  for (int e = 0; e < n; ++e) {
    const int i = t + e;
    const bool there = i >= 0 && i < vocab;
    const float pv = there ? as_float(p[i]) : 0.f, qv = there && q != nullptr ? as_float(q[i]) : 0.f;
    if (i != without) s += left.of(pv, qv);
  }
  return s;
}

// The sum of a lane's share of a stretch whose blocks of 16 bytes are all inside the row.  p is read at its own blocks; q, which may lie otherwise (rows of an odd
// vocabulary begin anywhere), at two blocks of its own for each, shifted by SHIFT tokens.
//
// Integer instructions in place of conversions, which have an eighth of their rate: the bits of a positive fp32 number, moved to the places of an fp64 one's
// exponent and mantissa, are that number times 2^-896, zero and subnormal ones too; and as integers they compare like the numbers.  The sum counts only if
// the largest of all bits, unsigned, is below those of infinity: then all were zeros or positive finite numbers.
constexpr double kUnscale = 0x1p+896;

template <class T, int SHIFT, bool WITH_Q>
struct Sum;
template <int SHIFT, bool WITH_Q>
struct Sum<float, SHIFT, WITH_Q> {
  static __device__ __forceinline__ double value(uint32_t bits) { return __hiloint2double(static_cast<int>(bits >> 3), static_cast<int>(bits << 29)); }
  static __device__ __forceinline__ bool usual(uint32_t largest) { return largest < 0x7f800000u; }
  static __device__ __forceinline__ void add(const uint4& p, const uint4 (&q)[2], double (&sums)[2], uint32_t& largest) {
    const uint32_t a[4] = {p.x, p.y, p.z, p.w}, b[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t m = a[j];
      if constexpr (WITH_Q) m = max(m, b[j + SHIFT]);
      largest = max(largest, m);
      if constexpr (WITH_Q) sums[j & 1] += value(m) - value(b[j + SHIFT]);
      else sums[j & 1] += value(m);
    }
  }
};
template <int SHIFT, bool WITH_Q>
struct Sum<__nv_bfloat16, SHIFT, WITH_Q> {  // two in a word
  static __device__ __forceinline__ double low(uint32_t w) { return __hiloint2double(static_cast<int>((w << 13) & 0x1fffe000u), 0); }
  static __device__ __forceinline__ double high(uint32_t w) { return __hiloint2double(static_cast<int>((w >> 3) & 0x1fffe000u), 0); }
  static __device__ __forceinline__ bool usual(uint32_t largest) { return (largest & 0xffffu) < 0x7f80u && (largest >> 16) < 0x7f80u; }
  static __device__ __forceinline__ void add(const uint4& p, const uint4 (&q)[2], double (&sums)[2], uint32_t& largest) {
    const uint32_t a[4] = {p.x, p.y, p.z, p.w}, w[8] = {q[0].x, q[0].y, q[0].z, q[0].w, q[1].x, q[1].y, q[1].z, q[1].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t m = a[j], b = 0;
      if constexpr (WITH_Q) {
        b = SHIFT % 2 == 0 ? w[j + SHIFT / 2] : __funnelshift_r(w[j + SHIFT / 2], w[j + SHIFT / 2 + 1], 16);
        m = max_u16x2(m, b);
      }
      largest = max_u16x2(largest, m);
      if constexpr (WITH_Q) {
        sums[0] += low(m) - low(b);
        sums[1] += high(m) - high(b);
      } else {
        sums[0] += low(m);
        sums[1] += high(m);
      }
    }
  }
};

// The first block of a row, and its tokens before the row.
template <class T>
struct Blocks {
  const uint4* first;
  int before;
  __device__ __forceinline__ explicit Blocks(const T* row)
      : first(reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(15))),
        before(static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))) {}
};

// How a row is cut: stretches of 32 * BLOCKS blocks of p's row as it lies in memory; the first may begin before the row.
template <class T, int BLOCKS>
struct Cut {
  static constexpr int B = 16 / sizeof(T), U = B * BLOCKS, kStretch = 32 * U;
  int before, stretches;
  __device__ __forceinline__ Cut(const T* row, int vocab) : before(Blocks<T>(row).before) { stretches = (vocab + before + kStretch - 1) / kStretch; }
  __device__ __forceinline__ int first_token(int k) const { return k * kStretch - before; }
};

// A warp's sum of stretch k.  EDGE: blocks that are not all inside the rows (q's second one among them), or have the refused token, are taken token by token.
template <class T, int BLOCKS, int SHIFT, bool WITH_Q, bool EDGE>
__device__ __forceinline__ double sum_blocks(const Left<T>& left, const uint4* p, const uint4* q, int first_token, int vocab) {
  using S = Sum<T, SHIFT, WITH_Q>;
  constexpr int B = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  p += lane, q += lane;
  uint4 a[BLOCKS], b[BLOCKS][2];
  bool inside[BLOCKS];
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) {
    inside[i] = true;
    if constexpr (EDGE) {
      const int t = first_token + (i * 32 + lane) * B;
      inside[i] = t >= B && t + 2 * B <= vocab && static_cast<unsigned>(left.without - t) >= static_cast<unsigned>(B);
    }
    a[i] = b[i][0] = b[i][1] = make_uint4(0, 0, 0, 0);
    if (inside[i]) {
      a[i] = __ldg(p + i * 32);
      if constexpr (WITH_Q) {
        b[i][0] = __ldg(q + i * 32);
        if constexpr (SHIFT > 0) b[i][1] = __ldg(q + i * 32 + 1);
      }
    }
  }
  double sums[2] = {0, 0}, others = 0;
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < BLOCKS; ++i) {
    S::add(a[i], b[i], sums, largest);
    if (EDGE && !inside[i]) others += sum_of_some(left.p, left.q, left.without, first_token + (i * 32 + lane) * B, B, vocab);
  }
  double sum = (sums[0] + sums[1]) * kUnscale + others;
  if (!__all_sync(kFull, S::usual(largest))) {  // a number that is no probability
    sum = 0;
#pragma unroll 1
    for (int i = 0; i < BLOCKS; ++i) sum += sum_of_some(left.p, left.q, left.without, first_token + (i * 32 + lane) * B, B, vocab);
  }
  return sum;
}
template <class T, int BLOCKS, bool EDGE, int SHIFT = 0>
__device__ __forceinline__ double sum_shifted(const Left<T>& left, const uint4* p, const uint4* q, int shift, int first_token, int vocab) {
  if constexpr (SHIFT + 1 < static_cast<int>(16 / sizeof(T))) {
    if (shift != SHIFT) return sum_shifted<T, BLOCKS, EDGE, SHIFT + 1>(left, p, q, shift, first_token, vocab);
  }
  return sum_blocks<T, BLOCKS, SHIFT, true, EDGE>(left, p, q, first_token, vocab);
}
template <class T, int BLOCKS>
__device__ __forceinline__ double sum_stretch(const Left<T>& left, int k, int vocab) {
  constexpr int B = 16 / sizeof(T), kStretch = 32 * B * BLOCKS;
  const Blocks<T> p(left.p), q(left.q);
  const int first_token = k * kStretch - p.before, q_token = q.before - p.before;  // q's first token of the stretch is so many behind a block's beginning
  const uint4* const at = p.first + static_cast<long long>(k) * (32 * BLOCKS);
  const uint4* const q_at = q.first + static_cast<long long>(k) * (32 * BLOCKS) + (q_token >> (B == 8 ? 3 : 2));
  const bool edge = first_token < B || first_token + kStretch + 2 * B > vocab || static_cast<unsigned>(left.without - first_token) < static_cast<unsigned>(kStretch);
  double sum;
  if (edge) {
    sum = left.q == nullptr ? sum_blocks<T, BLOCKS, 0, false, true>(left, at, at, first_token, vocab)
                            : sum_shifted<T, BLOCKS, true>(left, at, q_at, q_token & (B - 1), first_token, vocab);
  } else {
    sum = left.q == nullptr ? sum_blocks<T, BLOCKS, 0, false, false>(left, at, at, first_token, vocab)
                            : sum_shifted<T, BLOCKS, false>(left, at, q_at, q_token & (B - 1), first_token, vocab);
  }
  return warp_sum(sum);
}

// A request's rows and drafts, inside the tensors whatever the offsets say.
struct Request {
  long long row0, d0;
  int n;       // drafts that are looked at
  bool there;  // it has a row
  __device__ __forceinline__ Request(const VerifyArgs& a, int b) {
    row0 = clamp_ll(load_offset(a.row_offsets, b, a.off64), 0, a.rows);
    const long long row1 = clamp_ll(load_offset(a.row_offsets, b + 1, a.off64), row0, a.rows);
    d0 = clamp_ll(load_offset(a.draft_offsets, b, a.off64), 0, a.drafts);
    const long long d1 = clamp_ll(load_offset(a.draft_offsets, b + 1, a.off64), d0, a.drafts);
    n = static_cast<int>(clamp_ll(min(d1 - d0, row1 - row0 - 1), 0, a.max_drafts));
    there = row1 > row0;
  }
};
__device__ __forceinline__ long long token_of(const VerifyArgs& a, long long d) {
  return a.tokens64 ? static_cast<const long long*>(a.tokens)[d] : static_cast<const int*>(a.tokens)[d];
}
__device__ __forceinline__ void put(const VerifyArgs& a, int b, int j, long long token) {
  const long long at = static_cast<long long>(b) * (a.max_drafts + 1) + j;
  if (a.tokens64) static_cast<long long*>(a.out_tokens)[at] = token;
  else static_cast<int*>(a.out_tokens)[at] = static_cast<int>(token);
}

// How many drafts are accepted, by a warp.
template <class T>
__device__ __forceinline__ int accept(const VerifyArgs& a, const Request& r) {
  const T *const target = static_cast<const T*>(a.target), *const draft = static_cast<const T*>(a.draft);
  const int lane = threadIdx.x & 31;
  for (int j0 = 0; j0 < r.n; j0 += 32) {
    const int j = j0 + lane;
    bool refused = false;
    if (j < r.n) {
      const long long x = token_of(a, r.d0 + j);
      const double u = a.accept[r.d0 + j];
      refused = true;
      if (x >= 0 && x < a.vocab) {
        const double p = share(as_float(target[(r.row0 + j) * a.target_stride + x]));
        const double q = draft != nullptr ? static_cast<double>(share(as_float(draft[(r.d0 + j) * a.draft_stride + x]))) : 1.0;
        refused = !(u * q < p);
      }
    }
    const unsigned those = __ballot_sync(kFull, refused);
    if (those != 0) return j0 + __ffs(those) - 1;
  }
  return r.n;
}
// What is known then, by `threads` threads: all but the token that is drawn.
__device__ __forceinline__ void put_accepted(const VerifyArgs& a, const Request& r, int b, int accepted, int thread, int threads) {
  for (int j = thread; j <= a.max_drafts; j += threads)
    if (j != accepted || !r.there) put(a, b, j, j < accepted ? token_of(a, r.d0 + j) : -1);
  if (thread == 0) a.accepted[b] = accepted, a.refused[b] = r.n - accepted;
}
template <class T>
__device__ __forceinline__ Left<T> left_of(const VerifyArgs& a, const Request& r, int accepted) {
  Left<T> left{static_cast<const T*>(a.target) + (r.row0 + accepted) * a.target_stride, nullptr, -1};
  if (accepted < r.n) {
    if (a.draft != nullptr) left.q = static_cast<const T*>(a.draft) + (r.d0 + accepted) * a.draft_stride;
    else left.without = static_cast<int>(clamp_ll(token_of(a, r.d0 + accepted), -1, a.vocab));
  }
  return left;
}

// n sums become sums up to each one's end, by a warp; the last of them.
__device__ __forceinline__ double add_up(double* sums, int n) {
  const int lane = threadIdx.x & 31;
  double before = 0;
  for (int k = 0; k < n; k += 32) {
    double up_to = k + lane < n ? sums[k + lane] : 0;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const double o = __shfl_up_sync(kFull, up_to, s);
      if (lane >= s) up_to += o;
    }
    if (k + lane < n) sums[k + lane] = before + up_to;
    before += __shfl_sync(kFull, up_to, 31);
  }
  return before;
}
// The first of n sums up to each one's end that, with `base`, lies above the mark and above the one before it; if there is none (rounding, or a mark that is
// not below the total): the last that lies above the one before it.  By a warp.
__device__ __forceinline__ int find(const double* sums, int n, double base, double mark) {
  const int lane = threadIdx.x & 31;
  int last = 0;
  for (int k = 0; k < n; k += 32) {
    const double from = k + lane > 0 && k + lane < n ? sums[k + lane - 1] : 0, to = k + lane < n ? sums[k + lane] : 0;
    const bool some = k + lane < n && to > from;
    const unsigned with = __ballot_sync(kFull, some), those = __ballot_sync(kFull, some && base + to > mark);
    if (those != 0) return k + __ffs(those) - 1;
    if (with != 0) last = k + 31 - __clz(with);
  }
  return last;
}
// The token of stretch k at which the sum, `at_start` before the stretch, passes the mark.  By a CTA; its first warp returns it.
template <class T, int BLOCKS>
__device__ __forceinline__ int find_token(const VerifyArgs& a, const Left<T>& left, int k, double at_start, double mark, double* s_share) {
  using C = Cut<T, BLOCKS>;
  constexpr int U = C::U;
  const int first = C(left.p, a.vocab).first_token(k), lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < C::kStretch; i += blockDim.x) {
    const int at = first + i;
    s_share[i / U * (U + 1) + i % U] = at >= 0 && at < a.vocab ? left(at) : 0;
  }
  __syncthreads();
  if (threadIdx.x >= 32) return -1;
  // U tokens of the stretch for each lane, then one
  double sum[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < U; ++i) sum[i & 1] += s_share[lane * (U + 1) + i];
  sum[0] += sum[1];
  double up_to = sum[0];
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const double o = __shfl_up_sync(kFull, up_to, s);
    if (lane >= s) up_to += o;
  }
  unsigned with = __ballot_sync(kFull, sum[0] > 0), those = __ballot_sync(kFull, sum[0] > 0 && at_start + up_to > mark);
  const int row = those != 0 ? __ffs(those) - 1 : with != 0 ? 31 - __clz(with) : 0;
  const double at_row = at_start + __shfl_sync(kFull, up_to - sum[0], row);
  static_assert(U <= 32, "a lane has one of a row's tokens");
  const double mine = lane < U ? s_share[row * (U + 1) + lane] : 0;
  up_to = mine;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const double o = __shfl_up_sync(kFull, up_to, s);
    if (lane >= s) up_to += o;
  }
  with = __ballot_sync(kFull, mine > 0), those = __ballot_sync(kFull, mine > 0 && at_row + up_to > mark);
  return first + row * U + (those != 0 ? __ffs(those) - 1 : with != 0 ? 31 - __clz(with) : 0);
}

// ---- few requests

// (Short stretches, BLOCKS = 1: a few for each warp.)
template <class T, int BLOCKS>
__global__ void __launch_bounds__(kVerifyThreads, kVerifyCtas) gdpa_verify_kernel(const __grid_constant__ VerifyArgs a) {
  using C = Cut<T, BLOCKS>;
  __shared__ double s_sum[BLOCKS == 1 ? 128 : kMostVocab / C::kStretch + 1];
  __shared__ double s_total;  // of this CTA, for the cluster
  __shared__ double s_share[32 * (C::U + 1)];
  __shared__ int s_accepted, s_stretch;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / ranks, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Request r(a, b);
  const float sample = a.sample[b];
  if (warp == 0) {  // by every CTA for itself
    const int n = accept<T>(a, r);
    if (lane == 0) s_accepted = n;
  }
  __syncthreads();
  const int accepted = s_accepted;
  if (rank == 0) put_accepted(a, r, b, accepted, threadIdx.x, kVerifyThreads);
  if (!r.there) return;  // the same for the whole cluster
  Left<T> left = left_of<T>(a, r, accepted);
  const int stretches = C(left.p, a.vocab).stretches;
  const int k0 = static_cast<int>(static_cast<long long>(stretches) * rank / ranks);
  const int mine = static_cast<int>(static_cast<long long>(stretches) * (rank + 1) / ranks) - k0;
  double total, base, mark;
  int owner;
  for (;;) {
    for (int k = warp; k < mine; k += kVerifyWarps) {
      const double sum = sum_stretch<T, BLOCKS>(left, k0 + k, a.vocab);
      if (lane == 0) s_sum[k] = sum;
    }
    __syncthreads();
    if (warp == 0) {
      const double sum = add_up(s_sum, mine);
      if (lane == 0) s_total = sum;
    }
    // The CTA in whose stretches the sum passes its mark: the first whose end lies above it; if there is none, the last with a share.
    cluster.sync();
    const double of_lane = lane < ranks ? *cluster.map_shared_rank(&s_total, lane) : 0;
    cluster.sync();  // before a CTA ends or writes its sum again
    total = 0;
    for (int i = 0; i < ranks; ++i) total += __shfl_sync(kFull, of_lane, i);
    mark = static_cast<double>(sample) * total;
    double end = 0;
    base = 0, owner = -1;
    bool above = false;
    for (int i = 0; i < ranks && !above; ++i) {
      const double of_rank = __shfl_sync(kFull, of_lane, i);
      if (of_rank > 0) owner = i, base = end;
      end += of_rank;
      above = of_rank > 0 && end > mark;
    }
    if (total > 0) break;
    if (left.q == nullptr && left.without < 0) break;
    left.q = nullptr, left.without = -1;  // nothing is left of the difference
  }
  if (owner < 0) {  // nothing to draw from
    if (rank == 0 && threadIdx.x == 0) put(a, b, accepted, -1);
    return;
  }
  if (rank != owner) return;
  if (warp == 0) {
    const int k = find(s_sum, mine, base, mark);
    if (lane == 0) s_stretch = k;
  }
  __syncthreads();
  const int k = s_stretch, token = find_token<T, BLOCKS>(a, left, k0 + k, base + (k > 0 ? s_sum[k - 1] : 0), mark, s_share);
  if (threadIdx.x == 0) put(a, b, accepted, token);
}

// ---- many requests

constexpr int kManyBlocks = 2;  // blocks of a lane of a stretch

// What a request's token is drawn from, with the address of its stretches' sums in between; as the workspace has it.
struct Draw {
  const void* p;
  const void* q;
  int without;
  int stretches;  // 0: no row
};
template <class T>
__device__ __forceinline__ Left<T> left_of(const Draw& d) { return {static_cast<const T*>(d.p), static_cast<const T*>(d.q), d.without}; }

template <class T>
__global__ void __launch_bounds__(kVerifyThreads) gdpa_verify_accept_kernel(const __grid_constant__ VerifyArgs a) {
  const int b = blockIdx.x * kVerifyWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (b >= a.batch) return;
  const Request r(a, b);
  const int accepted = accept<T>(a, r);
  put_accepted(a, r, b, accepted, lane, 32);
  if (lane != 0) return;
  Draw d{nullptr, nullptr, -1, 0};
  if (r.there) {
    const Left<T> left = left_of<T>(a, r, accepted);
    d = Draw{left.p, left.q, left.without, Cut<T, kManyBlocks>(left.p, a.vocab).stretches};
  }
  static_cast<Draw*>(a.draws)[b] = d;
}

// A warp takes stretch after stretch, the w-th of every n of all requests' together: rows with and without a second one to read mix on every SM.
template <class T>
__global__ void __launch_bounds__(kVerifyThreads, kSumCtas) gdpa_verify_sum_kernel(const __grid_constant__ VerifyArgs a) {
  const int lane = threadIdx.x & 31;
  const unsigned most = static_cast<unsigned>(a.most_stretches), all = static_cast<unsigned>(a.batch) * most, step = gridDim.x * kVerifyWarps;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the draws
  const unsigned first = blockIdx.x * kVerifyWarps + (threadIdx.x >> 5), whole = step / most, part = step - whole * most;
  unsigned b = first / most, k = first - b * most;  // request and stretch
  const Draw* const draws = static_cast<const Draw*>(a.draws);
  Draw next{nullptr, nullptr, -1, 0};
  if (first < all) next = draws[b];
  for (unsigned i = first; i < all; i += step) {
    const Draw d = next;
    const unsigned now = k;
    b += whole, k += part;
    if (k >= most) k -= most, ++b;
    if (i + step < all) next = draws[b];
    if (now >= static_cast<unsigned>(d.stretches)) continue;
    const double sum = sum_stretch<T, kManyBlocks>(left_of<T>(d), static_cast<int>(now), a.vocab);
    if (lane == 0) a.sums[i] = sum;
  }
}

// Of n sums: their total, and the first one whose end lies above sample times that, or, if none does, the last with a share; and what lies before
// it.  By a CTA.
struct Found {
  double total, before, mark;
  int k;
};
__device__ __forceinline__ Found find_stretch(const double* sums, int n, double sample) {
  __shared__ double s_of_warp[kVerifyWarps], s_before[2][kVerifyWarps];
  __shared__ int s_k[2][kVerifyWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int each = (n + kVerifyThreads - 1) / kVerifyThreads, k0 = threadIdx.x * each, k1 = min(k0 + each, n);
  double own = 0;
  for (int k = k0; k < k1; ++k) own += sums[k];
  double up_to = own;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const double o = __shfl_up_sync(kFull, up_to, s);
    if (lane >= s) up_to += o;
  }
  if (lane == 31) s_of_warp[warp] = up_to;
  __syncthreads();
  Found f{0, 0, 0, 0};
  double run = __shfl_up_sync(kFull, up_to, 1);
  if (lane == 0) run = 0;
#pragma unroll
  for (int w = 0; w < kVerifyWarps; ++w) {
    if (w == warp) run += f.total;
    f.total += s_of_warp[w];
  }
  f.mark = sample * f.total;
  int at[2] = {-1, -1};  // the lane's first one above the mark, its last one with a share
  double before[2] = {0, 0};
  for (int k = k0; k < k1; ++k) {
    const double x = sums[k];
    if (x > 0) {
      at[1] = k, before[1] = run;
      if (at[0] < 0 && run + x > f.mark) at[0] = k, before[0] = run;
    }
    run += x;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const unsigned those = __ballot_sync(kFull, at[c] >= 0);
    const int of = c == 0 ? __ffs(those) - 1 : 31 - __clz(those);
    const int k = __shfl_sync(kFull, at[c], of & 31);
    const double x = __shfl_sync(kFull, before[c], of & 31);
    if (lane == 0) s_k[c][warp] = those != 0 ? k : -1, s_before[c][warp] = x;
  }
  __syncthreads();
  f.k = -1;
#pragma unroll
  for (int w = 0; w < kVerifyWarps; ++w)
    if (f.k < 0 && s_k[0][w] >= 0) f.k = s_k[0][w], f.before = s_before[0][w];
  if (f.k < 0) {
#pragma unroll
    for (int w = 0; w < kVerifyWarps; ++w)
      if (s_k[1][w] >= 0) f.k = s_k[1][w], f.before = s_before[1][w];
  }
  return f;
}

template <class T>
__global__ void __launch_bounds__(kVerifyThreads) gdpa_verify_draw_kernel(const __grid_constant__ VerifyArgs a) {
  using C = Cut<T, kManyBlocks>;
  __shared__ double s_sum[kMostVocab / C::kStretch + 1];
  __shared__ double s_share[32 * (C::U + 1)];
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const double sample = a.sample[b];
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the sums, and with them for the draws and what is accepted
  const Draw d = static_cast<const Draw*>(a.draws)[b];
  if (d.stretches == 0) return;
  const int accepted = a.accepted[b];
  Left<T> left = left_of<T>(d);
  for (int k = threadIdx.x; k < d.stretches; k += kVerifyThreads) s_sum[k] = a.sums[static_cast<long long>(b) * a.most_stretches + k];
  __syncthreads();
  Found f = find_stretch(s_sum, d.stretches, sample);
  if (f.k < 0 && (left.q != nullptr || left.without >= 0)) {  // nothing is left of the difference
    left.q = nullptr, left.without = -1;
    for (int k = warp; k < d.stretches; k += kVerifyWarps) {
      const double sum = sum_stretch<T, kManyBlocks>(left, k, a.vocab);
      if (lane == 0) s_sum[k] = sum;
    }
    __syncthreads();
    f = find_stretch(s_sum, d.stretches, sample);
  }
  const int token = f.k < 0 ? -1 : find_token<T, kManyBlocks>(a, left, f.k, f.before, f.mark, s_share);  // -1: nothing to draw from
  if (threadIdx.x == 0) put(a, b, accepted, token);
}

// ------------------------------------------------------------------------------------------ tokens that leave the cache
//
// The last dropped[b] tokens of each request leave; the blocks that none of its tokens needs any more go onto the stack of free blocks, in
// the order of the requests and of their tables (entries that are no block, -1, do not).  Tables are left as they are: what lies behind a
// request's length is not looked at.
//
// Latency is all of it.  A warp has four requests, up to 128 entries of each, all asked for at once and kept in registers until it is known how many go
// before them; where tables are wide, four chunks of requests: one request of 2^20 tokens in blocks of 16, all of which leave, 377 us by a warp, 19
// by many.  Up to 256 of those, a cluster of CTAs adds that up in shared memory.  More of them: one kernel counts, another, whose loads the end of the first
// overlaps, adds up the counts of the CTAs before its own (4096 requests with 64 entries each: 11 us; up to 256 a cluster is 2 us faster).
constexpr int kDropWarps = 8, kDropChunks = 4;

enum DropWay { kDropCluster, kDropCount, kDropStore };

template <DropWay WAY>
__global__ void __launch_bounds__(kDropWarps * 32) gdpa_drop_kernel(const __grid_constant__ DropArgs a) {
  __shared__ int s_count[kDropWarps];
  __shared__ int s_total;
  __shared__ long long s_before[kDropWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int S = 1 << a.block_shift;
  // the warp's chunks, and those of their entries that may go
  const unsigned v = (blockIdx.x * kDropWarps + warp) * kDropChunks + lane, b = v / static_cast<unsigned>(a.chunks);
  const int c = static_cast<int>(v - b * a.chunks);
  int from_here = 0, to_here = 0;
  if (lane < kDropChunks && b < static_cast<unsigned>(a.batch)) {
    const long long len = clamp_ll(load_offset(a.seq_lens, b, a.lens64), 0, 0x7fffff00);
    const long long after = len - clamp_ll(load_offset(a.dropped, b, a.dropped64), 0, len);
    if (WAY != kDropCount && c == 0) a.seq_lens_after[b] = static_cast<int>(after);
    const int keep = static_cast<int>(min((after + S - 1) >> a.block_shift, static_cast<long long>(a.table_width)));
    const int held = static_cast<int>(min((len + S - 1) >> a.block_shift, static_cast<long long>(a.table_width)));
    from_here = min(keep + c * a.chunk_entries, held);
    to_here = c + 1 == a.chunks ? held : min(from_here + a.chunk_entries, held);
  }
  int entry[kDropChunks][4];
#pragma unroll
  for (int i = 0; i < kDropChunks; ++i) {
    const int from = __shfl_sync(kFull, from_here, i), to = __shfl_sync(kFull, to_here, i);
    const int* const row = a.block_tables + static_cast<long long>(__shfl_sync(kFull, b, i)) * a.table_stride;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = from + 32 * u + lane;
      entry[i][u] = j < to ? row[j] : -1;
    }
  }
  // all of them in order: body(the lane's entry or -1, votes of the lanes that have one)
  auto walk = [&](auto body) {
#pragma unroll
    for (int i = 0; i < kDropChunks; ++i) {
      const int from = __shfl_sync(kFull, from_here, i), to = __shfl_sync(kFull, to_here, i);
#pragma unroll
      for (int u = 0; u < 4; ++u) body(entry[i][u], __ballot_sync(kFull, entry[i][u] >= 0));
      // a chunk with more
      const int* const row = a.block_tables + static_cast<long long>(__shfl_sync(kFull, b, i)) * a.table_stride;
      for (int j0 = from + 128; j0 < to; j0 += 512) {
        int e[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) e[u] = j0 + 32 * u + lane < to ? row[j0 + 32 * u + lane] : -1;
#pragma unroll
        for (int u = 0; u < 16; ++u) body(e[u], __ballot_sync(kFull, e[u] >= 0));
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

namespace {
// Whether a call takes the three kernels: where its rows keep the whole GPU busy.  One kernel against three, us, rows of bf16, cold (calls in a row): 64 requests of 32000
// tokens (4 MB) 14 and 16 (12 and 15), 32 of 131071 (8 MB) 18 and 20 (16 and 17), 256 of 32000 (16 MB) 22 and 22 (18 and 20), 256 of 131071 (67 MB) 55 and 43 (47 and 39).
bool many_requests(long long batch, long long vocab, int size) { return batch >= 32 && batch * vocab * size >= (8ll << 20); }
long long most_stretches(long long vocab, int size) { return (vocab * size + 15) / (32 * kManyBlocks * 16) + 1; }
}  // namespace

VerifyWorkspace verify_workspace(long long batch, long long vocab, int is_bf16) {
  const int size = is_bf16 ? 2 : 4;
  VerifyWorkspace w{0, 0};
  if (!many_requests(batch, vocab, size)) return w;
  w.sums = batch * static_cast<long long>(sizeof(Draw));
  w.bytes = w.sums + batch * most_stretches(vocab, size) * static_cast<long long>(sizeof(double));
  return w;
}

int launch_verify(VerifyArgs& a, int is_bf16, int sm_count, cudaStream_t stream) {
  const int size = is_bf16 ? 2 : 4;
  if (many_requests(a.batch, a.vocab, size)) {
    a.most_stretches = static_cast<int>(most_stretches(a.vocab, size));
    if (static_cast<long long>(a.batch) * a.most_stretches > 0x7fffffffll) return GDPA_ERR_LAUNCH_;
    auto launch = [&](auto type) -> int {
      using T = decltype(type);
      gdpa_verify_accept_kernel<T><<<(a.batch + kVerifyWarps - 1) / kVerifyWarps, kVerifyThreads, 0, stream>>>(a);
      if (cudaGetLastError() != cudaSuccess) return GDPA_ERR_LAUNCH_;
      int rc = launch_cluster(gdpa_verify_sum_kernel<T>, a, static_cast<unsigned>(kSumCtas * sm_count), kVerifyThreads, 0, stream);
      if (rc == 0) rc = launch_cluster(gdpa_verify_draw_kernel<T>, a, static_cast<unsigned>(a.batch), kVerifyThreads, 0, stream);
      return rc;
    };
    return is_bf16 ? launch(__nv_bfloat16{}) : launch(float{});
  }
  // CTAs of a request: as many as are resident at once with all requests', and as long as each has half a kilobyte for each warp
  unsigned ranks = 1;
  while (ranks < kMaxCluster && 2ll * a.batch * ranks <= static_cast<long long>(kVerifyCtas) * sm_count &&
         static_cast<long long>(a.vocab) * size > static_cast<long long>(ranks) * kVerifyWarps * 512)
    ranks *= 2;
  const unsigned grid = static_cast<unsigned>(a.batch) * ranks;
  auto launch = [&](auto type, auto blocks) {
    return launch_cluster(gdpa_verify_kernel<decltype(type), decltype(blocks)::value>, a, grid, kVerifyThreads, ranks, stream);
  };
  // short stretches where long ones would leave warps without one
  using Short = std::integral_constant<int, 1>;
  using Long = std::integral_constant<int, 4>;
  if (static_cast<long long>(a.vocab) * size < static_cast<long long>(ranks) * kVerifyWarps * 2048)
    return is_bf16 ? launch(__nv_bfloat16{}, Short{}) : launch(float{}, Short{});
  return is_bf16 ? launch(__nv_bfloat16{}, Long{}) : launch(float{}, Long{});
}

namespace {
// Chunks of a request: as many as give each 512 entries at least, and no more than 2^17 of them all together (a CTA reads the counts of all).
int drop_chunks(long long batch, int table_width) {
  const long long most = batch > 0 ? (1ll << 17) / batch : 1, wanted = table_width > 640 ? (table_width + 511) / 512 : 1;
  return static_cast<int>(most < 1 ? 1 : wanted < most ? wanted : most);
}
unsigned drop_ctas(long long chunks) { return static_cast<unsigned>((chunks + kDropWarps * kDropChunks - 1) / (kDropWarps * kDropChunks)); }
}  // namespace

long long drop_workspace_ints(long long batch, int table_width) {
  const unsigned ctas = drop_ctas(batch * drop_chunks(batch, table_width));
  return ctas <= kMaxCluster ? 0 : static_cast<long long>(ctas) * (kDropWarps + 1);
}

int launch_drop(DropArgs& a, cudaStream_t stream) {
  a.chunks = drop_chunks(a.batch, a.table_width);
  a.chunk_entries = (a.table_width + a.chunks - 1) / a.chunks;
  const unsigned ctas = a.batch > 0 ? drop_ctas(static_cast<long long>(a.batch) * a.chunks) : 1;
  if (ctas <= kMaxCluster) return launch_cluster(gdpa_drop_kernel<kDropCluster>, a, ctas, kDropWarps * 32, ctas, stream);
  gdpa_drop_kernel<kDropCount><<<ctas, kDropWarps * 32, 0, stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return GDPA_ERR_LAUNCH_;
  return launch_cluster(gdpa_drop_kernel<kDropStore>, a, ctas, kDropWarps * 32, 0, stream);
}

}  // namespace gdpa
