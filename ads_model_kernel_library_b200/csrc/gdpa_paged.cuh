// What the kernels of the attention over a paged cache share: items and how they are dealt out, the loader, the join of items that several
// CTAs had a part of.  A kernel's shape L says where its shared memory and barriers are.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "gdpa_common.cuh"
#include "gdpa_launch.h"

namespace gdpa {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kItemSlots = 4;
constexpr float kMax8 = 448.f;
constexpr float kNoMax = -3.0e38f;     // running maximum of a row that has seen no key
constexpr float kLeastScale = 7.888609e-31f;  // 2^-100, the least scale that the append writes
// What stands in the place of V's scale for a block that the table has not: a NaN that no arithmetic makes.
constexpr uint32_t kNoBlock = 0xffffffffu;
__device__ const uint32_t g_no_block = kNoBlock;
__device__ __forceinline__ bool no_block(float v_scale) { return __float_as_uint(v_scale) == kNoBlock; }

// One stretch of tiles of one item, as the loader publishes it.
struct PagedItem {
  int h;        // K / V head; -1 ends the walk, -2: a wait ran out
  int q_start;  // first query row of the request
  int past;     // position of its first query
  int row0;     // first (query, head of the group) row of the tile
  int rows;
  int len;      // tokens of the request
  int lo, hi;   // keys that any of the rows takes part with
  int tile0, tiles;
  int pieces;   // stretches the item is cut into
  int first;    // CTA of the first of them
  int b;        // request
};

// One more of the CTAs of an item: how many came before.  Release and acquire: what the caller's CTA wrote before its barrier is seen by
// whoever counts after it.
__device__ __forceinline__ int count_arrival(int* counter) {
  int old;
  asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
  return old;
}

struct KeyRange {
  int lo, hi;
};
// keys that query i takes part with; the first one's position is `past`
__device__ __forceinline__ KeyRange keys_of(int i, int past, int len, int causal, int window) {
  const int p = past + i;
  KeyRange r{0, len};
  if (causal) r.hi = min(r.hi, p + 1);
  if (window >= 0) r.lo = max(0, p - window), r.hi = min(r.hi, p + window + 1);
  if (r.hi <= r.lo) r.lo = r.hi = 0;
  return r;
}
// ... and any of queries i0 .. i1
__device__ __forceinline__ KeyRange keys_of_any(int i0, int i1, int past, int len, int causal, int window) {
  const int p0 = past + i0, p1 = past + i1;
  KeyRange r{0, len};
  if (causal) r.hi = min(r.hi, p1 + 1);
  if (window >= 0) r.lo = max(0, p0 - window), r.hi = min(r.hi, p1 + window + 1);
  if (r.hi <= r.lo) r.lo = r.hi = 0;
  return r;
}
__device__ __forceinline__ int tiles_of(const KeyRange& r) { return r.hi > r.lo ? (r.hi + kTile - 1) / kTile - r.lo / kTile : 0; }

// A NaN in V makes NaN of its column of O, for the rows that take part with its token.  Where all rows of a tile do, the products see to that; where
// some do not, the NaNs leave V before them (0 times NaN is NaN), and a stretch that had any asks here at its end: a bit for each of 32
// columns, c0 on, that holds a NaN at one of a row's keys [lo, hi) in those of the tiles that not all rows take part with ([all_lo, all_hi)).  From
// the cache once more: rare, and no place to remember it in (256 rows of 128 columns).
static __device__ __noinline__ uint32_t nan_columns(const PagedArgs& a, int b, int h, int tile0, int tiles, int lo, int hi, int all_lo, int all_hi, int c0) {
  const int* const table = a.block_tables + static_cast<long long>(b) * a.table_stride;
  uint32_t bits = 0;
  for (int t = tile0; t < tile0 + tiles; ++t) {
    if (t * kTile >= all_lo && (t + 1) * kTile <= all_hi) continue;
    for (int key = max(lo, t * kTile); key < min(hi, (t + 1) * kTile); ++key) {
      const int blk = table[key >> a.block_shift];
      if (blk < 0 || blk >= a.num_blocks) continue;
      const uint4* const v = reinterpret_cast<const uint4*>(a.v_cache + blk * a.v_strides[0] + (key & ((1 << a.block_shift) - 1)) * a.v_strides[1] +
                                                            h * a.v_strides[2] + c0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 u = v[i];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          bits |= (((__vcmpeq4(w[e] & 0x7f7f7f7fu, 0x7f7f7f7fu) & 0x08040201u) * 0x01010101u) >> 24) << (16 * i + 4 * e);
      }
    }
  }
  return bits;
}
// Sixteen bytes of V without their NaNs; whether there were any.
__device__ __forceinline__ bool drop_nans(uint4& u) {
  const uint32_t x = __vcmpeq4(u.x & 0x7f7f7f7fu, 0x7f7f7f7fu), y = __vcmpeq4(u.y & 0x7f7f7f7fu, 0x7f7f7f7fu),
                 z = __vcmpeq4(u.z & 0x7f7f7f7fu, 0x7f7f7f7fu), w = __vcmpeq4(u.w & 0x7f7f7f7fu, 0x7f7f7f7fu);
  u = make_uint4(u.x & ~x, u.y & ~y, u.z & ~z, u.w & ~w);
  return (x | y | z | w) != 0u;
}

struct Request {
  int q_start, q_len;
  int len;   // tokens that the table can hold, at most
  int past;  // position of the first query: the queries are the request's last tokens, those that the table has no place for among them
};
__device__ __forceinline__ Request load_request(const PagedArgs& a, int b) {
  long long q0 = load_offset(a.q_off, b, a.off64), q1 = load_offset(a.q_off, b + 1, a.off64);
  q0 = clamp_ll(q0, 0, a.total_q);
  q1 = clamp_ll(q1, q0, a.total_q);
  const long long most = static_cast<long long>(a.table_width) << a.block_shift;
  Request r;
  r.q_start = static_cast<int>(q0);
  r.q_len = static_cast<int>(min(q1 - q0, static_cast<long long>(a.max_q)));
  const long long len = clamp_ll(load_offset(a.seq_lens, b, a.lens64), 0, 1 << 30);
  r.len = static_cast<int>(min(len, most));
  r.past = static_cast<int>(len) - r.q_len;
  return r;
}

// What an item costs, in units: L::kItemUnits for its beginning and end, and for each of its KV tiles (one at least: a row tile without keys
// has zeros to write) one.
template <class L>
__device__ __forceinline__ long long units_of_item(int tiles) {
  return L::kItemUnits + max(1, tiles);
}
// ... and one K / V head of a request.
template <class L, int NMAX>
__device__ __forceinline__ long long units_of(const PagedArgs& a, const Request& r) {
  const int rows = r.q_len * a.group, nt = (rows + NMAX - 1) / NMAX;
  if (nt == 0) return 0;
  if (!a.causal && a.window < 0) return nt * units_of_item<L>(tiles_of(KeyRange{0, r.len}));
  long long n = 0;
  for (int t = 0; t < nt; ++t) {
    const int last = min(rows, (t + 1) * NMAX);
    n += units_of_item<L>(tiles_of(keys_of_any(t * NMAX / a.group, (last - 1) / a.group, r.past, r.len, a.causal, a.window)));
  }
  return n;
}
// CTAs that have a share of `all` units: no share is smaller than a unit, or a CTA between an item's first and last would have none of its
// tiles, and the join would wait for a piece that nobody makes.
__device__ __forceinline__ long long sharing_ctas(long long all) { return min(static_cast<long long>(gridDim.x), max(1ll, all)); }

template <int ACT>
__device__ __forceinline__ float act_one(float x, float m) {
  // x/2 erfc(-x / sqrt 2): 1 + erf would cancel where x is well below zero, and a row's scale brings such a P up when it has no larger
  if constexpr (ACT == ACT_GELU_ERF) return 0.5f * m * x * erfcf(x * -0.70710678118654752f);
  else return act_scaled<ACT>(x, m, 0.5f * m);
}
template <int ACT, int N>
__device__ __forceinline__ void act_all(float (&x)[N], float m) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = act_one<ACT>(x[i], m);
}
// x = act(x) * m for a run-time activation class
template <int N>
__device__ __forceinline__ void act_any(int act, float (&x)[N], float m) {
  switch (act) {
    case ACT_GELU_ERF: act_all<ACT_GELU_ERF>(x, m); break;
    case ACT_GELU_TANH: act_all<ACT_GELU_TANH>(x, m); break;
    case ACT_LEAKY_RELU: act_all<ACT_LEAKY_RELU>(x, m); break;
    case ACT_RELU: act_all<ACT_RELU>(x, m); break;
    case ACT_SILU: act_all<ACT_SILU>(x, m); break;
    case ACT_HARDSWISH: act_all<ACT_HARDSWISH>(x, m); break;
    case ACT_RELU_SQUARE: act_all<ACT_RELU_SQUARE>(x, m); break;
    default: act_all<ACT_RAW>(x, m); break;
  }
}

// Where a CTA's walk over the items begins.
struct PagedStart {
  long long all, before;  // all units; units before request b
  int b;
};

// A kernel's wait, by a whole warp: whether it ended.
#define PAGED_WAIT(bar_idx, parity, role)                                                                             \
  {                                                                                                                   \
    const bool ok_ = mbar_wait(bar_base + 8u * (bar_idx), (parity), abort_flag, a.status, ((bar_idx) << 8) | (role)); \
    if (!__all_sync(kFull, ok_)) goto role_done;                                                                      \
  }

// The element-wise warps meet at barriers of their own, so none of them may leave alone: a wait that runs out is recorded (the abort
// flag ends every later wait at once) and they go on, on whatever is there, to the end of the item, where they leave together.
#define PAGED_WAIT_ON(bar_idx, parity)                                                                                       \
  {                                                                                                                         \
    (void)mbar_wait(bar_base + 8u * (bar_idx), (parity), abort_flag, a.status, ((bar_idx) << 8) | ST_ROLE_ACT);              \
    __syncwarp();                                                                                                           \
  }

// A CTA of one of the kernels, as one of its warps sees it.
template <class L>
struct PagedCta {
  const PagedArgs& a;
  uint8_t* smem;
  uint32_t smem_base, bar_base;
  volatile int* abort_flag;
  int lane;
  uint32_t item_pos = 0;  // items this warp has taken or published

  __device__ __forceinline__ bool wait(int bar, uint32_t parity, int role) const {
    const bool ok = mbar_wait(bar_base + 8u * bar, parity, abort_flag, a.status, (bar << 8) | role);
    return __all_sync(kFull, ok);
  }
  __device__ __forceinline__ int4* slot() const { return reinterpret_cast<int4*>(smem + L::kRingOff + item_pos % kItemSlots * 64); }

  __device__ __forceinline__ PagedItem take_item(int role) {
    PagedItem it;
    it.h = -2;
    if (!wait(L::B_ITEM_FULL + item_pos % kItemSlots, (item_pos / kItemSlots) & 1u, role)) return it;
    const int4 x = slot()[0], y = slot()[1], z = slot()[2];
    const int b = slot()[3].x;
    it = PagedItem{warp_uniform(x.x), warp_uniform(x.y), warp_uniform(x.z), warp_uniform(x.w), warp_uniform(y.x), warp_uniform(y.y),
                   warp_uniform(y.z), warp_uniform(y.w), warp_uniform(z.x), warp_uniform(z.y), warp_uniform(z.z), warp_uniform(z.w), warp_uniform(b)};
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_base + 8u * (L::B_ITEM_EMPTY + item_pos % kItemSlots));
    ++item_pos;
    return it;
  }
  __device__ __forceinline__ bool publish(const PagedItem& it) {
    if (!wait(L::B_ITEM_EMPTY + item_pos % kItemSlots, ((item_pos / kItemSlots) & 1u) ^ 1u, ST_ROLE_LOAD)) return false;
    if (lane == 0) {
      slot()[0] = make_int4(it.h, it.q_start, it.past, it.row0);
      slot()[1] = make_int4(it.rows, it.len, it.lo, it.hi);
      slot()[2] = make_int4(it.tile0, it.tiles, it.pieces, it.first);
      slot()[3].x = it.b;
      mbar_arrive(bar_base + 8u * (L::B_ITEM_FULL + item_pos % kItemSlots));
    }
    ++item_pos;
    return true;
  }
};

// Where this CTA begins: every CTA sums the units of all requests (a run of them per thread) and looks for its own first one.  Called by
// all threads, with a barrier inside and one after it; `scan` is a scratch of a long long per warp.
template <class L, int NMAX>
__device__ __forceinline__ void find_start(const PagedArgs& a, long long* scan, PagedStart* start, int warp, int lane) {
  const int per = (a.batch + L::kThreads - 1) / L::kThreads;
  const int b0 = min(a.batch, static_cast<int>(threadIdx.x) * per), b1 = min(a.batch, b0 + per);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) sum += units_of<L, NMAX>(a, load_request(a, b)) * a.kv_heads;
  long long incl = sum;
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const long long o = __shfl_up_sync(kFull, incl, s);
    if (lane >= s) incl += o;
  }
  if (lane == 31) scan[warp] = incl;
  if (threadIdx.x == 0) *start = PagedStart{0, 0, a.batch};
  __syncthreads();
  long long all = 0, before = 0;
  for (int w = 0; w < L::kWarps; ++w) {
    before += w < warp ? scan[w] : 0;
    all += scan[w];
  }
  if (threadIdx.x == 0) start->all = all;
  const long long ctas = sharing_ctas(all);
  if (blockIdx.x < ctas) {
    const long long u0 = all * blockIdx.x / ctas;
    long long at = before + incl - sum;
    if (u0 >= at && u0 < at + sum) {
      for (int b = b0; b < b1; ++b) {
        const long long n = units_of<L, NMAX>(a, load_request(a, b)) * a.kv_heads;
        if (u0 < at + n) {
          start->before = at, start->b = b;
          break;
        }
        at += n;
      }
    }
  }
}

// The loader's role, by a whole warp: it walks the items of this CTA, publishes each before the tiles of the one before it are asked for, and
// asks for the tiles of their blocks, with the blocks' scales, and through `load_q(item)` for Q (which the kernel before this one
// makes: nothing of it is read before griddepcontrol.wait).
template <class L, int D, int NMAX, class F>
__device__ __forceinline__ void paged_load(PagedCta<L>& cta, const PagedStart* start, const CUtensorMap& tm_k, const CUtensorMap& tm_v, F load_q) {
  const PagedArgs& a = cta.a;
  const int lane = cta.lane;
  const uint32_t smem_base = cta.smem_base, bar_base = cta.bar_base;
  const long long all_units = start->all, ctas = sharing_ctas(all_units);
  uint32_t loaded = 0, loaded_v = 0;  // tiles asked for
  auto walk = [&]() -> bool {
    const int per_tile = kTile >> a.block_shift;  // blocks of a tile
    const int block_size = 1 << a.block_shift;
    uint32_t pos = 0;                             // tiles before this one
    const long long u0 = blockIdx.x < ctas ? all_units * blockIdx.x / ctas : 0, u1 = blockIdx.x < ctas ? all_units * (blockIdx.x + 1) / ctas : 0;
    // the walk: request, head and row tile that come next, units before them
    int wb = start->b - 1, wh = a.kv_heads, wt = 0, w_nt = 0, w_rows = 0;
    long long at = start->before;
    Request rq{0, 0, 0, 0};
    // the next item of which this CTA has tiles, published; h = -1 at the end
    auto next_item = [&](PagedItem& it) -> bool {
      it = PagedItem{};
      it.h = -1;
      while (at < u1) {
        if (wt >= w_nt) wt = 0, ++wh;
        if (wh >= a.kv_heads) {
          if (++wb >= a.batch) break;
          rq = load_request(a, wb);
          wh = 0;
          w_rows = rq.q_len * a.group;
          w_nt = (w_rows + NMAX - 1) / NMAX;
          if (w_nt == 0) {
            wh = a.kv_heads;
            continue;
          }
        }
        const int row0 = wt * NMAX, rows = min(NMAX, w_rows - row0);
        ++wt;
        const KeyRange r = keys_of_any(row0 / a.group, (row0 + rows - 1) / a.group, rq.past, rq.len, a.causal, a.window);
        const int n = tiles_of(r), n1 = max(1, n);
        const long long s = at + L::kItemUnits;  // where the tiles' units begin
        at = s + n1;
        // a tile belongs to the CTA that has its first unit
        auto tile_from = [&](long long u) { return static_cast<int>(min(max(u - s, 0ll), static_cast<long long>(n1))); };
        const int from = u0 <= s ? 0 : tile_from(u0), to = u1 <= s ? 0 : tile_from(u1);
        if (from >= to) continue;
        // the CTA that has unit u is the largest c with all * c / ctas <= u
        const int first = static_cast<int>(((s + 1) * ctas - 1) / all_units);
        const int pieces = static_cast<int>(((s + n1) * ctas - 1) / all_units) - first + 1;
        it = PagedItem{wh, rq.q_start, rq.past, row0, rows, rq.len, r.lo, r.hi, r.lo / kTile + from, n == 0 ? 0 : to - from, pieces, first, wb};
        break;
      }
      return cta.publish(it);
    };
    PagedItem it, ahead;
    if (!next_item(it)) return false;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (it.h >= 0 && it.tiles > 0 && !load_q(it)) return false;
    for (; it.h >= 0; it = ahead) {
      if (!next_item(ahead)) return false;
      const int n_blocks = min((it.len + block_size - 1) >> a.block_shift, a.table_width);
      const int* const table = a.block_tables + static_cast<long long>(it.b) * a.table_stride;
      int cached = 0, cached_at = -1;  // 32 entries of the table, from entry cached_at on
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages;
        const int p0 = (it.tile0 + j) * per_tile;
        if (cached_at < 0 || p0 + per_tile > cached_at + 32) {
          cached_at = p0;
          cached = cached_at + lane < n_blocks ? table[cached_at + lane] : -1;
        }
        const int blk = __shfl_sync(kFull, cached, (p0 - cached_at + lane) & 31);
        const bool valid = lane < per_tile && p0 + lane < n_blocks && blk >= 0 && blk < a.num_blocks;
        if (!cta.wait(L::B_KV_EMPTY + stage, ((pos / L::kStages) & 1u) ^ 1u, ST_ROLE_LOAD)) return false;
        const uint32_t bar = bar_base + 8u * (L::B_KV_FULL + stage);
        const unsigned n_valid = __popc(__ballot_sync(kFull, valid));
        if (lane == 0) mbar_arrive_expect_tx(bar, n_valid * block_size * D * (L::kOwnV ? 1 : 2));
        __syncwarp();
        const uint32_t dst = smem_base + L::kKvOff + stage * (L::kOwnV ? 1 : 2) * L::kTileBytes + lane * block_size * D;
        if (valid) {
          tma_load_4d(dst, &tm_k, bar, 0, 0, it.h, blk);
          if constexpr (!L::kOwnV) tma_load_4d(dst + L::kTileBytes, &tm_v, bar, 0, 0, it.h, blk);
        }
        // a block that is not there has a mark in the place of V's scale, which tells the others
        if (lane < per_tile) {
          const uint32_t sc = smem_base + L::kScaleOff + stage * 64 + lane * 4;
          const long long si = valid ? static_cast<long long>(blk) * a.kv_heads + it.h : 0;
          cp_async4(sc, a.k_scales + si, valid);
          cp_async4(sc + 32, valid ? static_cast<const void*>(a.v_scales + si) : &g_no_block, true);
        }
        cp_async_mbar_arrive(bar_base + 8u * (L::B_SC_FULL + stage));
        loaded = pos + 1;
        if constexpr (L::kOwnV) {  // V has places of its own
          const uint32_t v_stage = pos % L::kVStages;
          if (!cta.wait(L::B_V_EMPTY + v_stage, ((pos / L::kVStages) & 1u) ^ 1u, ST_ROLE_LOAD)) return false;
          const uint32_t v_bar = bar_base + 8u * (L::B_V_FULL + v_stage);
          if (lane == 0) mbar_arrive_expect_tx(v_bar, n_valid * block_size * D);
          __syncwarp();
          if (valid) tma_load_4d(smem_base + L::kVOff + v_stage * L::kTileBytes + lane * block_size * D, &tm_v, v_bar, 0, 0, it.h, blk);
          loaded_v = pos + 1;
        }
        // the next item's Q: its buffer is the last item's, which is done when this item's first stages have been used
        if (j == min(L::kStages, it.tiles - 1) && ahead.h >= 0 && ahead.tiles > 0 && !load_q(ahead)) return false;
      }
      if (it.tiles == 0 && ahead.h >= 0 && ahead.tiles > 0 && !load_q(ahead)) return false;
    }
    return true;
  };
  if (!walk()) {
    // after a wait that ran out: not before this CTA's own copies have landed (again with a limit)
    const uint64_t t0 = global_timer_ns();
    for (uint32_t k = loaded > L::kStages ? loaded - L::kStages : 0; k < loaded; ++k)
      while (!mbar_try_wait(bar_base + 8u * (L::B_KV_FULL + k % L::kStages), (k / L::kStages) & 1u) && global_timer_ns() - t0 < kWaitLimitNs) {
      }
    if constexpr (L::kOwnV)
      for (uint32_t k = loaded_v > L::kVStages ? loaded_v - L::kVStages : 0; k < loaded_v; ++k)
        while (!mbar_try_wait(bar_base + 8u * (L::B_V_FULL + k % L::kVStages), (k / L::kVStages) & 1u) && global_timer_ns() - t0 < kWaitLimitNs) {
        }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
}

// Joins the pieces of an item, by WARPS warps of the CTA that finished its piece last.  `row_at(r)`: where row r of O begins.
template <int D, int NMAX, bool SOFTMAX, int WARPS, class F>
__device__ __forceinline__ void paged_join(const PagedArgs& a, const PagedItem& it, int warp, int lane, F row_at) {
  // A warp has two rows: the weights of 32 pieces over its lanes, then the pieces in order.  What this takes is trips to L2: eight
  // pieces' values of both rows are asked for before the first is used, and with the pieces' statistics.
  constexpr int V = D / 32, kAhead = 8, kWarpsHere = WARPS;
  const auto slot_of = [&](int k) { return static_cast<long long>(2 * (it.first + k) + (k == 0 ? 1 : 0)); };
  for (int ra = warp; ra < it.rows; ra += 2 * kWarpsHere) {
    const int row[2] = {ra, min(ra + kWarpsHere, it.rows - 1)};
    float acc[2][V], m_all[2] = {kNoMax, kNoMax}, l_all[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < V; ++e) acc[0][e] = acc[1][e] = 0.f;
    if constexpr (SOFTMAX) {
      for (int k = lane; k < it.pieces; k += 32) {
#pragma unroll
        for (int x = 0; x < 2; ++x) m_all[x] = fmaxf(m_all[x], __ldcg(a.part_ml + slot_of(k) * 2 * NMAX + row[x]));
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) m_all[x] = warp_max(m_all[x]);
    }
    for (int k0 = 0; k0 < it.pieces; k0 += 32) {
      const int n = min(32, it.pieces - k0);
      float w[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        w[x] = lane < n ? 1.f : 0.f;
        if constexpr (SOFTMAX) {
          const float* const ml = a.part_ml + slot_of(k0 + min(lane, n - 1)) * 2 * NMAX + row[x];
          const float m = __ldcg(ml), l = __ldcg(ml + NMAX);
          const float half = ex2_approx(0.5f * (m - m_all[x]));  // twice: l is large where V's scales are small, and must not be lost before it is scaled
          w[x] *= half * half;
          if (lane < n) l_all[x] = fmaf(l * half, half, l_all[x]);
        }
      }
      for (int i0 = 0; i0 < n; i0 += kAhead) {
        float v[2][kAhead][V];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const float* const po = a.part_o + slot_of(k0 + min(i0 + i, n - 1)) * NMAX * D + lane * V;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if constexpr (V == 4) {
              const float4 u = __ldcg(reinterpret_cast<const float4*>(po + row[x] * D));
              v[x][i][0] = u.x, v[x][i][1] = u.y, v[x][i][2] = u.z, v[x][i][3] = u.w;
            } else {
              const float2 u = __ldcg(reinterpret_cast<const float2*>(po + row[x] * D));
              v[x][i][0] = u.x, v[x][i][1] = u.y;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (i0 + i < n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float wi = __shfl_sync(kFull, w[x], i0 + i);
#pragma unroll
              for (int e = 0; e < V; ++e) acc[x][e] = fmaf(wi, v[x][i][e], acc[x][e]);
            }
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float inv = 1.f;
      if constexpr (SOFTMAX) {
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) l_all[x] += __shfl_xor_sync(kFull, l_all[x], s);
        inv = l_all[x] > 0.f || l_all[x] != l_all[x] ? 1.f / l_all[x] : 0.f;
      }
      if (x == 0 || ra + kWarpsHere < it.rows) {
        uint32_t* const dst = reinterpret_cast<uint32_t*>(a.o + row_at(row[x]) + lane * V);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) dst[e] = pack_bf16x2(acc[x][2 * e] * inv, acc[x][2 * e + 1] * inv);
      }
    }
  }
}

// Launch of `kernel` that may begin while the kernel before it in the stream still runs (it waits for that one itself).
template <class... P, class... A>
int launch_after(void (*kernel)(P...), int grid, int threads, int smem, cudaStream_t stream, const A&... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  c.attrs = &early;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...) == cudaSuccess ? 0 : GDPA_ERR_LAUNCH_;
}

}  // namespace gdpa
