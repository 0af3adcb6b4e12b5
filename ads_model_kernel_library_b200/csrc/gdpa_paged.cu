// GDPA forward over a paged cache of 8-bit keys and values, for sm_100a:  O = act(Q K^T) * scale V  (or the softmax form) for the last
// queries of every request, K and V e4m3 with one fp32 scale per (block, head).
//
// This is the form for few queries (a step of generation: up to 64 rows), where the bytes of the cache bound it; many queries have the kernel
// of gdpa_paged_rows.cu.  It is transposed.  A tile is 128 cached tokens of one K / V head against N rows, the rows being the (query, head of
// the group) pairs that share this K / V head:
//     S^T [128 tokens x N] = K Q^T          tcgen05.mma kind::f8f6f4, A = the K tile as it lies in the cache
//     P^T = act(S^T) per token and row      a thread has one token: its scales are two registers, a mask is a compare
//     O^T [D x N] += V^T P^T                A = the V tile, MN-major, as it lies in the cache
// The cache bytes go from HBM through TMA into the tensor cores without a conversion, the 128-row side of the MMA is always full, and
// N is as small as the rows are few (16 or 64), where the untransposed form would compute 128 rows for one query.
//
// Both small operands have to be e4m3 as well, and one e4m3 value has four significant bits, none of them below 2^-9.  So Q is the sum of two:
// hi = e4m3(x), lo = e4m3(x - hi), both multiplied into the same accumulator.  For a bf16 Q (eight significant bits) scaled by a
// power of two per row the sum is exact (down to 2^-19 of the row's largest element).
//
// P is the sum of three, a = e4m3(x), b = e4m3(16 (x - a)), c = e4m3(32 (16 (x - a) - b)): each remainder is brought up to where the format has its
// bits (16 * 16 and 32 * 8 are the most that fit below 448), and has an accumulator of its own, O = A + B / 16 + C / 512: the parts are columns of
// one product, beside one another for each warpgroup.  That is float16's precision, and steps of 2^-18 where the row's largest is 64.  With hi and lo
// as for Q, what was 2^-16 of the largest P was zero and what is just above it off by a half, while the row's sum took it in full: a key 12 (nats) ahead of
// 4095 others, 0.97 of the weight, took 0.25 of the others' share away, one 13 ahead 0.55.  Two parts with their own accumulators would take 112 us
// where three take 116 (256 requests of up to 4096 tokens), but have steps of 2^-13, an eighth of what lies 12 below.  c only where a is subnormal,
// or multiplied only in tiles that have one: no faster.
//
// P^T is scaled per row so that its largest element (times V's block scale) lies at kTarget.  The scale, for the softmax the
// running maximum, is kept until a product would pass 448 (e4m3's largest): only then, and for the first tile, is the exact maximum
// taken and O rescaled, a vote of the warpgroup per tile and group of columns otherwise.  The exact value of a row's reference does
// not enter the result.
//
// Work: units are tiles, and four for an item's beginning and end; the units of all (request, K / V head, row tile) items in order are cut into equal stretches, one per CTA
// (persistent ones, as many as are resident), whatever the requests' lengths.  An item that is cut leaves partial sums in a workspace, and the
// CTA that finishes it last (an atomic count per item) joins them in the order of the pieces, so the result does not depend on who
// was last.  No CTA waits for another.
//
// Measured (one B200, us a pass of both kernels, calls back to back): 256 requests of up to 4096 tokens, a query each, 32 heads on 4: 117 (4.8 TB/s
// of cache); six of 32768 to 262144 tokens 81 (5.0 TB/s); one of 1500 tokens 14.3, a chain of trips to memory; up to four draft queries of 96 requests,
// head_dim 64, window 1024: 50, a chain of latencies per item.
//
// Roles: kGroups warpgroups (element-wise work, epilogue), one warp of TMA loads, one warp that issues MMAs.  A small kernel before this one
// splits Q and zeroes the items' counters; this one's beginning (barriers, tensor memory, the scan of the lengths) overlaps it.
#include <cuda_bf16.h>

#include <type_traits>

#include "gdpa_paged.cuh"

namespace gdpa {

namespace {

template <int D, int NMAX>
struct PagedShape {
  static constexpr int kCols = NMAX < 32 ? NMAX : 32;  // columns of a warpgroup
  static constexpr int kGroups = NMAX / kCols;         // warpgroups
  static constexpr int kCtasPerSm = NMAX > 16 ? 1 : D == 128 ? 2 : 3;
  static constexpr int kTileBytes = kTile * D;         // K or V tile
  static constexpr int kStages = NMAX <= 16 ? 3 : D == 128 ? 5 : 10;
  static constexpr int kQBytes = NMAX * D;             // hi, then lo
  static constexpr int kPBytes = NMAX * kTile;
  static constexpr int kWarps = 4 * kGroups + 2;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kLoadWarp = 4 * kGroups, kMmaWarp = kLoadWarp + 1;
  static constexpr int kTmemCols = NMAX <= 16 ? 128 : 512;  // S0, S1 of NMAX columns each, O: [warpgroup][part]
  static constexpr bool kOwnV = false;  // a stage has K and V
  static constexpr int kItemUnits = 4;                 // beginning and end, in tiles; 2 to 8: the same within 3 %, 4 the best by a little
  static constexpr float kTarget = 64.f;

  static constexpr int kKvOff = 0;                                  // [stage]{K, V}
  static constexpr int kQOff = kKvOff + kStages * 2 * kTileBytes;   // [2]{hi, lo}
  static constexpr int kPOff = kQOff + 2 * 2 * kQBytes;             // [warpgroup][part of P]
  static constexpr int kScaleOff = kPOff + 3 * kPBytes;             // float[stage][16]: K scales of up to 8 blocks, V scales
  static constexpr int kQaOff = kScaleOff + kStages * 64;           // float[2][NMAX]: factor of a row's scores
  static constexpr int kRefOff = kQaOff + 2 * NMAX * 4;             // float[NMAX]: minus the running maximum / multiplier of a row
  static constexpr int kFacOff = kRefOff + NMAX * 4;                // float[NMAX]
  static constexpr int kRedOff = kFacOff + NMAX * 4;                // float[4][NMAX]
  static constexpr int kRangeOff = kRedOff + 4 * NMAX * 4;          // int2[NMAX]: keys a row takes part with
  static constexpr int kRowOff = kRangeOff + NMAX * 8;              // long long[NMAX]: where a row of O begins
  static constexpr int kRingOff = kRowOff + NMAX * 8;               // int[kItemSlots][16]
  static constexpr int kBarOff = kRingOff + kItemSlots * 64;
  enum : int {
    B_KV_FULL = 0,
    B_KV_EMPTY = B_KV_FULL + kStages,
    B_SC_FULL = B_KV_EMPTY + kStages,
    B_S_FULL = B_SC_FULL + kStages,   // [2]
    B_P_FULL = B_S_FULL + 2,
    B_PV_DONE = B_P_FULL + 1,
    B_Q_FULL = B_PV_DONE + 1,         // [2]
    B_Q_EMPTY = B_Q_FULL + 2,         // [2]
    B_ITEM_FULL = B_Q_EMPTY + 2,      // [kItemSlots]
    B_ITEM_EMPTY = B_ITEM_FULL + kItemSlots,
    B_COUNT = B_ITEM_EMPTY + kItemSlots
  };
  static constexpr int kMiscOff = kBarOff + B_COUNT * 8;  // tmem address, abort flag, last-arrival flag, nan_item; then the scan's scratch
  static constexpr int kScanOff = kMiscOff + 16;          // long long[32] + start state
  static constexpr int kBytes = kScanOff + 32 * 8 + 48;
  static constexpr int kDynBytes = kBytes + 1024;
  static_assert(kCtasPerSm * (kDynBytes + 1024) <= 228 * 1024, "shared memory");
};

// The N columns' values over the warp's 32 lanes, reduced: lane i gets column i % N's result.  Halves change places (N - 1 shuffles).
template <int N, class F>
__device__ __forceinline__ float reduce_columns(float (&v)[N], int lane, F op) {
#pragma unroll
  for (int w = N / 2; w > 0; w >>= 1) {
    const bool upper = lane & w;
#pragma unroll
    for (int i = 0; i < w; ++i) {
      const float mine = upper ? v[i + w] : v[i], other = upper ? v[i] : v[i + w];
      v[i] = op(mine, __shfl_xor_sync(kFull, other, w));
    }
  }
  float r = v[0];
#pragma unroll
  for (int w = N; w < 32; w <<= 1) r = op(r, __shfl_xor_sync(kFull, r, w));
  return r;
}

template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_ld32(taddr, r);
  else tmem_ld16(taddr, r);
}
template <int N>
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[N]) {
  if constexpr (N == 32) tmem_st32(taddr, r);
  else tmem_st16(taddr, r);
}

template <int D, int NMAX, bool SOFTMAX>
__global__ void __launch_bounds__(PagedShape<D, NMAX>::kThreads, PagedShape<D, NMAX>::kCtasPerSm)
gdpa_paged_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                  const __grid_constant__ PagedArgs a) {
  using L = PagedShape<D, NMAX>;
  constexpr int kGroups = L::kGroups;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_base + L::kBarOff;
  volatile uint32_t* const tmem_ptr = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOff);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  volatile int* const last_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 8);
  volatile uint32_t* const nan_item = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOff + 12);  // the last item that had NaNs taken out of V, from 1
  const int warp = warp_uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::B_COUNT; ++i) {
      uint32_t n = 1;
      if (i >= L::B_SC_FULL && i < L::B_SC_FULL + L::kStages) n = 32;
      if (i == L::B_P_FULL) n = 128 * kGroups;
      if (i >= L::B_Q_FULL && i < L::B_Q_FULL + 2) n = 33;
      if (i >= L::B_Q_EMPTY && i < L::B_Q_EMPTY + 2) n = 1 + 4 * kGroups;
      if (i >= L::B_ITEM_EMPTY && i < L::B_ITEM_EMPTY + kItemSlots) n = 1 + 4 * kGroups;
      mbar_init(bar_base + 8u * i, n);
    }
    *abort_flag = 0;
    *nan_item = 0;
    mbar_fence_init();
  }
  if (warp == L::kMmaWarp) {
    tmem_alloc(smem_base + L::kMiscOff, L::kTmemCols);
    tmem_relinquish();
  }
  if (warp == L::kLoadWarp && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  PagedStart* const start = reinterpret_cast<PagedStart*>(smem + L::kScanOff + 32 * 8);
  find_start<L, NMAX>(a, reinterpret_cast<long long*>(smem + L::kScanOff), start, warp, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_ptr);
  PagedCta<L> cta{a, smem, smem_base, bar_base, abort_flag, lane};

  if (warp == L::kLoadWarp) {
    // ------------------------------------------------------------------ TMA loader, and the walk over the items
    // Q of an item (both halves of its values, all NMAX rows: those past the item's are another request's, or zeros) and its rows'
    // factors.
    uint32_t q_pos = 0;
    auto load_q = [&](const PagedItem& i) -> bool {
      const uint32_t buf = q_pos & 1u;
      if (!cta.wait(L::B_Q_EMPTY + buf, ((q_pos >> 1) & 1u) ^ 1u, ST_ROLE_LOAD)) return false;
      ++q_pos;
      const long long row = static_cast<long long>(i.q_start) * a.group + i.row0;
      const uint32_t bar = bar_base + 8u * (L::B_Q_FULL + buf), dst = smem_base + L::kQOff + buf * 2 * L::kQBytes;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, 2 * L::kQBytes);
        tma_load_3d(dst, &tm_q, bar, 0, static_cast<int>(row), i.h);
        tma_load_3d(dst + L::kQBytes, &tm_q, bar, 0, static_cast<int>(row), a.kv_heads + i.h);
      }
      for (int r = lane; r < NMAX; r += 32)
        cp_async4(smem_base + L::kQaOff + (buf * NMAX + r) * 4, a.qa + i.h * a.total_q * a.group + row + min(r, i.rows - 1), true);
      cp_async_mbar_arrive(bar);
      return true;
    };
    paged_load<L, D, NMAX>(cta, start, tm_k, tm_v, load_q);
  } else if (warp == L::kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr int kSwizzle = D == 128 ? 128 : 64;
    // K: rows of D bytes, K-major, eight rows after eight rows; V: the same bytes, MN-major (with 64 columns the second half of the
    // MMA's 128 rows repeats the first: its lanes of O are not read).
    const uint64_t dk0 = umma_smem_desc(smem_base + L::kKvOff, 16, 8 * D, kSwizzle);
    const uint64_t dv0 = umma_smem_desc(smem_base + L::kKvOff + L::kTileBytes, 0, 8 * D, kSwizzle);
    const uint64_t dq0 = umma_smem_desc(smem_base + L::kQOff, 16, 8 * D, kSwizzle);
    const uint64_t dp0 = umma_smem_desc(smem_base + L::kPOff, 128, 16 * kTile, 0);
    uint32_t pos = 0, q_pos = 0, pv_pos = 0;
    struct {
      int n16;
      uint32_t stage;
      bool accumulate, any;
    } owed{0, 0, false, false};  // the tile whose P V has not been issued
    auto issue_pv = [&]() -> bool {
      const bool ok = mbar_wait(bar_base + 8u * L::B_P_FULL, pv_pos & 1u, abort_flag, a.status, (L::B_P_FULL << 8) | ST_ROLE_MMA);
      if (!__all_sync(kFull, ok)) return false;
      ++pv_pos;
      tc_fence_after();
      const uint32_t idesc = umma_idesc(0, 0, 1, 1, kTile, 3 * 16 * owed.n16);
      const uint64_t dv = umma_desc_advance(dv0, owed.stage * 2 * L::kTileBytes);
#pragma unroll
      for (int kk = 0; kk < kTile / 32; ++kk)
        umma_ss_f8(tmem_base + 2 * NMAX, umma_desc_advance(dv, kk * 32 * D), umma_desc_advance(dp0, kk * 512), idesc, owed.accumulate || kk > 0 ? 1u : 0u);
      tc_commit(bar_base + 8u * (L::B_KV_EMPTY + owed.stage));
      tc_commit(bar_base + 8u * L::B_PV_DONE);
      owed.any = false;
      return true;
    };
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_MMA);
      if (it.h < 0) {
        if (it.h == -2) goto role_done;
        break;
      }
      if (it.tiles == 0) {
        // nothing of it is multiplied, but the element-wise warps take no further item before they have what is owed: a few items without keys in
        // a row fill the ring, and the next item with keys would never come
        if (owed.any && !issue_pv()) goto role_done;
        continue;
      }
      const int n16 = (it.rows + L::kCols - 1) / L::kCols * (L::kCols / 16);  // whole warpgroups' columns
      const uint32_t q_buf = q_pos & 1u;
      PAGED_WAIT(L::B_Q_FULL + q_buf, (q_pos >> 1) & 1u, ST_ROLE_MMA);
      ++q_pos;
      const uint32_t idesc = umma_idesc(0, 0, 0, 0, kTile, 16 * n16);
      const uint64_t dq = umma_desc_advance(dq0, q_buf * 2 * L::kQBytes);
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages;
        PAGED_WAIT(L::B_KV_FULL + stage, (pos / L::kStages) & 1u, ST_ROLE_MMA);
        tc_fence_after();
        const uint64_t dk = umma_desc_advance(dk0, stage * 2 * L::kTileBytes);
        const uint32_t s_tmem = tmem_base + (pos & 1u) * NMAX;
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk) {
          umma_ss_f8(s_tmem, umma_desc_advance(dk, kk * 32), umma_desc_advance(dq, kk * 32), idesc, kk > 0 ? 1u : 0u);
          umma_ss_f8(s_tmem, umma_desc_advance(dk, kk * 32), umma_desc_advance(dq, L::kQBytes + kk * 32), idesc, 1u);
        }
        tc_commit(bar_base + 8u * (L::B_S_FULL + (pos & 1u)));
        if (j + 1 == it.tiles) tc_commit(bar_base + 8u * (L::B_Q_EMPTY + q_buf));
        if (owed.any && !issue_pv()) goto role_done;
        owed = {n16, stage, j > 0, true};
      }
    }
    if (owed.any && !issue_pv()) goto role_done;
  } else {
    // ------------------------------------------------------------------ element-wise work and epilogue
    // Warpgroup wg has columns [wg * kCols, (wg + 1) * kCols) of the 128 tokens, a thread one token.
    constexpr int C = L::kCols;
    constexpr float kHeadroom = 2.8073549f + 0.001f;  // log2(448 / kTarget)
    static_assert(L::kTarget == 64.f, "kHeadroom");
    const int wg = warp >> 2, tid = threadIdx.x & 127, quarter = warp & 3, c0 = wg * C;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t o_tmem = tmem_base + 2 * NMAX + lane_base + 3 * c0;
    float* const ref = reinterpret_cast<float*>(smem + L::kRefOff) + c0;
    float* const fac = reinterpret_cast<float*>(smem + L::kFacOff) + c0;
    float* const red = reinterpret_cast<float*>(smem + L::kRedOff) + c0;  // [quarter * NMAX + column]
    int2* const range = reinterpret_cast<int2*>(smem + L::kRangeOff) + c0;
    long long* const row_at = reinterpret_cast<long long*>(smem + L::kRowOff) + c0;
    const int bar_wg = 4 + wg;
    uint32_t pos = 0, q_pos = 0;  // tiles, items with tiles
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_ACT);
      if (named_bar_or(3, 128 * kGroups, it.h < 0)) break;
      const int rows = min(C, it.rows - c0);  // of this warpgroup; none or fewer: it only keeps step
      if (tid < C) {
        const int g = it.row0 + c0 + tid, i = g / a.group;
        row_at[tid] = ((it.q_start + static_cast<long long>(i)) * a.heads + it.h * a.group + (g - i * a.group)) * D;
        const KeyRange r = tid < rows ? keys_of(i, it.past, it.len, a.causal, a.window) : KeyRange{0, 0};
        range[tid] = make_int2(r.lo, r.hi);
        ref[tid] = SOFTMAX ? -kNoMax : 1.f;
      }
      named_bar_sync(bar_wg, 128);
      if (it.tiles == 0) {
        // no row of the tile has a key
        for (int i = tid; i < rows * (D / 2); i += 128) reinterpret_cast<uint32_t*>(a.o + row_at[i / (D / 2)])[i % (D / 2)] = 0u;
        named_bar_sync(bar_wg, 128);
        continue;
      }
      const uint32_t q_buf = q_pos & 1u;
      const float* const qa = reinterpret_cast<const float*>(smem + L::kQaOff) + q_buf * NMAX + c0;
      uint64_t l[C / 2];  // row sums of this token's P, in pairs of columns
#pragma unroll
      for (int i = 0; i < C / 2; ++i) l[i] = 0ull;
      const int i0 = it.row0 / a.group, i1 = (it.row0 + it.rows - 1) / a.group;
      const KeyRange r0 = keys_of(i0, it.past, it.len, a.causal, a.window), r1 = keys_of(i1, it.past, it.len, a.causal, a.window);
      const int all_lo = max(r0.lo, r1.lo), all_hi = min(r0.hi, r1.hi);  // keys that every row takes part with (if any)
      PAGED_WAIT_ON(L::B_Q_FULL + q_buf, (q_pos >> 1) & 1u);
      ++q_pos;
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages, phase = (pos / L::kStages) & 1u;
        const int key0 = (it.tile0 + j) * kTile, key = key0 + tid;
        const bool first = j == 0;
        PAGED_WAIT_ON(L::B_SC_FULL + stage, phase);
        const float* const sc = reinterpret_cast<const float*>(smem + L::kScaleOff) + stage * 16 + (tid >> a.block_shift);
        const float ks = sc[0];
        float vs = sc[8];
        const bool out = key < it.lo || key >= it.hi || no_block(vs);  // no row takes part with this token
        bool poisoned = !out && !(vs <= 3.4028235e38f);                // a scale that is no number makes NaN of all rows that do
        if (out || poisoned) vs = 0.f;
        const bool every = key0 >= all_lo && key0 + kTile <= all_hi;  // the tile needs no mask but that of `out`
        const bool masked = !every || __any_sync(kFull, out || poisoned);
        PAGED_WAIT_ON(L::B_S_FULL + (pos & 1u), (pos >> 1) & 1u);
        tc_fence_after();
        if (masked && wg == 0) {
          // P of a token that takes no part is 0, and 0 times what its V row holds (an unused row, NaN) has to be 0
          PAGED_WAIT_ON(L::B_KV_FULL + stage, phase);
          uint4* const v_row = reinterpret_cast<uint4*>(smem + L::kKvOff + (2 * stage + 1) * L::kTileBytes + tid * D);
          if (out || poisoned) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) v_row[i] = make_uint4(0, 0, 0, 0);
          } else if (!every) {
            // some row may take part and some not: a NaN is put into the columns of those that do at the stretch's end
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              uint4 u = v_row[i];
              if (drop_nans(u)) v_row[i] = u, *nan_item = q_pos;
            }
          }
        }
        if (rows > 0) {
          const uint32_t s_tmem = tmem_base + (pos & 1u) * NMAX + lane_base + c0;
          const float m = SOFTMAX ? vs * L::kTarget : vs;
          float p[C];
          // the scores, times the row's and the block's factors (for the softmax less the row's reference)
          auto scores = [&](bool relative) {
            uint32_t raw[C];
            tmem_ld_cols(s_tmem, raw);
            tmem_wait_ld();
            tmem_regs_ready(raw);
            const uint64_t k2 = pack_f32x2(ks, ks);
#pragma unroll
            for (int i = 0; i < C; i += 4) {
              const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(qa + i);
              ulonglong2 r = make_ulonglong2(0, 0);
              if (relative) r = *reinterpret_cast<const ulonglong2*>(ref + i);
              uint64_t x0 = mul_f32x2(pack_f32x2(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1])), k2);
              uint64_t x1 = mul_f32x2(pack_f32x2(__uint_as_float(raw[i + 2]), __uint_as_float(raw[i + 3])), k2);
              x0 = relative ? fma_f32x2(x0, f.x, r.x) : mul_f32x2(x0, f.x);
              x1 = relative ? fma_f32x2(x1, f.y, r.y) : mul_f32x2(x1, f.y);
              unpack_f32x2(x0, p[i], p[i + 1]);
              unpack_f32x2(x1, p[i + 2], p[i + 3]);
            }
          };
          // P for the reference the rows have now; whether it fits e4m3
          auto compute = [&]() -> bool {
            scores(SOFTMAX);
            if constexpr (SOFTMAX) {
#pragma unroll
              for (int i = 0; i < C; ++i) p[i] = ex2_approx(p[i]);
            } else {
              act_any(a.act, p, a.scale);
#pragma unroll
              for (int i = 0; i < C; i += 4) {
                const float4 r = *reinterpret_cast<const float4*>(ref + i);
                p[i] *= r.x, p[i + 1] *= r.y, p[i + 2] *= r.z, p[i + 3] *= r.w;
              }
            }
            if (masked) {
#pragma unroll
              for (int i = 0; i < C; ++i) {
                const int2 rg = range[i];
                const bool in = !out && key >= rg.x && key < rg.y;
                p[i] = in ? (poisoned ? __uint_as_float(0x7fffffffu) : p[i]) : 0.f;
              }
            }
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < C; i += 2) most = SOFTMAX ? max3(most, p[i], p[i + 1]) : max3(most, fabsf(p[i]), fabsf(p[i + 1]));
            return most * m <= kMax8;
          };
          // With head_dim 64 the code of compute is there once, with 128 twice: three CTAs an SM are short of instructions, two wait for the
          // cache (draft_window 49.5 us and 52, decode_ragged 118 and 114.5).
#pragma unroll 1
          for (bool moved = false, next = !first;; next = moved = true) {
            if (next) {
              const bool fits = compute();
              if (moved || !named_bar_or(bar_wg, 128, !fits)) break;
            }
            // the exact reference of every column, and O and the row sums moved to it
            scores(false);
            if constexpr (SOFTMAX) {
              const float lv = log2f(fmaxf(vs, kLeastScale));
#pragma unroll
              for (int i = 0; i < C; ++i) p[i] += lv;
            } else {
              act_any(a.act, p, a.scale);
#pragma unroll
              for (int i = 0; i < C; ++i) p[i] = fabsf(p[i]) * vs;
            }
            if (masked) {
#pragma unroll
              for (int i = 0; i < C; ++i) {
                const int2 rg = range[i];
                p[i] = !out && key >= rg.x && key < rg.y ? p[i] : (SOFTMAX ? kNoMax : 0.f);
              }
            }
            const float most = reduce_columns<C>(p, lane, [](float x, float y) { return fmaxf(x, y); });
            if (lane < C) red[quarter * NMAX + lane] = most;
            if (!first) {
              PAGED_WAIT_ON(L::B_PV_DONE, (pos - 1) & 1u);  // O holds every tile before this one
              tc_fence_after();
            }
            named_bar_sync(bar_wg, 128);
            if (tid < C) {
              const float now = fmaxf(fmaxf(red[tid], red[NMAX + tid]), fmaxf(red[2 * NMAX + tid], red[3 * NMAX + tid]));
              // a column that fits keeps its reference: no row's bits depend on another row's values (the margin keeps the two ways
              // to say that one does not fit from differing)
              if constexpr (SOFTMAX) {
                const float old = -ref[tid];
                const float next = first || now - old > kHeadroom ? fmaxf(old, fminf(now, 3.0e38f)) : old;
                fac[tid] = first ? 0.f : ex2_approx(0.5f * (old - next));  // its root, taken twice: a row's sum is large where V's scales were small
                ref[tid] = -next;
              } else {
                // the largest power of two that keeps |P| times V's scale at or below the target; 2^100 for a row of zeros
                const float old = ref[tid];
                float next = 1.2676506e30f;
                if (now > 0.f) next = exp2f(fminf(fmaxf(floorf(log2f(L::kTarget / now)), -100.f), 100.f));
                if (!first) next = now * old > kMax8 * 1.001f ? fminf(next, old) : old;
                fac[tid] = first ? 0.f : next / old;
                ref[tid] = next;
              }
            }
            named_bar_sync(bar_wg, 128);
            if (!first) {
              if constexpr (SOFTMAX) {
#pragma unroll
                for (int i = 0; i < C; i += 2) {
                  const uint64_t f = pack_f32x2(fac[i], fac[i + 1]);
                  l[i / 2] = mul_f32x2(mul_f32x2(l[i / 2], f), f);
                }
              }
#pragma unroll 1
              for (int part = 0; part < 3; ++part) {
                uint32_t raw[C];
                tmem_ld_cols(o_tmem + part * C, raw);
                tmem_wait_ld();
                tmem_regs_ready(raw);
#pragma unroll
                for (int i = 0; i < C; i += 2) {
                  float2 f = *reinterpret_cast<const float2*>(fac + i);
                  if constexpr (SOFTMAX) f = make_float2(f.x * f.x, f.y * f.y);
                  raw[i] = __float_as_uint(__uint_as_float(raw[i]) * f.x);
                  raw[i + 1] = __float_as_uint(__uint_as_float(raw[i + 1]) * f.y);
                }
                tmem_st_cols(o_tmem + part * C, raw);
              }
              tmem_wait_st();
            }
            if constexpr (D == 128) {
              compute();
              break;
            }
          }
          // P, times V's scale, as the sum of three e4m3 values (see the top of this file)
          uint32_t w[3][C / 4], h[C / 2];
          const uint64_t m2 = pack_f32x2(m, m);
#pragma unroll
          for (int i = 0; i < C / 2; ++i) {
            const uint64_t x = pack_f32x2(p[2 * i], p[2 * i + 1]);
            if constexpr (SOFTMAX) l[i] = add_f32x2(l[i], x);
            float y0, y1;
            unpack_f32x2(mul_f32x2(x, m2), y0, y1);
            h[i] = pack_f16x2(y0, y1);
          }
#pragma unroll
          for (int part = 0; part < 3; ++part) {
            const uint32_t up = part == 0 ? 0x4c004c00u : 0x50005000u, down = up | 0x80008000u;  // 16, 32; exact, and so is what is left
#pragma unroll
            for (int i = 0; i < C / 4; ++i) {
              const uint16_t e0 = e4m3x2_from_f16x2(h[2 * i]), e1 = e4m3x2_from_f16x2(h[2 * i + 1]);
              w[part][i] = static_cast<uint32_t>(e0) | (static_cast<uint32_t>(e1) << 16);
              if (part < 2) {
                h[2 * i] = fma_f16x2(f16x2_from_e4m3x2(e0), down, mul_f16x2(h[2 * i], up));
                h[2 * i + 1] = fma_f16x2(f16x2_from_e4m3x2(e1), down, mul_f16x2(h[2 * i + 1], up));
              }
            }
          }
          if (pos > 0) PAGED_WAIT_ON(L::B_PV_DONE, (pos - 1) & 1u);  // P's buffer is free
          uint8_t* const dst = smem + L::kPOff + 3 * c0 * kTile + tid * 16;
#pragma unroll
          for (int c = 0; c < C / 16; ++c) {
#pragma unroll
            for (int part = 0; part < 3; ++part)
              *reinterpret_cast<uint4*>(dst + (part * C + c * 16) * kTile) =
                  make_uint4(w[part][4 * c], w[part][4 * c + 1], w[part][4 * c + 2], w[part][4 * c + 3]);
          }
        } else if (pos > 0) {
          // a warpgroup without columns waits too: its arrival for the next tile must not count for this one
          PAGED_WAIT_ON(L::B_PV_DONE, (pos - 1) & 1u);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(bar_base + 8u * L::B_P_FULL);
      }
      // ---- the end of the stretch: row sums over the 128 tokens' threads, then O
      if (lane == 0) mbar_arrive(bar_base + 8u * (L::B_Q_EMPTY + q_buf));
      if constexpr (SOFTMAX) {
        float sums[C];
#pragma unroll
        for (int i = 0; i < C / 2; ++i) unpack_f32x2(l[i], sums[2 * i], sums[2 * i + 1]);
        const float sum = reduce_columns<C>(sums, lane, [](float x, float y) { return x + y; });
        if (lane < C) red[quarter * NMAX + lane] = sum;
      }
      PAGED_WAIT_ON(L::B_PV_DONE, (pos - 1) & 1u);
      tc_fence_after();
      named_bar_sync(bar_wg, 128);
      const bool cut = it.pieces > 1;
      const int part = 2 * blockIdx.x + (static_cast<int>(blockIdx.x) == it.first ? 1 : 0);
      if (tid < rows) {
        const float sum = SOFTMAX ? red[tid] + red[NMAX + tid] + red[2 * NMAX + tid] + red[3 * NMAX + tid] : 1.f;
        if (cut) {
          float* const ml = a.part_ml + static_cast<long long>(part) * 2 * NMAX + c0;
          ml[tid] = -ref[tid];
          ml[NMAX + tid] = sum;
          fac[tid] = SOFTMAX ? 1.f / L::kTarget : 1.f / ref[tid];
        } else {
          fac[tid] = SOFTMAX ? (sum > 0.f || sum != sum ? 1.f / (sum * L::kTarget) : 0.f) : 1.f / ref[tid];
        }
      }
      named_bar_sync(bar_wg, 128);
      if (rows > 0) {
        uint32_t raw[3][C];
#pragma unroll
        for (int part = 0; part < 3; ++part) tmem_ld_cols(o_tmem + part * C, raw[part]);
        tmem_wait_ld();
#pragma unroll
        for (int part = 0; part < 3; ++part) tmem_regs_ready(raw[part]);
        if (tid < D) {
          float* const po = a.part_o + (static_cast<long long>(part) * NMAX + c0) * D + tid;
#pragma unroll
          for (int i = 0; i < C; ++i) {
            if (i < rows) {
              const float v = fmaf(fmaf(__uint_as_float(raw[2][i]), 1.f / 32.f, __uint_as_float(raw[1][i])), 1.f / 16.f, __uint_as_float(raw[0][i])) * fac[i];
              if (cut) po[i * D] = v;
              else a.o[row_at[i] + tid] = __float2bfloat16_rn(v);
            }
          }
          if (*nan_item == q_pos) {
            for (int i = 0; i < rows; ++i) {
              if (((nan_columns(a, it.b, it.h, it.tile0, it.tiles, range[i].x, range[i].y, all_lo, all_hi, tid & ~31) >> (tid & 31)) & 1u) == 0u) continue;
              if (cut) po[i * D] = __uint_as_float(0x7fffffffu);
              else a.o[row_at[i] + tid] = __ushort_as_bfloat16(0x7fffu);
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      if (!cut) {
        named_bar_sync(bar_wg, 128);  // the next item writes over fac and row_at
      } else {
        // the last of the item's CTAs joins the pieces
        named_bar_sync(3, 128 * kGroups);
        if (threadIdx.x == 0) *last_flag = count_arrival(a.counters + it.first) == it.pieces - 1;
        named_bar_sync(3, 128 * kGroups);
        if (*last_flag) {
          paged_join<D, NMAX, SOFTMAX, 4 * kGroups>(a, it, warp, lane, [&](int r) { return reinterpret_cast<const long long*>(smem + L::kRowOff)[r]; });
        }
        named_bar_sync(3, 128 * kGroups);
      }
    }
  }
role_done:
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == L::kMmaWarp) tmem_dealloc(tmem_base, L::kTmemCols);
}

// Q in the form the tensor cores take it, for the kernel after this one: rows of one K / V head one after the other (query, head of the
// group), each scaled by a power of two to a largest element in (224, 448] and split in two e4m3 values, hi first, all rows' lo behind; their
// factors; and the item counters, zeroed.  A row that is not finite becomes zeros with a factor of NaN.
template <int D>
__global__ void __launch_bounds__(256) gdpa_paged_prepare_kernel(const PagedArgs a, uint8_t* q8, int ctas) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // that kernel waits before it reads any of this
  constexpr int kLanes = D / 8;  // lanes of one row, 16 bytes each
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < ctas; i += 256) a.counters[i] = 0;
  const long long n = a.total_q * a.heads, rows = a.total_q * a.group;  // of one K / V head
  const int c8 = threadIdx.x % kLanes;
  const long long row0 = static_cast<long long>(blockIdx.x) * (256 / kLanes) + threadIdx.x / kLanes;
  for (long long i = row0; i - threadIdx.x / kLanes < n; i += static_cast<long long>(gridDim.x) * (256 / kLanes)) {
    const long long t = min(i, n - 1) / a.heads;
    const int hd = static_cast<int>(min(i, n - 1) - t * a.heads), h = hd / a.group;
    const uint4 u = *reinterpret_cast<const uint4*>(a.q + t * a.q_strides[0] + hd * a.q_strides[1] + c8 * 8);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max_u16x2(top, w[e] & 0x7fff7fffu);
    top = max(top & 0xffffu, top >> 16);
#pragma unroll
    for (int s = kLanes / 2; s > 0; s >>= 1) top = max(top, __shfl_xor_sync(kFull, top, s));
    const bool finite = top < 0x7f80u;
    const int k = max(static_cast<int>(top >> 7) - 127 - 8 + ((top & 0x7fu) > 0x60u ? 1 : 0), -100);
    const float inv = __uint_as_float(static_cast<uint32_t>(127 - k) << 23);
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint16_t eh[2], el[2];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const uint32_t v = finite ? w[2 * e + f] : 0u;
        const uint32_t x = pack_f16x2(__uint_as_float(v << 16) * inv, __uint_as_float(v & 0xffff0000u) * inv);  // exact but for what lies 2^-24 below
        eh[f] = e4m3x2_from_f16x2(x);
        el[f] = e4m3x2_from_f16x2(sub_f16x2(x, f16x2_from_e4m3x2(eh[f])));
      }
      hi[e] = __byte_perm(eh[0], eh[1], 0x5410);
      lo[e] = __byte_perm(el[0], el[1], 0x5410);
    }
    if (i < n) {
      const long long r = h * rows + t * a.group + (hd - h * a.group);
      *reinterpret_cast<uint2*>(q8 + r * D + c8 * 8) = make_uint2(hi[0], hi[1]);
      *reinterpret_cast<uint2*>(q8 + (a.kv_heads * rows + r) * D + c8 * 8) = make_uint2(lo[0], lo[1]);
      const float s = __uint_as_float(static_cast<uint32_t>(k + 127) << 23) * (a.act == ACT_SOFTMAX ? a.scale * 1.4426950408889634f : 1.f);
      if (c8 == 0) a.qa[r] = finite ? s : __uint_as_float(0x7fffffffu);
    }
  }
}

template <int D, int NMAX>
int launch(const PagedLaunch& l) {
  using L = PagedShape<D, NMAX>;
  auto go = [&](auto kernel) -> int {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynBytes) != cudaSuccess) return GDPA_ERR_LAUNCH_;
    return launch_after(kernel, l.grid, L::kThreads, L::kDynBytes, l.stream, l.tm_q, l.tm_k, l.tm_v, l.args);
  };
  return l.args.act == ACT_SOFTMAX ? go(gdpa_paged_kernel<D, NMAX, true>) : go(gdpa_paged_kernel<D, NMAX, false>);
}

}  // namespace

int paged_ctas_per_sm(int rows, int head_dim) {
  return rows > 16 ? 1 : head_dim == 128 ? PagedShape<128, 16>::kCtasPerSm : PagedShape<64, 16>::kCtasPerSm;
}

int launch_paged(const PagedLaunch& l, int head_dim) {
  const long long blocks = (l.args.total_q * l.args.heads * (head_dim / 8) + 255) / 256;
  const int grid = static_cast<int>(blocks < 4096 ? blocks : 4096);
  if (head_dim == 128) gdpa_paged_prepare_kernel<128><<<grid, 256, 0, l.stream>>>(l.args, l.q8, l.grid);
  else gdpa_paged_prepare_kernel<64><<<grid, 256, 0, l.stream>>>(l.args, l.q8, l.grid);
  if (cudaGetLastError() != cudaSuccess) return GDPA_ERR_LAUNCH_;
  auto go = [&](auto dim) -> int {
    constexpr int D = decltype(dim)::value;
    return l.rows == 16 ? launch<D, 16>(l) : launch<D, 64>(l);
  };
  if (l.rows > 64) return launch_paged_rows(l, head_dim);
  return head_dim == 128 ? go(std::integral_constant<int, 128>{}) : go(std::integral_constant<int, 64>{});
}

}  // namespace gdpa
