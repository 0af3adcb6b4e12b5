// The attention over a paged 8-bit cache (gdpa_paged.cu) for many queries: candidates of a request, chunks of a prompt.  The form is the
// ordinary one, a row of scores to a thread:
//     S [128 rows x 64 tokens] = Q K^T       kind::f8f6f4, A = Q (two e4m3 planes in shared memory), B = the K tile as it lies in the cache
//     P = act(S) in registers, float16       a thread has a row: its maximum, sum and reference are its own, nothing is exchanged
//     O [128 rows x D] += P V                kind::f16, A = P in tensor memory over its own S, B = V in float16, MN-major
// A work item is 256 rows (two row tiles) of one (request, K / V head), a KV tile 128 tokens, taken in two halves: while a row tile's warps have
// one half of its scores the tensor cores have the other, the products with V of the tile and the scores of the next.
//
// P in one float16 instead of two e4m3 values: the products take as long (half the rate, once instead of twice) and leave 2^-11 of a value,
// and P takes one conversion for two elements, not four; V, which then has to be float16, is one conversion of 128 x D elements for all rows
// of a tile, by warps of their own.  A token's scales are the same for a whole row of threads, two registers
// for 16 tokens.  P is an FMA, an exponential and, for the product, V's scale; the row's sum is taken without it, so that blocks of small values (of zeros
// above all, whose scale is the least there is) keep their weight beside blocks of large ones.
//
// The reference of a row (the running maximum; for the other activations a power of two that P is multiplied by) is set so that the largest P
// lies in (32, 64], and moves when 64 tokens' |P| sum up to 65504, float16's largest, or more: the sum that the softmax takes anyhow is the
// whole test.  Then, for the first tokens of a stretch and where a mask leaves tokens out, the scores, which are still there, are gone through
// again: once for the sum and maximum under the masks, once for P.  Both forms do the same arithmetic, so no row's bits depend on its neighbours.
//
// Measured (one B200, caches cold): causal chunks of 256 to 1024 queries 373 us, candidates (64 to 1024, SiLU) 655 us; the transposed form with
// 128 rows 757 and 917, this form with P in two e4m3 values 478 and 815.  128 tokens against 256 rows take 2.4 to 2.5 us whatever the
// activation, against 128 rows 1.85 (2.2 with one place for V as it comes from the cache: its next tile then waited for the conversion).
// No pipe is near its end (exponentials 30 %, tensor 25 %, ALU 25 %, issue 39 % on chunks); what bounds it is the way of 64 tokens from the products with Q to
// those with V and back, with two warps on a scheduler.  No faster (against 427, 724 then): an MMA warp for each row tile (429, 743); a row tile's two halves one
// after the other (433, 735); scores of 128 tokens at once (438, 730); the row tiles' warps taking strict turns (507, 967); 16 element-wise
// warps, half a row each, with two converting V, who are then late (600, 1110).
//
// Roles: warps 0-3 and 4-7 the element-wise work and epilogue of row tiles 0 and 1, warp 8 TMA loads and the walk, warp 9 MMAs, warps 10-13
// V to float16, with zeros for tokens that no query may see (0 times NaN is NaN), and for NaNs where some see the token and some do not.
#include <cuda_bf16.h>

#include "gdpa_paged.cuh"

namespace gdpa {

namespace {

constexpr int kRows = 256;  // of an item

template <int D>
struct RowsShape {
  static constexpr int kTileBytes = kTile * D;               // K or V tile, or a plane of a row tile of Q
  static constexpr int kStages = D == 128 ? 2 : 4;           // of K and the scales
  static constexpr bool kOwnV = true;
  static constexpr int kVStages = 2;
  static constexpr int kActWarps = 8, kConvertWarps = 4, kWarps = kActWarps + 2 + kConvertWarps, kThreads = 32 * kWarps;
  static constexpr int kLoadWarp = kActWarps, kMmaWarp = kActWarps + 1, kConvertWarp = kActWarps + 2;
  static constexpr int kItemUnits = 4;  // beginning and end, in tiles.  Chunks / candidates, us: 1 454 / 803, 2 427 / 724, 3 410 / 682, 4 396 / 629, 6 399 / 642, 10 410 / 669
  static constexpr float kTarget = 64.f;
  static constexpr int kKvOff = 0;                                 // [stage] K
  static constexpr int kVOff = kStages * kTileBytes;               // [V stage] V as it is in the cache
  static constexpr int kV16Off = kVOff + kVStages * kTileBytes;            // V in float16: [D / 64][128 tokens][64]
  static constexpr int kQOff = kV16Off + 2 * kTileBytes;           // [2][row tile]{hi, lo}
  static constexpr int kScaleOff = kQOff + 8 * kTileBytes;         // float[stage][16]: K scales of up to 8 blocks, V scales
  static constexpr int kPoisonOff = kScaleOff + kStages * 64;      // uint16[8]: tokens whose V row held a NaN
  static constexpr int kRingOff = kPoisonOff + 16;         // int[kItemSlots][16]
  static constexpr int kBarOff = kRingOff + kItemSlots * 64;
  enum : int {
    B_KV_FULL = 0,
    B_KV_EMPTY = B_KV_FULL + kStages,
    B_SC_FULL = B_KV_EMPTY + kStages,
    B_V_FULL = B_SC_FULL + kStages,
    B_V_EMPTY = B_V_FULL + kVStages,
    B_V_READY = B_V_EMPTY + kVStages,  // [half]: V in float16
    B_V_DONE = B_V_READY + 2,   // [half]
    B_S_FULL = B_V_DONE + 2,  // [row tile][half]
    B_P_FULL = B_S_FULL + 4,         // [row tile][half]
    B_PV_DONE = B_P_FULL + 4,        // [row tile][half]
    B_Q_FULL = B_PV_DONE + 4,        // [2]
    B_Q_EMPTY = B_Q_FULL + 2,        // [2]
    B_ITEM_FULL = B_Q_EMPTY + 2,     // [kItemSlots]
    B_ITEM_EMPTY = B_ITEM_FULL + kItemSlots,
    B_COUNT = B_ITEM_EMPTY + kItemSlots
  };
  static constexpr int kMiscOff = kBarOff + B_COUNT * 8;  // tmem address, abort flag, last-arrival flag, pad
  static constexpr int kScanOff = (kMiscOff + 16 + 15) / 16 * 16;
  static constexpr int kBytes = kScanOff + 32 * 8 + 48;
  static constexpr int kDynBytes = kBytes + 1024;
  static_assert(kDynBytes <= 227 * 1024, "shared memory");
};

template <int D, int ACT>
__global__ void __launch_bounds__(RowsShape<D>::kThreads, 1)
gdpa_paged_rows_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       const __grid_constant__ PagedArgs a) {
  using L = RowsShape<D>;
  constexpr bool SOFTMAX = ACT == ACT_SOFTMAX;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_base + L::kBarOff;
  volatile uint32_t* const tmem_ptr = reinterpret_cast<volatile uint32_t*>(smem + L::kMiscOff);
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 4);
  volatile int* const last_flag = reinterpret_cast<volatile int*>(smem + L::kMiscOff + 8);
  const int warp = warp_uniform(threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::B_COUNT; ++i) {
      uint32_t n = 1;
      if (i >= L::B_SC_FULL && i < L::B_SC_FULL + L::kStages) n = 32;
      if (i >= L::B_V_EMPTY && i < L::B_V_READY + 2) n = L::kConvertWarps;  // V_EMPTY, V_READY
      if (i >= L::B_P_FULL && i < L::B_P_FULL + 4) n = L::kActWarps / 2;
      if (i >= L::B_ITEM_EMPTY && i < L::B_ITEM_EMPTY + kItemSlots) n = L::kActWarps + 1 + L::kConvertWarps;
      mbar_init(bar_base + 8u * i, n);
    }
    *abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == L::kMmaWarp) {
    tmem_alloc(smem_base + L::kMiscOff, 512);
    tmem_relinquish();
  }
  if (warp == L::kLoadWarp && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  PagedStart* const start = reinterpret_cast<PagedStart*>(smem + L::kScanOff + 32 * 8);
  find_start<L, kRows>(a, reinterpret_cast<long long*>(smem + L::kScanOff), start, warp, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = warp_uniform(*tmem_ptr);  // S0, S1 of 128 columns each (two halves), O0, O1
  PagedCta<L> cta{a, smem, smem_base, bar_base, abort_flag, lane};

  if (warp == L::kLoadWarp) {
    // ------------------------------------------------------------------ TMA loader, and the walk over the items
    uint32_t q_pos = 0;
    auto load_q = [&](const PagedItem& i) -> bool {
      const uint32_t buf = q_pos & 1u;
      if (!cta.wait(L::B_Q_EMPTY + buf, ((q_pos >> 1) & 1u) ^ 1u, ST_ROLE_LOAD)) return false;
      ++q_pos;
      const long long row = static_cast<long long>(i.q_start) * a.group + i.row0;
      const uint32_t bar = bar_base + 8u * (L::B_Q_FULL + buf);
      const int tiles = i.rows > kTile ? 2 : 1;
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, tiles * 2 * L::kTileBytes);
        for (int t = 0; t < tiles; ++t)
          for (int plane = 0; plane < 2; ++plane)
            tma_load_3d(smem_base + L::kQOff + (4 * buf + 2 * t + plane) * L::kTileBytes, &tm_q, bar, 0, static_cast<int>(row) + t * kTile, plane * a.kv_heads + i.h);
      }
      return true;
    };
    paged_load<L, D, kRows>(cta, start, tm_k, tm_v, load_q);
  } else if (warp == L::kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr int kSwizzle = D == 128 ? 128 : 64;
    constexpr uint32_t kIdescQK = umma_idesc(0, 0, 0, 0, kTile, kTile / 2), kIdescPV = umma_idesc(0, 0, 0, 1, kTile, D);  // e4m3 there, float16 here
    const uint64_t dk0 = umma_smem_desc(smem_base + L::kKvOff, 16, 8 * D, kSwizzle);
    const uint64_t dv0 = umma_smem_desc_sw128(smem_base + L::kV16Off, kTile * 128, 1024);
    const uint64_t dq0 = umma_smem_desc(smem_base + L::kQOff, 16, 8 * D, kSwizzle);
    uint32_t pos = 0, q_pos = 0, p_phase = 0;
    auto issue_qk = [&](int s, int h, uint32_t stage, uint32_t buf) {  // scores of row tile s with tokens 64 h .. of the tile
      const uint64_t dk = umma_desc_advance(dk0, stage * L::kTileBytes + h * L::kTileBytes / 2),
                     dq = umma_desc_advance(dq0, (2 * buf + s) * 2 * L::kTileBytes);
      const uint32_t d = tmem_base + s * kTile + h * (kTile / 2);
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        umma_ss_f8(d, umma_desc_advance(dq, kk * 32), umma_desc_advance(dk, kk * 32), kIdescQK, kk > 0 ? 1u : 0u);
        umma_ss_f8(d, umma_desc_advance(dq, L::kTileBytes + kk * 32), umma_desc_advance(dk, kk * 32), kIdescQK, 1u);
      }
      tc_commit(bar_base + 8u * (L::B_S_FULL + 2 * s + h));
    };
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_MMA);
      if (it.h < 0) {
        if (it.h == -2) goto role_done;
        break;
      }
      if (it.tiles == 0) continue;
      const int nst = it.rows > kTile ? 2 : 1;
      const uint32_t buf = q_pos & 1u;
      PAGED_WAIT(L::B_Q_FULL + buf, (q_pos >> 1) & 1u, ST_ROLE_MMA);
      ++q_pos;
      PAGED_WAIT(L::B_KV_FULL + pos % L::kStages, (pos / L::kStages) & 1u, ST_ROLE_MMA);
      tc_fence_after();
      for (int h = 0; h < 2; ++h)
        for (int s = 0; s < nst; ++s) issue_qk(s, h, pos % L::kStages, buf);
      if (it.tiles == 1) tc_commit(bar_base + 8u * (L::B_Q_EMPTY + buf));
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages, next = (pos + 1) % L::kStages;
        const bool more = j + 1 < it.tiles;
        for (int h = 0; h < 2; ++h) {
          for (int s = 0; s < nst; ++s) {
            PAGED_WAIT(L::B_P_FULL + 2 * s + h, (p_phase >> s) & 1u, ST_ROLE_MMA);
            if (h == 1) p_phase ^= 1u << s;
            if (s == 0) PAGED_WAIT(L::B_V_READY + h, pos & 1u, ST_ROLE_MMA);
            tc_fence_after();
            const uint32_t o = tmem_base + 256 + s * kTile, p = tmem_base + s * kTile + h * (kTile / 2);
#pragma unroll
            for (int kk = 0; kk < kTile / 32; ++kk)
              umma_ts_f16(o, p + kk * 8, umma_desc_advance(dv0, (h * 4 + kk) * 16 * 128), kIdescPV, j > 0 || h > 0 || kk > 0 ? 1u : 0u);
            if (s == nst - 1) tc_commit(bar_base + 8u * (L::B_V_DONE + h));
            tc_commit(bar_base + 8u * (L::B_PV_DONE + 2 * s + h));
            if (more) {
              if (h == 0 && s == 0) PAGED_WAIT(L::B_KV_FULL + next, ((pos + 1) / L::kStages) & 1u, ST_ROLE_MMA);
              tc_fence_after();
              issue_qk(s, h, next, buf);
            }
          }
        }
        tc_commit(bar_base + 8u * (L::B_KV_EMPTY + stage));
        if (j + 2 == it.tiles) tc_commit(bar_base + 8u * (L::B_Q_EMPTY + buf));
      }
    }
  } else if (warp >= L::kConvertWarp) {
    // ------------------------------------------------------------------ V to float16; rows that must not be seen, to zeros
    constexpr int kChunks = D / 16, kTokens = 32 / kChunks, kSteps = 16 / kTokens;  // 16 bytes of a row to a lane, tokens of a warp at once
    const int w = warp - L::kConvertWarp, chunk = lane % kChunks, t_lane = lane / kChunks, other = chunk >> 2;
    // where a lane's 16 bytes are, as the copy's swizzle has them, and where their 16 values go: eight lanes at once to as many groups of banks,
    // for which the second panel's halves are written in the other order
    auto from_of = [&](uint32_t pos, int t) { return L::kVOff + pos % L::kVStages * L::kTileBytes + t * D + (D == 128 ? chunk ^ (t & 7) : chunk ^ ((t >> 1) & 3)) * 16; };
    auto to_of = [&](int t, int k) { return L::kV16Off + other * (kTile * 128) + t * 128 + ((2 * (chunk & 3) + (other ^ k)) ^ (t & 7)) * 16; };
    auto put = [&](int t, const uint4& u) {
      const uint32_t v[4] = {u.x, u.y, u.z, u.w};
      uint32_t f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = f16x2_from_e4m3x2(static_cast<uint16_t>(v[e] & 0xffffu));
        f[2 * e + 1] = f16x2_from_e4m3x2(static_cast<uint16_t>(v[e] >> 16));
      }
      const uint4 lo = make_uint4(f[0], f[1], f[2], f[3]), hi = make_uint4(f[4], f[5], f[6], f[7]);
      *reinterpret_cast<uint4*>(smem + to_of(t, 0)) = other ? hi : lo;
      *reinterpret_cast<uint4*>(smem + to_of(t, 1)) = other ? lo : hi;
    };
    uint32_t pos = 0;
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_FIX);
      if (it.h < 0) {
        if (it.h == -2) goto role_done;
        break;
      }
      const KeyRange r0 = keys_of(it.row0 / a.group, it.past, it.len, a.causal, a.window),
                     r1 = keys_of((it.row0 + it.rows - 1) / a.group, it.past, it.len, a.causal, a.window);
      const int all_lo = max(r0.lo, r1.lo), all_hi = min(r0.hi, r1.hi);  // keys that every row takes part with (if any)
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages;
        const int key0 = (it.tile0 + j) * kTile;
        PAGED_WAIT(L::B_SC_FULL + stage, (pos / L::kStages) & 1u, ST_ROLE_FIX);
        PAGED_WAIT(L::B_V_FULL + pos % L::kVStages, (pos / L::kVStages) & 1u, ST_ROLE_FIX);
        const float* const sv = reinterpret_cast<const float*>(smem + L::kScaleOff) + stage * 16 + 8;
        const bool every = key0 >= all_lo && key0 + kTile <= all_hi;
        const bool checks = !every || __any_sync(kFull, lane < kTile >> a.block_shift && no_block(sv[lane & 7]));
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          const int t0 = half * 64 + w * 16 + t_lane;
          PAGED_WAIT(L::B_V_DONE + half, (pos & 1u) ^ 1u, ST_ROLE_FIX);  // the products with the tile before
          if (!checks) {
            uint4 u[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) u[i] = *reinterpret_cast<const uint4*>(smem + from_of(pos, t0 + i * kTokens));
#pragma unroll
            for (int i = 0; i < kSteps; ++i) put(t0 + i * kTokens, u[i]);
          } else {
            unsigned poison = 0;
#pragma unroll 1
            for (int i = 0; i < kSteps; ++i) {
              const int t = t0 + i * kTokens, key = key0 + t;
              uint4 u = *reinterpret_cast<const uint4*>(smem + from_of(pos, t));
              const bool out = key < it.lo || key >= it.hi || no_block(sv[t >> a.block_shift]);
              // some row may take part with this token and some not: a NaN is put into the columns of those that do at the stretch's end
              if (!every && !out && drop_nans(u)) poison |= 1u << (i * kTokens + t_lane);
              if (out) u = make_uint4(0, 0, 0, 0);
              put(t, u);
            }
            poison = __reduce_or_sync(kFull, poison);
            if (lane == 0) reinterpret_cast<uint16_t*>(smem + L::kPoisonOff)[half * 4 + w] = static_cast<uint16_t>(poison);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(bar_base + 8u * (L::B_V_READY + half));
            if (half == 1) mbar_arrive(bar_base + 8u * (L::B_V_EMPTY + pos % L::kVStages));
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ element-wise work and epilogue: a row to a thread
    constexpr float kLogTarget = 6.f;
    static_assert(L::kTarget == 64.f, "kLogTarget");
    constexpr float kMostSum = 65504.f;  // of 64 |P|: then each has its place in a float16
    const int qt = warp >> 2, quarter = warp & 3;
    const int r = qt * kTile + quarter * 32 + lane;  // row of the item
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_rows = tmem_base + qt * kTile + lane_base, o_tmem = tmem_base + 256 + qt * kTile + lane_base;
    uint32_t pos = 0, done = 0;  // tiles, tiles of this row tile
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the rows' factors are read below
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_ACT);
      if (named_bar_or(3, 32 * L::kActWarps, it.h < 0)) break;
      const int g = it.row0 + r, i = g / a.group;
      const bool live = r < it.rows;
      __nv_bfloat16* const o_row = a.o + ((it.q_start + static_cast<long long>(i)) * a.heads + it.h * a.group + (g - i * a.group)) * D;
      if (it.tiles == 0) {
        if (live)
          for (int e = 0; e < D / 8; ++e) reinterpret_cast<uint4*>(o_row)[e] = make_uint4(0, 0, 0, 0);
        continue;
      }
      const bool tile_live = qt * kTile < it.rows, warp_live = qt * kTile + quarter * 32 < it.rows;
      const KeyRange rg = live ? keys_of(i, it.past, it.len, a.causal, a.window) : KeyRange{0, 0};
      const KeyRange rf = keys_of(it.row0 / a.group, it.past, it.len, a.causal, a.window),
                     rl = keys_of((it.row0 + it.rows - 1) / a.group, it.past, it.len, a.causal, a.window);
      const int all_lo = max(rf.lo, rl.lo), all_hi = min(rf.hi, rl.hi);
      const float qa = __ldcg(a.qa + (static_cast<long long>(it.h) * a.total_q + it.q_start) * a.group + it.row0 + min(r, it.rows - 1));
      float ref = SOFTMAX ? kNoMax : 1.2676506e30f, l = 0.f;  // running maximum / multiplier; sum of P
      bool nan_seen = false;                                  // a token of this row had NaNs taken out of V
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages, phase = (pos / L::kStages) & 1u;
        if (!tile_live) continue;  // neither S nor P of this row tile in the item
        const int key0 = (it.tile0 + j) * kTile;
        PAGED_WAIT_ON(L::B_SC_FULL + stage, phase);
        const float* const sc = reinterpret_cast<const float*>(smem + L::kScaleOff) + stage * 16;
        const bool every = key0 >= all_lo && key0 + kTile <= all_hi;
        // ... or a block that the table has not
        const bool masked = !every || __any_sync(kFull, lane < kTile >> a.block_shift && no_block(sc[8 + (lane & 7)]));
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          PAGED_WAIT_ON(L::B_S_FULL + 2 * qt + half, done & 1u);
          tc_fence_after();
          if (warp_live) {
            const uint32_t s_tmem = s_rows + half * (kTile / 2);
            if (!every) PAGED_WAIT_ON(L::B_V_READY + half, pos & 1u);  // with the tokens whose V held a NaN
            const uint16_t* const poison = reinterpret_cast<const uint16_t*>(smem + L::kPoisonOff) + half * 4;
            const int my_key0 = key0 + half * (kTile / 2);
            const int from = rg.lo - my_key0, to = rg.hi - my_key0;  // columns of this half of the row that count
            // columns 16 i .. of this half's scores
            auto factors = [&](int i, float& kf, float& vs) {
              const int b = (half * (kTile / 2) + i * 16) >> a.block_shift;
              kf = sc[b] * qa;
              vs = no_block(sc[8 + b]) ? 0.f : sc[8 + b];
            };
            auto first_bits = [](int n) { return n >= 16 ? 0xffffu : n <= 0 ? 0u : (1u << n) - 1u; };
            auto part_of = [&](int i) -> uint32_t {  // a bit for each of the 16
              return no_block(sc[8 + ((half * (kTile / 2) + i * 16) >> a.block_shift)]) ? 0u : first_bits(to - i * 16) & ~first_bits(from - i * 16);
            };
            // P of 16 scores (for the softmax without V's scale: its sum is of these), and its sum (of |P|), the same in both forms below: no row's
            // bits depend on what another row asks for
            auto products = [&](const uint32_t (&s)[16], float kf, float vs, float (&y)[16]) {
              const float off = kLogTarget - ref;
              float m = a.scale * vs * ref;
              if (fabsf(m) > 3.4028235e38f) m = copysignf(3.4028235e38f, m);  // a row of zeros stays one
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float x = __uint_as_float(s[e]);
                y[e] = SOFTMAX ? ex2_approx(fmaf(x, kf, off)) : act_one<ACT>(x * kf, m);
              }
            };
            auto scaled = [&](float (&y)[16], float vs) {
              if constexpr (SOFTMAX) {
                const uint64_t v2 = pack_f32x2(vs, vs);
#pragma unroll
                for (int e = 0; e < 16; e += 2) unpack_f32x2(mul_f32x2(pack_f32x2(y[e], y[e + 1]), v2), y[e], y[e + 1]);
              }
            };
            auto sum_of = [&](const float (&y)[16]) {
              float p[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) p[e] = (fabsf(y[e]) + fabsf(y[e + 4])) + (fabsf(y[e + 8]) + fabsf(y[e + 12]));
              return (p[0] + p[1]) + (p[2] + p[3]);
            };
            uint32_t w[32];                 // P in float16
            float sum = 0.f, weights = 0.f;  // of |P|; of P before V's scale
            const bool first = j == 0 && half == 0;
            const float before = ref;
            bool again = masked || first;
            if (!again) {
              uint32_t s[4][16];
#pragma unroll
              for (int i = 0; i < 4; ++i) tmem_ld16(s_tmem + i * 16, s[i]);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 4; ++i) tmem_regs_ready(s[i]);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float kf, vs, y[16];
                factors(i, kf, vs);
                products(s[i], kf, vs, y);
                const float part = sum_of(y);
                sum = SOFTMAX ? fmaf(part, vs, sum) : sum + part;
                if constexpr (SOFTMAX) weights = fmaf(part, 1.f / L::kTarget, weights);
                scaled(y, vs);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[8 * i + e] = pack_f16x2(y[2 * e], y[2 * e + 1]);
              }
            }
            again = again || __any_sync(kFull, !(sum < kMostSum));
            if (again) {
              // with masks, or a reference that is new or has to move
              auto pass = [&](bool keep) {
                sum = weights = 0.f;
                float top = SOFTMAX ? kNoMax : 0.f;  // the largest |P| without the reference (softmax: its logarithm)
#pragma unroll 1
                for (int i = 0; i < 4; ++i) {
                  const uint32_t in = masked ? part_of(i) : 0xffffu;
                  if (!every && (poison[i] & in) != 0u) nan_seen = true;
                  uint32_t s[16];
                  float kf, vs, y[16];
                  tmem_ld16(s_tmem + i * 16, s);
                  tmem_wait_ld();
                  tmem_regs_ready(s);
                  factors(i, kf, vs);
                  products(s, kf, vs, y);
#pragma unroll
                  for (int e = 0; e < 16; ++e) y[e] = (in >> e) & 1u ? y[e] : 0.f;
                  const float part = sum_of(y);
                  const bool number = fabsf(vs) <= 3.4028235e38f;  // a scale that is none makes NaN of the rows that take part, and of no other
                  sum = SOFTMAX ? fmaf(part, number ? vs : 0.f, sum) : sum + part;
                  if constexpr (SOFTMAX) weights = fmaf(part, 1.f / L::kTarget, weights);
                  if (keep) {
                    scaled(y, vs);
                    if (!number) {
#pragma unroll
                      for (int e = 0; e < 16; ++e) y[e] = (in >> e) & 1u ? y[e] : 0.f;
                    }
                    uint32_t p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = pack_f16x2(y[2 * e], y[2 * e + 1]);
                    tmem_st8(s_tmem + i * 8, p);
                  } else {
                    const float log_vs = __log2f(fmaxf(vs, kLeastScale));
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                      const float x = __uint_as_float(s[e]) * kf, t = SOFTMAX ? x + log_vs : fabsf(act_one<ACT>(x, a.scale)) * vs;
                      top = fmaxf(top, (in >> e) & 1u ? t : kNoMax);
                    }
                  }
                }
                return top;
              };
              const float top = pass(false);
              // ... to a largest P in (target / 2, target]
              if (!(sum < kMostSum)) {
                if constexpr (SOFTMAX) ref = ceilf(fminf(top, 1.0e30f));
                else ref = top > 0.f ? exp2f(fminf(fmaxf(floorf(log2f(L::kTarget / top)), -100.f), 100.f)) : 1.2676506e30f;
              }
              pass(true);
            } else {
              tmem_st32(s_tmem, w);
            }
            if constexpr (SOFTMAX) {
              const float root = ex2_approx(0.5f * (before - ref));  // twice: the sum is large where V's scales were small
              l = fmaf(l * root, root, weights);
            }
            if (!first && __any_sync(kFull, ref != before)) {
              const float f = SOFTMAX ? ex2_approx(before - ref) : ref / before;
              PAGED_WAIT_ON(L::B_PV_DONE + 2 * qt + (half ^ 1), (half ? done : done - 1) & 1u);  // O holds every token before these
              tc_fence_after();
#pragma unroll 1
              for (int b = 0; b < D / 32; ++b) {
                uint32_t o[32];
                tmem_ld32(o_tmem + b * 32, o);
                tmem_wait_ld();
                tmem_regs_ready(o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st32(o_tmem + b * 32, o);
              }
            }
            tmem_wait_st();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_base + 8u * (L::B_P_FULL + 2 * qt + half));
        }
        ++done;
      }
      // ---- the end of the stretch
      const bool cut = it.pieces > 1;
      const int part = 2 * blockIdx.x + (static_cast<int>(blockIdx.x) == it.first ? 1 : 0);
      if (warp_live) {
        PAGED_WAIT_ON(L::B_PV_DONE + 2 * qt + 1, (done - 1) & 1u);
        tc_fence_after();
        float f;
        if (cut) f = SOFTMAX ? 1.f / L::kTarget : 1.f / ref;
        else f = SOFTMAX ? (l > 0.f || l != l ? 1.f / (l * L::kTarget) : 0.f) : 1.f / ref;
        if (cut && live) {
          float* const ml = a.part_ml + static_cast<long long>(part) * 2 * kRows;
          ml[r] = ref;
          ml[kRows + r] = l;
        }
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_tmem + c * 32, o);
          tmem_wait_ld();
          tmem_regs_ready(o);
          if (live && cut) {
            float4* const dst = reinterpret_cast<float4*>(a.part_o + (static_cast<long long>(part) * kRows + r) * D + c * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[e] = make_float4(__uint_as_float(o[4 * e]) * f, __uint_as_float(o[4 * e + 1]) * f, __uint_as_float(o[4 * e + 2]) * f,
                                   __uint_as_float(o[4 * e + 3]) * f);
          } else if (live) {
            uint4* const dst = reinterpret_cast<uint4*>(o_row + c * 32);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) w[x] = pack_bf16x2(__uint_as_float(o[8 * e + 2 * x]) * f, __uint_as_float(o[8 * e + 2 * x + 1]) * f);
              dst[e] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (nan_seen) {
          for (int c = 0; c < D; c += 32) {
            for (uint32_t nans = nan_columns(a, it.b, it.h, it.tile0, it.tiles, rg.lo, rg.hi, all_lo, all_hi, c); nans != 0u; nans &= nans - 1u) {
              const int e = c + __ffs(nans) - 1;
              if (cut) a.part_o[(static_cast<long long>(part) * kRows + r) * D + e] = __uint_as_float(0x7fffffffu);
              else o_row[e] = __ushort_as_bfloat16(0x7fffu);
            }
          }
        }
        __syncwarp();
        tc_fence_before();
      }
      if (cut) {
        // the last of the item's CTAs joins the pieces
        named_bar_sync(3, 32 * L::kActWarps);
        if (threadIdx.x == 0) *last_flag = count_arrival(a.counters + it.first) == it.pieces - 1;
        named_bar_sync(3, 32 * L::kActWarps);
        if (*last_flag)
          paged_join<D, kRows, SOFTMAX, L::kActWarps>(a, it, warp, lane, [&](int row) {
            const int at = it.row0 + row, q = at / a.group;
            return ((it.q_start + static_cast<long long>(q)) * a.heads + it.h * a.group + (at - q * a.group)) * D;
          });
        named_bar_sync(3, 32 * L::kActWarps);
      }
    }
  }
role_done:
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == L::kMmaWarp) tmem_dealloc(tmem_base, 512);
}

template <int D>
int launch(const PagedLaunch& l) {
  using L = RowsShape<D>;
  auto go = [&](auto kernel) -> int {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynBytes) != cudaSuccess) return GDPA_ERR_LAUNCH_;
    return launch_after(kernel, l.grid, L::kThreads, L::kDynBytes, l.stream, l.tm_q, l.tm_k, l.tm_v, l.args);
  };
  switch (l.args.act) {
    case ACT_SOFTMAX: return go(gdpa_paged_rows_kernel<D, ACT_SOFTMAX>);
    case ACT_GELU_ERF: return go(gdpa_paged_rows_kernel<D, ACT_GELU_ERF>);
    case ACT_GELU_TANH: return go(gdpa_paged_rows_kernel<D, ACT_GELU_TANH>);
    case ACT_LEAKY_RELU: return go(gdpa_paged_rows_kernel<D, ACT_LEAKY_RELU>);
    case ACT_RELU: return go(gdpa_paged_rows_kernel<D, ACT_RELU>);
    case ACT_SILU: return go(gdpa_paged_rows_kernel<D, ACT_SILU>);
    case ACT_HARDSWISH: return go(gdpa_paged_rows_kernel<D, ACT_HARDSWISH>);
    case ACT_RELU_SQUARE: return go(gdpa_paged_rows_kernel<D, ACT_RELU_SQUARE>);
    default: return go(gdpa_paged_rows_kernel<D, ACT_RAW>);
  }
}

}  // namespace

int launch_paged_rows(const PagedLaunch& l, int head_dim) { return head_dim == 128 ? launch<128>(l) : launch<64>(l); }

}  // namespace gdpa
