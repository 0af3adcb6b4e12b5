// The attention over a paged 8-bit cache (gdpa_paged.cu) for many queries: candidates of a request, chunks of a prompt.  There the tensor
// cores and the element-wise work bound it, and the form is the ordinary one, a row of scores to a thread:
//     S [128 rows x 128 tokens] = Q K^T      A = Q (two e4m3 planes in shared memory), B = the K tile
//     P = act(S) in registers                a thread has a row: its maximum, sum and reference are its own, nothing is exchanged
//     O [128 rows x D] += P V                A = P (two e4m3 planes) in tensor memory over its own S, B = the V tile, MN-major
// A work item is 256 rows (two row tiles) of one (request, K / V head); the tiles' element-wise warps and MMAs take turns, one tile's
// MMAs under the other's exponentials.  A token's scales are the same for a whole row of threads: for each block of 16 tokens and more
// the score's factor and the reference less log2 of V's scale are two registers, so that P times V's scale is one FMA and one
// exponential.  A first look at a tile's scores (one maximum in two of them, of the numbers as they are) says whether a product would pass
// 448 for the reference that a row has; only then it moves (by whole powers of two) and the row's O and sum with it.
//
// Against the transposed form on 128 rows (one B200): candidates (SiLU) 917 us, causal chunks 757 us there.
//
// Roles: warps 0-3 and 4-7 the element-wise work and epilogue of row tiles 0 and 1, warp 8 TMA loads and the walk, warp 9 MMAs, warp 10
// overwrites V rows that no query may see with zeros (0 times NaN is NaN) before the products with V.
#include <cuda_bf16.h>

#include "gdpa_paged.cuh"

namespace gdpa {

namespace {

constexpr int kRows = 256;  // of an item

template <int D>
struct RowsShape {
  static constexpr int kTileBytes = kTile * D;               // K or V tile, or a plane of a row tile of Q
  static constexpr int kStages = D == 128 ? 2 : 4;
  static constexpr int kWarps = 11, kThreads = 32 * kWarps;
  static constexpr int kLoadWarp = 8, kMmaWarp = 9, kFixWarp = 10;
  static constexpr int kItemUnits = 2, kMostTileUnits = 1;
  static constexpr __host__ __device__ int tile_units(int) { return 1; }
  static constexpr float kTarget = 64.f;
  static constexpr int kKvOff = 0;                                 // [stage]{K, V}
  static constexpr int kQOff = kStages * 2 * kTileBytes;           // [2][row tile]{hi, lo}
  static constexpr int kScaleOff = kQOff + 8 * kTileBytes;         // float[stage][16]: K scales of up to 8 blocks, V scales
  static constexpr int kPoisonOff = kScaleOff + kStages * 64;      // uint[stage][4]: tokens whose V row held a NaN
  static constexpr int kQaOff = kPoisonOff + kStages * 16;         // float[2][kRows]
  static constexpr int kRingOff = kQaOff + 2 * kRows * 4;              // int[kItemSlots][16]
  static constexpr int kBarOff = kRingOff + kItemSlots * 64;
  enum : int {
    B_KV_FULL = 0,
    B_KV_EMPTY = B_KV_FULL + kStages,
    B_SC_FULL = B_KV_EMPTY + kStages,
    B_V_READY = B_SC_FULL + kStages,
    B_S_FULL = B_V_READY + kStages,  // [2]
    B_P_FULL = B_S_FULL + 2,         // [2]
    B_PV_DONE = B_P_FULL + 2,        // [2]
    B_Q_FULL = B_PV_DONE + 2,        // [2]
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
                       const PagedArgs a) {
  using L = RowsShape<D>;
  constexpr bool SOFTMAX = ACT == ACT_SOFTMAX;
  constexpr PagedMufu kMufu = SOFTMAX ? MUFU_EX2 : ACT == ACT_SILU || ACT == ACT_GELU_TANH ? MUFU_TANH : MUFU_NONE;
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
      if (i >= L::B_P_FULL && i < L::B_P_FULL + 2) n = 4;
      if (i >= L::B_Q_FULL && i < L::B_Q_FULL + 2) n = 33;
      if (i >= L::B_Q_EMPTY && i < L::B_Q_EMPTY + 2) n = 1 + 8;
      if (i >= L::B_ITEM_EMPTY && i < L::B_ITEM_EMPTY + kItemSlots) n = 10;
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
  const uint32_t tmem_base = warp_uniform(*tmem_ptr);  // S0, S1 of 128 columns each, O0, O1
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
      for (int r = lane; r < kRows; r += 32)
        cp_async4(smem_base + L::kQaOff + (buf * kRows + r) * 4, a.qa + i.h * a.total_q * a.group + row + min(r, i.rows - 1), true);
      cp_async_mbar_arrive(bar);
      return true;
    };
    paged_load<L, D, kRows>(cta, start, tm_k, tm_v, load_q);
  } else if (warp == L::kMmaWarp) {
    // ------------------------------------------------------------------ MMA issuer
    constexpr int kSwizzle = D == 128 ? 128 : 64;
    constexpr uint32_t kIdescQK = umma_idesc(0, 0, 0, 0, kTile, kTile), kIdescPV = umma_idesc(0, 0, 0, 1, kTile, D);
    const uint64_t dk0 = umma_smem_desc(smem_base + L::kKvOff, 16, 8 * D, kSwizzle);
    const uint64_t dv0 = umma_smem_desc(smem_base + L::kKvOff + L::kTileBytes, 0, 8 * D, kSwizzle);
    const uint64_t dq0 = umma_smem_desc(smem_base + L::kQOff, 16, 8 * D, kSwizzle);
    uint32_t pos = 0, q_pos = 0, p_phase = 0;
    auto issue_qk = [&](int s, uint32_t stage, uint32_t buf) {
      const uint64_t dk = umma_desc_advance(dk0, stage * 2 * L::kTileBytes), dq = umma_desc_advance(dq0, (2 * buf + s) * 2 * L::kTileBytes);
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        umma_ss_f8(tmem_base + s * kTile, umma_desc_advance(dq, kk * 32), umma_desc_advance(dk, kk * 32), kIdescQK, kk > 0 ? 1u : 0u);
        umma_ss_f8(tmem_base + s * kTile, umma_desc_advance(dq, L::kTileBytes + kk * 32), umma_desc_advance(dk, kk * 32), kIdescQK, 1u);
      }
      tc_commit(bar_base + 8u * (L::B_S_FULL + s));
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
      for (int s = 0; s < nst; ++s) issue_qk(s, pos % L::kStages, buf);
      if (it.tiles == 1) tc_commit(bar_base + 8u * (L::B_Q_EMPTY + buf));
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages, next = (pos + 1) % L::kStages;
        const bool more = j + 1 < it.tiles;
        for (int s = 0; s < nst; ++s) {
          PAGED_WAIT(L::B_P_FULL + s, (p_phase >> s) & 1u, ST_ROLE_MMA);
          p_phase ^= 1u << s;
          if (s == 0) PAGED_WAIT(L::B_V_READY + stage, (pos / L::kStages) & 1u, ST_ROLE_MMA);
          tc_fence_after();
          const uint64_t dv = umma_desc_advance(dv0, stage * 2 * L::kTileBytes);
          const uint32_t o = tmem_base + 256 + s * kTile, p = tmem_base + s * kTile;
#pragma unroll
          for (int kk = 0; kk < kTile / 32; ++kk) {
            const uint64_t dvk = umma_desc_advance(dv, kk * 32 * D);
            umma_ts_f8(o, p + kk * 32, dvk, kIdescPV, j > 0 || kk > 0 ? 1u : 0u);
            umma_ts_f8(o, p + kk * 32 + 8, dvk, kIdescPV, 1u);
          }
          tc_commit(bar_base + 8u * (L::B_PV_DONE + s));
          if (more) {
            if (s == 0) PAGED_WAIT(L::B_KV_FULL + next, ((pos + 1) / L::kStages) & 1u, ST_ROLE_MMA);
            tc_fence_after();
            issue_qk(s, next, buf);
          }
        }
        tc_commit(bar_base + 8u * (L::B_KV_EMPTY + stage));
        if (j + 2 == it.tiles) tc_commit(bar_base + 8u * (L::B_Q_EMPTY + buf));
      }
    }
  } else if (warp == L::kFixWarp) {
    // ------------------------------------------------------------------ V rows that must not be seen
    uint32_t pos = 0;
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_FIX);
      if (it.h < 0) {
        if (it.h == -2) goto role_done;
        break;
      }
      const KeyRange r0 = keys_of(it.row0 / a.group, it.q_len, it.len, a.causal, a.window),
                     r1 = keys_of((it.row0 + it.rows - 1) / a.group, it.q_len, it.len, a.causal, a.window);
      const int all_lo = max(r0.lo, r1.lo), all_hi = min(r0.hi, r1.hi);  // keys that every row takes part with (if any)
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages, phase = (pos / L::kStages) & 1u;
        const int key0 = (it.tile0 + j) * kTile;
        PAGED_WAIT(L::B_SC_FULL + stage, phase, ST_ROLE_FIX);
        PAGED_WAIT(L::B_KV_FULL + stage, phase, ST_ROLE_FIX);
        const float* const sv = reinterpret_cast<const float*>(smem + L::kScaleOff) + stage * 16 + 8;
        const bool every = key0 >= all_lo && key0 + kTile <= all_hi;
        bool touched = false;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          const int t = 32 * i + lane, key = key0 + t;
          const bool out = key < it.lo || key >= it.hi || sv[t >> a.block_shift] == 0.f;
          uint4* const v_row = reinterpret_cast<uint4*>(smem + L::kKvOff + (2 * stage + 1) * L::kTileBytes + t * D);
          bool bad = false;
          if (!every && !out) {
            // some row may take part with this token and some not: a NaN goes into P of those that do
            for (int e = 0; e < D / 16; ++e) {
              const uint4 u = v_row[e];
              bad |= (__vcmpeq4(u.x & 0x7f7f7f7fu, 0x7f7f7f7fu) | __vcmpeq4(u.y & 0x7f7f7f7fu, 0x7f7f7f7fu) |
                      __vcmpeq4(u.z & 0x7f7f7f7fu, 0x7f7f7f7fu) | __vcmpeq4(u.w & 0x7f7f7f7fu, 0x7f7f7f7fu)) != 0u;
            }
          }
          if (out || bad)
            for (int e = 0; e < D / 16; ++e) v_row[e] = make_uint4(0, 0, 0, 0);
          touched |= out || bad;
          const unsigned poison = __ballot_sync(kFull, bad);
          if (lane == 0) reinterpret_cast<unsigned*>(smem + L::kPoisonOff)[stage * 4 + i] = poison;
        }
        if (touched) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_base + 8u * (L::B_V_READY + stage));
      }
    }
  } else {
    // ------------------------------------------------------------------ element-wise work and epilogue: a row to a thread
    constexpr float kHeadroom = 2.8073549f + 0.001f;  // log2(448 / kTarget)
    constexpr float kLogTarget = 6.f;
    static_assert(L::kTarget == 64.f, "kHeadroom, kLogTarget");
    const int qt = warp >> 2, quarter = warp & 3;
    const int r = qt * kTile + quarter * 32 + lane;  // row of the item
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_tmem = tmem_base + qt * kTile + lane_base, o_tmem = tmem_base + 256 + qt * kTile + lane_base;
    uint32_t pos = 0, q_pos = 0, done = 0;  // tiles, items with tiles, tiles of this row tile
    while (true) {
      const PagedItem it = cta.take_item(ST_ROLE_ACT);
      if (named_bar_or(3, 256, it.h < 0)) break;
      const int g = it.row0 + r, i = g / a.group;
      const bool live = r < it.rows;
      __nv_bfloat16* const o_row = a.o + ((it.q_start + static_cast<long long>(i)) * a.heads + it.h * a.group + (g - i * a.group)) * D;
      if (it.tiles == 0) {
        if (live)
          for (int e = 0; e < D / 8; ++e) reinterpret_cast<uint4*>(o_row)[e] = make_uint4(0, 0, 0, 0);
        continue;
      }
      const bool tile_live = qt * kTile < it.rows, warp_live = qt * kTile + quarter * 32 < it.rows;
      const KeyRange rg = live ? keys_of(i, it.q_len, it.len, a.causal, a.window) : KeyRange{0, 0};
      const KeyRange rf = keys_of(it.row0 / a.group, it.q_len, it.len, a.causal, a.window),
                     rl = keys_of((it.row0 + it.rows - 1) / a.group, it.q_len, it.len, a.causal, a.window);
      const int all_lo = max(rf.lo, rl.lo), all_hi = min(rf.hi, rl.hi);
      const uint32_t buf = q_pos & 1u;
      PAGED_WAIT_ON(L::B_Q_FULL + buf, (q_pos >> 1) & 1u);
      ++q_pos;
      const float qa = reinterpret_cast<const float*>(smem + L::kQaOff)[buf * kRows + r];
      float ref = SOFTMAX ? kNoMax : 1.f, l = 0.f;  // running maximum / multiplier; sum of P
      for (int j = 0; j < it.tiles; ++j, ++pos) {
        const uint32_t stage = pos % L::kStages, phase = (pos / L::kStages) & 1u;
        if (!tile_live) continue;  // neither S nor P of this row tile in the item
        const int key0 = (it.tile0 + j) * kTile;
        PAGED_WAIT_ON(L::B_SC_FULL + stage, phase);
        PAGED_WAIT_ON(L::B_S_FULL + qt, done & 1u);
        tc_fence_after();
        if (warp_live) {
          const float* const sc = reinterpret_cast<const float*>(smem + L::kScaleOff) + stage * 16;
          const bool every = key0 >= all_lo && key0 + kTile <= all_hi;
          if (!every) PAGED_WAIT_ON(L::B_V_READY + stage, phase);  // with the tokens whose V held a NaN
          const unsigned* const poison = reinterpret_cast<const unsigned*>(smem + L::kPoisonOff) + stage * 4;
          bool missing = false;  // a block that the table has not
#pragma unroll 1
          for (int b = 0; b < kTile >> a.block_shift; ++b) missing |= sc[8 + b] == 0.f;
          const bool masked = !every || missing;
          const int from = rg.lo - key0, to = rg.hi - key0;  // columns of this row that count
          // columns 32 c .. of the scores; `h`: which 16 of them
          auto factors = [&](int c, int h, float& kf, float& vs) {
            const int b = (c * 32 + h * 16) >> a.block_shift;
            kf = sc[b] * qa;
            vs = fmaxf(sc[8 + b], kLeastScale);
          };
          auto first_bits = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
          auto part_of = [&](int c) -> uint32_t {  // a bit for each of the 32
            uint32_t m = first_bits(to - c * 32) & ~first_bits(from - c * 32);
            if (sc[8 + ((c * 32) >> a.block_shift)] == 0.f) m &= 0xffff0000u;
            if (sc[8 + ((c * 32 + 16) >> a.block_shift)] == 0.f) m &= 0x0000ffffu;
            return m;
          };
          // ---- first look: how large this tile's P, times V's scale, gets (softmax: its logarithm).  Monotone in the score on its positive side,
          // |activation| is bounded by a constant on the other (exactly so, or 0.38 at most).
          float top = SOFTMAX ? kNoMax : 0.f;
          const bool flip = SOFTMAX && a.scale < 0.f;  // then the smallest product is the largest score
          auto look = [&](float most, float least, float kf, float vs) {
            if constexpr (SOFTMAX) {
              const float m = (flip ? least : most) * kf;
              top = fmaxf(top, (flip ? -least : most) > kNoMax ? m + __log2f(vs) : kNoMax);
            } else {
              float p = fabsf(act_one<ACT>(fmaxf(most * kf, 0.f), a.scale)), n = fmaxf(-least * kf, 0.f);
              if constexpr (ACT == ACT_RAW || ACT == ACT_LEAKY_RELU) p = fmaxf(p, fabsf(act_one<ACT>(-n, a.scale)));
              else if constexpr (ACT != ACT_RELU && ACT != ACT_RELU_SQUARE) p = fmaxf(p, fminf(n, 0.375f) * fabsf(a.scale));
              top = fmaxf(top, p * vs);
            }
          };
          if (!masked) {
            uint32_t s[2][16];
            tmem_ld16(s_tmem, s[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              tmem_wait_ld();
              tmem_regs_ready(s[i & 1]);
              if (i < 7) tmem_ld16(s_tmem + (i + 1) * 16, s[(i + 1) & 1]);
              float m[2], n[2] = {0.f, 0.f};
              const float* const x = reinterpret_cast<const float*>(s[i & 1]);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                m[e] = n[e] = x[8 * e];
                if (!flip) m[e] = max3(max3(max3(m[e], x[8 * e + 1], x[8 * e + 2]), x[8 * e + 3], x[8 * e + 4]), x[8 * e + 5], fmaxf(x[8 * e + 6], x[8 * e + 7]));
                if (flip || !SOFTMAX)
                  n[e] = -max3(max3(max3(-n[e], -x[8 * e + 1], -x[8 * e + 2]), -x[8 * e + 3], -x[8 * e + 4]), -x[8 * e + 5], fmaxf(-x[8 * e + 6], -x[8 * e + 7]));
              }
              float kf, vs;
              factors(i / 2, i & 1, kf, vs);
              look(fmaxf(m[0], m[1]), fminf(n[0], n[1]), kf, vs);
            }
          } else {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              const uint32_t in = part_of(c);
              uint32_t s[32];
              tmem_ld32(s_tmem + c * 32, s);
              tmem_wait_ld();
              tmem_regs_ready(s);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float kf, vs, most = kNoMax, least = -kNoMax;
                factors(c, h, kf, vs);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float x = __uint_as_float(s[16 * h + e]);
                  const bool part = (in >> (16 * h + e)) & 1u;
                  most = fmaxf(most, part ? x : kNoMax), least = fminf(least, part ? x : -kNoMax);
                }
                if (SOFTMAX || most > kNoMax) look(most, least, kf, vs);
              }
            }
          }
          // ---- the reference moves to a largest P in (target / 2, target], where there is none yet or where P would not fit
          bool moves;
          if constexpr (SOFTMAX) moves = top > kNoMax && (ref == kNoMax || top - ref > kHeadroom);
          else moves = j == 0 || top * ref > kMax8;
          if (__any_sync(kFull, moves)) {
            float f = 1.f;
            if (moves) {
              float next;
              if constexpr (SOFTMAX) {
                next = ceilf(fminf(top, 1.0e30f));
                f = ref == kNoMax ? 0.f : ex2_approx(ref - next);
              } else {
                next = top > 0.f ? exp2f(fminf(fmaxf(floorf(log2f(L::kTarget / top)), -100.f), 100.f)) : 1.2676506e30f;
                f = next / ref;
              }
              ref = next;
            }
            l *= f;
            if (j > 0) {
              PAGED_WAIT_ON(L::B_PV_DONE + qt, (done - 1) & 1u);  // O holds every tile before this one
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
              tmem_wait_st();
            }
          }
          // ---- P, over its own scores: of 32 tokens the hi plane, then the lo plane
          if (!masked) {
            // sixteen columns after sixteen, the special functions of one under the conversions of the one before, without a branch
            uint32_t w[16], s[2][16];
            float y[16], sum = 0.f;
            tmem_ld16(s_tmem, s[0]);
#pragma unroll
            for (int i = 0; i < 9; ++i) {
              float u[16], z[16], kf = 0.f, vs = 0.f;
              if (i < 8) {
                tmem_wait_ld();
                tmem_regs_ready(s[i & 1]);
                if (i < 7) tmem_ld16(s_tmem + (i + 1) * 16, s[(i + 1) & 1]);
                factors(i / 2, i & 1, kf, vs);
                const float off = SOFTMAX ? __log2f(vs) + kLogTarget - ref : 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  z[e] = SOFTMAX ? 0.f : __uint_as_float(s[i & 1][e]) * kf;
                  if constexpr (SOFTMAX) u[e] = fmaf(__uint_as_float(s[i & 1][e]), kf, off);
                  else if constexpr (ACT == ACT_SILU) u[e] = 0.5f * z[e];
                  else if constexpr (ACT == ACT_GELU_TANH) u[e] = z[e] * fmaf(z[e] * z[e], 0.7978845608028654f * 0.044715f, 0.7978845608028654f);
                  else u[e] = 0.f;
                }
              }
              if (i == 0) {
                mufu_all<kMufu>(u);
              } else {
                uint32_t w_hi[4], w_lo[4];
                if (i < 8) split_e4m3_and<kMufu>(y, w_hi, w_lo, u);
                else split_e4m3(y, w_hi, w_lo);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * ((i - 1) & 1) + e] = w_hi[e], w[8 + 4 * ((i - 1) & 1) + e] = w_lo[e];
                if ((i & 1) == 0) tmem_st16(s_tmem + (i / 2 - 1) * 32, w);
              }
              if (i < 8) {
                const float m = a.scale * vs * ref;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  if constexpr (SOFTMAX) y[e] = u[e];
                  else if constexpr (kMufu == MUFU_TANH) y[e] = fmaf(z[e] * (0.5f * m), u[e], z[e] * (0.5f * m));
                  else y[e] = act_one<ACT>(z[e], m);
                }
                if constexpr (SOFTMAX) {
                  float p[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) p[e] = (y[e] + y[e + 4]) + (y[e + 8] + y[e + 12]);
                  sum = fmaf((p[0] + p[1]) + (p[2] + p[3]), __fdividef(1.f, vs * L::kTarget), sum);
                }
              }
            }
            if constexpr (SOFTMAX) l += sum;
          } else {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              const uint32_t in = part_of(c), bad = every ? 0u : poison[c] & in;
              uint32_t s[32], w[16];
              tmem_ld32(s_tmem + c * 32, s);
              tmem_wait_ld();
              tmem_regs_ready(s);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float kf, vs, y[16];
                uint32_t w_hi[4], w_lo[4];
                factors(c, h, kf, vs);
                const float off = SOFTMAX ? __log2f(vs) + kLogTarget - ref : 0.f, m = a.scale * vs * ref;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  y[e] = SOFTMAX ? fmaf(__uint_as_float(s[16 * h + e]), kf, off) : act_one<ACT>(__uint_as_float(s[16 * h + e]) * kf, m);
                if constexpr (SOFTMAX) mufu_all<MUFU_EX2>(y);
#pragma unroll
                for (int e = 0; e < 16; ++e) y[e] = (in >> (16 * h + e)) & 1u ? y[e] : 0.f;
                if (bad != 0u) {
#pragma unroll
                  for (int e = 0; e < 16; ++e) y[e] = (bad >> (16 * h + e)) & 1u ? __uint_as_float(0x7fffffffu) : y[e];
                }
                if constexpr (SOFTMAX) {
                  float p[4];
#pragma unroll
                  for (int e = 0; e < 4; ++e) p[e] = (y[e] + y[e + 4]) + (y[e + 8] + y[e + 12]);
                  l = fmaf((p[0] + p[1]) + (p[2] + p[3]), __fdividef(1.f, vs * L::kTarget), l);
                }
                split_e4m3(y, w_hi, w_lo);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * h + e] = w_hi[e], w[8 + 4 * h + e] = w_lo[e];
              }
              tmem_st16(s_tmem + c * 32, w);
            }
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_base + 8u * (L::B_P_FULL + qt));
        ++done;
      }
      // ---- the end of the stretch
      if (lane == 0) mbar_arrive(bar_base + 8u * (L::B_Q_EMPTY + buf));
      const bool cut = it.pieces > 1;
      const int part = 2 * blockIdx.x + (static_cast<int>(blockIdx.x) == it.first ? 1 : 0);
      if (warp_live) {
        PAGED_WAIT_ON(L::B_PV_DONE + qt, (done - 1) & 1u);
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
        tc_fence_before();
      }
      if (cut) {
        // the last of the item's CTAs joins the pieces
        named_bar_sync(3, 256);
        if (threadIdx.x == 0) *last_flag = count_arrival(a.counters + it.first) == it.pieces - 1;
        named_bar_sync(3, 256);
        if (*last_flag)
          paged_join<D, kRows, SOFTMAX, 8>(a, it, warp, lane, [&](int row) {
            const int at = it.row0 + row, q = at / a.group;
            return ((it.q_start + static_cast<long long>(q)) * a.heads + it.h * a.group + (at - q * a.group)) * D;
          });
        named_bar_sync(3, 256);
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
