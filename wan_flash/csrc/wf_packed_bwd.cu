// Backward attention over packed sequences (sm_100a): dK/dV-stationary, dQ by
// fp32 reductions, grouped heads, causal or not.
//
// For one tile of 128 keys of one sequence and key-value head the main kernel
// walks units u = (q head of the group, tile of 128 query rows that sees some
// of the keys) and forms
//     S^T  = K Q^T                      P^T = exp2(S^T * scale_log2 - lse * log2(e))
//     dP^T = V dO^T                     dS^T = P^T * (dP^T - D),  D = rowsum(o * dO)
//     dV  += P^T dO                     dK  += dS^T Q         dQ_tile += dS K
// dK and dV of all the q heads of a group stay in tensor memory over the whole
// walk, so the gradients of shared heads need no reduction and no atomics.
//
// Bound: shared-memory traffic of the five products and the dQ staging, as in
// wf_bwd_main_kernel, whose pipeline, roles and layouts this is (one CTA per
// key tile; the elementwise warpgroups, the dQ warpgroup, one MMA and one TMA
// warp).  What differs:
//
//   items     The plan's key tiles, sorted by falling number of units (causal:
//             the first keys of a sequence are seen by all its rows).  A long
//             walk comes as several pieces; each leaves fp32 partial dK and dV
//             of its own, summed in a fixed order by the convert.
//   masks     Key r of the tile is seen by query rows >= need + r.  Only units
//             whose rows start below need + 127 compare; masked scores become
//             -inf before the exponential.
//   isolation -lse * log2(e) and D come from padded tiles (-inf and 0 behind
//             the sequence's end), so those columns have P = dS = 0; the rows of
//             Q, dO and K behind the ends, which belong to a neighbour or to
//             padding and may be NaN, are zeroed in shared memory before a
//             product sums over them, and so are rows of Q and dO that see no
//             key at all.
//   dQ        The fp32 accumulator is tiled by the plan's query tiles, so no
//             tile holds rows of two sequences, but a tile has only its own rows
//             (rounded up to 8) of it: many short sequences need little more than one
//             long one.  In ordered mode every tile gets its contributions key tile
//             by key tile (bitwise reproducible).
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

// The dQ accumulator of a query tile: [2 halves of 64 columns][rows / 8][16 groups
// of 4 columns][8 rows], so a half of the tile is one run however many rows it has.
// (Rows with a pitch of their own, or a reduction per 8 columns, made the main
// kernel's dQ warpgroup 9 to 17 % slower: full attention over 7800 tokens 1075 -> 1170
// to 1260 us.)  Against 64 KiB a tile, 2500 sequences of 20 tokens with 40 heads take
// 7.8 ms and 1.7 GB of workspace instead of 9.4 ms and 7.8 GB, full attention 0.5 % more.
__device__ __forceinline__ int packed_dq_rows(int rows) { return min(128, (rows + 7) & ~7); }
// First float of query tile `tile`, which starts at packed row x, of q head h.  The
// tiles before it start 8 places apart beside their rows, so rounding finds room.
__device__ __forceinline__ size_t packed_dq_place(size_t dq_rows, int h, int x, int tile) {
  return ((size_t)h * dq_rows + (x & ~7) + 8 * (size_t)tile) * 128;
}

// Preprocess: D = rowsum((o + residual) * dO), -lse * log2(e), and the zeroed dQ
// accumulator.  Bound: HBM (1036 bytes per row and head, 1292 with the residual).  grid (2 * tiles,
// h), 256 threads: 64 rows of one tile, 16 threads per row.
__global__ void __launch_bounds__(256) wf_packed_pre_kernel(PackedBwdParams p, const __nv_bfloat16* __restrict__ o,
                                                            const __nv_bfloat16* __restrict__ res,
                                                            const __nv_bfloat16* __restrict__ dO,
                                                            const float* __restrict__ lse) {
  griddep_launch_dependents();
  griddep_wait();  // the plan
  const int tile = blockIdx.x >> 1, half = blockIdx.x & 1, h = blockIdx.y;
  if (tile >= p.head[1].x) return;
  const int4 w = p.q_tiles[tile];
  if (!w.z) return;  // rows outside any sequence
  const size_t at = (size_t)h * p.q_tile_stride + tile;
  const int sub = threadIdx.x & 15, rr = threadIdx.x >> 4;
#pragma unroll
  for (int pass = 0; pass < 4; ++pass) {
    const int r = half * 64 + pass * 16 + rr;
    float acc = 0.f;
    if (r < w.y) {
      const size_t off = ((size_t)(w.x + r) * p.h + h) * 128 + sub * 8;
      const uint4 a = ldg_u4(o + off);
      const uint4 c = ldg_u4(dO + off);
      acc = bf16_dot2(a.x, c.x) + bf16_dot2(a.y, c.y) + bf16_dot2(a.z, c.z) + bf16_dot2(a.w, c.w);
      if (res != nullptr) {
        const uint4 b = ldg_u4(res + off);
        acc += bf16_dot2(b.x, c.x) + bf16_dot2(b.y, c.y) + bf16_dot2(b.z, c.z) + bf16_dot2(b.w, c.w);
      }
    }
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (sub == 0) {
      float nl2 = -INFINITY;  // pad rows and rows that see nothing: P = 0
      if (r < w.y) {
        const float l = lse[(size_t)h * p.total_q + w.x + r];
        if (l == -INFINITY) acc = 0.f; else nl2 = -(l * 1.4426950408889634f);
      }
      p.dpsum[at * 128 + r] = acc;
      p.neg_lse_log2[at * 128 + r] = nl2;
    }
  }
  float4* const acc_tile = reinterpret_cast<float4*>(p.dq_accum + packed_dq_place(p.dq_rows, h, w.x, tile));
  const int end = 32 * packed_dq_rows(w.y);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at4 = half * 2048 + i * 256 + (int)threadIdx.x;
    if (at4 < end) acc_tile[at4] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
}

// The units of an item's walk one by one, forwards or backwards: (q head g of
// the group, query tile m), m fastest.  Only the start divides.
struct PackedWalk {
  int m_begin, m_end, g, m, step;
  __device__ __forceinline__ PackedWalk(const PackedBwdItem& w, bool reverse) {
    const int i = w.first + (reverse ? w.count - 1 : 0);
    m_begin = w.m_begin;
    m_end = w.m_begin + w.m_count;
    g = i / w.m_count;
    m = m_begin + (i - g * w.m_count);
    step = reverse ? -1 : 1;
  }
  __device__ __forceinline__ void next() {
    m += step;
    if (m == m_end) m = m_begin, ++g;
    else if (m < m_begin) m = m_end - 1, --g;
  }
};

// The causal kernel zeroes rows through a call, the other in line: 16384 causal
// 2.54 ms in line, 2.44 by the call; 7800 full 1.04 in line, 1.11 by the call.
__device__ __noinline__ void packed_zero_rows_call(uint32_t tile, int first, int none) {
  packed_zero_rows(tile, first, none);
}
template <bool kCausal>
__device__ __forceinline__ void packed_bwd_zero(uint32_t tile, int first, int none) {
  if constexpr (kCausal) packed_zero_rows_call(tile, first, none);
  else packed_zero_rows(tile, first);
}

template <bool kCausal>
__global__ void __launch_bounds__(bwd::kThreads, 1)
    wf_packed_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                         PackedBwdParams p) {
  using namespace bwd;
  extern __shared__ uint8_t smem_raw[];
  const uintptr_t raw = reinterpret_cast<uintptr_t>(smem_raw);
  uint8_t* smem = reinterpret_cast<uint8_t*>((raw + 1023) & ~uintptr_t(1023));
  griddep_launch_dependents();
  if ((uint32_t)(reinterpret_cast<uintptr_t>(smem) - raw) + kSmemUsed > dynamic_smem_size()) {
    // the aligned layout does not fit: report and leave (uniform for the CTA)
    if (threadIdx.x == 0) atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_SMEM_ALIGN);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + kOffBar;
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kOffAbort);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + kOffTmemHolder);
  const int warp = (int)warp_id();
  const int lane = (int)lane_id();

  // (Setting up barriers and tensor memory before this wait slowed full attention
  // over 7800 tokens by 4 %: the grid has room for more items than there are.)
  griddep_wait();  // the plan's lists, and what the preprocess wrote
  if ((int)blockIdx.x >= p.head[0].x * p.h_kv) return;
  int kvh;
  const PackedBwdItem w = p.items[packed_locate(p.items, (int)blockIdx.x, p.h_kv, kvh)];
  // successive waves of CTAs walk in alternating directions and start on the
  // query tiles that the previous wave touched last (still in L2).  The item's
  // place inside its bucket comes from atomics, so its tile number stands in
  // for it here: the direction, and with it the sums' order, is the item's own.
  const unsigned about = (unsigned)(w.bucket * p.h_kv + kvh * w.bucket_items + min(w.nb, w.bucket_items - 1));
  const bool reverse = !p.ordered && p.wave > 0 && ((about / (unsigned)p.wave) & 1u);
  const int cnt = w.count;
  if (cnt <= 0) {
    // no query row sees these keys, or rows outside any sequence
    const uint32_t fill = p.head[0].y ? 0x7fff7fffu : 0u;  // NaN where the offsets were impossible
    for (int i = threadIdx.x; i < w.rows * 16; i += kThreads) {
      const size_t off = ((size_t)(w.k0 + (i >> 4)) * p.h_kv + kvh) * 128 + (i & 15) * 8;
      st_global_v4(p.dk + off, fill, fill, fill, fill);
      st_global_v4(p.dv + off, fill, fill, fill, fill);
    }
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < kNumBars; ++i) {
      const bool ew = (i == kBarPReady || i == kBarDsReady);
      const uint32_t count = ew ? 256u : (i == kBarDqDrained || i == kBarXchgDone || i == kBarXchgFull) ? 128u : 1u;
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  // first place of q head g of the group, query tile m, in the tiled workspaces
  auto q_place = [&](int g, int m) -> size_t {
    return (size_t)(kvh * p.group + g) * p.q_tile_stride + w.qtile + m;
  };

  if (warp >= 14) {
    regs_dec<kRegsOther>();  // idle warps of warpgroup 3
  } else if (warp == 13) {
    regs_dec<kRegsOther>();
    // ------------------------------------------------------------------ TMA
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      tma_prefetch_desc(&tm_do);
      mbar_expect_tx(bar(kBarKvFull), 2 * kTileBytes);
      for (int x = 0; x < 2; ++x) {
        tma_load_4d(sbase + kOffK + x * kBoxBytes, &tm_k, bar(kBarKvFull), x * 64, w.k0, kvh, 0);
        tma_load_4d(sbase + kOffV + x * kBoxBytes, &tm_v, bar(kBarKvFull), x * 64, w.k0, kvh, 0);
      }
      int issued0 = 0, issued1 = 0, issued_do = 0;  // completed uses per buffer (for the abort drain)
      PackedWalk at(w, reverse);
      for (int u = 0; u < cnt; ++u, at.next()) {
        const int st = u & 1, use = u >> 1;
        const int g = at.g, m = at.m;
        const int row = w.q0 + m * 128, h = kvh * p.group + g;
        if (use > 0 && !mbar_wait(bar(kBarQEmpty + st), (use - 1) & 1, abort_flag, kRoleBwdLoad, 3 + st)) break;
        const uint32_t qfull = bar(kBarQFull + st);
        mbar_expect_tx(qfull, kTileBytes + 1024);
        for (int x = 0; x < 2; ++x)
          tma_load_4d(sbase + kOffQ + st * kTileBytes + x * kBoxBytes, &tm_q, qfull, x * 64, row, h, 0);
        bulk_load(sbase + kOffLse + st * 512, p.neg_lse_log2 + q_place(g, m) * 128, 512, qfull);
        bulk_load(sbase + kOffD + st * 512, p.dpsum + q_place(g, m) * 128, 512, qfull);
        if (st) issued1 = use + 1; else issued0 = use + 1;
        // dO has one buffer: refill it once dV of the previous unit has read it
        if (u > 0 && !mbar_wait(bar(kBarDoEmpty), (u - 1) & 1, abort_flag, kRoleBwdLoad, 6)) break;
        mbar_expect_tx(bar(kBarDoFull), kTileBytes);
        for (int x = 0; x < 2; ++x)
          tma_load_4d(sbase + kOffdO + x * kBoxBytes, &tm_do, bar(kBarDoFull), x * 64, row, h, 0);
        issued_do = u + 1;
      }
      if (*abort_flag) {
        mbar_wait_drain(bar(kBarKvFull), 0);
        if (issued0 > 0) mbar_wait_drain(bar(kBarQFull + 0), (issued0 - 1) & 1);
        if (issued1 > 0) mbar_wait_drain(bar(kBarQFull + 1), (issued1 - 1) & 1);
        if (issued_do > 0) mbar_wait_drain(bar(kBarDoFull), (issued_do - 1) & 1);
      }
    }
  } else if (warp == 12) {
    regs_dec<kRegsOther>();
    // ------------------------------------------------------------------ MMA
    constexpr uint32_t id_kk = idesc_bf16(128, 128, 0, 0);  // A, B K-major
    constexpr uint32_t id_kb = idesc_bf16(128, 128, 0, 1);  // A K-major (or TMEM), B MN-major
    constexpr uint32_t id_mm = idesc_bf16(128, 128, 1, 1);  // A, B MN-major
    const uint32_t tS = tmem, tdP = tmem + 128, tdV = tmem + 256, tdK = tmem + 384;
    const uint64_t dK_k = sdesc(sbase + kOffK, 16, 1024);
    const uint64_t dV_k = sdesc(sbase + kOffV, 16, 1024);
    const uint64_t dK_mn = sdesc(sbase + kOffK, kBoxBytes, 1024);
    const uint64_t dS_mn = sdesc(sbase + kOffdS, kBoxBytes, 1024);
    auto koff = [](int ks) -> uint32_t { return (uint32_t)((ks >> 2) * kBoxBytes + (ks & 3) * 32); };
    auto moff = [](int ks) -> uint32_t { return (uint32_t)(ks * 2048); };
    PackedWalk at(w, reverse);  // the unit whose S^T is issued next
    int rows_s = 128, rows_dp = 128;  // query rows of the units of the last S^T and of the next dP^T
    int none_s = 0, none_dp = 0;      // their first rows that see no key at all (causal, more queries than keys)
    // only a sequence's first key tile walks a query tile with such rows
    const int none = kCausal && w.nb == 0 ? w.need : 0;
    auto issue_s = [&](int u) {  // S^T = K Q^T
      const uint32_t sq = sbase + kOffQ + (u & 1) * kTileBytes;
      rows_s = w.lq - at.m * 128;
      if constexpr (kCausal) none_s = none - at.m * 128;
      at.next();
      if (rows_s < 128 || none_s > 0) packed_bwd_zero<kCausal>(sq, rows_s, none_s);  // dK sums over the query rows
      const uint64_t q_k = sdesc(sq, 16, 1024);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) mma_ss_e(tS, desc_add(dK_k, koff(ks)), desc_add(q_k, koff(ks)), id_kk, ks > 0);
      mma_commit_e(bar(kBarSFull));
    };
    const uint64_t do_k = sdesc(sbase + kOffdO, 16, 1024);
    const uint64_t do_mn = sdesc(sbase + kOffdO, kBoxBytes, 1024);
    auto issue_dp = [&]() {  // dP^T = V dO^T
      if (rows_dp < 128 || none_dp > 0)
        packed_bwd_zero<kCausal>(sbase + kOffdO, rows_dp, none_dp);  // dV sums over the query rows too
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) mma_ss_e(tdP, desc_add(dV_k, koff(ks)), desc_add(do_k, koff(ks)), id_kk, ks > 0);
      mma_commit_e(bar(kBarDpFull));
    };
    bool ok = mbar_wait_warp(bar(kBarKvFull), 0, abort_flag, kRoleBwdMma, 0) &&
              mbar_wait_warp(bar(kBarQFull + 0), 0, abort_flag, kRoleBwdMma, 1) &&
              mbar_wait_warp(bar(kBarDoFull), 0, abort_flag, kRoleBwdMma, 5);
    if (ok) {
      tc_fence_after();
      if (w.rows < 128) packed_bwd_zero<kCausal>(sbase + kOffK, w.rows, 0);  // dQ sums over the keys
      rows_dp = w.lq - at.m * 128;
      if constexpr (kCausal) none_dp = none - at.m * 128;
      issue_dp();
      issue_s(0);
    }
    for (int u = 0; u < cnt && ok; ++u) {
      const int st = u & 1;
      // dV += P^T dO   (P^T from TMEM: query 0-63 in columns [0,32), 64-127 in [64,96))
      if (!(ok = mbar_wait_warp(bar(kBarPReady), u & 1, abort_flag, kRoleBwdMma, 7))) break;
      tc_fence_after();
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        mma_ts_e(tdV, tS + (ks >> 2) * 64 + (ks & 3) * 8, desc_add(do_mn, moff(ks)), id_kb, (u > 0 || ks > 0) ? 1u : 0u);
      mma_commit_e(bar(kBarDoEmpty));  // dO(u) is read by dP(u) and dV(u) only
      // S^T(u+1): the S columns are free once dV(u) has read P^T(u)
      if (u + 1 < cnt) {
        if (!(ok = mbar_wait_warp(bar(kBarQFull + ((u + 1) & 1)), ((u + 1) >> 1) & 1, abort_flag, kRoleBwdMma, 1)))
          break;
        tc_fence_after();
        issue_s(u + 1);
      }
      // dK += dS^T Q
      if (!(ok = mbar_wait_warp(bar(kBarDsReady), u & 1, abort_flag, kRoleBwdMma, 8))) break;
      tc_fence_after();
      const uint64_t q_mn = sdesc(sbase + kOffQ + st * kTileBytes, kBoxBytes, 1024);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        mma_ts_e(tdK, tdP + (ks >> 2) * 64 + (ks & 3) * 8, desc_add(q_mn, moff(ks)), id_kb, (u > 0 || ks > 0) ? 1u : 0u);
      mma_commit_e(bar(kBarQEmpty + st));
      // dQ_tile = dS K   (same dS bytes read MN-major) into the dP^T columns
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) mma_ss_e(tdP, desc_add(dS_mn, moff(ks)), desc_add(dK_mn, moff(ks)), id_mm, ks > 0);
      mma_commit_e(bar(kBarDqFull));
      mma_commit_e(bar(kBarDsEmpty));
      // dP^T(u+1) once dQ(u) has been read out of those columns and dO(u+1) is in
      if (u + 1 < cnt) {
        if (!(ok = mbar_wait_warp(bar(kBarDqDrained), u & 1, abort_flag, kRoleBwdMma, 11))) break;
        if (!(ok = mbar_wait_warp(bar(kBarDoFull), (u + 1) & 1, abort_flag, kRoleBwdMma, 5))) break;
        tc_fence_after();
        rows_dp = rows_s, none_dp = none_s;  // S^T(u+1) has been issued
        issue_dp();
      }
    }
    if (ok) mma_commit_e(bar(kBarDkvFull));
    mma_commit_e(bar(kBarDrain));
    mbar_wait_drain(bar(kBarDrain), 0);
  } else if (warp < 8) {
    regs_inc<kRegsEw>();
    // ---------------------------------------------- elementwise warpgroups
    const int half = warp >> 2;   // 0: query columns [0,64), 1: [64,128)
    const int wq = warp & 3;      // TMEM lane quadrant: key rows [32 wq, 32 wq + 32)
    // 16x256b TMEM reads: thread t holds key rows 32 wq + 16 g + 8 e + t/4 and, in
    // repetition j, query columns 64 half + 8 j + 2 (t%4) + {0, 1}
    const int tq = lane & 3;
    const int tr = lane >> 2;
    auto kv_row = [&](int g, int e) -> int { return wq * 32 + 16 * g + 8 * e + tr; };
    bool kv_ok[2][2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 2; ++e) kv_ok[g][e] = kv_row(g, e) < w.rows;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    constexpr uint32_t kLane16 = 16u << 16;
    const uint32_t tS = tmem + lane_base + (uint32_t)(half * 64);
    const uint32_t tdP = tmem + lane_base + 128u + (uint32_t)(half * 64);
    const float sl2 = p.scale_log2;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    const uint32_t sdS = sbase + kOffdS + (uint32_t)half * kBoxBytes;
    bool ok = true;
    PackedWalk at(w, reverse);
    for (int u = 0; u < cnt; ++u, at.next()) {
      const int st = u & 1;
      const float* snl = reinterpret_cast<const float*>(smem + kOffLse + st * 512) + half * 64 + 2 * tq;
      const float* sD = reinterpret_cast<const float*>(smem + kOffD + st * 512) + half * 64 + 2 * tq;
      if (!(ok = mbar_wait(bar(kBarSFull), u & 1, abort_flag, kRoleEw, 5))) break;
      // -lse*log2(e) / D of this unit arrived with Q (already complete; this
      // wait makes the bulk-copied bytes visible to these threads)
      if (!(ok = mbar_wait(bar(kBarQFull + st), (u >> 1) & 1, abort_flag, kRoleEw, 1))) break;
      tc_fence_after();
      uint32_t s[2][32];
      tmem_ld_16x256b_x8(tS, s[0]);
      tmem_ld_16x256b_x8(tS + kLane16, s[1]);
      uint64_t nl[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 L = *reinterpret_cast<const float2*>(snl + 8 * j);
        nl[j] = f2_pack(L.x, L.y);
      }
      tmem_wait_ld();
      reg_fence32(s[0]);
      reg_fence32(s[1]);
      if constexpr (kCausal) {
        // key row r is seen by the unit's columns >= below + r (a copy of the
        // exponentials' loop with the compares in it ran 12 % slower, compares
        // in a kernel for both kinds cost full attention 5 %)
        const int below = w.need - at.m * 128;
        if (below > -127) {
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int first = below + kv_row(g, e) - half * 64 - 2 * tq;
#pragma unroll
              for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  if (8 * j + i < first) s[g][4 * j + 2 * e + i] = __float_as_uint(-INFINITY);
            }
        }
      }
      // P^T = 2^(S^T * scale_log2 + neg_lse_log2[q]); rounded to bf16 as the
      // dV product's operand, kept in fp32 for dS.  Rows past the keys' end are zeroed.
      uint64_t pp[2][16];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint64_t x = f2_fma(f2_pack(__uint_as_float(s[g][4 * j + 2 * e]), __uint_as_float(s[g][4 * j + 2 * e + 1])),
                                      sl2x2, nl[j]);
            pp[g][2 * j + e] = exp2_mufu2(x);
            float p0, p1;
            f2_unpack(pp[g][2 * j + e], p0, p1);
            pk[2 * j + e] = kv_ok[g][e] ? pack_bf16(p0, p1) : 0u;
          }
        tmem_st_16x128b_x8(tS + (g ? kLane16 : 0u), pk);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar(kBarPReady));
      // dS^T = P^T * (dP^T - D[q])
      if (!(ok = mbar_wait(bar(kBarDpFull), u & 1, abort_flag, kRoleEw, 6))) break;
      tc_fence_after();
      uint32_t dp[2][32];
      tmem_ld_16x256b_x8(tdP, dp[0]);
      tmem_ld_16x256b_x8(tdP + kLane16, dp[1]);
      tmem_wait_ld();
      reg_fence32(dp[0]);
      reg_fence32(dp[1]);
      tc_fence_before();  // the dP columns are read; dQ(u) may overwrite them after dS_ready
      if (u > 0 && !(ok = mbar_wait(bar(kBarDsEmpty), (u - 1) & 1, abort_flag, kRoleEw, 9))) break;
      const uint64_t m1x2 = f2_pack(-1.f, -1.f);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 D = *reinterpret_cast<const float2*>(sD + 8 * j);
          const uint64_t d2 = f2_pack(D.x, D.y);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint64_t dpp = f2_pack(__uint_as_float(dp[g][4 * j + 2 * e]), __uint_as_float(dp[g][4 * j + 2 * e + 1]));
            float d0, d1;
            f2_unpack(f2_mul(pp[g][2 * j + e], f2_fma(d2, m1x2, dpp)), d0, d1);
            pk[2 * j + e] = kv_ok[g][e] ? pack_bf16(d0, d1) : 0u;
            // row of dS^T in shared memory for the dQ MMA (128B-swizzled
            // [kv][q] box of this half): 4 bytes of the 16-byte chunk j
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(sdS + sw128_offset((uint32_t)kv_row(g, e), (uint32_t)j) +
                                                          4u * (uint32_t)tq),
                         "r"(pk[2 * j + e])
                         : "memory");
          }
        }
        tmem_st_16x128b_x8(tdP + (g ? kLane16 : 0u), pk);
      }
      fence_proxy_async_smem();
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar(kBarDsReady));
    }
    // ----------------------------------------------------------- epilogue
    // WG A writes dV (unscaled), WG B writes dK (scaled by softmax_scale)
    const int r = wq * 32 + lane;  // 32x32b reads: thread = one key row
    if (ok) ok = mbar_wait(bar(kBarDkvFull), 0, abort_flag, kRoleEpi, 12);
    if (ok) {
      tc_fence_after();
      const uint32_t tsrc = tmem + lane_base + (half ? 384u : 256u);
      const float mul = half ? p.scale : 1.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t a[32];
        tmem_ld32(tsrc + c * 32, a);
        tmem_wait_ld();
        reg_fence32(a);
        if (w.part < 0) {
          if (r < w.rows) {
            __nv_bfloat16* row = (half ? p.dk : p.dv) + ((size_t)(w.k0 + r) * p.h_kv + kvh) * 128;
#pragma unroll
            for (int v = 0; v < 4; ++v)
              st_global_v4(row + c * 32 + v * 8,
                           pack_bf16(__uint_as_float(a[8 * v + 0]) * mul, __uint_as_float(a[8 * v + 1]) * mul),
                           pack_bf16(__uint_as_float(a[8 * v + 2]) * mul, __uint_as_float(a[8 * v + 3]) * mul),
                           pack_bf16(__uint_as_float(a[8 * v + 4]) * mul, __uint_as_float(a[8 * v + 5]) * mul),
                           pack_bf16(__uint_as_float(a[8 * v + 6]) * mul, __uint_as_float(a[8 * v + 7]) * mul));
          }
        } else {
          float* dst = (half ? p.dk_part : p.dv_part) + ((size_t)w.part * p.h_kv + kvh) * 16384 +
                       (size_t)(r >> 6) * 8192 + (size_t)(r & 63) * 4;
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<float4*>(dst + (size_t)(c * 8 + g) * 256) =
                make_float4(__uint_as_float(a[4 * g + 0]) * mul, __uint_as_float(a[4 * g + 1]) * mul,
                            __uint_as_float(a[4 * g + 2]) * mul, __uint_as_float(a[4 * g + 3]) * mul);
        }
      }
    }
  } else {
    regs_inc<kRegsDq>();
    // ------------------------------------------------------- dQ warpgroup
    // dQ(u) leaves TMEM into registers, goes through a 32 KB staging buffer in
    // two column halves and is reduced into the accumulator by one bulk
    // reduction per half
    const int wq = warp & 3;
    const int r = wq * 32 + lane;  // query row within the tile
    const uint32_t tQ = tmem + ((uint32_t)(wq * 32) << 16) + 128u;  // dQ lives in the dP^T columns
    const uint32_t sx = sbase + kOffX;
    uint8_t* xb = smem + kOffX;
    const bool leader = (threadIdx.x == 256);
    PackedWalk at(w, reverse);
    for (int u = 0; u < cnt; ++u, at.next()) {
      if (!mbar_wait(bar(kBarDqFull), u & 1, abort_flag, kRoleDq, 10)) break;
      tc_fence_after();
      uint32_t q[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(tQ + c * 32, q[c]);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 4; ++c) reg_fence32(q[c]);
      tc_fence_before();
      mbar_arrive(bar(kBarDqDrained));
      float* dst = p.dq_accum + packed_dq_place(p.dq_rows, kvh * p.group + at.g, w.q0 + at.m * 128, w.qtile + at.m);
      int* const sem = p.ordered ? p.sem + q_place(at.g, at.m) : nullptr;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // the staging buffer is free once the previous bulk reduction has read it
        if (leader) bulk_wait_read_all();
        mbar_arrive(bar(kBarXchgDone));
        if (!mbar_wait(bar(kBarXchgDone), (2 * u + half) & 1, abort_flag, kRoleDq, 16)) break;
#pragma unroll
        for (int cc = 0; cc < 2; ++cc)
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<uint4*>(xb + (((r >> 3) * 16 + cc * 8 + g) * 8 + (r & 7)) * 16) =
                make_uint4(q[2 * half + cc][4 * g + 0], q[2 * half + cc][4 * g + 1], q[2 * half + cc][4 * g + 2],
                           q[2 * half + cc][4 * g + 3]);
        fence_proxy_async_smem();
        mbar_arrive(bar(kBarXchgFull));
        if (leader) {
          if (!mbar_wait(bar(kBarXchgFull), (2 * u + half) & 1, abort_flag, kRoleDq, 15)) break;
          if (sem != nullptr && half == 0) {
            // the sequence's key tiles 0..nb-1 add to this query tile first
            if (!counter_wait_eq(sem, w.nb, abort_flag, kRoleDq, 20)) break;
            fence_proxy_async_global();
          }
          const int rows = packed_dq_rows(w.lq - at.m * 128);
          bulk_reduce_add_f32(dst + half * rows * 64, sx, (uint32_t)rows * 256);
          bulk_commit_group();
          if (sem != nullptr && half == 1) {
            bulk_wait_all();  // the reductions have landed in global memory
            fence_proxy_async_global();
            st_release_gpu(sem, w.nb + 1);
          }
        }
      }
      if (*abort_flag) break;
    }
    if (leader) bulk_wait_all();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

// fp32 tiles -> bf16 rows, times a scale: the dQ accumulator, and the sums of
// the pieces' partial dK and dV in a fixed order.  Rows of dQ outside any
// sequence become 0 (NaN where the offsets were impossible).
// Bound: HBM.  A thread turns two groups of four columns of a row into 16 bytes;
// a warp has 8 rows x 4 such chunks, so it reads 128-byte runs and writes 64-byte
// runs without a detour through shared memory, eight loads a thread in flight.
// grid dq_blocks + 2 * split_blocks, 256 threads: 64 rows x 128 columns of one head.
__global__ void __launch_bounds__(256) wf_packed_convert_kernel(PackedConvertParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const bool split = blockIdx.x >= p.dq_blocks;
  unsigned i = split ? blockIdx.x - p.dq_blocks : blockIdx.x;
  const bool is_dv = split && i >= p.split_blocks;
  if (is_dv) i -= p.split_blocks;
  const int half = (int)(i & 1);
  const int heads = split ? p.h_kv : p.h;
  const int t = (int)(i >> 1) / heads, h = (int)(i >> 1) - t * heads;
  if (t >= (split ? p.head[0].z : p.head[1].x)) return;
  const int4 w = split ? p.split_tiles[t] : p.q_tiles[t];  // first row, rows, first part / inside, parts
  const int rows = w.y - half * 64;
  if (rows <= 0) return;
  __nv_bfloat16* const out = (!split ? p.dq : is_dv ? p.dv : p.dk) + ((size_t)(w.x + half * 64) * heads + h) * 128;
  const size_t row_stride = (size_t)heads * 128;
  // this thread's rows r + 8 k' and chunks c + 4 k'' of the 64 x 16
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = (lane >> 2) + 8 * warp, c = lane & 3;
  if (!split && w.z == 0) {
    const uint32_t fill = p.head[1].y ? 0x7fff7fffu : 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r < rows) st_global_v4(out + r * row_stride + (c + 4 * k) * 8, fill, fill, fill, fill);
    return;
  }
  if (r >= rows) return;
  const int parts = split ? w.w : 1;
  // the two layouts: a part's 64 rows lie behind each other in a group of four columns
  const int group_step = split ? 64 : 8, half_step = split ? 1024 : 16 * packed_dq_rows(w.y);
  const float4* src =
      split ? reinterpret_cast<const float4*>((is_dv ? p.dv_part : p.dk_part) + ((size_t)w.z * heads + h) * 16384) +
                  half * 2048 + r
            : reinterpret_cast<const float4*>(p.dq_accum + packed_dq_place(p.dq_rows, h, w.x, t)) +
                  (half * 8 + (r >> 3)) * 128 + (r & 7);
  const size_t step = (size_t)heads * 4096;
  float4 v[4][2];
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int g = 0; g < 2; ++g) v[k][g] = src[(k >> 1) * half_step + (2 * (c + 4 * (k & 1)) + g) * group_step];
  for (int s = 1; s < parts; ++s) {
    src += step;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 x = src[(2 * (c + 4 * k) + g) * 64];
        v[k][g].x += x.x, v[k][g].y += x.y, v[k][g].z += x.z, v[k][g].w += x.w;
      }
  }
  const float scale = split ? 1.f : p.scale;  // dk was scaled where it left the tensor core
#pragma unroll
  for (int k = 0; k < 4; ++k)
    st_global_v4(out + r * row_stride + (c + 4 * k) * 8, pack_bf16(v[k][0].x * scale, v[k][0].y * scale),
                 pack_bf16(v[k][0].z * scale, v[k][0].w * scale), pack_bf16(v[k][1].x * scale, v[k][1].y * scale),
                 pack_bf16(v[k][1].z * scale, v[k][1].w * scale));
}

}  // namespace wf
