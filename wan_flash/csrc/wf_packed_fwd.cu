// Forward attention over packed sequences (sm_100a): sequences of different
// lengths one behind the other, grouped heads, causal or not.
//
//     S = q k^T / sqrt(128), row i of a sequence sees keys j <= i + lk - lq
//     (causal) or all of them; o = softmax(S) v; lse.
//
// Bound: the tensor pipe and, level with it, the MUFU exponentials need as many
// cycles for a 128 x 128 block of S; each is busy 52 to 56 % of the time, the rest is
// the chain scores -> probabilities -> product of a tile that the other one does
// not always cover, and the uneven end of the last round.  The inner pipeline is
// that of wf_fwd_kernel: two 128-row query tiles per CTA, S and O in tensor
// memory, P written over S in two halves, one MMA warp, one TMA warp, one
// thread per query row.  What differs:
//
//   items     A work item is one record of the plan (up to 256 query rows of
//             one sequence) and one head; the grid is persistent.  The list is
//             sorted by falling number of key blocks and CTAs draw from it with
//             a counter, longest first, so ragged and causal items end level.
//             Warp 11 draws an item when the TMA warp comes to the last block of
//             the one before (three blocks before the tensor core does) and
//             hands the record to the other roles through a ring in shared
//             memory.  Drawing four items ahead cost 16 % on causal 7800.
//   walk      Key blocks from the last visible one down: the blocks that need
//             masks (the ragged end, the causal diagonal) come first, the rest
//             runs without a compare.  A record of at most 128 rows drives one
//             of the two tiles only, and the first tile starts at its own
//             diagonal (a block later than the second).
//   pieces    Where few tiles would leave SMs idle (a short query behind a long
//             prefix), the plan cuts their walks; a piece leaves its unnormalised
//             O, reference maximum and row sum in fp32, and
//             wf_packed_fwd_join_kernel adds the pieces in a fixed order.
//   masks     A row's visible keys are a count; the block loop compares it
//             with the block's end and masks by column.  A row whose blocks so
//             far are all masked keeps -inf as its maximum and exponentiates
//             against 0; a row that sees nothing ends with l = 0 and is
//             written as o = 0, lse = -inf.
//   isolation Tiles are cut at the sequence, TMA boxes are not: rows behind
//             the end belong to the next sequence or to padding and may hold
//             NaN.  For K that is harmless (their scores are masked by a
//             select), for V 0 * NaN is not: the MMA warp zeroes those rows of
//             the box in shared memory before its product.  Short O tiles are
//             copied out row by row instead of by tensor store.
//   residual  For training, what rounding o to bf16 took away is written too
//             (bf16): the backward's D = rowsum(o * dO) then has 16 bits of o.
//             In rows with few keys the error of an 8-bit o in D is as large as
//             dS's own rounding (dq 1.7 times the error of one rounding, 1.4 with
//             the residual); it costs 256 bytes a row and head each way.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

namespace pfwd {
constexpr int kThreads = 384;
constexpr uint32_t kRegsSoftmax = 208;
constexpr uint32_t kRegsOther = 88;
constexpr int kKvSlots = 4;
constexpr uint32_t kBoxBytes = 128 * 128;
constexpr uint32_t kTileBytes = 2 * kBoxBytes;
constexpr uint32_t kOffQ = 0;
constexpr uint32_t kOffKV = 2 * kTileBytes;
constexpr uint32_t kOffOStage = kOffKV + kKvSlots * kTileBytes;
constexpr uint32_t kOffBar = kOffOStage + kTileBytes;
constexpr int kBarQFull = 0;                       // + tile
constexpr int kBarQEmpty = 2;                      // + tile
constexpr int kBarKvFull = 4;                      // + slot
constexpr int kBarKvEmpty = kBarKvFull + kKvSlots;
constexpr int kBarSFull = kBarKvEmpty + kKvSlots;  // + tile
constexpr int kBarPFull = kBarSFull + 2;           // + 2 * tile + half
constexpr int kBarOFull = kBarPFull + 4;           // + tile
constexpr int kBarDrain = kBarOFull + 2;
constexpr int kBarOStaged = kBarDrain + 1;
// A stage use n is freed on barrier n & 3: a warpgroup that waits for use n - 1
// may not have seen the uses before it freed (up to two of the other warpgroup
// and its own last), and one barrier's parity could not tell them apart.  Its
// own last use but one is always freed, so four barriers can.
constexpr int kBarOStageFree = kBarOStaged + 1;    // + use & 3
constexpr int kItemSlots = 4;
constexpr int kBarItemFull = kBarOStageFree + 4;         // + slot
constexpr int kBarItemEmpty = kBarItemFull + kItemSlots; // + slot; one arrival per reader
constexpr int kItemReaders = 11;                         // 8 softmax warps, MMA, TMA, store
constexpr int kBarItemNext = kBarItemEmpty + kItemSlots; // the TMA warp is at its item's last block
constexpr int kNumBars = kBarItemNext + 1;
constexpr uint32_t kOffItems = kOffBar + ((kNumBars * 8 + 15) & ~15);
constexpr uint32_t kOffTmemHolder = kOffItems + kItemSlots * 64;
constexpr uint32_t kOffAbort = kOffTmemHolder + 4;
constexpr uint32_t kSmemUsed = kOffAbort + 4;
constexpr uint32_t kSmemBytes = kSmemUsed + 1024;
static_assert(kSmemBytes <= 232448, "packed forward shared memory exceeds the per-CTA limit");
}  // namespace pfwd

// A drawn item as the roles read it.
struct __align__(16) PackedFwdItem {
  PackedFwdTile w;
  int h;      // q head; -1: no items left
  int skip0;  // blocks of the walk that no row of tile 0 sees (but one block is walked at least)
  int bad;    // kDirect: the offsets were impossible
  int pad;
};
static_assert(sizeof(PackedFwdItem) == 64, "four 16-byte words");

// Zero rows [0, none) and [first, 128) of a 128-row tile of two 64-column boxes
// (a converged warp; the swizzle permutes 16-byte chunks inside a row only),
// and order the stores before the tensor core's reads.
__device__ __forceinline__ void packed_zero_rows(uint32_t tile, int first, int none = 0) {
  for (int i = (none > 0 ? 0 : first * 8) + (int)lane_id(); i < 128 * 8; i += 32) {
    if (i >= none * 8 && i < first * 8) continue;
    st_shared_v4(tile + i * 16, 0u, 0u, 0u, 0u);
    st_shared_v4(tile + 128 * 128 + i * 16, 0u, 0u, 0u, 0u);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// kDirect: there is no plan, CTA i works on tile i / h, head i % h (465 tokens in
// five sequences, 12 heads: 16.5 us with a plan, 12.4 without).  A kernel of its
// own: with both schedulers in one, long calls ran 2 % slower.
template <bool kDirect>
__global__ void __launch_bounds__(pfwd::kThreads, 1)
    wf_packed_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                         const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                         const __grid_constant__ CUtensorMap tm_res, PackedFwdParams p) {
  using namespace pfwd;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t bar0 = sbase + kOffBar;
  auto bar = [&](int i) -> uint32_t { return bar0 + 8u * (uint32_t)i; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kOffAbort);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + kOffTmemHolder);
  const int warp = (int)warp_id();
  const int lane = (int)lane_id();

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar(kBarQFull + t), 1);
      mbar_init(bar(kBarQEmpty + t), 1);
      mbar_init(bar(kBarSFull + t), 1);
      mbar_init(bar(kBarPFull + 2 * t), 4);  // one arrival per softmax warp
      mbar_init(bar(kBarPFull + 2 * t + 1), 4);
      mbar_init(bar(kBarOFull + t), 1);
      mbar_init(bar(kBarOStageFree + t), 1);
      mbar_init(bar(kBarOStageFree + 2 + t), 1);
    }
    for (int s = 0; s < kKvSlots; ++s) {
      mbar_init(bar(kBarKvFull + s), 1);
      mbar_init(bar(kBarKvEmpty + s), 1);
    }
    for (int s = 0; s < kItemSlots; ++s) {
      mbar_init(bar(kBarItemFull + s), 1);
      mbar_init(bar(kBarItemEmpty + s), kItemReaders);
    }
    mbar_init(bar(kBarItemNext), 1);
    mbar_init(bar(kBarDrain), 1);
    mbar_init(bar(kBarOStaged), 4);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int passes = p.res != nullptr ? 2 : 1;  // o, and what its rounding took away
  // a programmatic dependent of the plan kernel, whose lists are read from here
  // on, or of whatever ran before.  The join, if one follows, may take its place on SMs as they fall free.
  griddep_launch_dependents();
  griddep_wait();
  // The k-th item of this CTA, for a whole warp (or, one = true, for one thread
  // that alone stands for its warp).  False: no more, or abort.
  auto get_item = [&](int k, PackedFwdItem& x, uint32_t role, bool one) -> bool {
    const int slot = k % kItemSlots;
    const bool ok = one ? mbar_wait(bar(kBarItemFull + slot), (uint32_t)(k / kItemSlots) & 1, abort_flag, role, 60)
                        : mbar_wait_warp(bar(kBarItemFull + slot), (uint32_t)(k / kItemSlots) & 1, abort_flag, role, 60);
    if (!ok) return false;
    x = reinterpret_cast<const PackedFwdItem*>(smem + kOffItems)[slot];
    if (one) mbar_arrive(bar(kBarItemEmpty + slot));
    else mbar_arrive_warp(bar(kBarItemEmpty + slot));
    return x.h >= 0;
  };

  if (warp == 11) {
    regs_dec<kRegsOther>();
    // ------------------------------------------------------ item scheduler
    auto set_skip0 = [&](PackedFwdItem& x) {
      const int seen0 = min(x.w.off + 127, x.w.klen);  // keys that the last row of tile 0 sees
      if (p.causal && x.w.rows > 128 && seen0 > 0)
        x.skip0 = max(0, min(x.w.j_last + 1 - (seen0 + 127) / 128, x.w.n_blocks - 1));
    };
    if constexpr (kDirect) {  // the one item of this CTA, and the end
      auto write_item = [&](int slot, const PackedFwdItem& x) {
        reinterpret_cast<PackedFwdItem*>(smem + kOffItems)[slot] = x;
        mbar_arrive(bar(kBarItemFull + slot));
      };
      PackedFwdItem x = {};
      PlanView v = {p.q_off, p.k_off, p.n, p.total_q, p.total_k, false, p.causal != 0};
      const int t = (int)blockIdx.x / p.h;
      const bool some = plan_direct_tile(v, t, x.w);
      if (lane == 0) {
        x.bad = v.bad;
        if (some) {
          x.h = (int)blockIdx.x - t * p.h;
          set_skip0(x);
          write_item(0, x);
        }
        x.h = -1;
        write_item(some ? 1 : 0, x);
      }
    } else if (lane == 0) {
      const int n_items = p.head->x * p.h;
      int next = (int)blockIdx.x;
      for (int k = 0;; ++k) {
        PackedFwdItem x = {};
        x.h = -1;
        if (next < n_items) {
          x.w = p.tiles[packed_locate(p.tiles, next, p.h, x.h)];
          set_skip0(x);
        }
        const int slot = k % kItemSlots;
        if (k >= kItemSlots && !mbar_wait(bar(kBarItemEmpty + slot), (uint32_t)(k / kItemSlots - 1) & 1, abort_flag,
                                          kRoleSchedule, 61))
          break;
        reinterpret_cast<PackedFwdItem*>(smem + kOffItems)[slot] = x;
        mbar_arrive(bar(kBarItemFull + slot));
        if (x.h < 0) break;
        if (!mbar_wait(bar(kBarItemNext), (uint32_t)k & 1, abort_flag, kRoleSchedule, 62)) break;
        next = (int)gridDim.x + atomicAdd(p.counter, 1);
      }
    }
  } else if (warp == 10) {
    regs_dec<kRegsOther>();
    // ------------------------------------------------------------ O store
    if (lane == 0) tma_prefetch_desc(&tm_o);
    int n = 0;  // tiles stored
    bool ok = true;
    PackedFwdItem x;
    for (int k = 0; ok && get_item(k, x, kRoleStore, false); ++k) {
      const PackedFwdTile& w = x.w;
      const int h = x.h;
      if (w.n_blocks == 0 || w.part >= 0) continue;
      const int stores = (w.rows > 128 ? 2 : 1) * passes;
      for (int i = 0; i < stores; ++i, ++n) {
        const int t = i / passes;
        const bool res = i - t * passes != 0;
        ok = mbar_wait_warp(bar(kBarOStaged), (uint32_t)n & 1, abort_flag, kRoleStore, 50 + t);
        if (!ok) break;
        const int rows = w.rows - t * 128;
        if (rows >= 128) {
          if (lane == 0) {
            for (int c = 0; c < 2; ++c)
              tma_store_4d(res ? &tm_res : &tm_o, sbase + kOffOStage + c * kBoxBytes, c * 64, w.q0 + t * 128, h, 0);
            bulk_commit_group();
            bulk_wait_read_all();
          }
        } else {
          // rows behind the sequence's end belong to the next one: copy the
          // valid ones, two rows of 16 chunks per pass
          __nv_bfloat16* const out = res ? p.res : p.o;
          const int c = lane & 15;
          for (int r = lane >> 4; r < rows; r += 2) {
            const uint4 v = *reinterpret_cast<const uint4*>(smem + kOffOStage + (c >> 3) * kBoxBytes +
                                                            sw128_offset((uint32_t)r, (uint32_t)(c & 7)));
            *reinterpret_cast<uint4*>(out + ((size_t)(w.q0 + t * 128 + r) * p.h + h) * 128 + c * 8) = v;
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarOStageFree + (n & 3)));
      }
    }
    if (lane == 0) bulk_wait_all();
  } else if (warp == 9) {
    regs_dec<kRegsOther>();
    // ------------------------------------------------------------------ TMA
    if (lane == 0) {
      tma_prefetch_desc(&tm_q);
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      int q_issued[2] = {0, 0};
      int issued[kKvSlots] = {0, 0, 0, 0};
      int u = 0;  // K/V units (K and V of a block alternate)
      bool ok = true;
      PackedFwdItem x;
      for (int k = 0; ok && get_item(k, x, kRoleLoad, true); ++k) {
        const PackedFwdTile& w = x.w;
        const int h = x.h, kvh = h / p.group;
        if (w.n_blocks == 0) mbar_arrive(bar(kBarItemNext));
        for (int it = 0; it < w.n_blocks && ok; ++it) {
          if (it == w.n_blocks - 1) mbar_arrive(bar(kBarItemNext));
          const int j = w.j_last - it;
          for (int kv = 0; kv < 2 && ok; ++kv, ++u) {  // 0 = K, 1 = V
            const int slot = u % kKvSlots;
            const int use = u / kKvSlots;
            if (use > 0) ok = mbar_wait(bar(kBarKvEmpty + slot), (use - 1) & 1, abort_flag, kRoleLoad, 100 + slot);
            if (!ok) break;
            mbar_expect_tx(bar(kBarKvFull + slot), kTileBytes);
            for (int c = 0; c < 2; ++c)
              tma_load_4d(sbase + kOffKV + slot * kTileBytes + c * kBoxBytes, kv ? &tm_v : &tm_k,
                          bar(kBarKvFull + slot), c * 64, w.k0 + j * 128, kvh, 0);
            issued[slot] = use + 1;
            if (it == 0 && kv == 0) {
              for (int t = 0; t * 128 < w.rows && ok; ++t) {
                if (q_issued[t] > 0)
                  ok = mbar_wait(bar(kBarQEmpty + t), (q_issued[t] - 1) & 1, abort_flag, kRoleLoad, 90 + t);
                if (!ok) break;
                mbar_expect_tx(bar(kBarQFull + t), kTileBytes);
                for (int c = 0; c < 2; ++c)
                  tma_load_4d(sbase + kOffQ + t * kTileBytes + c * kBoxBytes, &tm_q, bar(kBarQFull + t), c * 64,
                              w.q0 + t * 128, h, 0);
                q_issued[t]++;
              }
            }
          }
        }
      }
      if (*abort_flag) {
        // drain: let every issued copy land before the CTA can exit
        for (int t = 0; t < 2; ++t)
          if (q_issued[t] > 0) mbar_wait_drain(bar(kBarQFull + t), (q_issued[t] - 1) & 1);
        for (int s = 0; s < kKvSlots; ++s)
          if (issued[s] > 0) mbar_wait_drain(bar(kBarKvFull + s), (issued[s] - 1) & 1);
      }
    }
  } else if (warp == 8) {
    regs_dec<kRegsOther>();
    // ------------------------------------------------------------------ MMA
    // converged warp: all lanes wait and form descriptors, elected lanes issue
    constexpr uint32_t idesc_qk = idesc_bf16(128, 128, 0, 0);
    constexpr uint32_t idesc_pv = idesc_bf16(128, 128, 0, 1);
    const uint32_t sQ = sbase + kOffQ;
    const uint32_t sKV = sbase + kOffKV;
    bool ok = true;
    int pv_phase[2] = {0, 0};
    int q_phase[2] = {0, 0};
    auto issue_s = [&](int t, int slot_k) {
      const uint32_t d = tmem + (uint32_t)(t * 128);
      const uint64_t a0 = sdesc(sQ + t * kTileBytes, 16, 1024);
      const uint64_t b0 = sdesc(sKV + slot_k * kTileBytes, 16, 1024);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const uint32_t off = (uint32_t)((ks >> 2) * kBoxBytes + (ks & 3) * 32);
        mma_ss_e(d, desc_add(a0, off), desc_add(b0, off), idesc_qk, ks > 0);
      }
    };
    auto issue_pv = [&](int t, int slot_v, bool acc) -> bool {
      const uint32_t d = tmem + 256u + (uint32_t)(t * 128);
      const uint32_t a = tmem + (uint32_t)(t * 128);
      const uint64_t b0 = sdesc(sKV + slot_v * kTileBytes, kBoxBytes, 1024);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!mbar_wait_warp(bar(kBarPFull + 2 * t + half), (uint32_t)pv_phase[t] & 1, abort_flag, kRoleMma,
                            20 + 2 * t + half))
          return false;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const int ks = half * 4 + kk;
          mma_ts_e(d, a + ks * 8, desc_add(b0, (uint32_t)(ks * 2048)), idesc_pv, (acc || ks > 0) ? 1u : 0u);
        }
      }
      pv_phase[t]++;
      return true;
    };
    // One flat pipeline over the blocks of all items: block g issues PV_t(g-1)
    // before S_t(g) for each tile that the block has.  An item without blocks
    // issues PV(g-1) too: the softmax warps that wait for it read no item until
    // then, and with the ring full none with blocks would come.
    int g = 0;
    bool pending = false;               // PV of block g-1 is not issued yet
    bool prev[2] = {false, false};      // tiles that block g-1 has
    bool prev_acc[2] = {false, false};  // ... and adds to (not its first block)
    int prev_keys = 128;                // keys of block g-1 that exist for its item (128 but for the last block)
    bool prev_last = false;
    auto wait_v = [&]() -> bool {  // V of block g-1, its rows behind the last visible key zeroed
      const int uv = 2 * (g - 1) + 1, slot_v = uv % kKvSlots;
      if (!mbar_wait_warp(bar(kBarKvFull + slot_v), (uv / kKvSlots) & 1, abort_flag, kRoleMma, 10 + slot_v))
        return false;
      if (prev_keys < 128) packed_zero_rows(sKV + slot_v * kTileBytes, prev_keys);
      return true;
    };
    auto flush = [&]() -> bool {
      if (!pending) return true;
      pending = false;
      const int slot_v = (2 * g + kKvSlots - 1) % kKvSlots;
      if (!wait_v()) return false;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!prev[t]) continue;
        if (!issue_pv(t, slot_v, prev_acc[t])) return false;
        if (prev_last) mma_commit_e(bar(kBarOFull + t));
      }
      mma_commit_e(bar(kBarKvEmpty + slot_v));
      return true;
    };
    PackedFwdItem x;
    x.h = 0;
    for (int k = 0; ok && get_item(k, x, kRoleMma, false); ++k) {
      const PackedFwdTile& w = x.w;
      if (w.n_blocks == 0) ok = flush();
      for (int it = 0; it < w.n_blocks && ok; ++it, ++g) {
        const int uk = 2 * g, slot_k = uk % kKvSlots;
        ok = mbar_wait_warp(bar(kBarKvFull + slot_k), (uk / kKvSlots) & 1, abort_flag, kRoleMma, 10 + slot_k);
        if (!ok) break;
        tc_fence_after();
        const int slot_v = (2 * g + kKvSlots - 1) % kKvSlots;  // of block g-1
        if (pending && !(ok = wait_v())) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok) break;
          if (pending && prev[t]) {
            if (!(ok = issue_pv(t, slot_v, prev_acc[t]))) break;
            if (prev_last) mma_commit_e(bar(kBarOFull + t));
          }
          if (pending && t == 1) mma_commit_e(bar(kBarKvEmpty + slot_v));
          const int first = t == 0 ? x.skip0 : 0;
          prev[t] = t * 128 < w.rows && it >= first;
          prev_acc[t] = it > first;
          if (prev[t]) {
            if (it == first) {
              ok = mbar_wait_warp(bar(kBarQFull + t), (uint32_t)q_phase[t] & 1, abort_flag, kRoleMma, t);
              if (!ok) break;
              q_phase[t]++;
              tc_fence_after();
            }
            issue_s(t, slot_k);
            mma_commit_e(bar(kBarSFull + t));
            if (it == w.n_blocks - 1) mma_commit_e(bar(kBarQEmpty + t));
          }
        }
        if (ok) mma_commit_e(bar(kBarKvEmpty + slot_k));
        pending = true;
        prev_last = (it == w.n_blocks - 1);
        prev_keys = min(128, w.klen - (w.j_last - it) * 128);
      }
    }
    if (ok && x.h < 0) ok = flush();  // (an abort leaves another item in x)
    // drain the tensor pipe before TMEM can be released
    mma_commit_e(bar(kBarDrain));
    mbar_wait_drain(bar(kBarDrain), 0);
  } else {
    regs_inc<kRegsSoftmax>();
    // -------------------------------------------------------------- softmax
    const int t = warp >> 2;  // query tile
    const int wq = warp & 3;  // TMEM lane quadrant
    const int r = wq * 32 + lane;
    const uint32_t role = t ? kRoleSoftmax1 : kRoleSoftmax0;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lane_base + (uint32_t)(t * 128);
    const uint32_t tO = tmem + lane_base + 256u + (uint32_t)(t * 128);
    const float sl2 = p.scale_log2;
    const float thr = p.rescale_threshold;
    bool ok = true;
    int s_waits = 0;    // S_t tiles consumed
    int o_waits = 0;    // items of this tile that had keys
    int stage_use = 0;  // O tiles of both tiles staged before this item
    const bool listed_bad = kDirect ? false : p.head->y != 0;
    PackedFwdItem x;
    for (int k = 0; ok && get_item(k, x, role, false); ++k) {
      const PackedFwdTile& w = x.w;
      const int h = x.h;
      const int row = t * 128 + r;  // within the record
      if (w.n_blocks == 0) {
        // nothing to attend (or rows outside any sequence): o = 0, lse = -inf;
        // NaN where the offsets were impossible
        const bool bad = kDirect ? x.bad != 0 : listed_bad;
        const uint32_t fill = bad ? 0x7fff7fffu : 0u;
        for (int i = (int)threadIdx.x; i < w.rows * 16; i += 256) {
          const size_t at = ((size_t)(w.q0 + (i >> 4)) * p.h + h) * 128 + (i & 15) * 8;
          st_global_v4(p.o + at, fill, fill, fill, fill);
          if (passes == 2) st_global_v4(p.res + at, fill, fill, fill, fill);
        }
        if (row < w.rows) p.lse[(size_t)h * p.total_q + w.q0 + row] = bad ? __int_as_float(0x7fffffff) : -INFINITY;
        continue;
      }
      const int use0 = stage_use + t * passes;
      if (w.part < 0) stage_use += (w.rows > 128 ? 2 : 1) * passes;
      if (t * 128 >= w.rows) continue;
      const int seen = p.causal ? min(max(w.off + row, 0), w.klen) : w.klen;  // keys that this row sees
      float m_s = -INFINITY;  // running reference max, in scaled log2 units
      float l = 0.f;          // running row sum (relative to m_s)
      const int first = t == 0 ? x.skip0 : 0;
      for (int it = first; it < w.n_blocks; ++it, ++s_waits) {
        ok = mbar_wait(bar(kBarSFull + t), (uint32_t)s_waits & 1, abort_flag, role, 30 + t);
        if (!ok) break;
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tS + c * 32, s[c]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) reg_fence32(s[c]);
        const int left = seen - (w.j_last - it) * 128;  // keys of this block that the row sees
        if (left < 128) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= left) s[c][i] = __float_as_uint(-INFINITY);
        }
        __syncwarp();
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            mx[i & 3] = fmax3(mx[i & 3], __uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1]));
        const float mnew_s = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
        if (it == first) {
          m_s = mnew_s;
        } else {
          // move the reference max only when the row max grew past the rescale
          // threshold, or was -inf (a row whose blocks were all masked so far:
          // l and O are 0, the factor 2^-inf = 0)
          const bool need = mnew_s - m_s > thr;
          if (__any_sync(0xffffffffu, need)) {
            const float factor = need ? ex2_approx(m_s - mnew_s) : 1.f;
            if (need) {
              l *= factor;
              m_s = mnew_s;
            }
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(tO + c * 16, o);
              tmem_wait_ld();
              reg_fence16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tmem_st16(tO + c * 16, o);
            }
          }
        }
        const float ref = m_s == -INFINITY ? 0.f : m_s;
        const uint64_t sl2x2 = f2_pack(sl2, sl2), negx2 = f2_pack(-ref, -ref);
        float bsum = fwd_exp_half(s, 0, tS, sl2x2, negx2);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive_warp(bar(kBarPFull + 2 * t));
        bsum += fwd_exp_half(s, 2, tS, sl2x2, negx2);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive_warp(bar(kBarPFull + 2 * t + 1));
        l += bsum;
      }
      // --------------------------------------------------------- epilogue
      if (ok) ok = mbar_wait(bar(kBarOFull + t), (uint32_t)o_waits & 1, abort_flag, role, 40 + t);
      if (!ok) break;
      ++o_waits;
      tc_fence_after();
      if (w.part >= 0) {
        // a piece of the walk: its O as it stands, row by row coalesced
        const size_t slot = (size_t)w.part * p.h + h;
        float4* dst = p.part_o + (slot * 2 + t) * 4096 + r;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
          reg_fence32(o);
#pragma unroll
          for (int g = 0; g < 8; ++g)
            dst[(c * 8 + g) * 128] = make_float4(__uint_as_float(o[4 * g]), __uint_as_float(o[4 * g + 1]),
                                                 __uint_as_float(o[4 * g + 2]), __uint_as_float(o[4 * g + 3]));
        }
        p.part_ml[slot * 256 + row] = make_float2(m_s, l);
        continue;
      }
      const float inv = 1.f / l;
      const uint32_t stage = sbase + kOffOStage + (uint32_t)r * 128u;
#pragma unroll 1
      for (int pass = 0; pass < passes; ++pass) {
        const int use = use0 + pass;
        if (use > 0)
          ok = mbar_wait(bar(kBarOStageFree + ((use - 1) & 3)), (uint32_t)((use - 1) >> 2) & 1, abort_flag, role, 45 + t);
        if (!ok) break;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t o[32];
          tmem_ld32(tO + c * 32, o);
          tmem_wait_ld();
          reg_fence32(o);
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = __uint_as_float(o[2 * i]) * inv, y = __uint_as_float(o[2 * i + 1]) * inv;
            uint32_t v = pack_bf16(x, y);
            if (pass) v = pack_bf16(x - __uint_as_float(v << 16), y - __uint_as_float(v & 0xffff0000u));
            pk[i] = l == 0.f ? 0u : v;
          }
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const uint32_t chunk = (uint32_t)((c & 1) * 4 + v);
            st_shared_v4(stage + (uint32_t)(c >> 1) * kBoxBytes + ((chunk ^ ((uint32_t)r & 7u)) << 4), pk[4 * v],
                         pk[4 * v + 1], pk[4 * v + 2], pk[4 * v + 3]);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kBarOStaged));
      }
      if (!ok) break;
      if (row < w.rows)
        p.lse[(size_t)h * p.total_q + w.q0 + row] = l == 0.f ? -INFINITY : (m_s + log2f(l)) * 0.69314718055994531f;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_dealloc(tmem, 512);
}

// Joins the pieces of the split tiles: o = sum_i w_i O_i / sum_i w_i l_i with
// w_i = 2^(m_i - max m).  Bound: L2 (520 bytes a row and piece).  grid (8 *
// split tiles, h), 256 threads: 32 rows x 128 columns.
__global__ void __launch_bounds__(256) wf_packed_fwd_join_kernel(PackedFwdJoinParams p) {
  __shared__ float tile[32][132];
  griddep_launch_dependents();
  griddep_wait();
  const int t = blockIdx.x >> 3, row0 = (blockIdx.x & 7) * 32, h = blockIdx.y;
  if (t >= p.head->z) return;
  const int4 w = p.split_tiles[t];  // first row, rows, first part, parts
  if (row0 >= w.y) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = row0 + lane;
  float top = -INFINITY;
  for (int i = 0; i < w.w; ++i) top = fmaxf(top, p.part_ml[((size_t)(w.z + i) * p.h + h) * 256 + row].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float l = 0.f;
  float4 x[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) x[g] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < w.w; ++i) {
    const size_t slot = (size_t)(w.z + i) * p.h + h;
    const float2 ml = p.part_ml[slot * 256 + row];
    if (ml.y == 0.f) continue;  // the row sees none of this piece's keys (whose values may be anything)
    const float f = ex2_approx(ml.x - ref);
    l += f * ml.y;
    const float4* src = p.part_o + (slot * 2 + (row >> 7)) * 4096 + (row & 127);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 y = src[(warp * 4 + g) * 128];
      x[g].x += f * y.x, x[g].y += f * y.y, x[g].z += f * y.z, x[g].w += f * y.w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: 0
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float* d = &tile[lane][(warp * 4 + g) * 4];
    d[0] = l == 0.f ? 0.f : x[g].x * inv, d[1] = l == 0.f ? 0.f : x[g].y * inv;
    d[2] = l == 0.f ? 0.f : x[g].z * inv, d[3] = l == 0.f ? 0.f : x[g].w * inv;
  }
  if (warp == 0 && row < w.y)
    p.lse[(size_t)h * p.total_q + w.x + row] = l == 0.f ? -INFINITY : (top + log2f(l)) * 0.69314718055994531f;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int idx = threadIdx.x + i * 256;  // 32 rows x 16 chunks of 8
    const int rw = idx >> 4, ch = idx & 15;
    if (row0 + rw >= w.y) continue;
    const float* v = &tile[rw][ch * 8];
    uint32_t o[4], r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = pack_bf16(v[2 * k], v[2 * k + 1]);
      r[k] = pack_bf16(v[2 * k] - __uint_as_float(o[k] << 16), v[2 * k + 1] - __uint_as_float(o[k] & 0xffff0000u));
    }
    const size_t at = ((size_t)(w.x + row0 + rw) * p.h + h) * 128 + ch * 8;
    st_global_v4(p.o + at, o[0], o[1], o[2], o[3]);
    if (p.res != nullptr) st_global_v4(p.res + at, r[0], r[1], r[2], r[3]);
  }
}

}  // namespace wf
