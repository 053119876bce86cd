// Work lists of the packed attention kernels, made on the device from the
// sequence offsets (the host never reads them, so nothing synchronises and a
// captured graph may be replayed with other offsets).
//
// One CTA per list.  The rows [0, total) fall into n + 2 segments: the rows
// before the first sequence, the n sequences, the rows behind the last; every
// segment is cut into tiles of T rows.  A scan over the segments gives each
// its first tile; each tile finds its segment by binary search.  Lists whose
// tiles differ in cost (forward query tiles, backward key tiles) are sorted by
// falling cost, a counting sort on the number of 128-row blocks the tile
// walks: CTAs that take their items in turn then end together although
// sequences are ragged and causal tiles grow with their row.
//
// Offsets that fall, start below 0 or end behind the tensor set the device
// error word; the lists then hold only rows outside any sequence, with
// status 1 (the kernels write NaN there).
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanBuckets = 1024;

struct PlanShared {
  int warp_sum[32];
  int carry;
  int bad;
  int hist[kPlanBuckets];
};

// Exclusive block scan of one int per thread; returns the prefix, *total the sum.
__device__ int plan_scan(PlanShared& sh, int x, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) sh.warp_sum[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = sh.warp_sum[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += up;
    }
    sh.warp_sum[lane] = w;
  }
  __syncthreads();
  const int before = warp ? sh.warp_sum[warp - 1] : 0;
  *total = sh.warp_sum[31];
  __syncthreads();
  return before + incl - x;
}

// Segment s of rows [0, total): start and length.  Segments 1..n are the sequences.
__device__ __forceinline__ void plan_segment(const int* off, int n, int total, bool bad, int s, int& start, int& len) {
  if (bad) {  // everything lies outside any sequence
    start = 0;
    len = s == 0 ? total : 0;
    return;
  }
  const int a = s == 0 ? 0 : __ldg(off + s - 1), b = s <= n ? __ldg(off + s) : total;
  start = a;
  len = (s == 0 ? __ldg(off) : b) - a;
}

__device__ bool plan_offsets_bad(const int* off, int n, int total) {
  bool bad = false;
  for (int s = threadIdx.x; s <= n; s += kPlanThreads) {
    const int x = __ldg(off + s);
    if (x < 0 || x > total || (s > 0 && x < __ldg(off + s - 1))) bad = true;
  }
  return __syncthreads_or(bad);
}

// base[s] = first tile of segment s (s = 0..n+1), base[n+2] = number of tiles
__device__ int plan_bases(PlanShared& sh, const int* off, int n, int total, bool bad, int tile, int* base) {
  int carry = 0;
  for (int s0 = 0; s0 < n + 2; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int start, len = 0;
    if (s < n + 2) plan_segment(off, n, total, bad, s, start, len);
    int sum;
    const int before = plan_scan(sh, (len + tile - 1) / tile, &sum);
    if (s < n + 2) base[s] = carry + before;
    carry += sum;
  }
  if (threadIdx.x == 0) base[n + 2] = carry;
  __syncthreads();
  return carry;
}

// The segment that tile t belongs to: the last s with base[s] <= t.
__device__ int plan_find(const int* base, int n, int t) {
  int lo = 0, hi = n + 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (base[mid] <= t) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Forward tile t: kFwdTileRows query rows.
__device__ PackedFwdTile plan_fwd_tile(const PackedPlanParams& p, bool bad, const int* base, int t) {
  const int s = plan_find(base, p.n, t);
  int qs, lq;
  plan_segment(p.q_off, p.n, p.total_q, bad, s, qs, lq);
  const int m0 = (t - base[s]) * 256;
  PackedFwdTile w;
  w.q0 = qs + m0;
  w.rows = min(256, lq - m0);
  w.k0 = w.klen = w.off = w.n_blocks = w.pad0 = w.pad1 = 0;
  if (!bad && s >= 1 && s <= p.n) {
    const int ks = __ldg(p.k_off + s - 1), lk = __ldg(p.k_off + s) - ks;
    w.k0 = ks;
    w.off = p.causal ? m0 + lk - lq + 1 : lk;  // keys that the tile's first row sees (causal: may be negative)
    w.klen = p.causal ? max(0, w.off + w.rows - 1) : lk;
    w.n_blocks = (w.klen + 127) / 128;
  }
  return w;
}

// Backward key tile t: 128 key rows, and the query tiles that see them.
__device__ PackedKTile plan_k_tile(const PackedPlanParams& p, bool bad, const int* kbase, const int* qbase, int t) {
  const int s = plan_find(kbase, p.n, t);
  int ks, lk;
  plan_segment(p.k_off, p.n, p.total_k, bad, s, ks, lk);
  const int n0 = (t - kbase[s]) * 128;
  PackedKTile w;
  w.k0 = ks + n0;
  w.rows = min(128, lk - n0);
  w.q0 = w.lq = w.m_begin = w.m_count = w.qtile = w.need = 0;
  w.nb = t - kbase[s];
  w.pad0 = w.pad1 = w.pad2 = 0;
  if (!bad && s >= 1 && s <= p.n) {
    const int qs = __ldg(p.q_off + s - 1), lq = __ldg(p.q_off + s) - qs;
    w.q0 = qs;
    w.lq = lq;
    w.qtile = qbase[s];
    w.need = p.causal ? n0 - lk + lq : -0x40000000;  // first query row that sees the tile's first key (may be negative)
    w.m_begin = max(w.need, 0) / 128;
    w.m_count = max(0, (lq + 127) / 128 - w.m_begin);
  }
  return w;
}

}  // namespace

// grid 1 (forward) or 2 (backward: block 0 the key tiles, block 1 the query tiles)
__global__ void __launch_bounds__(kPlanThreads) wf_packed_plan_kernel(PackedPlanParams p) {
  __shared__ PlanShared sh;
  griddep_launch_dependents();
  const bool bad = plan_offsets_bad(p.q_off, p.n, p.total_q) | plan_offsets_bad(p.k_off, p.n, p.total_k);
  if (bad && threadIdx.x == 0 && atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_INVALID_ARG) == 0u) {
    g_err_info[0] = g_err_info[1] = g_err_info[3] = 0u;
    g_err_info[2] = kRolePackedPlan;
  }
  const bool q_list = p.backward && blockIdx.x == 1;
  int* const base = p.base + (q_list ? 2 * (p.n + 3) : 0);
  const bool k_list = p.backward && !q_list;
  const int n_tiles = k_list ? plan_bases(sh, p.k_off, p.n, p.total_k, bad, 128, base)
                             : plan_bases(sh, p.q_off, p.n, p.total_q, bad, p.backward ? 128 : 256, base);
  if (q_list) {  // in the order of the rows: the index is the tile's place in the fp32 workspaces
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
      const int s = plan_find(base, p.n, t);
      int qs, lq;
      plan_segment(p.q_off, p.n, p.total_q, bad, s, qs, lq);
      const int m0 = (t - base[s]) * 128;
      p.q_tiles[t] = make_int4(qs + m0, min(128, lq - m0), !bad && s >= 1 && s <= p.n, 0);
    }
    if (threadIdx.x == 0) p.head[1] = make_int4(n_tiles, bad, 0, 0);
    return;
  }
  int* const qbase = p.base + (p.n + 3);
  if (k_list) plan_bases(sh, p.q_off, p.n, p.total_q, bad, 128, qbase);
  if (p.ordered) {
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) p.k_tiles[t] = plan_k_tile(p, bad, base, qbase, t);
  } else {
    for (int i = threadIdx.x; i < kPlanBuckets; i += kPlanThreads) sh.hist[i] = 0;
    __syncthreads();
    auto bucket = [&](int cost) { return kPlanBuckets - 1 - min(cost >> p.cost_shift, kPlanBuckets - 1); };
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
      const int cost = k_list ? plan_k_tile(p, bad, base, qbase, t).m_count : plan_fwd_tile(p, bad, base, t).n_blocks;
      atomicAdd(&sh.hist[bucket(cost)], 1);
    }
    __syncthreads();
    static_assert(kPlanBuckets == kPlanThreads, "one bucket per thread");
    int sum;
    const int first = plan_scan(sh, sh.hist[threadIdx.x], &sum);
    sh.hist[threadIdx.x] = first;
    __syncthreads();
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
      if (k_list) {
        const PackedKTile w = plan_k_tile(p, bad, base, qbase, t);
        p.k_tiles[atomicAdd(&sh.hist[bucket(w.m_count)], 1)] = w;
      } else {
        const PackedFwdTile w = plan_fwd_tile(p, bad, base, t);
        p.fwd_tiles[atomicAdd(&sh.hist[bucket(w.n_blocks)], 1)] = w;
      }
    }
  }
  if (threadIdx.x == 0) p.head[0] = make_int4(n_tiles, bad, 0, 0);
}

}  // namespace wf
