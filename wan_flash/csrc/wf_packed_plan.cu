// Work lists of the packed attention kernels, made on the device from the
// sequence offsets (the host never reads them, so nothing synchronises and a
// captured graph may be replayed with other offsets).
//
// One CTA per list.  The rows [0, total) fall into n + 2 segments: the rows
// before the first sequence, the n sequences, the rows behind the last; every
// segment is cut into tiles of T rows.  A scan over the segments gives each
// its first tile; each tile finds its segment by binary search.
//
// Items (forward: query tiles; backward: key tiles, or pieces of one) are
// sorted by falling cost in a counting sort, so CTAs that take them in turn end
// together although sequences are ragged and causal tiles grow with their row.
// Items of equal cost form a bucket, and inside a bucket the kernels run head
// by head (packed_locate): the tiles of one sequence and head, which read the
// same keys (backward: queries), run side by side.
//
// Pieces: a backward key tile with a long walk over (query tile, q head) units is
// cut into pieces whose partial dK and dV a convert sums, so one long sequence
// fills the GPU as evenly as many; a forward walk over key blocks is cut where
// few tiles (a short query behind a long prefix) would leave SMs idle, and a
// join adds its partial results.
//
// Offsets that fall, start below 0 or end behind the tensor set the device
// error word; the lists then hold only rows outside any sequence, with
// status 1 (the kernels write NaN there).
//
// Bound: latency (a chain of barriers, dependent loads and cold code).  Up to
// 2045 sequences the offsets and scans stay in shared memory; a thread keeps
// the record of its first tile in registers over the passes; 256 threads
// because most calls have fewer tiles and barriers cost by the warp.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanBuckets = 256;
constexpr int kPlanSmall = 2048;  // n + 3 up to this: offsets and tile bases in shared memory
static_assert(kPlanBuckets == kPlanThreads, "one bucket per thread in the scan");

struct PlanShared {
  int warp_sum[kPlanThreads / 32];
  int start[kPlanBuckets + 1];
  int cursor[kPlanBuckets];
  unsigned long long units;
  int most, items, parts, split_tiles;
  int q_off[kPlanSmall], k_off[kPlanSmall], base0[kPlanSmall], base1[kPlanSmall];
};

// Exclusive block scan of one int per thread; returns the prefix, *total the sum.
__device__ __noinline__ int plan_scan(PlanShared& sh, int x, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += up;
  }
  if (lane == 31) sh.warp_sum[warp] = incl;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 32; ++i) {
    const int s = sh.warp_sum[i];
    if (i < warp) before += s;
    sum += s;
  }
  __syncthreads();
  *total = sum;
  return before + incl - x;
}

// Segment s of rows [0, total): start and length.  Segments 1..n are the sequences.
__device__ __forceinline__ void plan_segment(const int* off, int n, int total, bool bad, int s, int& start, int& len) {
  if (bad) {  // everything lies outside any sequence
    start = 0;
    len = s == 0 ? total : 0;
    return;
  }
  start = s == 0 ? 0 : off[s - 1];
  len = (s <= n ? off[s] : total) - start;
}

__device__ __forceinline__ bool plan_bad(const int* off, int s, int total) {
  return off[s] < 0 || off[s] > total || (s > 0 && off[s] < off[s - 1]);
}

// base[s] = first tile of segment s (s = 0..n+1), base[n+2] = number of tiles
__device__ __noinline__ int plan_bases(PlanShared& sh, const int* off, int n, int total, bool bad, int tile, int* base) {
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

struct PlanView {
  const int* q_off;
  const int* k_off;
  int n, total_q, total_k;
  bool bad, causal;
};

// Forward tile i of segment s: up to 256 query rows.
__device__ __forceinline__ PackedFwdTile plan_fwd_tile_of(const PlanView& p, int s, int i) {
  int qs, lq;
  plan_segment(p.q_off, p.n, p.total_q, p.bad, s, qs, lq);
  const int m0 = i * 256;
  PackedFwdTile w;
  w.q0 = qs + m0;
  w.rows = min(256, lq - m0);
  w.k0 = w.klen = w.off = w.n_blocks = w.j_last = w.bucket = w.bucket_items = w.pad0 = w.pad1 = 0;
  w.part = -1;
  if (!p.bad && s >= 1 && s <= p.n) {
    const int ks = p.k_off[s - 1], lk = p.k_off[s] - ks;
    w.k0 = ks;
    w.off = p.causal ? m0 + lk - lq + 1 : lk;  // keys that the tile's first row sees (causal: may be negative)
    w.klen = p.causal ? max(0, w.off + w.rows - 1) : lk;
    w.n_blocks = (w.klen + 127) / 128;
    w.j_last = w.n_blocks - 1;
  }
  return w;
}

__device__ __noinline__ PackedFwdTile plan_fwd_tile(const PlanView& p, const int* base, int t) {
  const int s = plan_find(base, p.n, t);
  return plan_fwd_tile_of(p, s, t - base[s]);
}

__device__ __forceinline__ void plan_report_bad() {
  if (atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_INVALID_ARG) == 0u) {
    g_err_info[0] = g_err_info[1] = g_err_info[3] = 0u;
    g_err_info[2] = kRolePackedPlan;
  }
}

// Forward tile t without a plan, by one converged warp; bad: impossible offsets.
// False: there is no such tile.
__device__ __forceinline__ bool plan_direct_tile(PlanView& p, int t, PackedFwdTile& w) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  for (int s = lane; s <= p.n; s += 32) bad |= plan_bad(p.q_off, s, p.total_q) || plan_bad(p.k_off, s, p.total_k);
  p.bad = __any_sync(0xffffffffu, bad);
  if (p.bad && lane == 0) plan_report_bad();
  int carry = 0;
  for (int s0 = 0; s0 < p.n + 2; s0 += 32) {
    int start, len = 0;
    if (s0 + lane < p.n + 2) plan_segment(p.q_off, p.n, p.total_q, p.bad, s0 + lane, start, len);
    const int tiles = (len + 255) / 256;
    int incl = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    const int first = carry + incl - tiles;
    const unsigned here = __ballot_sync(0xffffffffu, t >= first && t < first + tiles);
    if (here) {
      const int src = __ffs(here) - 1;
      w = plan_fwd_tile_of(p, s0 + src, t - __shfl_sync(0xffffffffu, first, src));
      return true;
    }
    carry += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// Backward key tile t: 128 key rows, and the query tiles that see them.
__device__ __noinline__ PackedBwdItem plan_k_tile(const PlanView& p, const int* kbase, const int* qbase, int t) {
  const int s = plan_find(kbase, p.n, t);
  int ks, lk;
  plan_segment(p.k_off, p.n, p.total_k, p.bad, s, ks, lk);
  const int n0 = (t - kbase[s]) * 128;
  PackedBwdItem w;
  w.k0 = ks + n0;
  w.rows = min(128, lk - n0);
  w.q0 = w.lq = w.qtile = w.m_begin = w.m_count = w.need = 0;
  w.nb = t - kbase[s];
  w.first = w.count = 0;
  w.part = -1;
  w.bucket = w.bucket_items = w.pad0 = w.pad1 = 0;
  if (!p.bad && s >= 1 && s <= p.n) {
    const int qs = p.q_off[s - 1], lq = p.q_off[s] - qs;
    w.q0 = qs;
    w.lq = lq;
    w.qtile = qbase[s];
    w.need = p.causal ? n0 - lk + lq : -0x40000000;  // first query row that sees the tile's first key (may be negative)
    w.m_begin = max(w.need, 0) / 128;
    w.m_count = max(0, (lq + 127) / 128 - w.m_begin);
  }
  return w;
}

// Adds to sh.units and raises sh.most by every thread's values (one atomic a warp).
__device__ __noinline__ void plan_totals(PlanShared& sh, unsigned long long units, int most) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) units += __shfl_xor_sync(0xffffffffu, units, d);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) {
    atomicAdd(&sh.units, units);
    atomicMax(&sh.most, most);
  }
  __syncthreads();
}

// The smallest chunk from `from` on with which all walks, cut into pieces of at
// most chunk, make at most `sms` items over `heads` heads; `most` (whole walks)
// where none does.
template <typename Cost>
__device__ int plan_fit(PlanShared& sh, int n_tiles, int heads, int sms, int most, long long from, Cost&& cost) {
  int chunk = (int)min(from, (long long)max(most, 1));
  while (chunk < most) {
    int mine = 0, items;
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads)
      mine += max(1, (int)(((unsigned)cost(t) + (unsigned)chunk - 1u) / (unsigned)chunk));
    plan_scan(sh, mine, &items);
    if ((long long)items * heads <= sms) return chunk;
    chunk = min((long long)most, (long long)chunk + chunk / 8 + 1);
  }
  return max(most, 1);
}

// Buckets of falling cost: sizes from count(add), their starts in sh.start.
template <typename Count>
__device__ void plan_buckets(PlanShared& sh, int n_tiles, int shift, Count&& count) {
  for (int i = threadIdx.x; i < kPlanBuckets; i += kPlanThreads) sh.cursor[i] = 0;
  __syncthreads();
  for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads)
    count(t, [&](int cost) { atomicAdd(&sh.cursor[kPlanBuckets - 1 - (cost >> shift)], 1); });
  __syncthreads();
  int sum;
  const int first = plan_scan(sh, sh.cursor[threadIdx.x], &sum);
  sh.start[threadIdx.x] = sh.cursor[threadIdx.x] = first;
  if (threadIdx.x == 0) sh.start[kPlanBuckets] = sum;
  __syncthreads();
}
// A place for an item of that cost, and its bucket.
template <typename Item>
__device__ int plan_place(PlanShared& sh, int cost, int shift, Item& w) {
  const int b = kPlanBuckets - 1 - (cost >> shift);
  w.bucket = sh.start[b];
  w.bucket_items = sh.start[b + 1] - sh.start[b];
  return atomicAdd(&sh.cursor[b], 1);
}

// The next free place, for an item of a list that is not sorted.
template <typename Item>
__device__ int plan_next(PlanShared& sh, Item& w) {
  w.bucket = atomicAdd(&sh.items, 1);
  w.bucket_items = 1;
  return w.bucket;
}

}  // namespace

// grid 1 (forward) or 2 (backward: block 0 the items, block 1 the query tiles)
__global__ void __launch_bounds__(kPlanThreads) wf_packed_plan_kernel(PackedPlanParams p) {
  __shared__ PlanShared sh;
  // a programmatic dependent of whatever ran before
  griddep_wait();
  griddep_launch_dependents();  // (only now: the next kernels' read-only loads must not meet that one's writes)
  const bool small = p.n + 3 <= kPlanSmall;
  if (threadIdx.x == 0) sh.units = 0ull, sh.most = sh.items = sh.parts = sh.split_tiles = 0;
  if (small) {
    for (int s = threadIdx.x; s <= p.n; s += kPlanThreads) {
      sh.q_off[s] = p.q_off[s];
      sh.k_off[s] = p.k_off[s];
    }
  }
  __syncthreads();
  PlanView v;
  v.q_off = small ? sh.q_off : p.q_off;
  v.k_off = small ? sh.k_off : p.k_off;
  v.n = p.n, v.total_q = p.total_q, v.total_k = p.total_k, v.causal = p.causal != 0;
  bool bad = false;
  for (int s = threadIdx.x; s <= p.n; s += kPlanThreads)
    bad |= plan_bad(v.q_off, s, p.total_q) || plan_bad(v.k_off, s, p.total_k);
  v.bad = __syncthreads_or(bad);
  if (v.bad && threadIdx.x == 0) plan_report_bad();
  int* const base0 = small ? sh.base0 : p.base + (blockIdx.x ? 2 * (p.n + 3) : 0);
  int* const base1 = small ? sh.base1 : p.base + (p.n + 3);  // block 0 of the backward only

  if (!p.backward) {
    const int n_tiles = plan_bases(sh, v.q_off, p.n, p.total_q, v.bad, 256, base0);
    PackedFwdTile mine = {};  // this thread's first tile
    if ((int)threadIdx.x < n_tiles) mine = plan_fwd_tile(v, base0, threadIdx.x);
    auto tile = [&](int t) { return t < kPlanThreads ? mine : plan_fwd_tile(v, base0, t); };
    const bool few = (long long)n_tiles * p.h <= p.sms;  // all items run at once: no need to sort
    if (few && !p.may_split) {
      for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
        PackedFwdTile w = tile(t);
        w.bucket = t;
        w.bucket_items = 1;
        p.fwd_tiles[t] = w;
      }
      if (threadIdx.x == 0) p.head[0] = make_int4(n_tiles, v.bad, 0, 0);
      return;
    }
    int most = 0;
    unsigned long long blocks = 0;
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
      most = max(most, tile(t).n_blocks);
      blocks += tile(t).n_blocks;
    }
    plan_totals(sh, blocks, most);
    most = sh.most;
    int chunk = max(most, 1);
    if (p.may_split && most > kPackedFwdMinChunk) {
      // an SM's even share of the blocks; a longer walk alone would be the time
      const long long share = (long long)(sh.units * p.h + p.sms - 1) / p.sms;
      if (2LL * n_tiles * p.h <= p.sms)  // at most one piece per SM
        chunk = plan_fit(sh, n_tiles, p.h, p.sms, most, max((long long)kPackedFwdMinChunk, share),
                         [&](int t) { return tile(t).n_blocks; });
      else
        chunk = (int)min((long long)most, max((long long)kPackedFwdMinChunk, share + share / 8 + 1));
      if (chunk + kPackedFwdJoinCost > most) chunk = most;  // the join would take what the cut saves
    }
    int shift = 0;
    while ((min(most, chunk) >> shift) >= kPlanBuckets) ++shift;
    auto pieces_of = [&](int n) { return n > chunk ? (n + chunk - 1) / chunk : 1; };
    if (!few)
      plan_buckets(sh, n_tiles, shift, [&](int t, auto add) {
        const int n = tile(t).n_blocks, s = pieces_of(n), even = n / s, more = n - even * s;
        for (int i = 0; i < s; ++i) add(even + (i < more ? 1 : 0));
      });
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
      PackedFwdTile w = tile(t);
      const int n = w.n_blocks, s = pieces_of(n), even = n / s, more = n - even * s;
      int part = -1;
      if (s > 1) {  // any place will do: the parts of a tile are joined in their order
        part = atomicAdd(&sh.parts, s);
        p.split_tiles[atomicAdd(&sh.split_tiles, 1)] = make_int4(w.q0, w.rows, part, s);
      }
      for (int i = 0; i < s; ++i) {
        w.n_blocks = even + (i < more ? 1 : 0);
        w.j_last = (i + 1) * even + min(i + 1, more) - 1;
        w.part = s > 1 ? part + i : -1;
        const int at = few ? plan_next(sh, w) : plan_place(sh, w.n_blocks, shift, w);
        p.fwd_tiles[at] = w;
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) p.head[0] = make_int4(few ? sh.items : sh.start[kPlanBuckets], v.bad, sh.split_tiles, 0);
    return;
  }
  if (blockIdx.x == 1) {
    // query tiles, in the order of the rows: the index is the tile's place in the fp32 workspaces
    const int n_tiles = plan_bases(sh, v.q_off, p.n, p.total_q, v.bad, 128, base0);
    for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
      const int s = plan_find(base0, p.n, t);
      int qs, lq;
      plan_segment(v.q_off, p.n, p.total_q, v.bad, s, qs, lq);
      const int m0 = (t - base0[s]) * 128;
      p.q_tiles[t] = make_int4(qs + m0, min(128, lq - m0), !v.bad && s >= 1 && s <= p.n, 0);
    }
    if (threadIdx.x == 0) p.head[1] = make_int4(n_tiles, v.bad, 0, 0);
    return;
  }
  const int n_tiles = plan_bases(sh, v.k_off, p.n, p.total_k, v.bad, 128, base0);
  plan_bases(sh, v.q_off, p.n, p.total_q, v.bad, 128, base1);
  PackedBwdItem mine = {};  // this thread's first key tile
  if ((int)threadIdx.x < n_tiles) mine = plan_k_tile(v, base0, base1, threadIdx.x);
  auto tile = [&](int t) { return t < kPlanThreads ? mine : plan_k_tile(v, base0, base1, t); };
  unsigned long long units = 0;
  int most = 0;
  for (int t = threadIdx.x; t < n_tiles; t += kPlanThreads) {
    const int u = tile(t).m_count * p.group;
    units += u;
    most = max(most, u);
  }
  plan_totals(sh, units, most);
  most = sh.most;
  int chunk;
  bool one_round = false;  // all items run at once: no need to sort
  if (p.nsplit > 0) {
    chunk = max(1, (int)(((unsigned)most + p.nsplit - 1) / p.nsplit));
  } else {
    // pieces of half an SM's even share, so their uneven ends even out ...
    chunk = (int)min((unsigned long long)0x7fffffff,
                     max((unsigned long long)kPackedMinChunkFull, sh.units * p.h_kv / p.pieces + 1));
    if ((long long)n_tiles * p.h_kv <= p.sms) {
      // ... or at most one piece per SM: the longest then is the time.  Each piece costs kPackedPieceCost units too
      const int share = (int)((sh.units * p.h_kv + p.sms - 1) / p.sms);
      const int one = plan_fit(sh, n_tiles, p.h_kv, p.sms, most, max(kPackedMinChunk, share),
                               [&](int t) { return tile(t).m_count * p.group; });
      if (one + kPackedPieceCost <= share + share / chunk * kPackedPieceCost + kPackedPieceCost + chunk / 2) {
        chunk = one;
        one_round = !p.ordered;
      }
    }
  }
  // a walk of u units in s pieces: the first u % s have one unit more
  auto pieces_of = [&](int u) { return u > chunk ? (int)(((unsigned)u + (unsigned)chunk - 1u) / (unsigned)chunk) : 1; };
  int shift = 0;
  while ((min(most, chunk) >> shift) >= kPlanBuckets) ++shift;
  if (!p.ordered && !one_round)
    plan_buckets(sh, n_tiles, shift, [&](int t, auto add) {
      const int u = tile(t).m_count * p.group, s = pieces_of(u), even = u / s, more = u - even * s;
      for (int i = 0; i < s; ++i) add(even + (i < more ? 1 : 0));
    });
  int items = 0;
  for (int t0 = 0; t0 < n_tiles; t0 += kPlanThreads) {
    const int t = t0 + threadIdx.x;
    PackedBwdItem w;
    int u = 0, s = 0, at = 0;
    if (t < n_tiles) {
      w = tile(t);
      u = w.m_count * p.group;
      s = pieces_of(u);
    }
    if (p.ordered) {
      int sum;
      at = items + plan_scan(sh, s, &sum);
      items += sum;
    }
    int part = -1;
    if (s > 1) {  // any place will do: the parts of a tile are summed in their order
      part = atomicAdd(&sh.parts, s);
      p.split_tiles[atomicAdd(&sh.split_tiles, 1)] = make_int4(w.k0, w.rows, part, s);
    }
    const int even = s ? u / s : 0, more = u - even * s;
    for (int i = 0; i < s; ++i) {
      w.first = i * even + min(i, more);
      w.count = even + (i < more ? 1 : 0);
      w.part = s > 1 ? part + i : -1;
      int place = at + i;  // ordered: key tiles as they stand, one after the other
      w.bucket = place;
      w.bucket_items = 1;
      if (one_round) place = plan_next(sh, w);
      else if (!p.ordered) place = plan_place(sh, w.count, shift, w);
      p.items[place] = w;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const int n_items = p.ordered ? items : one_round ? sh.items : sh.start[kPlanBuckets];
    p.head[0] = make_int4(n_items, v.bad, sh.split_tiles, 0);
  }
}

// Work index i (of items * heads) -> item and head: bucket by bucket, inside a
// bucket head by head.  The item at place i / heads lies in the right bucket.
template <typename Item>
__device__ __forceinline__ int packed_locate(const Item* list, int i, int heads, int& head) {
  const int at = i / heads;
  const int first = list[at].bucket, n = list[at].bucket_items;
  const int r = i - first * heads;
  head = r / n;
  return first + (r - head * n);
}

}  // namespace wf
