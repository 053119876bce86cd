// C entries of packed attention (declared in include/wan_flash.h): argument
// checks, workspace layout, tensor maps and launches.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

namespace {

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Tiles of `rows` rows that [0, total) and n sequences can need at most: a
// ragged one per sequence, and per run of rows before and behind them; each has
// a row, so empty sequences need none.
long long packed_max_tiles(long long total, long long n, int rows) { return std::min(total, total / rows + n + 2); }

// Whether the forward goes without a plan; by the most tiles that there can be.
bool packed_fwd_direct(int n, int total_q, int total_k, int h, int sms) {
  const long long items = packed_max_tiles(total_q, n, 256) * h;
  if (n > kPackedDirectSeqs) return false;
  if (total_k <= 128 * kPackedDirectBlocks) return items <= kPackedDirectItems * sms;
  return total_k <= 128 * kPackedDirectMoreBlocks && 2 * items <= kPackedDirectItems * sms &&
         (n > 1 || 2LL * ((total_q + 255) / 256) * h > sms);
}

// Whether the plan may cut forward walks: where the query rows make few items
// and a walk can be long enough to gain from it.  Its pieces are no shorter than
// an SM's even share of all blocks (items: one per SM more than whole walks;
// partial results: two per SM), so the bounds hold whatever the lengths.
bool packed_fwd_may_split(int total_q, int total_k, int h, int sms) {
  return (long long)((total_q + 255) / 256) * h <= (long long)kPackedFwdSplitItems * sms &&
         total_k > 128 * (kPackedFwdMinChunk + kPackedFwdJoinCost);
}

struct PackedFwdWorkspace {  // byte offsets
  size_t head = 0, base, tiles, split_tiles, part_ml, part_o, bytes;
  bool may_split, direct;  // direct: no plan, and no workspace
  PackedFwdWorkspace(int n, int total_q, int total_k, int h, int sms) {
    direct = packed_fwd_direct(n, total_q, total_k, h, sms);
    may_split = !direct && packed_fwd_may_split(total_q, total_k, h, sms);
    const size_t items = may_split ? (size_t)sms : 0;
    base = 256;
    tiles = align256(base + (size_t)3 * (n + 3) * 4);
    split_tiles = align256(tiles + (packed_max_tiles(total_q, n, 256) + items) * sizeof(PackedFwdTile));
    part_ml = align256(split_tiles + items * sizeof(int4));
    part_o = part_ml + 2 * items * 256 * sizeof(float2);
    bytes = direct ? 0 : part_o + 2 * items * 8192 * sizeof(float4);
  }
};

// Items, split key tiles and partial tiles (per key-value head) that the plan
// can make at most.  It cuts walks of more than `chunk` units, and chunk is at
// least kPackedMinChunk and, few tiles or many, units * h_kv / pieces: sum ceil(u
// / chunk) <= tiles + units / chunk, and a cut tile has at most 2 u / chunk parts.
struct PackedBwdBounds {
  long long pieces, items, split_tiles, parts;
  PackedBwdBounds(int n, int total_q, int total_k, int h, int h_kv, int nsplit, int sms) {
    const long long q_tiles = packed_max_tiles(total_q, n, 128), k_tiles = packed_max_tiles(total_k, n, 128);
    const long long group = h_kv ? h / h_kv : 0;
    pieces = (long long)sms * kPackedPiecesPerSm;
    const long long units = group * q_tiles * k_tiles;
    const long long cuts = std::min(units / kPackedMinChunk, pieces / std::max(h_kv, 1)) + 1;
    // a piece has a unit at least, and a walk those of one sequence
    const long long set = std::min<long long>(nsplit, std::max(group * ((total_q + 127LL) / 128), 1LL));
    items = nsplit > 0 ? k_tiles * set : k_tiles + cuts;
    split_tiles = nsplit > 0 ? k_tiles : std::min(k_tiles, cuts);
    parts = nsplit > 0 ? (set > 1 ? k_tiles * set : 0) : 2 * cuts;
  }
};

struct PackedBwdWorkspace {  // byte offsets
  size_t head = 0, base, items, q_tiles, split_tiles, neg_lse_log2, dpsum, dq_accum, dk_part, dv_part, sem,
      sem_bytes, bytes;
  size_t q_tile_stride, dq_rows;
  PackedBwdWorkspace(int n, int total_q, int total_k, int h, int h_kv, const wf_packed_bwd_cfg* cfg, int sms) {
    const PackedBwdBounds most(n, total_q, total_k, h, h_kv, cfg->nsplit, sms);
    q_tile_stride = (size_t)packed_max_tiles(total_q, n, 128);
    dq_rows = (size_t)total_q + 8 * q_tile_stride;  // a tile's rows are rounded up to 8
    const size_t q_all = q_tile_stride * h, parts = (size_t)most.parts * h_kv;
    base = 256;
    items = align256(base + (size_t)3 * (n + 3) * 4);
    q_tiles = align256(items + (size_t)most.items * sizeof(PackedBwdItem));
    split_tiles = align256(q_tiles + q_tile_stride * sizeof(int4));
    neg_lse_log2 = align256(split_tiles + (size_t)most.split_tiles * sizeof(int4));
    dpsum = neg_lse_log2 + q_all * 512;
    dq_accum = align256(dpsum + q_all * 512);
    dk_part = dq_accum + dq_rows * h * 512;
    dv_part = dk_part + parts * 65536;
    sem = dv_part + parts * 65536;
    sem_bytes = cfg->deterministic ? q_all * 4 : 0;
    bytes = sem + sem_bytes;
  }
};

int packed_bwd_cfg_check(const wf_packed_bwd_cfg* cfg) {
  if (!cfg) return fail(WF_ERR_INVALID_ARG, "null cfg");
  if (cfg->nsplit < 0 || cfg->nsplit > 1024)
    return fail(WF_ERR_INVALID_ARG, "nsplit=%d outside [0, 1024]", cfg->nsplit);
  return WF_OK;
}

int packed_check(int n, int total_q, int total_k, int h, int h_kv, int causal) {
  if (n < 0 || total_q < 0 || total_k < 0 || h < 0 || h_kv < 0) return fail(WF_ERR_INVALID_ARG, "negative size");
  if (causal != 0 && causal != 1) return fail(WF_ERR_INVALID_ARG, "causal %d not in {0, 1}", causal);
  if (h_kv == 0 ? h != 0 : h % h_kv != 0)
    return fail(WF_ERR_INVALID_ARG, "h=%d is not a multiple of h_kv=%d", h, h_kv);
  if (h > 65535) return fail(WF_ERR_UNSUPPORTED, "h=%d exceeds 65535", h);
  // tile coordinates and item numbers are 32-bit
  if (n > (1 << 24) || total_q > (1 << 30) || total_k > (1 << 30))
    return fail(WF_ERR_UNSUPPORTED, "n=%d, total_q=%d, total_k=%d exceed 2^24 sequences of 2^30 rows", n, total_q,
                total_k);
  if (packed_max_tiles(total_q, n, 128) * h > 0x7fffffffLL || packed_max_tiles(total_k, n, 128) * h > 0x7fffffffLL)
    return fail(WF_ERR_UNSUPPORTED, "too many (tile, head) items");
  return WF_OK;
}

}  // namespace

cudaError_t packed_setup() {
  cudaError_t e = cudaSuccess;
  for (auto k : {wf_packed_fwd_kernel<false>, wf_packed_fwd_kernel<true>})
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pfwd::kSmemBytes);
  for (auto k : {wf_packed_bwd_kernel<false>, wf_packed_bwd_kernel<true>})
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bwd::kSmemBytes);
  return e;
}

}  // namespace wf

using namespace wf;

extern "C" int wf_packed_fwd_workspace(int n, int total_q, int total_k, int h, size_t* bytes) {
  if (!bytes) return fail(WF_ERR_INVALID_ARG, "null pointer");
  int rc, dev;
  if ((rc = packed_check(n, total_q, total_k, h, h ? 1 : 0, 0))) return rc;
  if ((rc = device_setup(&dev))) return rc;
  *bytes = PackedFwdWorkspace(n, total_q, total_k, h, g_dev_sms[dev]).bytes;
  return WF_OK;
}

extern "C" int wf_packed_fwd(const void* q, const void* k, const void* v, const int* q_offsets, const int* k_offsets,
                             void* o, void* o_residual, float* lse, void* workspace, size_t workspace_bytes, int n,
                             int total_q, int total_k, int h, int h_kv, int causal, void* stream) {
  return wf_packed_fwd_with(q, k, v, q_offsets, k_offsets, o, o_residual, lse, workspace, workspace_bytes, n, total_q,
                            total_k, h, h_kv, causal, nullptr, stream);
}

extern "C" int wf_packed_fwd_with(const void* q, const void* k, const void* v, const int* q_offsets,
                                  const int* k_offsets, void* o, void* o_residual, float* lse, void* workspace,
                                  size_t workspace_bytes, int n, int total_q, int total_k, int h, int h_kv, int causal,
                                  const wf_fwd_cfg* cfg, void* stream) {
  int rc = packed_check(n, total_q, total_k, h, h_kv, causal);
  if (rc) return rc;
  if (cfg && cfg->num_sms < 0) return fail(WF_ERR_INVALID_ARG, "num_sms %d < 0", cfg->num_sms);
  if (total_q == 0 || h == 0) return WF_OK;
  if (!q || !o || !lse || !q_offsets || !k_offsets || (!workspace && workspace_bytes) || (total_k > 0 && (!k || !v)))
    return fail(WF_ERR_INVALID_ARG, "null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(o_residual) ||
      !aligned16(workspace) || (reinterpret_cast<uintptr_t>(lse) & 3) || (reinterpret_cast<uintptr_t>(q_offsets) & 3) ||
      (reinterpret_cast<uintptr_t>(k_offsets) & 3))
    return fail(WF_ERR_MISALIGNED, "q/k/v/o/o_residual/workspace must be 16-byte aligned, lse and offsets 4-byte"
                                    " aligned");
  int dev;
  if ((rc = device_setup(&dev))) return rc;
  const int sms = g_dev_sms[dev];
  const PackedFwdWorkspace ws(n, total_q, total_k, h, sms);
  if (workspace_bytes < ws.bytes)
    return fail(WF_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", workspace_bytes, ws.bytes);
  CUtensorMap mq, mk, mv, mo, mr;
  // with no keys at all nothing is loaded: q stands in for the maps of k and v
  if ((rc = make_bshd_map(&mq, q, 1, total_q, h)) || (rc = make_bshd_map(&mo, o, 1, total_q, h)) ||
      (o_residual && (rc = make_bshd_map(&mr, o_residual, 1, total_q, h))) ||
      (rc = make_bshd_map(&mk, total_k ? k : q, 1, total_k ? total_k : total_q, total_k ? h_kv : h)) ||
      (rc = make_bshd_map(&mv, total_k ? v : q, 1, total_k ? total_k : total_q, total_k ? h_kv : h)))
    return rc;
  if (!o_residual) mr = mo;  // never used
  uint8_t* const w = reinterpret_cast<uint8_t*>(workspace);
  PackedPlanParams pp = {};
  pp.q_off = q_offsets, pp.k_off = k_offsets;
  pp.n = n, pp.total_q = total_q, pp.total_k = total_k, pp.causal = causal;
  pp.head = reinterpret_cast<int4*>(w + ws.head);
  pp.base = reinterpret_cast<int*>(w + ws.base);
  pp.fwd_tiles = reinterpret_cast<PackedFwdTile*>(w + ws.tiles);
  pp.split_tiles = reinterpret_cast<int4*>(w + ws.split_tiles);
  pp.h = h, pp.sms = sms;
  pp.may_split = ws.may_split ? 1 : 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const long long most_items = packed_max_tiles(total_q, n, 256) * h;
  cudaError_t e = cudaSuccess;
  if (!ws.direct) e = launch_ex(wf_packed_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, true, 1u, pp);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed plan launch");
  PackedFwdParams p = {};
  p.head = pp.head;
  p.tiles = pp.fwd_tiles;
  p.counter = &pp.head->w;
  p.o = reinterpret_cast<__nv_bfloat16*>(o);
  p.res = reinterpret_cast<__nv_bfloat16*>(o_residual);
  p.lse = lse;
  p.total_q = total_q, p.h = h, p.group = h / h_kv, p.causal = causal;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt(128.0));
  p.rescale_threshold = cfg ? cfg->rescale_threshold : 8.0f;
  p.part_o = reinterpret_cast<float4*>(w + ws.part_o);
  p.part_ml = reinterpret_cast<float2*>(w + ws.part_ml);
  p.q_off = q_offsets, p.k_off = k_offsets, p.n = n, p.total_k = total_k;
  // the CTAs draw whatever items the plan makes: up to one per SM more where it may cut
  const int ctas = cfg && cfg->num_sms > 0 ? cfg->num_sms : sms;
  const int grid = (int)(ws.direct ? most_items : std::min<long long>(most_items + (ws.may_split ? sms : 0), ctas));
  e = launch_ex(ws.direct ? wf_packed_fwd_kernel<true> : wf_packed_fwd_kernel<false>, dim3(grid), dim3(pfwd::kThreads), pfwd::kSmemBytes, st, true, 1u, mq,
                            mk, mv, mo, mr, p);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed_fwd launch");
  if (ws.may_split) {
    PackedFwdJoinParams j = {};
    j.head = pp.head;
    j.split_tiles = pp.split_tiles;
    j.part_o = p.part_o, j.part_ml = p.part_ml;
    j.o = p.o, j.res = p.res, j.lse = lse;
    j.total_q = total_q, j.h = h;
    // split tiles * h <= SMs: every one adds an item to those of whole walks
    e = launch_ex(wf_packed_fwd_join_kernel, dim3(8 * std::max(1, sms / h), h), dim3(256), 0, st, true, 1u, j);
    if (e != cudaSuccess) return cuda_fail(e, "wf_packed_fwd join launch");
  }
  return launch_check("wf_packed_fwd launch");
}

extern "C" int wf_packed_bwd_workspace(int n, int total_q, int total_k, int h, int h_kv, const wf_packed_bwd_cfg* cfg,
                                       size_t* bytes) {
  if (!bytes) return fail(WF_ERR_INVALID_ARG, "null pointer");
  int rc, dev;
  if ((rc = packed_check(n, total_q, total_k, h, h_kv, 0)) || (rc = packed_bwd_cfg_check(cfg))) return rc;
  if ((rc = device_setup(&dev))) return rc;
  *bytes = PackedBwdWorkspace(n, total_q, total_k, h, h_kv, cfg, g_dev_sms[dev]).bytes;
  return WF_OK;
}

extern "C" int wf_packed_bwd(const void* q, const void* k, const void* v, const void* o,
                             const void* o_residual, const float* lse, const void* dO, const int* q_offsets,
                             const int* k_offsets, void* dq, void* dk, void* dv,
                             void* workspace, size_t workspace_bytes, int n, int total_q, int total_k, int h, int h_kv,
                             int causal, const wf_packed_bwd_cfg* cfg, void* stream) {
  wf_bwd_cfg all = {};
  if (cfg) all.nsplit = cfg->nsplit, all.deterministic = cfg->deterministic;
  return wf_packed_bwd_with(q, k, v, o, o_residual, lse, dO, q_offsets, k_offsets, dq, dk, dv, workspace,
                            workspace_bytes, n, total_q, total_k, h, h_kv, causal, cfg ? &all : nullptr, stream);
}

extern "C" int wf_packed_bwd_with(const void* q, const void* k, const void* v, const void* o,
                                  const void* o_residual, const float* lse, const void* dO, const int* q_offsets,
                                  const int* k_offsets, void* dq, void* dk, void* dv, void* workspace,
                                  size_t workspace_bytes, int n, int total_q, int total_k, int h, int h_kv, int causal,
                                  const wf_bwd_cfg* all, void* stream) {
  int rc;
  if ((rc = packed_check(n, total_q, total_k, h, h_kv, causal))) return rc;
  if (!all) return fail(WF_ERR_INVALID_ARG, "null cfg");
  const wf_packed_bwd_cfg sizes = {all->nsplit, all->deterministic}, *const cfg = &sizes;
  if ((rc = packed_bwd_cfg_check(cfg))) return rc;
  const bool pdl = !all->pdl_off;
  if (h == 0 || (total_q == 0 && total_k == 0)) return WF_OK;
  if (total_q == 0 || total_k == 0)
    return fail(WF_ERR_UNSUPPORTED, "no queries or no keys: the caller must zero the gradients");
  if (!q || !k || !v || !o || !lse || !dO || !q_offsets || !k_offsets || !dq || !dk || !dv || !workspace)
    return fail(WF_ERR_INVALID_ARG, "null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(o_residual) ||
      !aligned16(dO) || !aligned16(dq) ||
      !aligned16(dk) || !aligned16(dv) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(lse) & 3) ||
      (reinterpret_cast<uintptr_t>(q_offsets) & 3) || (reinterpret_cast<uintptr_t>(k_offsets) & 3))
    return fail(WF_ERR_MISALIGNED, "tensors and workspace must be 16-byte aligned, lse and offsets 4-byte"
                                    " aligned");
  int dev;
  if ((rc = device_setup(&dev))) return rc;
  const int sms = g_dev_sms[dev];
  const PackedBwdBounds most(n, total_q, total_k, h, h_kv, cfg->nsplit, sms);
  const PackedBwdWorkspace ws(n, total_q, total_k, h, h_kv, cfg, sms);
  if (workspace_bytes < ws.bytes)
    return fail(WF_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", workspace_bytes, ws.bytes);
  const long long dq_blocks = 2LL * ws.q_tile_stride * h, split_blocks = most.parts ? 2LL * most.split_tiles * h_kv : 0;
  if (most.items * h_kv > 0x7fffffffLL || dq_blocks + 2 * split_blocks > 0x7fffffffLL)
    return fail(WF_ERR_UNSUPPORTED, "%lld work items exceed the grid limit", most.items * h_kv);
  CUtensorMap mq, mk, mv, mdo;
  if ((rc = make_bshd_map(&mq, q, 1, total_q, h)) || (rc = make_bshd_map(&mk, k, 1, total_k, h_kv)) ||
      (rc = make_bshd_map(&mv, v, 1, total_k, h_kv)) || (rc = make_bshd_map(&mdo, dO, 1, total_q, h)))
    return rc;
  uint8_t* const w = reinterpret_cast<uint8_t*>(workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  PackedPlanParams pp = {};
  pp.q_off = q_offsets, pp.k_off = k_offsets;
  pp.n = n, pp.total_q = total_q, pp.total_k = total_k, pp.causal = causal;
  pp.backward = 1;
  pp.ordered = cfg->deterministic ? 1 : 0;
  pp.h = h, pp.group = h / h_kv, pp.h_kv = h_kv, pp.sms = sms;
  pp.nsplit = cfg->nsplit;
  pp.pieces = (int)most.pieces;
  pp.head = reinterpret_cast<int4*>(w + ws.head);
  pp.base = reinterpret_cast<int*>(w + ws.base);
  pp.items = reinterpret_cast<PackedBwdItem*>(w + ws.items);
  pp.q_tiles = reinterpret_cast<int4*>(w + ws.q_tiles);
  pp.split_tiles = reinterpret_cast<int4*>(w + ws.split_tiles);
  PackedBwdParams p = {};
  p.head = pp.head;
  p.items = pp.items;
  p.q_tiles = pp.q_tiles;
  p.neg_lse_log2 = reinterpret_cast<float*>(w + ws.neg_lse_log2);
  p.dpsum = reinterpret_cast<float*>(w + ws.dpsum);
  p.dq_accum = reinterpret_cast<float*>(w + ws.dq_accum);
  p.dk = reinterpret_cast<__nv_bfloat16*>(dk);
  p.dv = reinterpret_cast<__nv_bfloat16*>(dv);
  p.dk_part = reinterpret_cast<float*>(w + ws.dk_part);
  p.dv_part = reinterpret_cast<float*>(w + ws.dv_part);
  p.sem = reinterpret_cast<int*>(w + ws.sem);
  p.q_tile_stride = ws.q_tile_stride, p.dq_rows = ws.dq_rows;
  p.total_q = total_q, p.h = h, p.h_kv = h_kv, p.group = h / h_kv;
  p.ordered = pp.ordered;
  p.wave = sms;
  p.scale = (float)(1.0 / std::sqrt(128.0));
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt(128.0));
  if (ws.sem_bytes) {
    const cudaError_t e = cudaMemsetAsync(p.sem, 0, ws.sem_bytes, st);
    if (e != cudaSuccess) return cuda_fail(e, "wf_packed_bwd counters");
  }
  cudaError_t e = launch_ex(wf_packed_plan_kernel, dim3(2), dim3(kPlanThreads), 0, st, pdl, 1u, pp);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed plan launch");
  e = launch_ex(wf_packed_pre_kernel, dim3((unsigned)(2 * ws.q_tile_stride), h), dim3(256), 0, st, pdl, 1u, p,
                reinterpret_cast<const __nv_bfloat16*>(o), reinterpret_cast<const __nv_bfloat16*>(o_residual),
                reinterpret_cast<const __nv_bfloat16*>(dO), lse);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed_bwd preprocess launch");
  e = launch_ex(causal ? wf_packed_bwd_kernel<true> : wf_packed_bwd_kernel<false>,
                dim3((unsigned)(most.items * h_kv)), dim3(bwd::kThreads), bwd::kSmemBytes, st, pdl, 1u, mq, mk, mv, mdo,
                p);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed_bwd launch");
  PackedConvertParams c = {};
  c.head = pp.head;
  c.q_tiles = pp.q_tiles, c.split_tiles = pp.split_tiles;
  c.dq_accum = p.dq_accum, c.dk_part = p.dk_part, c.dv_part = p.dv_part;
  c.dq = reinterpret_cast<__nv_bfloat16*>(dq), c.dk = p.dk, c.dv = p.dv;
  c.dq_blocks = (unsigned)dq_blocks, c.split_blocks = (unsigned)split_blocks;
  c.dq_rows = ws.dq_rows;
  c.h = h, c.h_kv = h_kv;
  c.scale = p.scale;
  e = launch_ex(wf_packed_convert_kernel, dim3((unsigned)(dq_blocks + 2 * split_blocks)), dim3(256), 0, st, pdl, 1u,
                c);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed_bwd convert launch");
  return launch_check("wf_packed_bwd launch");
}
