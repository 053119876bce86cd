// C entries of packed attention (declared in include/wan_flash.h): argument
// checks, workspace layout, tensor maps and launches.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

namespace {

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Tiles of `rows` rows that [0, total) and n sequences can need at most: a
// ragged one per sequence, and per run of rows before and behind them.
long long packed_max_tiles(long long total, long long n, int rows) { return total / rows + n + 2; }

struct PackedFwdWorkspace {  // byte offsets
  size_t head = 0, base, tiles, bytes;
  PackedFwdWorkspace(int n, int total_q) {
    base = 256;
    tiles = align256(base + (size_t)3 * (n + 3) * 4);
    bytes = tiles + (size_t)packed_max_tiles(total_q, n, 256) * sizeof(PackedFwdTile);
  }
};

int packed_check(int n, int total_q, int total_k, int h, int h_kv, int causal) {
  if (n < 0 || total_q < 0 || total_k < 0 || h < 0 || h_kv < 0) return fail(WF_ERR_INVALID_ARG, "negative size");
  if (causal != 0 && causal != 1) return fail(WF_ERR_INVALID_ARG, "causal %d not in {0, 1}", causal);
  if (h_kv == 0 ? h != 0 : h % h_kv != 0)
    return fail(WF_ERR_INVALID_ARG, "h=%d is not a multiple of h_kv=%d", h, h_kv);
  if (h > 65535) return fail(WF_ERR_UNSUPPORTED, "h=%d exceeds 65535", h);
  // tile coordinates and item numbers are 32-bit
  if (n > (1 << 24) || total_q > (1 << 30) || total_k > (1 << 30))
    return fail(WF_ERR_UNSUPPORTED, "n=%d, total_q=%d, total_k=%d exceed 2^24 sequences of 2^30 rows", n, total_q, total_k);
  if (packed_max_tiles(total_q, n, 128) * h > 0x7fffffffLL || packed_max_tiles(total_k, n, 128) * h > 0x7fffffffLL)
    return fail(WF_ERR_UNSUPPORTED, "too many (tile, head) items");
  return WF_OK;
}

int plan_shift(int total) {
  int shift = 0;
  while (((total / 128 + 1) >> shift) >= kPlanBuckets) ++shift;
  return shift;
}

}  // namespace

cudaError_t packed_setup() {
  return cudaFuncSetAttribute(wf_packed_fwd_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pfwd::kSmemBytes);
}

}  // namespace wf

using namespace wf;

extern "C" int wf_packed_fwd_workspace(int n, int total_q, size_t* bytes) {
  if (!bytes) return fail(WF_ERR_INVALID_ARG, "null pointer");
  int rc = packed_check(n, total_q, 0, 1, 1, 0);
  if (rc) return rc;
  *bytes = PackedFwdWorkspace(n, total_q).bytes;
  return WF_OK;
}

extern "C" int wf_packed_fwd(const void* q, const void* k, const void* v, const int* q_offsets, const int* k_offsets,
                             void* o, float* lse, void* workspace, size_t workspace_bytes, int n, int total_q,
                             int total_k, int h, int h_kv, int causal, void* stream) {
  int rc = packed_check(n, total_q, total_k, h, h_kv, causal);
  if (rc) return rc;
  if (total_q == 0 || h == 0) return WF_OK;
  if (!q || !o || !lse || !q_offsets || !k_offsets || !workspace || (total_k > 0 && (!k || !v)))
    return fail(WF_ERR_INVALID_ARG, "null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(lse) & 3) || (reinterpret_cast<uintptr_t>(q_offsets) & 3) ||
      (reinterpret_cast<uintptr_t>(k_offsets) & 3))
    return fail(WF_ERR_MISALIGNED, "q/k/v/o/workspace must be 16-byte aligned, lse and offsets 4-byte aligned");
  const PackedFwdWorkspace ws(n, total_q);
  if (workspace_bytes < ws.bytes)
    return fail(WF_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", workspace_bytes, ws.bytes);
  int dev;
  if ((rc = device_setup(&dev))) return rc;
  CUtensorMap mq, mk, mv, mo;
  // with no keys at all nothing is loaded: q stands in for the maps of k and v
  if ((rc = make_bshd_map(&mq, q, 1, total_q, h)) || (rc = make_bshd_map(&mo, o, 1, total_q, h)) ||
      (rc = make_bshd_map(&mk, total_k ? k : q, 1, total_k ? total_k : total_q, total_k ? h_kv : h)) ||
      (rc = make_bshd_map(&mv, total_k ? v : q, 1, total_k ? total_k : total_q, total_k ? h_kv : h)))
    return rc;
  uint8_t* const w = reinterpret_cast<uint8_t*>(workspace);
  PackedPlanParams pp = {};
  pp.q_off = q_offsets, pp.k_off = k_offsets;
  pp.n = n, pp.total_q = total_q, pp.total_k = total_k, pp.causal = causal;
  pp.cost_shift = plan_shift(total_k);
  pp.head = reinterpret_cast<int4*>(w + ws.head);
  pp.base = reinterpret_cast<int*>(w + ws.base);
  pp.fwd_tiles = reinterpret_cast<PackedFwdTile*>(w + ws.tiles);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  wf_packed_plan_kernel<<<1, kPlanThreads, 0, st>>>(pp);
  if ((rc = launch_check("wf_packed plan launch"))) return rc;
  PackedFwdParams p = {};
  p.head = pp.head;
  p.tiles = pp.fwd_tiles;
  p.o = reinterpret_cast<__nv_bfloat16*>(o);
  p.lse = lse;
  p.total_q = total_q, p.h = h, p.group = h / h_kv, p.causal = causal;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt(128.0));
  p.rescale_threshold = 8.0f;
  const long long items = packed_max_tiles(total_q, n, 256) * h;
  const int grid = (int)std::min<long long>(items, g_dev_sms[dev]);
  cudaError_t e = launch_ex(wf_packed_fwd_kernel, dim3(grid), dim3(pfwd::kThreads), pfwd::kSmemBytes, st, true, 1u, mq,
                            mk, mv, mo, p);
  if (e != cudaSuccess) return cuda_fail(e, "wf_packed_fwd launch");
  return launch_check("wf_packed_fwd launch");
}
