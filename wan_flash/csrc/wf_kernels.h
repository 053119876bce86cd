// Kernel parameter blocks and launch-side declarations shared by the kernel
// translation units and the C ABI (wf_capi.cu).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace wf {

struct FwdParams {
  float* lse[2];           // per KV segment: (b, h, sq) natural-log LSE
  int sq, h;
  int skv[2];              // per KV segment (segment 1 only in the two-context kernel)
  int n_blocks[2];         // ceil(skv / 128)
  int n_pairs;             // ceil(sq / 256): work items per (batch, head)
  int n_items;             // b * h * n_pairs
  float scale_log2;        // log2(e) / sqrt(128)
  float rescale_threshold; // log2 units
};

struct BwdParams {
  const float* neg_lse_log2;  // (b, h, sq_rounded): -lse * log2(e), -inf on pad rows
  const float* dpsum;      // (b, h, sq_rounded)
  float* dq_accum;         // tiled, b*h*sq_rounded*128
  void* dk;                // bf16 (b, skv, h, 128) or fp32 tiled accumulator
  void* dv;
  int sq, skv, h;
  int sq_rounded, m_blocks, n_blocks, skv_rounded;
  int n_blocks_padded;     // n_blocks rounded up to the 2-CTA cluster size
  int accum_dkv;           // 1: dk/dv are fp32 tiled accumulators (split-M)
  int m_chunk;             // split-M: m-blocks per CTA
  float scale;             // 1/sqrt(128)
  float scale_log2;        // log2(e)/sqrt(128)
  int* dq_sem;             // deterministic: (b*h, m_blocks) dQ contributions added so far
  int* dkv_sem;            // deterministic, split-M: (b*h, n_blocks) splits added so far
  int deterministic;
  int wave;                // CTAs resident at once (one per SM): the serpentine walk's period
};

template <int kMode>
__global__ void wf_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k0,
                              const __grid_constant__ CUtensorMap tm_v0, const __grid_constant__ CUtensorMap tm_o0,
                              const __grid_constant__ CUtensorMap tm_k1, const __grid_constant__ CUtensorMap tm_v1,
                              const __grid_constant__ CUtensorMap tm_o1, FwdParams p);
__global__ void wf_fwd2_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k64,
                               const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                               FwdParams p);
__global__ void wf_bwd_main_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                                   BwdParams p);
__global__ void wf_bwd2_main_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_q64,
                                    const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                                    const __grid_constant__ CUtensorMap tm_do,
                                    const __grid_constant__ CUtensorMap tm_do64, BwdParams p);
__global__ void wf_bwd_pre_kernel(const __nv_bfloat16* __restrict__ o, const __nv_bfloat16* __restrict__ dO,
                                  const float* __restrict__ lse, float* __restrict__ dpsum,
                                  float* __restrict__ neg_lse_log2, float* __restrict__ dq_accum, int sq,
                                  int sq_rounded, int h);
__global__ void wf_convert_kernel(const float* __restrict__ accum, __nv_bfloat16* __restrict__ out, float scale,
                                  int s, int s_rounded, int h);

// ---- packed sequences (wf_packed_*.cu) ----
// Work records that the plan kernel writes and the packed kernels read.
struct __align__(16) PackedFwdTile {  // up to 256 query rows of one sequence
  int q0, rows;   // first row in the packed tensor, rows
  int k0;         // the sequence's first key row
  int klen;       // keys that the tile's last row sees; 0: nothing to attend, the rows are filled
  int off;        // causal: keys that row 0 of the tile sees (row r: off + r); may be negative
  int n_blocks;   // 128-key blocks of this piece of the walk (the whole walk: ceil(klen / 128))
  int j_last;     // the piece's last block; the walk goes down from it
  int part;       // place of the piece's partial result; -1: the whole walk, written as the result
  int bucket, bucket_items;  // place and number of the items of equal cost
  int pad0, pad1;
};
struct __align__(16) PackedBwdItem {  // up to 128 key rows of one sequence, and a piece of their walk
  int k0, rows;   // first row in the packed tensor, rows
  int q0, lq;     // the sequence's query rows
  int qtile;      // the sequence's first query tile (place in lse's and D's padded tiles)
  int m_begin, m_count;  // query tiles of the sequence that see some of these keys
  int need;       // first query row of the sequence that sees the tile's first key (key r: need + r)
  int nb;         // place of the tile in its sequence
  int first, count;      // units (q head of the group, query tile) of this piece
  int part;       // place of the piece's partial dK and dV; -1: the whole walk, written as the result
  int bucket, bucket_items;
  int pad0, pad1;
};
struct PackedPlanParams {
  const int* q_off;
  const int* k_off;
  int n, total_q, total_k;
  int causal, backward, ordered;
  int h, group, h_kv;
  int sms;
  int may_split;            // forward: the workspace has room for partial results
  int nsplit;               // > 0: pieces of the longest walk; 0: by `pieces`
  int pieces;               // sets the smallest piece: the whole work (over all key-value heads) in so many
  int4* head;               // [0] {items, status, split key tiles, draw counter}, [1] (backward) {query tiles, status}
  int* base;                // scratch: 3 * (n + 3)
  PackedFwdTile* fwd_tiles;
  PackedBwdItem* items;
  int4* q_tiles;            // {first row, rows, 1 inside a sequence, 0}
  int4* split_tiles;        // {first row, rows, first part, parts}
};
// Backward pieces: about two per SM's even share, of 8 units at least; or,
// with few key tiles, as many as make one item per SM, of 2 units at least.  A
// piece's own cost (prologue, K and V, partial dK and dV) is about two units.
constexpr int kPackedMinChunk = 2;
constexpr int kPackedMinChunkFull = 8;
constexpr int kPackedPiecesPerSm = 2;
constexpr int kPackedPieceCost = 2;
// Forward pieces: of at least 8 blocks (16 us), of an SM's even share of all
// blocks or, with few tiles, as many as make one item per SM; only where the
// longest walk gets shorter by more than the join's cost in blocks.
constexpr int kPackedFwdMinChunk = 8;
constexpr int kPackedFwdJoinCost = 4;
// Forward calls without a plan: every CTA finds its own tile, the segments 32 at
// a time.  The plan and the join are worth 4 to 8 us; what they would even out is
// worth less up to 3 items per SM with walks of at most 12 blocks (30 drawn calls
// each: 20.5 -> 16.8 us in the geometric mean up to 1.3 items per SM, 21.6 -> 17.9 up to
// 2, 23.4 -> 20.5 up to 3; none up to 5, a loss of 5 % above), and up to half as many
// items with walks of at most 16 blocks (1537 to 2048 keys, 14 calls each, against the
// plan: -28 % with ten sequences of about one length, -21 % with three, -3 % with one
// long sequence among ten, 14 % more at worst).  One sequence alone is one walk, which the plan cuts
// where its tiles leave half the SMs idle: there 36.5 us with it and 38.5 without,
// 36.5 and 41.0 at worst; with more tiles 48 and 40.
constexpr int kPackedDirectSeqs = 126;
constexpr int kPackedDirectBlocks = 12, kPackedDirectMoreBlocks = 16;
constexpr int kPackedDirectItems = 3;  // per SM
constexpr int kPackedFwdSplitItems = 4;  // per SM: with more items the longest walk is not the time
struct PackedFwdParams {
  const int4* head;
  const PackedFwdTile* tiles;
  int* counter;             // items drawn beyond the first of every CTA; the plan sets it to 0
  __nv_bfloat16* o;
  __nv_bfloat16* res;       // what rounding o to bf16 took away, like o; or null
  float* lse;               // (h, total_q)
  float4* part_o;           // (parts, h) x [2 tiles][32 groups of 4 columns][128 rows]: unnormalised O
  float2* part_ml;          // (parts, h, 256): reference max (scaled log2 units) and row sum
  const int* q_off;         // without a plan only, like k_off, n and total_k
  const int* k_off;
  int n, total_k;
  int total_q, h, group, causal;
  float scale_log2, rescale_threshold;
};
struct PackedFwdJoinParams {
  const int4* head;
  const int4* split_tiles;
  const float4* part_o;
  const float2* part_ml;
  __nv_bfloat16* o;
  __nv_bfloat16* res;
  float* lse;
  int total_q, h;
};
struct PackedBwdParams {
  const int4* head;
  const PackedBwdItem* items;
  const int4* q_tiles;
  float* neg_lse_log2;      // (h, q_tile_stride, 128): -lse * log2(e), -inf behind the sequence's end
  float* dpsum;             // (h, q_tile_stride, 128)
  float* dq_accum;          // (h, dq_rows, 128) fp32, by query tiles
  __nv_bfloat16* dk;        // (total_k, h_kv, 128)
  __nv_bfloat16* dv;
  float* dk_part;           // (parts, h_kv) tiles of 16384 fp32
  float* dv_part;
  int* sem;                 // ordered: (h, q_tile_stride) key tiles added so far
  size_t q_tile_stride, dq_rows;
  int total_q, h, h_kv, group, ordered, wave;
  float scale, scale_log2;
};
struct PackedConvertParams {
  const int4* head;
  const int4* q_tiles;
  const int4* split_tiles;
  const float* dq_accum;
  const float* dk_part;     // (parts, h_kv) tiles
  const float* dv_part;
  __nv_bfloat16* dq;
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  size_t dq_rows;
  unsigned dq_blocks, split_blocks;  // 2 * tiles * heads
  int h, h_kv;
  float scale;
};
cudaError_t packed_setup();

// per-device kernel attributes of the operators that bring their own entry points
cudaError_t decode_setup();

// role ids recorded with a device error by the operators without mbarrier roles
enum : uint32_t { kRoleRope = 21, kRoleDecode = 22, kRolePackedPlan = 23, kRoleSchedule = 24 };

size_t fwd_smem_bytes();
size_t fwd2_smem_bytes();
size_t bwd_smem_bytes();
size_t bwd2_smem_bytes();

// wf_fwd with cluster_m = 0 (auto), one KV context, one item per CTA: true =
// the CTA-pair kernel.
constexpr bool kFwdPairDefault = true;
// wf_bwd_main with cluster_n = 0 (auto): true = the CTA-pair kernel.
constexpr bool kBwdPairDefault = false;

constexpr int kFwdThreads = 384;
// wf_fwd with scheduler = 0 (auto): persistent grid when KV has at most this
// many 128-key blocks.
constexpr int kFwdPersistMaxBlocks = 64;
constexpr int kBwdThreads = 512;

}  // namespace wf
