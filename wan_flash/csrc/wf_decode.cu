// Attention of one new token per sequence over a paged key-value cache:
// wf_decode (declared in include/wan_flash.h).
//
//     o[b, h] = softmax(q[b, h] K_b^T / sqrt(128)) V_b,   lse[b, h]
// with K_b, V_b the first lengths[b] tokens of sequence b, token t in slot
// t % page_size of page page_table[b][t / page_size].
//
// Bound: HBM (512 bytes of K and V per token and key-value head against
// 512 * h / h_kv flops).  The q heads of one key-value head are served by
// one read of its K and V; tensor cores (mma.sync) do the products so that
// grouped heads cost no more issue slots than one head: S^T = K q^T has 16
// tokens as M and 8 q heads as N, O^T = V^T P^T 16 dims as M, so nothing is
// padded beyond 8 heads.  tcgen05's M of 64-128 rows would leave the tensor
// pipe as idle and add a trip through tensor memory.
//
// Loads: 16-byte cp.async into per-warp rings, 16 lanes to a row of 256 bytes.
// Lane j of a warp finds the page of token j of the next tile and hands its
// place round as a 32-bit count of 16-byte units, so a row costs a shuffle and
// a multiply-add.  (64-bit places cost 900 instructions a 16-token tile, which
// bounded the kernel: eight warps an SM do not hide that many dependent ones.
// One 256-byte bulk copy per lane cost 512 and no less time: bulk copies take
// their addresses one lane after the other.)
//
// Split: the work is cut by tiles of 64 tokens, not by sequences.  The tiles
// of all (sequence, key-value head[, block of heads]) rows stand one behind
// the other and every CTA takes an equal run of them, whatever the lengths;
// a row that spans several CTAs leaves partial results (running maximum,
// sum, unnormalised O, all fp32) which a second kernel joins in a fixed
// order, so results do not depend on timing.  Where the page table is short and
// the rows are few, a CTA takes a whole row instead.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

namespace dec {
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 64;                       // tokens of a CTA's tile: 16 per warp
constexpr uint32_t kRowBytes = 256 + 16;        // a token's 128 dims; 16 bytes more spread ldmatrix over the banks
constexpr uint32_t kHalfBytes = 16 * kRowBytes; // 16 tokens of K (or V)
constexpr uint32_t kStageBytes = 2 * kHalfBytes;
constexpr int kMaxHeads = 32;                   // q heads of a row (4 n-tiles of 8)
// Tables of at most so many tokens, with no more rows than CTAs: a CTA takes a
// whole row and no join follows.  One launch less is 2 us of a call; on the
// device 12 rows of 300 tokens take 8.2 us either way, 12 of 512 10.3 against 8.7, of
// 1024 16.4 against 10.3, ragged ones (up to 512 tokens) in 144 rows 10.3 against
// 12.3, 432 rows 16.4 against 20.5.  With more rows than SMs ragged rows of up to
// 1024 tokens still gain (192 rows 20.5 against 18.3, 288 20.6 against 25.2, 432 27.3
// against 35.9), of up to 2048 not always (192 rows 38 against 29).  With 32 heads a
// row 512 tokens take 18.5 against 16.4.
constexpr int whole_tokens(int heads_per_row, bool more_rows_than_sms) {
  return (heads_per_row <= 16 ? 512 : 256) << more_rows_than_sms;
}
// Per-warp ring of 16-token K and V tiles, and CTAs per SM, for rows of kN x 8
// heads.  8 heads: 12 warps with one tile ahead beat 8 with two (48 ragged
// streams 138 us against 140, 75600-token caches 221 against 228); more heads
// need more registers than 12 warps have.  From 24 heads on q is read from
// shared memory tile by tile: its fragments (64 registers at 32 heads) spilled.
template <int kN>
struct Shape {
  static constexpr int kStages = kN == 1 ? 2 : 3;
  static constexpr int kCtasPerSm = kN == 1 ? 3 : 2;
  static constexpr bool kQShared = kN >= 3;
  static constexpr uint32_t kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr uint32_t kOffML = kRingBytes;  // [warp][head] running max, then sum
  static constexpr uint32_t kOffQ = kOffML + 2 * kWarps * kMaxHeads * 4;
  static constexpr uint32_t kSmemBytes = kOffQ + (kQShared ? kN * 8 * kRowBytes : 0);
  static_assert(kCtasPerSm * (kSmemBytes + 2048) <= 233472, "the CTAs of an SM fit in its shared memory");
};
constexpr int ctas_per_sm(int heads_per_row) { return heads_per_row <= 8 ? Shape<1>::kCtasPerSm : Shape<2>::kCtasPerSm; }
constexpr int kOPitch = 132;                    // floats per head in the join buffer (128 + 4 against bank conflicts)
static_assert(16 * kOPitch * 4 <= kStageBytes, "a round of the join fits in a stage");
}  // namespace dec

struct DecodeParams {
  const __nv_bfloat16* q;    // (b, h, 128)
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  unsigned page_stride[2], slot_stride[2], head_stride[2];  // K, V, in units of 16 bytes
  const int* page_table;
  long long table_stride;
  const int* lengths;
  __nv_bfloat16* o;          // (b, h, 128)
  float* lse;                // (b, h)
  float* part_o;             // (2 * ctas, heads_per_row, 128) unnormalised O
  float* part_ml;            // (2 * ctas, heads_per_row, 2) running max (scaled log2 units) and sum
  int4* join;                // per CTA: row that starts there and ends elsewhere (or -1), last CTA of it
  int b, h, h_kv, group;     // group = h / h_kv
  int blocks;                // blocks of heads_per_row q heads per key-value head
  int heads_per_row;
  int n_pages, page_size, max_pages;
  int whole;                 // CTA i works on row i, no row is split
  float scale_log2;
};

namespace {

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  // bytes 0: the 16 bytes become zeros and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A length outside [0, max_pages * page_size] counts as 0 tokens (its rows
// are written as NaN).
__device__ __forceinline__ bool decode_length_ok(const DecodeParams& p, int len) {
  return len >= 0 && (long long)len <= (long long)p.max_pages * p.page_size;
}
__device__ __forceinline__ int decode_length(const DecodeParams& p, int seq) {
  const int len = p.lengths[seq];
  return decode_length_ok(p, len) ? len : 0;
}
__device__ __forceinline__ int decode_tiles(int len) { return (len + dec::kTile - 1) / dec::kTile; }

// A CTA's run of one row: tiles [t0, t1) of (sequence, key-value head, block of heads).
struct DecodeRun {
  int seq, len, n_tiles, row, t0, t1;
  long long seq_at;  // tiles before the sequence
  long long row_at;  // tiles before the row
};

// The run that starts at tile `at` < hi; r holds the run before it, or the
// sequence to look from.  False where the lengths changed under the call.
__device__ bool decode_next_run(const DecodeParams& p, int rows_per_seq, long long at, long long hi, DecodeRun& r) {
  r.len = decode_length(p, r.seq);
  r.n_tiles = decode_tiles(r.len);
  while (at >= r.seq_at + (long long)r.n_tiles * rows_per_seq) {
    if (r.seq + 1 >= p.b) return false;
    r.seq_at += (long long)r.n_tiles * rows_per_seq;
    ++r.seq;
    r.len = decode_length(p, r.seq);
    r.n_tiles = decode_tiles(r.len);
  }
  r.row = (int)((at - r.seq_at) / r.n_tiles);
  r.row_at = r.seq_at + (long long)r.row * r.n_tiles;
  r.t0 = (int)(at - r.row_at);
  r.t1 = (int)min((long long)r.n_tiles, hi - r.row_at);
  return true;
}

}  // namespace

// kN: n-tiles of 8 q heads that a row has.
template <int kN>
__global__ void __launch_bounds__(dec::kThreads, dec::Shape<kN>::kCtasPerSm)
    wf_decode_kernel(DecodeParams p) {
  using namespace dec;
  constexpr int kStages = Shape<kN>::kStages;
  constexpr bool kQShared = Shape<kN>::kQShared;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_scan[kWarps + 1];
  __shared__ long long s_start[2];  // tiles before the first sequence of this CTA's run; that sequence
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sbase = smem_u32(smem);
  const int rows_per_seq = p.h_kv * p.blocks;
  // A programmatic dependent of whatever ran before: 48 ragged streams 142.2 ->
  // 139.7 us, 75600-token caches 219.0 -> 216.9.  The join leaves the way free only
  // as it ends: with the next call's CTAs up around its blocks those cost 15 % more.
  // (Plain loads from here on, not read-only ones, which may move above the wait.)
  griddep_launch_dependents();
  griddep_wait();

  // ---- this CTA's run [lo, hi) of the tiles of all rows
  long long total = 0, ctas = 1, lo, hi;
  if (p.whole) {  // (counted from the row's sequence on)
    const int seq = (int)blockIdx.x / rows_per_seq;
    const int n = decode_tiles(decode_length(p, seq));
    lo = (long long)((int)blockIdx.x - seq * rows_per_seq) * n;
    hi = lo + n;
    if (threadIdx.x == 0) s_start[0] = 0, s_start[1] = seq;
  } else {
    const int per_thread = (p.b + kThreads - 1) / kThreads;
    const int s0 = min(p.b, (int)threadIdx.x * per_thread), s1 = min(p.b, s0 + per_thread);
    long long mine = 0;
    for (int s = s0; s < s1; ++s) mine += (long long)decode_tiles(decode_length(p, s)) * rows_per_seq;
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += up;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    before += incl - mine;
    // with fewer tiles than CTAs the first `total` CTAs take one each, so a row's CTAs are neighbours
    ctas = min((long long)gridDim.x, max(total, 1LL));
    const long long cta = min((long long)blockIdx.x, ctas);
    lo = total * cta / ctas, hi = total * min(cta + 1, ctas) / ctas;
    if (lo < hi && before <= lo && lo < before + mine) {
      long long at = before;
      for (int s = s0; s < s1; ++s) {
        const long long t = (long long)decode_tiles(decode_length(p, s)) * rows_per_seq;
        if (lo < at + t) {
          s_start[0] = at;
          s_start[1] = s;
          break;
        }
        at += t;
      }
    }
  }
  __syncthreads();

  // ---- sequences with nothing cached: o = 0, lse = -inf (NaN where the length is impossible)
  for (int s = blockIdx.x; s < p.b; s += gridDim.x) {
    const int len = p.lengths[s];
    if (len > 0 && decode_length_ok(p, len)) continue;
    const bool bad = !decode_length_ok(p, len);
    if (bad && threadIdx.x == 0 && atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_INVALID_ARG) == 0u) {
      g_err_info[0] = (unsigned)s;
      g_err_info[1] = (unsigned)len;
      g_err_info[2] = kRoleDecode;
      g_err_info[3] = 1u;
    }
    uint4 fill = make_uint4(0u, 0u, 0u, 0u);
    if (bad) fill = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
    uint4* dst = reinterpret_cast<uint4*>(p.o + (long long)s * p.h * 128);
    for (int i = threadIdx.x; i < p.h * 16; i += kThreads) dst[i] = fill;
    for (int i = threadIdx.x; i < p.h; i += kThreads)
      p.lse[(long long)s * p.h + i] = bad ? __int_as_float(0x7fffffff) : -INFINITY;
  }
  if (lo >= hi) {
    if (threadIdx.x == 0 && !p.whole) p.join[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }

  const uint32_t ring = sbase + warp * (kStages * kStageBytes);
  float* const s_m = reinterpret_cast<float*>(smem + Shape<kN>::kOffML);
  float* const s_l = s_m + kWarps * kMaxHeads;
  int4 join = make_int4(-1, 0, 0, 0);

  // ---- the loader: this warp's tokens of the CTA's tiles one after the other,
  // kStages - 1 tiles ahead of the products and on into the next rows.  Of tile t a
  // warp has tokens 64 t + 16 warp + [0, 16); lane j (and 16 + j) steps token j
  // through the pages; lanes 0-15 (16-31) copy the 16-byte chunks of the even
  // (odd) rows.
  DecodeRun ahead;
  ahead.seq = (int)s_start[1];
  ahead.seq_at = s_start[0];
  long long ahead_at = lo;
  const int* table = nullptr;
  const char* src_k = nullptr;
  const char* src_v = nullptr;
  const int step_pages = kTile / p.page_size, step_slots = kTile - step_pages * p.page_size;
  int tok = 0, last = 0, pg = 0, slot = 0, page = 0;
  auto open_run = [&]() {
    if (!decode_next_run(p, rows_per_seq, ahead_at, hi, ahead)) {
      ahead_at = hi;
      last = 0;
      return;
    }
    const int kvh = ahead.row / p.blocks;
    table = p.page_table + (long long)ahead.seq * p.table_stride;
    src_k = reinterpret_cast<const char*>(p.k) + ((long long)kvh * p.head_stride[0] + (lane & 15)) * 16;
    src_v = reinterpret_cast<const char*>(p.v) + ((long long)kvh * p.head_stride[1] + (lane & 15)) * 16;
    tok = ahead.t0 * kTile + warp * 16 + (lane & 15);  // of the next tile to send for
    last = min(ahead.len, ahead.t1 * kTile);
    pg = tok / p.page_size;
    slot = tok - pg * p.page_size;
    page = tok < last ? table[pg] : 0;
  };
  open_run();
  const uint32_t dst0 = ring + (lane >> 4) * kRowBytes + (lane & 15) * 16;
  auto load = [&](int stage) -> bool {  // whether the tile had a bad page
    bool bad = false;
    if (ahead_at < hi) {
      const bool there = tok < last;
      const bool ok = there && page >= 0 && page < p.n_pages;
      if (there && !ok) {
        bad = true;
        if (atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_INVALID_ARG) == 0u) {
          g_err_info[0] = (unsigned)ahead.seq;
          g_err_info[1] = (unsigned)page;
          g_err_info[2] = kRoleDecode;
          g_err_info[3] = 2u;
        }
      }
      const unsigned at_k = (unsigned)page * p.page_stride[0] + (unsigned)slot * p.slot_stride[0];
      const unsigned at_v = (unsigned)page * p.page_stride[1] + (unsigned)slot * p.slot_stride[1];
      const unsigned here = __ballot_sync(0xffffffffu, ok);
      const uint32_t dst = dst0 + stage * kStageBytes;
      if (here == 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 2 * i + (lane >> 4);
          const unsigned ak = __shfl_sync(0xffffffffu, at_k, r), av = __shfl_sync(0xffffffffu, at_v, r);
          cp_async16(dst + i * 2 * kRowBytes, src_k + (unsigned long long)ak * 16);
          cp_async16(dst + i * 2 * kRowBytes + kHalfBytes, src_v + (unsigned long long)av * 16);
        }
      } else {  // rows behind the end (and of bad pages) become zeros: 0 * NaN would reach the V product
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 2 * i + (lane >> 4);
          const unsigned ak = __shfl_sync(0xffffffffu, at_k, r), av = __shfl_sync(0xffffffffu, at_v, r);
          const bool row_ok = (here >> r) & 1;
          cp_async16(dst + i * 2 * kRowBytes, src_k + (row_ok ? (unsigned long long)ak * 16 : 0), row_ok ? 16 : 0);
          cp_async16(dst + i * 2 * kRowBytes + kHalfBytes, src_v + (row_ok ? (unsigned long long)av * 16 : 0),
                     row_ok ? 16 : 0);
        }
      }
      if (++ahead_at < ahead.row_at + ahead.t1) {
        tok += kTile;
        pg += step_pages;
        slot += step_slots;
        if (slot >= p.page_size) slot -= p.page_size, ++pg;
        page = tok < last ? table[pg] : 0;
      } else if (ahead_at < hi) {
        open_run();
      }
    }
    cp_async_commit();
    return bad;
  };
  // bad pages of the tiles in flight, one bit a stage
  unsigned bad_stage = 0;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i)
    if (load(i)) bad_stage |= 1u << i;
  int stage = kStages - 1, fill = kStages - 2;

  DecodeRun run;
  run.seq = (int)s_start[1];
  run.seq_at = s_start[0];
  for (long long at = lo; at < hi;) {
    if (!decode_next_run(p, rows_per_seq, at, hi, run)) break;
    const int kvh = run.row / p.blocks;
    const int head0 = kvh * p.group + (run.row - kvh * p.blocks) * p.heads_per_row;
    const int n_heads = min(p.heads_per_row, (kvh + 1) * p.group - head0);

    // q as the B operand of S^T = K q^T: lane holds head lane/4, dims 16 ks + 2 (lane%4) + {0, 1, 8, 9}
    uint32_t qf[kQShared ? 1 : kN][8][2];
    const uint4* const q_rows = reinterpret_cast<const uint4*>(p.q + ((long long)run.seq * p.h + head0) * 128);
    if constexpr (kQShared) {
      for (int i = threadIdx.x; i < kN * 8 * 16; i += kThreads) {
        const uint4 x = i < n_heads * 16 ? q_rows[i] : make_uint4(0u, 0u, 0u, 0u);
        *reinterpret_cast<uint4*>(smem + Shape<kN>::kOffQ + (i >> 4) * kRowBytes + (i & 15) * 16) = x;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        const int hd = n * 8 + (lane >> 2);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(q_rows + hd * 16) + (lane & 3);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qf[n][ks][0] = hd < n_heads ? src[ks * 8] : 0u;
          qf[n][ks][1] = hd < n_heads ? src[ks * 8 + 4] : 0u;
        }
      }
    }
    float m[kN][2], l[kN][2], acc[kN][8][4];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][d][i] = 0.f;
    }
    bool bad = false;
    for (int t = run.t0; t < run.t1; ++t) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      if (++stage == kStages) stage = 0;
      if (bad_stage >> stage & 1) bad = true;
      // refill the stage that the previous step read (every lane is past it)
      if (++fill == kStages) fill = 0;
      bad_stage &= ~(1u << fill);
      if (load(fill)) bad_stage |= 1u << fill;
      const uint32_t sk = ring + stage * kStageBytes, sv = sk + kHalfBytes;
      const int tok0 = t * kTile + warp * 16;
      if (tok0 >= run.len) continue;  // this warp has no token in the row's last tile
      // S^T (16 tokens x 8 heads per n-tile); up to 16 heads in two chains of four
      // products (with more the heads' own chains overlap)
      float s[kN][4], s2[kN][4];
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][i] = s2[n][i] = 0.f;
      {
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8;  // matrices 0, 2: tokens 0-7; 1, 3: tokens 8-15
        const uint32_t row = sk + r * kRowBytes + ((lane >> 4) << 4);  // matrices 2, 3: dims 8-15 of the step
        if constexpr (kQShared) {
          const uint32_t sq = sbase + Shape<kN>::kOffQ + (lane & 7) * kRowBytes + ((lane >> 3) << 4);
#pragma unroll
          for (int ks = 0; ks < 8; ks += 2) {
            uint32_t a0[4], a1[4];
            ldmatrix_x4(row + ks * 32, a0);
            ldmatrix_x4(row + ks * 32 + 32, a1);
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              uint32_t b[4];  // the head tile's fragments of steps ks and ks + 1
              ldmatrix_x4(sq + n * 8 * kRowBytes + ks * 32, b);
              mma_16816(s[n], a0, b[0], b[1]);
              mma_16816(s[n], a1, b[2], b[3]);
            }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            uint32_t a[4];
            ldmatrix_x4(row + ks * 32, a);
#pragma unroll
            for (int n = 0; n < kN; ++n) mma_16816((ks & 1) ? s2[n] : s[n], a, qf[n][ks][0], qf[n][ks][1]);
          }
        }
      }
      // online softmax over the tokens: rows lane/4 and lane/4 + 8, heads 2 (lane%4) + {0, 1}
      const bool in0 = tok0 + (lane >> 2) < run.len, in1 = tok0 + (lane >> 2) + 8 < run.len;
      uint32_t pb[kN][2], pl[kN][2];
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = kQShared ? s[n][i] : s[n][i] + s2[n][i];
          s[n][i] = (i < 2 ? in0 : in1) ? x * p.scale_log2 : -INFINITY;
        }
        float pr[4];
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(s[n][e], s[n][2 + e]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(m[n][e], mx);
          const float ref = mn == -INFINITY ? 0.f : mn;
          f[e] = ex2_approx(m[n][e] - ref);
          m[n][e] = mn;
          pr[e] = ex2_approx(s[n][e] - ref);
          pr[2 + e] = ex2_approx(s[n][2 + e] - ref);
          l[n][e] = l[n][e] * f[e] + pr[e] + pr[2 + e];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            acc[n][d][0] *= f[0];
            acc[n][d][1] *= f[1];
            acc[n][d][2] *= f[0];
            acc[n][d][3] *= f[1];
          }
        }
        // P^T (tokens x heads) to the B operand of O^T = V^T P^T: 8x8
        // transposes within the warp.  P goes as a pair of bf16, its upper half
        // cut off and the rest (2^-16 of the value is lost; a single bf16
        // loses as much as o's own rounding, and 75600-token caches take 219.2 us
        // against 218.2, 32 heads a row 82.5 against 79.2); the sum l keeps the fp32 values.
        // The rest is never negative, nor 0 (P's last bit is set, an fp32 step): an
        // infinite V times either would make NaN of the infinity that P V is.
        auto rest = [](float x) {
          return __uint_as_float(__float_as_uint(x) | 1u) - __uint_as_float(__float_as_uint(x) & 0xffff0000u);
        };
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = pr[2 * i], y = pr[2 * i + 1];
          pb[n][i] = movmatrix_trans((__float_as_uint(x) >> 16) | (__float_as_uint(y) & 0xffff0000u));
          pl[n][i] = pack_bf16(rest(x), rest(y));
          if constexpr (kN > 2) pl[n][i] = movmatrix_trans(pl[n][i]);  // else behind the first products
        }
      }
      // O^T (16 dims x 8 heads) += V^T P^T, up to 8 independent products in a row
      {
        constexpr int kDims = kN == 1 ? 8 : kN == 2 ? 4 : 2;
        const int r = (lane & 7) + (lane >> 4) * 8;        // matrices 0, 1: tokens 0-7; 2, 3: tokens 8-15
        const uint32_t row = sv + r * kRowBytes + (((lane >> 3) & 1) << 4);  // matrices 1, 3: dims 8-15 of the tile
#pragma unroll
        for (int d0 = 0; d0 < 8; d0 += kDims) {
          uint32_t a[kDims][4];
#pragma unroll
          for (int d = 0; d < kDims; ++d) ldmatrix_x4_trans(row + (d0 + d) * 32, a[d]);
#pragma unroll
          for (int n = 0; n < kN; ++n) {
#pragma unroll
            for (int d = 0; d < kDims; ++d) mma_16816(acc[n][d0 + d], a[d], pb[n][0], pb[n][1]);
            if (kN <= 2 && d0 == 0) pl[n][0] = movmatrix_trans(pl[n][0]), pl[n][1] = movmatrix_trans(pl[n][1]);
#pragma unroll
            for (int d = 0; d < kDims; ++d) mma_16816(acc[n][d0 + d], a[d], pl[n][0], pl[n][1]);
          }
        }
      }
    }
    bad = __any_sync(0xffffffffu, bad);
    // ---- join the four warps' results.  Each warp's O goes through its ring's
    // stage that was read last (the others hold the next tiles): 16 heads a round.
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = l[n][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (bad) x = __int_as_float(0x7fffffff);
        if (lane < 4) {
          s_m[warp * kMaxHeads + n * 8 + 2 * lane + e] = m[n][e];
          s_l[warp * kMaxHeads + n * 8 + 2 * lane + e] = x;
        }
      }
    __syncthreads();
    const bool whole = run.t0 == 0 && run.t1 == run.n_tiles;
    const int part = 2 * blockIdx.x + (run.t0 == 0 ? 1 : 0);
#pragma unroll
    for (int n0 = 0; n0 < kN; n0 += 2) {
      float* const s_o = reinterpret_cast<float*>(smem + stage * kStageBytes);
      constexpr int kWarpFloats = kStages * kStageBytes / 4;
#pragma unroll
      for (int n = n0; n < (n0 + 2 < kN ? n0 + 2 : kN); ++n) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int hd = n * 8 + 2 * (lane & 3) + e;
          float top = s_m[hd];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w * kMaxHeads + hd]);
          f[e] = ex2_approx(m[n][e] - (top == -INFINITY ? 0.f : top));
        }
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s_o[warp * kWarpFloats + ((n - n0) * 8 + 2 * (lane & 3) + (i & 1)) * kOPitch + d * 16 + (lane >> 2) +
                (i >> 1) * 8] = acc[n][d][i] * f[i & 1];
      }
      __syncthreads();
      // thread = 4 dims of a head; a warp writes one head's 128
      for (int hd = n0 * 8 + warp; hd < min(n_heads, n0 * 8 + 16); hd += kWarps) {
        float top = s_m[hd];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, s_m[w * kMaxHeads + hd]);
        const float ref = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          sum += s_l[w * kMaxHeads + hd] * ex2_approx(s_m[w * kMaxHeads + hd] - ref);
          const float4 y = *reinterpret_cast<const float4*>(s_o + w * kWarpFloats + (hd - n0 * 8) * kOPitch + lane * 4);
          x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        if (whole) {
          const float inv = 1.f / sum;  // a row with tokens has a sum >= 1 (or NaN)
          uint2 w2;
          w2.x = pack_bf16(x.x * inv, x.y * inv);
          w2.y = pack_bf16(x.z * inv, x.w * inv);
          const long long out = (long long)run.seq * p.h + head0 + hd;
          *reinterpret_cast<uint2*>(p.o + out * 128 + lane * 4) = w2;
          if (lane == 0) p.lse[out] = (top + log2f(sum)) * 0.69314718055994531f;
        } else {
          const long long out = (long long)part * p.heads_per_row + hd;
          *reinterpret_cast<float4*>(p.part_o + out * 128 + lane * 4) = x;
          if (lane == 0) *reinterpret_cast<float2*>(p.part_ml + out * 2) = make_float2(top, sum);
        }
      }
      __syncthreads();  // the join's stage is read: the next round, or the loader, may write it
    }
    if (run.t0 == 0 && run.t1 < run.n_tiles) {
      // the CTA whose run holds the row's last tile ends it
      const long long end = run.row_at + run.n_tiles - 1;
      long long e = (end * ctas) / total;
      while (total * (e + 1) / ctas <= end) ++e;
      while (total * e / ctas > end) --e;
      join = make_int4(head0, n_heads, (int)min(e, ctas - 1), run.seq);
    }
    at = run.row_at + run.t1;
  }
  cp_async_wait<0>();
  if (threadIdx.x == 0 && !p.whole) p.join[blockIdx.x] = join;
}

// Joins the rows that span several CTAs: block (c, head) takes the row that
// starts in CTA c's run (slot 1 of c, slot 0 of the CTAs behind it); block
// (c, y) its heads y, y + gridDim.y, ...
__global__ void __launch_bounds__(256) wf_decode_join_kernel(DecodeParams p) {
  griddep_wait();
  const int c = blockIdx.x;
  const int4 j = p.join[c];
  if (j.x < 0) return;
  const int n = j.z - c + 1;
  __shared__ float s_red[8];
  __shared__ float4 s_acc[8][32];
  __shared__ float s_sum[8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int hd = blockIdx.y; hd < j.y; hd += gridDim.y) {
    auto slot = [&](int i) -> long long { return (long long)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * p.heads_per_row + hd; };
    float top = -INFINITY;
    for (int i = threadIdx.x; i < n; i += 256) top = fmaxf(top, p.part_ml[slot(i) * 2]);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) s_red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_red[w]);
    const float ref = top == -INFINITY ? 0.f : top;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int i = warp; i < n; i += 8) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(i) * 2);
      const float4 y = *reinterpret_cast<const float4*>(p.part_o + slot(i) * 128 + lane * 4);
      const float f = ex2_approx(ml.x - ref);
      sum += ml.y * f;
      x.x += y.x * f, x.y += y.y * f, x.z += y.z * f, x.w += y.w * f;
    }
    s_acc[warp][lane] = x;
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      sum = 0.f;
      x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float4 y = s_acc[w][lane];
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        sum += s_sum[w];
      }
      const float inv = 1.f / sum;
      uint2 w2;
      w2.x = pack_bf16(x.x * inv, x.y * inv);
      w2.y = pack_bf16(x.z * inv, x.w * inv);
      const long long out = (long long)j.w * p.h + j.x + hd;
      *reinterpret_cast<uint2*>(p.o + out * 128 + lane * 4) = w2;
      if (lane == 0) p.lse[out] = (top + log2f(sum)) * 0.69314718055994531f;
    }
    __syncthreads();
  }
}

namespace {

int decode_rows(int h, int h_kv, int* blocks, int* heads_per_row) {
  if (h < 1 || h_kv < 1 || h % h_kv) return fail(WF_ERR_INVALID_ARG, "h=%d is not a multiple of h_kv=%d", h, h_kv);
  const int group = h / h_kv;
  *blocks = (group + dec::kMaxHeads - 1) / dec::kMaxHeads;
  *heads_per_row = (group + *blocks - 1) / *blocks;
  return WF_OK;
}

template <int kN>
int decode_launch(const DecodeParams& p, int ctas, cudaStream_t st) {
  if (p.whole) ctas = p.b * p.h_kv * p.blocks;
  using dec::Shape;
  cudaError_t e = launch_ex(wf_decode_kernel<kN>, dim3(ctas), dim3(dec::kThreads), Shape<kN>::kSmemBytes, st, true, 1u, p);
  if (e != cudaSuccess) return cuda_fail(e, "wf_decode launch");
  if (!p.whole) e = launch_ex(wf_decode_join_kernel, dim3(ctas, std::min(p.heads_per_row, 8)), dim3(256), 0, st, true, 1u, p);
  if (e != cudaSuccess) return cuda_fail(e, "wf_decode join launch");
  return launch_check("wf_decode join launch");
}

// Whether every row is one CTA's.
bool decode_whole(int b, int h_kv, int blocks, int heads_per_row, int max_pages, int page_size, int sms) {
  const long long rows = (long long)b * h_kv * blocks;
  return rows <= (long long)sms * dec::ctas_per_sm(heads_per_row) &&
         (long long)max_pages * page_size <= dec::whole_tokens(heads_per_row, rows > sms);
}

// workspace: join descriptors, then (max, sum) pairs, then O of two partial rows per CTA
size_t decode_workspace_bytes(int ctas, int heads_per_row) {
  return (size_t)ctas * 16 + (size_t)2 * ctas * heads_per_row * (8 + 512);
}

}  // namespace

// One-time per-device set-up (from device_setup, with that device current).
cudaError_t decode_setup() {
  auto smem = [](auto* k, uint32_t bytes) {
    return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  };
  cudaError_t e = smem(wf_decode_kernel<1>, dec::Shape<1>::kSmemBytes);
  if (e == cudaSuccess) e = smem(wf_decode_kernel<2>, dec::Shape<2>::kSmemBytes);
  if (e == cudaSuccess) e = smem(wf_decode_kernel<3>, dec::Shape<3>::kSmemBytes);
  if (e == cudaSuccess) e = smem(wf_decode_kernel<4>, dec::Shape<4>::kSmemBytes);
  return e;
}
}  // namespace wf

extern "C" int wf_decode_workspace(int b, int h, int h_kv, int max_pages, int page_size, size_t* bytes) {
  using namespace wf;
  if (!bytes) return fail(WF_ERR_INVALID_ARG, "null pointer");
  if (b < 0 || max_pages < 0 || page_size < 1)
    return fail(WF_ERR_INVALID_ARG, "b %d, max_pages %d, page_size %d", b, max_pages, page_size);
  int blocks, heads, dev, rc;
  if ((rc = decode_rows(h, h_kv, &blocks, &heads))) return rc;
  if ((rc = device_setup(&dev))) return rc;
  *bytes = decode_whole(b, h_kv, blocks, heads, max_pages, page_size, g_dev_sms[dev])
               ? 0
               : decode_workspace_bytes(g_dev_sms[dev] * dec::ctas_per_sm(heads), heads);
  return WF_OK;
}

extern "C" int wf_decode(const void* q, const void* k_cache, const void* v_cache, const int* page_table,
                         const int* lengths, void* o, float* lse, void* workspace, size_t workspace_bytes, int b, int h,
                         int h_kv, const wf_decode_cfg* cfg, void* stream) {
  using namespace wf;
  if (b < 0 || h < 0 || h_kv < 0) return fail(WF_ERR_INVALID_ARG, "negative size");
  if (!cfg) return fail(WF_ERR_INVALID_ARG, "null cfg");
  if (cfg->n_pages < 0 || cfg->page_size < 1 || cfg->max_pages < 0)
    return fail(WF_ERR_INVALID_ARG, "n_pages %d, page_size %d, max_pages %d", cfg->n_pages, cfg->page_size, cfg->max_pages);
  if ((long long)cfg->page_size * cfg->max_pages > 0x7fffffffLL - 1024)
    return fail(WF_ERR_UNSUPPORTED, "max_pages * page_size = %lld tokens exceed 2^31 - 1025",
                (long long)cfg->page_size * cfg->max_pages);
  for (long long x : {cfg->k_page_stride, cfg->k_slot_stride, cfg->k_head_stride, cfg->v_page_stride, cfg->v_slot_stride,
                      cfg->v_head_stride})
    if (x < 0 || x >= (8LL << 32))
      return fail(WF_ERR_UNSUPPORTED, "cache stride of %lld elements outside [0, 2^35)", x);
  // places within a cache are 32-bit counts of 16 bytes
  for (int i = 0; i < 2; ++i) {
    const double reach = (double)cfg->n_pages * (double)(i ? cfg->v_page_stride : cfg->k_page_stride) +
                         (double)cfg->page_size * (double)(i ? cfg->v_slot_stride : cfg->k_slot_stride);
    if (reach >= 8.0 * 4294967296.0)
      return fail(WF_ERR_UNSUPPORTED, "a cache of %.3g elements exceeds 2^35 (64 GiB)", reach);
  }
  if (b == 0 || h == 0) return WF_OK;
  DecodeParams p;
  int rc, dev;
  if ((rc = decode_rows(h, h_kv, &p.blocks, &p.heads_per_row))) return rc;
  if (!q || !lengths || !o || !lse || (!workspace && workspace_bytes) || (cfg->max_pages > 0 && !page_table) ||
      (cfg->n_pages > 0 && (!k_cache || !v_cache)))
    return fail(WF_ERR_INVALID_ARG, "null pointer");
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(o) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(lse) & 3) || (reinterpret_cast<uintptr_t>(lengths) & 3) ||
      (reinterpret_cast<uintptr_t>(page_table) & 3) || cfg->k_page_stride % 8 || cfg->k_slot_stride % 8 ||
      cfg->k_head_stride % 8 || cfg->v_page_stride % 8 || cfg->v_slot_stride % 8 || cfg->v_head_stride % 8)
    return fail(WF_ERR_MISALIGNED, "q/k_cache/v_cache/o/workspace and the caches' strides must be multiples of 16 bytes");
  if ((rc = device_setup(&dev))) return rc;
  const int ctas = g_dev_sms[dev] * dec::ctas_per_sm(p.heads_per_row);
  p.whole = decode_whole(b, h_kv, p.blocks, p.heads_per_row, cfg->max_pages, cfg->page_size, g_dev_sms[dev]);
  const size_t need = p.whole ? 0 : decode_workspace_bytes(ctas, p.heads_per_row);
  if (workspace_bytes < need)
    return fail(WF_ERR_INVALID_ARG, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.k = reinterpret_cast<const __nv_bfloat16*>(k_cache);
  p.v = reinterpret_cast<const __nv_bfloat16*>(v_cache);
  p.page_stride[0] = (unsigned)(cfg->k_page_stride / 8), p.page_stride[1] = (unsigned)(cfg->v_page_stride / 8);
  p.slot_stride[0] = (unsigned)(cfg->k_slot_stride / 8), p.slot_stride[1] = (unsigned)(cfg->v_slot_stride / 8);
  p.head_stride[0] = (unsigned)(cfg->k_head_stride / 8), p.head_stride[1] = (unsigned)(cfg->v_head_stride / 8);
  p.page_table = page_table;
  p.table_stride = cfg->table_stride;
  p.lengths = lengths;
  p.o = reinterpret_cast<__nv_bfloat16*>(o);
  p.lse = lse;
  p.join = reinterpret_cast<int4*>(workspace);
  p.part_ml = reinterpret_cast<float*>(p.join + ctas);
  p.part_o = p.part_ml + (size_t)2 * ctas * p.heads_per_row * 2;
  p.b = b, p.h = h, p.h_kv = h_kv, p.group = h / h_kv;
  p.n_pages = cfg->n_pages, p.page_size = cfg->page_size, p.max_pages = cfg->max_pages;
  p.scale_log2 = (float)(1.4426950408889634 / std::sqrt(128.0));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch ((p.heads_per_row + 7) / 8) {
    case 1: return decode_launch<1>(p, ctas, st);
    case 2: return decode_launch<2>(p, ctas, st);
    case 3: return decode_launch<3>(p, ctas, st);
    default: return decode_launch<4>(p, ctas, st);
  }
}
