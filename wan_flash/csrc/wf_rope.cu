// Rotary positions with three axes (time, height, width) of q and k, both in
// one launch: wf_rope (declared in include/wan_flash.h).
//
// Pair i of a 128-dim head turns by the angle whose cosine and sine the
// table holds at row positions[token][axis(i)], column i:
//     y[2i]   = x[2i] c - x[2i+1] s        y[2i+1] = x[2i] s + x[2i+1] c
// and the backward is the turn by the negative angle (s -> -s).
//
// Bound: HBM.  Every value is read once and written once; three flops a
// value are nothing.  The angles are not computed here: a table row is 512
// bytes, a whole video's rows fit in L1 / L2, and its fp64-made entries keep
// far positions exact to fp32 rounding, which sincosf of an fp32 product
// would not.  A thread keeps its token's cosines and sines in registers and
// walks heads with six rows' loads in flight: with the table looked up row by
// row the kernel issued 178 instructions a warp row and ran at its issue rate,
// 75 % of the copy rate; this one runs at 90 to 99 %.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

// Rows of a thread's walk, at least (below, its prologue of position and table
// shows), and rows in flight per thread.  75600 tokens, 40 + 40 heads, bf16 (5
// rows a thread): 571 us with 3 rows in flight, 530 with 4, 483 with 6 (6.41
// TB/s), 530 with 8; 32760 tokens, 12 + 12 heads: 80 us as 3 rows a thread, 69 as 6.
constexpr int kRopeMinRows = 5;
constexpr int kRopeBatch = 6;

struct RopeParams {
  const void* src[2];          // q, k
  void* dst[2];                // contiguous (b, s, h, 128)
  long long stride_b[2], stride_s[2], stride_h[2];  // of src, in elements
  int heads[2];
  const float2* table;         // (max_pos, 64) of (cos, sin)
  const int* positions;        // (s, 3), or (b, s, 3) with pos_stride_b = 3 s
  long long pos_stride_b;
  int b, s, max_pos;
  int pair_end0, pair_end1;    // pairs [0, end0) time, [end0, end1) height, [end1, 64) width
  float sign;                  // +1 forward, -1 backward
  int lanes;                   // rows of one token that a block works on side by side (a power of two)
};

template <typename T>
struct RopeVec;  // 16 bytes of a head: kPairs pairs
template <>
struct RopeVec<__nv_bfloat16> {
  static constexpr int kPairs = 4;
  __device__ static void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ static uint4 pack(const float (&x)[8]) {
    // the one rounding: the turned fp32 pair to bf16
    return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
  }
};
template <>
struct RopeVec<float> {
  static constexpr int kPairs = 2;
  __device__ static void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

// Plain loads throughout, not read-only ones: the kernel before may still be
// writing what this one reads when its blocks come up.
__device__ __forceinline__ uint4 ld_stream_u4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// A row (one head of one token) is 16 (bf16) or 32 (fp32) threads of 16
// bytes, so 256 threads hold 16 (8) rows: `lanes` rows of each of 16 / lanes (8 /
// lanes) tokens.  A thread walks rows lane, lane + lanes, ... of its token, the
// heads of q and then of k.  Block (x, y): those tokens of batch item y.
template <typename T>
__global__ void __launch_bounds__(256) wf_rope_kernel(RopeParams p) {
  constexpr int kPairs = RopeVec<T>::kPairs;
  constexpr int kThreadsPerRow = 64 / kPairs;
  constexpr int kRows = 256 / kThreadsPerRow;
  constexpr int kBatch = kRopeBatch;
  // a programmatic dependent of whatever ran before: its blocks come up while
  // that drains (480p forward and gradients 139 -> 135 us, one token 14.8 -> 14.3)
  griddep_launch_dependents();
  griddep_wait();
  const int c = threadIdx.x % kThreadsPerRow;
  const int place = threadIdx.x / kThreadsPerRow;
  const int lane = place & (p.lanes - 1);
  const int bb = blockIdx.y;
  const long long ss = (long long)blockIdx.x * (kRows / p.lanes) + place / p.lanes;
  if (ss >= p.s) return;
  const int hq = p.heads[0], rows = hq + p.heads[1];
  const T* const q = reinterpret_cast<const T*>(p.src[0]) + bb * p.stride_b[0] + ss * p.stride_s[0] + c * (2 * kPairs);
  const T* const k = reinterpret_cast<const T*>(p.src[1]) + bb * p.stride_b[1] + ss * p.stride_s[1] + c * (2 * kPairs);
  const long long tok = (long long)bb * p.s + ss;
  T* const oq = reinterpret_cast<T*>(p.dst[0]) + tok * hq * 128 + c * (2 * kPairs);
  T* const ok = reinterpret_cast<T*>(p.dst[1]) + tok * p.heads[1] * 128 + c * (2 * kPairs);
  uint4 v[kBatch];
  auto load = [&](int row0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int row = row0 + i * p.lanes;
      if (row < rows) v[i] = ld_stream_u4(row < hq ? q + row * p.stride_h[0] : k + (row - hq) * p.stride_h[1]);
    }
  };
  load(lane);
  // this thread's pairs of its token
  const int* const pp = p.positions + bb * p.pos_stride_b + 3 * ss;
  const int pos0 = pp[0], pos1 = pp[1], pos2 = pp[2];
  const bool still = (pos0 | pos1 | pos2) < 0;  // padding: passes bit for bit
  // (an axis without pairs turns nothing and reads no row)
  const int most = max(p.pair_end0 > 0 ? pos0 : 0,
                       max(p.pair_end1 > p.pair_end0 ? pos1 : 0, p.pair_end1 < 64 ? pos2 : 0));
  float cs[kPairs], sn[kPairs];
  if (still || most >= p.max_pos) {
    // outside the table: no value is right; say so in the error word too
    if (!still && lane == 0 && c == 0 && atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_INVALID_ARG) == 0u) {
      g_err_info[0] = blockIdx.x;
      g_err_info[1] = (unsigned)bb;
      g_err_info[2] = kRoleRope;
      g_err_info[3] = (unsigned)most;
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) cs[j] = sn[j] = __int_as_float(0x7fffffff);
  } else {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int pair = c * kPairs + j;
      const int pos = pair < p.pair_end0 ? pos0 : pair < p.pair_end1 ? pos1 : pos2;
      const float2 t = p.table[(long long)pos * 64 + pair];
      cs[j] = t.x;
      sn[j] = t.y * p.sign;
    }
  }
  for (int row0 = lane; row0 < rows; row0 += kBatch * p.lanes) {
    if (row0 != lane) load(row0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int row = row0 + i * p.lanes;
      if (row >= rows) break;
      float x[2 * kPairs];
      RopeVec<T>::unpack(v[i], x);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float a = x[2 * j], b = x[2 * j + 1];
        x[2 * j] = a * cs[j] - b * sn[j];
        x[2 * j + 1] = a * sn[j] + b * cs[j];
      }
      const uint4 turned = RopeVec<T>::pack(x);
      T* const dst = row < hq ? oq + row * 128 : ok + (row - hq) * 128;
      *reinterpret_cast<uint4*>(dst) = still ? v[i] : turned;
    }
  }
}

}  // namespace wf

extern "C" int wf_rope(const void* q, const void* k, void* q_out, void* k_out, const float* table,
                       const int* positions, int b, int s, int h, int h_kv, const wf_rope_cfg* cfg, void* stream) {
  using namespace wf;
  if (b < 0 || s < 0 || h < 0 || h_kv < 0) return fail(WF_ERR_INVALID_ARG, "negative size");
  if (!cfg) return fail(WF_ERR_INVALID_ARG, "null cfg");
  if (cfg->dtype != WF_BF16 && cfg->dtype != WF_FP32) return fail(WF_ERR_UNSUPPORTED, "dtype %d", cfg->dtype);
  if (cfg->max_pos < 1) return fail(WF_ERR_INVALID_ARG, "max_pos %d < 1", cfg->max_pos);
  if (cfg->pairs_t < 0 || cfg->pairs_h < 0 || cfg->pairs_t > 64 || cfg->pairs_h > 64 - cfg->pairs_t)
    return fail(WF_ERR_INVALID_ARG, "pairs_t %d + pairs_h %d outside [0, 64]", cfg->pairs_t, cfg->pairs_h);
  if (h > 65535 || h_kv > 65535 || b > 65535)
    return fail(WF_ERR_UNSUPPORTED, "h=%d / h_kv=%d / b=%d exceed 65535", h, h_kv, b);
  if (b == 0 || s == 0 || h + h_kv == 0) return WF_OK;
  if (!table || !positions || (h > 0 && (!q || !q_out)) || (h_kv > 0 && (!k || !k_out)))
    return fail(WF_ERR_INVALID_ARG, "null pointer");
  const long long per16 = cfg->dtype == WF_BF16 ? 8 : 4;  // elements in 16 bytes
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) ||
      !aligned16(table) || (reinterpret_cast<uintptr_t>(positions) & 3) ||
      cfg->q_stride_b % per16 || cfg->q_stride_s % per16 || cfg->q_stride_h % per16 || cfg->k_stride_b % per16 ||
      cfg->k_stride_s % per16 || cfg->k_stride_h % per16)
    return fail(WF_ERR_MISALIGNED, "q/k/outputs and their strides and the table must be multiples of 16 bytes");
  int dev, rc;
  if ((rc = device_setup(&dev))) return rc;
  RopeParams p;
  p.src[0] = q, p.src[1] = k, p.dst[0] = q_out, p.dst[1] = k_out;
  p.stride_b[0] = cfg->q_stride_b, p.stride_s[0] = cfg->q_stride_s, p.stride_h[0] = cfg->q_stride_h;
  p.stride_b[1] = cfg->k_stride_b, p.stride_s[1] = cfg->k_stride_s, p.stride_h[1] = cfg->k_stride_h;
  p.heads[0] = h, p.heads[1] = h_kv;
  p.table = reinterpret_cast<const float2*>(table);
  p.positions = positions;
  p.pos_stride_b = cfg->pos_stride_b;
  p.b = b, p.s = s, p.max_pos = cfg->max_pos;
  p.pair_end0 = cfg->pairs_t, p.pair_end1 = cfg->pairs_t + cfg->pairs_h;
  p.sign = cfg->inverse ? -1.f : 1.f;
  // the widest split of a token's rows that gives a thread kRopeMinRows of them
  // and leaves at most an eighth of the row places empty (24 rows: 4 lanes of 6)
  const int heads = h + h_kv;
  int lanes = cfg->dtype == WF_BF16 ? 16 : 8;
  const int rows_per_block = lanes;
  while (lanes > 1 && (heads < kRopeMinRows * lanes || ((heads + lanes - 1) / lanes * lanes - heads) * 8 > heads))
    lanes >>= 1;
  p.lanes = lanes;
  const int tokens_per_block = rows_per_block / lanes;
  const dim3 grid((unsigned)((s + (long long)tokens_per_block - 1) / tokens_per_block), b);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const cudaError_t e = launch_ex(cfg->dtype == WF_BF16 ? wf_rope_kernel<__nv_bfloat16> : wf_rope_kernel<float>, grid,
                                  dim3(256), 0, st, true, 1u, p);
  if (e != cudaSuccess) return cuda_fail(e, "wf_rope launch");
  return launch_check("wf_rope launch");
}
