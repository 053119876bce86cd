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
// would not.
#include "wf_common.cuh"
#include "wf_kernels.h"

namespace wf {

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
  int tokens_per_block;
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

// One block: tokens_per_block tokens, all heads of q and k of each.  A row
// (one head of one token) is 16 (bf16) or 32 (fp32) threads of 16 bytes.
template <typename T>
__global__ void __launch_bounds__(256) wf_rope_kernel(RopeParams p) {
  constexpr int kPairs = RopeVec<T>::kPairs;
  constexpr int kThreadsPerRow = 64 / kPairs;
  constexpr int kRowsPerPass = 256 / kThreadsPerRow;
  const int c = threadIdx.x % kThreadsPerRow;
  const int heads = p.heads[0] + p.heads[1];
  const long long n_tokens = (long long)p.b * p.s;
  const long long tok0 = (long long)blockIdx.x * p.tokens_per_block;
  const int tokens = (int)min((long long)p.tokens_per_block, n_tokens - tok0);
  const int rows = tokens * heads;
  for (int row = threadIdx.x / kThreadsPerRow; row < rows; row += kRowsPerPass) {
    const int lt = row / heads;
    const long long tok = tok0 + lt;
    const int hh = row - lt * heads;
    const int which = hh >= p.heads[0] ? 1 : 0;
    const int h = which ? hh - p.heads[0] : hh;
    const int bb = (int)(tok / p.s);
    const int ss = (int)(tok - (long long)bb * p.s);
    const T* src = reinterpret_cast<const T*>(which ? p.src[1] : p.src[0]) +
                   (long long)bb * (which ? p.stride_b[1] : p.stride_b[0]) +
                   (long long)ss * (which ? p.stride_s[1] : p.stride_s[0]) +
                   (long long)h * (which ? p.stride_h[1] : p.stride_h[0]) + c * (2 * kPairs);
    const uint4 v = ldg_u4(src);
    const int* pp = p.positions + (long long)bb * p.pos_stride_b + 3LL * ss;
    const int pos0 = __ldg(pp), pos1 = __ldg(pp + 1), pos2 = __ldg(pp + 2);
    uint4 out = v;
    if ((pos0 | pos1 | pos2) >= 0) {
      float x[2 * kPairs];
      RopeVec<T>::unpack(v, x);
      if (max(pos0, max(pos1, pos2)) >= p.max_pos) {
        // outside the table: no value is right; say so in the error word too
        if (atomicCAS(&g_err_code, 0u, (unsigned)WF_ERR_INVALID_ARG) == 0u) {
          g_err_info[0] = (unsigned)ss;
          g_err_info[1] = (unsigned)bb;
          g_err_info[2] = kRoleRope;
          g_err_info[3] = (unsigned)max(pos0, max(pos1, pos2));
        }
#pragma unroll
        for (int i = 0; i < 2 * kPairs; ++i) x[i] = __int_as_float(0x7fffffff);
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int pair = c * kPairs + i;
          const int pos = pair < p.pair_end0 ? pos0 : pair < p.pair_end1 ? pos1 : pos2;
          const float2 cs = __ldg(p.table + (long long)pos * 64 + pair);
          const float sn = cs.y * p.sign;
          const float a = x[2 * i], b2 = x[2 * i + 1];
          x[2 * i] = a * cs.x - b2 * sn;
          x[2 * i + 1] = a * sn + b2 * cs.x;
        }
      }
      out = RopeVec<T>::pack(x);
    }
    T* dst = reinterpret_cast<T*>(which ? p.dst[1] : p.dst[0]) +
             (tok * (which ? p.heads[1] : p.heads[0]) + h) * 128 + c * (2 * kPairs);
    *reinterpret_cast<uint4*>(dst) = out;
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
  if (h > 65535 || h_kv > 65535) return fail(WF_ERR_UNSUPPORTED, "h=%d / h_kv=%d exceed 65535", h, h_kv);
  if (b == 0 || s == 0 || h + h_kv == 0) return WF_OK;
  if (!table || !positions || (h > 0 && (!q || !q_out)) || (h_kv > 0 && (!k || !k_out)))
    return fail(WF_ERR_INVALID_ARG, "null pointer");
  const long long per16 = cfg->dtype == WF_BF16 ? 8 : 4;  // elements in 16 bytes
  if (!aligned16(q) || !aligned16(k) || !aligned16(q_out) || !aligned16(k_out) ||
      (reinterpret_cast<uintptr_t>(table) & 7) || (reinterpret_cast<uintptr_t>(positions) & 3) ||
      cfg->q_stride_b % per16 || cfg->q_stride_s % per16 || cfg->q_stride_h % per16 || cfg->k_stride_b % per16 ||
      cfg->k_stride_s % per16 || cfg->k_stride_h % per16)
    return fail(WF_ERR_MISALIGNED, "q/k/outputs and their strides must be multiples of 16 bytes, the table of 8");
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
  const int heads = h + h_kv;
  p.tokens_per_block = std::max(1, 64 / heads);
  const long long n_tokens = (long long)b * s;
  const long long grid = (n_tokens + p.tokens_per_block - 1) / p.tokens_per_block;
  if (grid > 0x7fffffffLL) return fail(WF_ERR_UNSUPPORTED, "%lld tokens exceed the grid limit", n_tokens);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (cfg->dtype == WF_BF16)
    wf_rope_kernel<__nv_bfloat16><<<(unsigned)grid, 256, 0, st>>>(p);
  else
    wf_rope_kernel<float><<<(unsigned)grid, 256, 0, st>>>(p);
  return launch_check("wf_rope launch");
}
