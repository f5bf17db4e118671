// What the kernels of differential attention share: their arguments and the
// range of keys that a group of queries sees.
#pragma once

#include <math.h>
#include <stdint.h>

#include "../../include/katab200.h"
#include "kb_numeric.cuh"

namespace kb {

struct DiffArgs {
  kb_diff_attention_desc d;
  const uint16_t *q, *k, *v;
  const float *lambda, *gamma;
  const int32_t* kv_lens;
  const uint8_t* key_mask;
  uint16_t* out;
  float scale_log2;  // scale * log2(e): the kernels' exponentials are powers of two
  // Partial results of keys split over blocks (workspace), per row (b, i, h),
  // split and map: {running maximum (log2 units), sum}, and 2 head_dim value sums.
  float2* part_ml;
  float* part_o;
};

// Strides of dimensions of extent 1 are set to 0, so no address depends on them.
inline DiffArgs make_diff_args(const kb_diff_attention_desc& desc, const uint16_t* q, const uint16_t* k,
                               const uint16_t* v, const float* lambda, const float* gamma, const int32_t* kv_lens,
                               const uint8_t* key_mask, uint16_t* out) {
  DiffArgs a{desc, q, k, v, lambda, gamma, kv_lens, key_mask, out, desc.scale * 1.4426950408889634f,
             nullptr, nullptr};
  kb_diff_attention_desc& d = a.d;
  if (!kv_lens && d.window >= d.kv_len) d.window = 0;  // hides nothing
  if (d.batch == 1) d.q_batch = d.k_batch = d.v_batch = d.out_batch = d.mask_batch = 0;
  if (d.q_len == 1) d.q_token = d.out_token = 0;
  if (d.kv_len <= 1) d.k_token = d.v_token = 0;
  if (d.heads == 1) d.q_head = d.out_head = 0;
  if (d.kv_heads == 1) d.k_head = d.v_head = 0;
  return a;
}

// Keys of sequence b, kv_lens clamped to what K and V hold, and the position of
// its query 0: kv_lens - q_len, negative when there are more queries than keys.
// A sequence longer than K and V hold keeps its positions (up to where those of
// a tile's unused rows would pass 31 bits).
__device__ __forceinline__ int key_count(const DiffArgs& a, int b, int& off) {
  const int n = a.kv_lens ? max(0, min(a.kv_lens[b], 0x7fffff00)) : a.d.kv_len;
  off = n - a.d.q_len;
  return min(n, a.d.kv_len);
}

// [first, last): the keys that some of the queries i0..i1 of a sequence of n
// keys sees, before the key mask.  first may lie past the last key.
__device__ __forceinline__ void key_range_n(const kb_diff_attention_desc& d, int n, int off, int i0, int i1, int& first,
                                            int& last) {
  first = 0;
  last = n;
  if (d.causal) {
    last = max(0, min(n, off + i1 + 1));
    if (d.window) first = max(d.window, off + i0 + 1) - d.window;
  }
}

__device__ __forceinline__ int64_t row_index(const DiffArgs& a, int b, int i, int h) {
  return (static_cast<int64_t>(b) * a.d.q_len + i) * a.d.heads + h;
}

// A row's result from both maps' sums `acc` (kE dims per lane, dims lane kE..)
// and weights `ll`: the weighted difference, its norm, one rounding.  Whole warps.
// A row that saw no key is zero whatever eps and gamma are (0 / sqrt(0) is not).
template <int kE>
__device__ __forceinline__ void finish_row(const DiffArgs& a, int b, int i, int h, int lane, const float (&acc)[2][kE],
                                           const float (&ll)[2]) {
  const bool seen = ll[0] != 0.0f || ll[1] != 0.0f;
  const float w0 = ll[0] == 0.0f ? 0.0f : 1.0f / ll[0];  // 0: no key was seen
  const float w1 = ll[1] == 0.0f ? 0.0f : a.lambda[h] / ll[1];
  float r[kE], ss = 0.0f;
#pragma unroll
  for (int e = 0; e < kE; ++e) {
    r[e] = acc[0][e] * w0 - acc[1][e] * w1;
    ss = fmaf(r[e], r[e], ss);
  }
  float f = a.d.out_scale;
  if (a.gamma) {
#pragma unroll
    for (int x = 16; x; x >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, x);
    f *= 1.0f / sqrtf(ss / (32 * kE) + a.d.eps);
  }
  uint16_t* out = a.out + b * a.d.out_batch + i * a.d.out_token + h * a.d.out_head + lane * kE;
  uint32_t w[kE / 2];
#pragma unroll
  for (int e = 0; e < kE; e += 2) {
    const float g0 = a.gamma ? a.gamma[lane * kE + e] : 1.0f, g1 = a.gamma ? a.gamma[lane * kE + e + 1] : 1.0f;
    w[e / 2] = seen ? pack16x2(make_float2(r[e] * f * g0, r[e + 1] * f * g1), a.d.dtype == KB_DT_F16) : 0u;
  }
  if constexpr (kE == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(out) = w[0];
}

template <int kE>
__device__ __forceinline__ void write_partial(const DiffArgs& a, int splits, int split, int b, int i, int h, int lane,
                                              const float (&acc)[2][kE], const float (&mm)[2], const float (&ll)[2]) {
  const int64_t at = (row_index(a, b, i, h) * splits + split) * 2;
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    if (lane == 0) a.part_ml[at + m] = make_float2(mm[m], ll[m]);
    float* dst = a.part_o + (at + m) * (32 * kE) + lane * kE;
    if constexpr (kE == 4) *reinterpret_cast<float4*>(dst) = make_float4(acc[m][0], acc[m][1], acc[m][2], acc[m][3]);
    else *reinterpret_cast<float2*>(dst) = make_float2(acc[m][0], acc[m][1]);
  }
}

// Blocks of a tile of few queries that join their keys within a cluster (the
// portable cluster size); more of them go through the workspace.
constexpr int kMostCluster = 8;

int diff_decode_launch(const DiffArgs& a, int splits, cudaStream_t s);
// wait_limit_ns: a test's limit of its waits on work (0: kWaitLimitNs).
int diff_tc_launch(const DiffArgs& a, int splits, unsigned* status, uint32_t wait_limit_ns, cudaStream_t s);
int diff_combine_launch(const DiffArgs& a, int splits, cudaStream_t s);
int smem_opt_in(const void* kernel, int bytes);

}  // namespace kb
