// What the kernels of differential attention share: their arguments and the
// range of keys that a group of queries sees.
#pragma once

#include <stdint.h>

#include "../../include/katab200.h"

namespace kb {

struct DiffArgs {
  kb_diff_attention_desc d;
  const uint16_t *q, *k, *v;
  const float *lambda, *gamma;
  const int32_t* kv_lens;
  const uint8_t* key_mask;
  uint16_t* out;
  float scale_log2;  // scale * log2(e): the kernels' exponentials are powers of two
};

// Strides of dimensions of extent 1 are set to 0, so no address depends on them.
inline DiffArgs make_diff_args(const kb_diff_attention_desc& desc, const uint16_t* q, const uint16_t* k,
                               const uint16_t* v, const float* lambda, const float* gamma, const int32_t* kv_lens,
                               const uint8_t* key_mask, uint16_t* out) {
  DiffArgs a{desc, q, k, v, lambda, gamma, kv_lens, key_mask, out, desc.scale * 1.4426950408889634f};
  kb_diff_attention_desc& d = a.d;
  if (d.batch == 1) d.q_batch = d.k_batch = d.v_batch = d.out_batch = d.mask_batch = 0;
  if (d.q_len == 1) d.q_token = d.out_token = 0;
  if (d.kv_len <= 1) d.k_token = d.v_token = 0;
  if (d.heads == 1) d.q_head = d.out_head = 0;
  if (d.kv_heads == 1) d.k_head = d.v_head = 0;
  return a;
}

// Keys of sequence b, kv_lens clamped to what K and V hold.
__device__ __forceinline__ int key_count(const DiffArgs& a, int b) {
  return a.kv_lens ? max(0, min(a.kv_lens[b], a.d.kv_len)) : a.d.kv_len;
}

// [first, last): the keys that some of the queries i0..i1 of a sequence of n
// keys sees, before the key mask.
__device__ __forceinline__ void key_range_n(const kb_diff_attention_desc& d, int n, int i0, int i1, int& first,
                                            int& last) {
  first = 0;
  last = n;
  if (d.causal) {
    const int off = n - d.q_len;  // position of query 0, negative when there are more queries than keys
    last = max(0, min(n, off + i1 + 1));
    if (d.window) first = max(0, off + i0 + 1 - d.window);
  }
}
__device__ __forceinline__ void key_range(const DiffArgs& a, int b, int i0, int i1, int& first, int& last) {
  key_range_n(a.d, key_count(a, b), i0, i1, first, last);
}

}  // namespace kb
