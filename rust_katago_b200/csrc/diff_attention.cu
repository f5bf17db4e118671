// Differential attention (kb_diff_attention): the difference of two softmax
// maps over shared values,
//   o = softmax(s q1 K1^T) V - lambda softmax(s q2 K2^T) V,
// then out = out_scale * gamma * o / sqrt(mean(o^2) + eps).
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "kb_diff.cuh"
#include "kb_internal.h"
#include "kb_numeric.cuh"

namespace kb {
namespace {

// Joins the parts of a row whose keys were split over blocks.  A block per row:
// the parts are dealt to its warps in order, each weighted by 2^(its maximum -
// the row's), and the warps' sums are added in order.  (One warp per row took
// longer over 100 parts than the keys did.)
constexpr int kJoinWarps = 8;

template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) diff_combine_kernel(const DiffArgs a, int splits) {
  constexpr int kE = 2 * D / 32;
  __shared__ float o_sh[kJoinWarps][2][2 * D], l_sh[kJoinWarps][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int h = static_cast<int>(row % a.d.heads);
  const int64_t bi = row / a.d.heads;
  float acc[2][kE], ll[2];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const float2* ml = a.part_ml + row * splits * 2 + m;
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, ml[2 * s].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    ll[m] = 0.0f;
#pragma unroll
    for (int e = 0; e < kE; ++e) acc[m][e] = 0.0f;
    const float* part = a.part_o + (row * splits * 2 + m) * (2 * D) + lane * kE;
#pragma unroll 4
    for (int s = warp; s < splits; s += kJoinWarps) {
      const float2 v = ml[2 * s];
      // A part that saw no key: its value sums may not have been written.  (A
      // NaN sum without a maximum is a row of NaN scores and has to go on.)
      if (v.x == -INFINITY && v.y == 0.0f) continue;
      const float f = exp2f(v.x - top);
      ll[m] += f * v.y;
      float o[kE];
      if constexpr (kE == 4) *reinterpret_cast<float4*>(o) = *reinterpret_cast<const float4*>(part + s * (4 * D));
      else *reinterpret_cast<float2*>(o) = *reinterpret_cast<const float2*>(part + s * (4 * D));
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[m][e] = fmaf(f, o[e], acc[m][e]);
    }
#pragma unroll
    for (int e = 0; e < kE; ++e) o_sh[warp][m][lane * kE + e] = acc[m][e];
    if (lane == 0) l_sh[warp][m] = ll[m];
  }
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int w = 1; w < kJoinWarps; ++w) {
      ll[m] += l_sh[w][m];
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[m][e] += o_sh[w][m][lane * kE + e];
    }
  finish_row<kE>(a, static_cast<int>(bi / a.d.q_len), static_cast<int>(bi % a.d.q_len), h, lane, acc, ll);
}

// How a call runs.  The kernel for few queries takes 16 rows (queries x heads of
// a group) a tile and reads K and V once for each; the one for many takes 128
// queries of one head.  Over the same keys a tile of the former costs about 3/4
// of one of the latter (32 sequences of 2,000 keys: 20 queries 64 against 42 us,
// 8 queries of 4 grouped heads 107 against 261 us), so the sums of tiles decide.
// A call of few tiles and short keys is all latency, where the former is quicker
// as long as its clusters fit one wave (one sequence of 1,000 keys: 32 tiles, 120
// queries of 4 heads, 14 against 21 us; 36 tiles, 96 queries of 6, 24 against 22;
// 48 tiles, 128 queries of 6, 26 and 26; 361 queries and keys: 23 tiles, 1 head, 11
// against 13, 46 tiles, 2 heads, 12 against 14, 138 tiles, 6 heads, 15 against 14).
// With longer keys it is not (24 tiles on 4,096 keys, 64 queries of 6 heads, 22
// against 21; 36 tiles on 2,048 keys 29 against 23).
struct Plan {
  bool few = false;
  int splits = 1;
  bool joined = false;  // by the kernel itself: no workspace
};

constexpr int kShortTiles = 36, kShortKeys = 2048;
constexpr int kFewKeys = 128;       // keys per block of four warps, at least
constexpr int kClusterKeys = 4096;  // up to here the join's launch costs more than blocks left idle
constexpr int kTileKeys = 128;
constexpr int kTilesPerPart = 4, kMostParts = 32;

Plan make_plan(const kb_diff_attention_desc& d) {
  Plan p;
  const int64_t rows = static_cast<int64_t>(d.q_len) * (d.heads / d.kv_heads);
  int dev = 0;
  cudaGetDevice(&dev);
  int64_t keys = d.kv_len;
  if (d.window && keys > static_cast<int64_t>(d.window) + d.q_len) keys = static_cast<int64_t>(d.window) + d.q_len;
  const int64_t few_tiles = (rows + 15) / 16 * d.kv_heads, many_tiles = (d.q_len + 127) / 128 * static_cast<int64_t>(d.heads);
  p.few = few_tiles * 3 <= many_tiles * 4 || (few_tiles * d.batch <= kShortTiles && keys <= kShortKeys) || keys == 0;
  if (p.few) {
    const int64_t units = static_cast<int64_t>(d.batch) * (rows <= 8 ? d.kv_heads : few_tiles);
    const int64_t most = (keys + kFewKeys - 1) / kFewKeys;
    // One wave of the two blocks that an SM holds; with more tiles than that
    // has room for, about two waves of smaller blocks, which even out lengths.
    const int64_t slots = 2 * static_cast<int64_t>(num_sms(dev));
    int64_t s = 2 * units <= slots ? slots / units : (2 * slots + units - 1) / units;
    // A cluster's worth serves when it gives every SM a block, or when the
    // keys are so few that the second launch would cost more.
    if (s > kMostCluster && (units * kMostCluster >= num_sms(dev) || keys <= kClusterKeys)) s = kMostCluster;
    if (s > most) s = most;
    p.splits = static_cast<int>(s < 1 ? 1 : s > 1024 ? 1024 : s);
    p.joined = p.splits <= kMostCluster;
  } else {
    // Parts of the keys so that the items fill the SMs evenly: rounds of items
    // times an item's time, plus the join, in microseconds (a tile of 128 keys
    // 2, as the prompt takes; an item's start and end 2.5, the join 4 and its
    // bytes, fitted to the order of the choices: the times themselves come out
    // low where parts are short, 119 for 361 tokens on three 16,001-key caches
    // that take 148).
    const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys, sms = num_sms(dev);
    const int64_t units = static_cast<int64_t>(d.batch) * many_tiles;
    const double part_bytes = static_cast<double>(d.batch) * d.q_len * d.heads * 32.0 * d.head_dim;
    double best = 0.0;
    for (int64_t s = 1; s <= kMostParts && (s == 1 || tiles / s >= kTilesPerPart); ++s) {
      const double rounds = static_cast<double>((units * s + sms - 1) / sms);
      const double us = rounds * (2.0 * static_cast<double>((tiles + s - 1) / s) + 2.5) +
                        (s > 1 ? 4.0 + part_bytes * static_cast<double>(s) / 5e6 : 0.0);
      if (s == 1 || us < 0.95 * best) best = us, p.splits = static_cast<int>(s);
    }
  }
  return p;
}

size_t partial_bytes(const kb_diff_attention_desc& d, int splits, size_t* o_offset) {
  const size_t parts = static_cast<size_t>(d.batch) * d.q_len * d.heads * splits * 2;
  const size_t at = (parts * sizeof(float2) + 127) / 128 * 128;
  if (o_offset) *o_offset = at;
  return at + parts * 2 * d.head_dim * sizeof(float);
}

int bad(const char* what) {
  set_error(std::string("kb_diff_attention: ") + what);
  return KB_E_INVALID;
}

int check_desc(const kb_diff_attention_desc* desc) {
  if (!desc) return bad("null descriptor");
  const kb_diff_attention_desc& d = *desc;
  if (d.dtype != KB_DT_F16 && d.dtype != KB_DT_BF16) return bad("dtype must be KB_DT_F16 or KB_DT_BF16");
  if (d.head_dim != 32 && d.head_dim != 64) return bad("head_dim must be 32 or 64");
  if (d.batch < 0 || d.q_len < 0 || d.kv_len < 0) return bad("batch, q_len and kv_len must not be negative");
  // (2^26 keys take a block about a second, below the limit of the kernels' waits.)
  if (d.batch > 65535 || d.q_len > (1 << 26) || d.kv_len > (1 << 26) || d.heads > 1024)
    return bad("at most 65535 sequences, 2^26 queries, 2^26 keys and 1024 heads");
  if (d.heads < 1 || d.kv_heads < 1 || d.heads % d.kv_heads) return bad("heads must be a multiple of kv_heads");
  if (d.window < 0 || (d.window > 0 && !d.causal)) return bad("a window must be positive and causal");
  if (!(d.scale > 0.0f) || !isfinite(d.scale) || !isfinite(d.out_scale) || !(d.eps >= 0.0f))
    return bad("a positive scale, a finite out_scale and eps >= 0 expected");
  const int64_t most = int64_t(1) << 38;
  auto ok = [&](int64_t stride, int64_t extent) { return extent <= 1 || (stride >= 0 && stride < most && stride % 8 == 0); };
  if (!ok(d.q_batch, d.batch) || !ok(d.q_token, d.q_len) || !ok(d.q_head, d.heads) || !ok(d.q_map, 2) ||
      !ok(d.k_batch, d.batch) || !ok(d.k_token, d.kv_len) || !ok(d.k_head, d.kv_heads) || !ok(d.k_map, 2) ||
      !ok(d.v_batch, d.batch) || !ok(d.v_token, d.kv_len) || !ok(d.v_head, d.kv_heads) ||
      !ok(d.out_batch, d.batch) || !ok(d.out_token, d.q_len) || !ok(d.out_head, d.heads))
    return bad("strides must be multiples of 8 elements, not negative and below 2^38");
  if ((d.q_len > 1 && d.q_token == 0) || (d.kv_len > 1 && (d.k_token == 0 || d.v_token == 0)))
    return bad("tokens cannot be broadcast");
  // out's dimensions nest: each steps over all that the smaller ones span.
  struct Dim {
    int64_t stride, extent;
  } dims[3] = {{d.out_batch, d.batch}, {d.out_token, d.q_len}, {d.out_head, d.heads}};
  std::sort(dims, dims + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  int64_t span = 2 * d.head_dim;
  for (const Dim& m : dims) {
    if (m.extent <= 1) continue;
    if (m.stride < span) return bad("out's rows must not overlap");
    span = m.stride > most / m.extent ? most : span + m.stride * (m.extent - 1);  // (no stride reaches `most`)
  }
  if (d.mask_batch < 0 || d.mask_batch > most) return bad("mask_batch");
  return KB_OK;
}

}  // namespace

int diff_combine_launch(const DiffArgs& a, int splits, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(a.d.batch) * a.d.q_len * a.d.heads;
  const unsigned grid = static_cast<unsigned>(rows);
  if (a.d.head_dim == 64) diff_combine_kernel<64><<<grid, 32 * kJoinWarps, 0, s>>>(a, splits);
  else diff_combine_kernel<32><<<grid, 32 * kJoinWarps, 0, s>>>(a, splits);
  return check_cuda(cudaGetLastError(), "differential attention join launch");
}

// Allow `kernel` to use `bytes` of dynamic shared memory on the current device.
int smem_opt_in(const void* kernel, int bytes) {
  return check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                    "differential attention smem attribute");
}

}  // namespace kb

extern "C" int kb_diff_attention_workspace(const kb_diff_attention_desc* desc, size_t* bytes) {
  using namespace kb;
  const int rc = check_desc(desc);
  if (rc) return rc;
  if (!bytes) return bad("null bytes");
  *bytes = 0;
  if (desc->batch == 0 || desc->q_len == 0) return KB_OK;
  const Plan p = make_plan(*desc);
  if (p.splits > 1 && !p.joined) *bytes = partial_bytes(*desc, p.splits, nullptr);
  return KB_OK;
}

namespace kb {
namespace {

int run(const kb_diff_attention_desc* desc, const uint16_t* q, const uint16_t* k, const uint16_t* v, const float* lambda,
        const float* gamma, const int32_t* kv_lens, const uint8_t* key_mask, uint16_t* out, void* workspace,
        size_t workspace_bytes, uint32_t* status, uint32_t wait_limit_ns, uintptr_t stream) {
  const int rc = check_desc(desc);
  if (rc) return rc;
  const kb_diff_attention_desc& d = *desc;
  if (d.batch == 0 || d.q_len == 0) return KB_OK;
  if (!q || !lambda || !out || (d.kv_len > 0 && (!k || !v))) return bad("null pointer");
  for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k), static_cast<const void*>(v),
                        static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (reinterpret_cast<uintptr_t>(p) % 16) return bad("q, k, v, out and workspace must be 16-byte aligned");
  for (const void* p : {static_cast<const void*>(lambda), static_cast<const void*>(gamma),
                        static_cast<const void*>(kv_lens), static_cast<const void*>(status)})
    if (reinterpret_cast<uintptr_t>(p) % 4) return bad("lambda, gamma, kv_lens and status must be 4-byte aligned");
  if (out == q || out == k || out == v) return bad("out must not be an input");
  size_t need = 0;
  kb_diff_attention_workspace(desc, &need);
  if (need > workspace_bytes || (need && !workspace)) {
    set_error("kb_diff_attention: workspace of " + std::to_string(need) + " bytes needed");
    return KB_E_INVALID;
  }
  DiffArgs a = make_diff_args(d, q, k, v, lambda, gamma, kv_lens, key_mask, out);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Plan p = make_plan(d);
  if (need) {
    size_t at = 0;
    partial_bytes(d, p.splits, &at);
    a.part_ml = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + at);
  }
  const int rc2 = p.few ? diff_decode_launch(a, p.splits, s) : diff_tc_launch(a, p.splits, status, wait_limit_ns, s);
  return rc2 || !need ? rc2 : diff_combine_launch(a, p.splits, s);
}

}  // namespace
}  // namespace kb

extern "C" int kb_diff_attention(const kb_diff_attention_desc* desc, const uint16_t* q, const uint16_t* k,
                                 const uint16_t* v, const float* lambda, const float* gamma, const int32_t* kv_lens,
                                 const uint8_t* key_mask, uint16_t* out, void* workspace, size_t workspace_bytes,
                                 uint32_t* status, uintptr_t stream) {
  return kb::run(desc, q, k, v, lambda, gamma, kv_lens, key_mask, out, workspace, workspace_bytes, status, 0, stream);
}

extern "C" int kb_test_diff_attention_wait_limit(const kb_diff_attention_desc* desc, const uint16_t* q,
                                                 const uint16_t* k, const uint16_t* v, const float* lambda,
                                                 uint16_t* out, void* workspace, size_t workspace_bytes,
                                                 unsigned long long wait_limit_ns, uint32_t* status, uintptr_t stream) {
  using namespace kb;
  if (!status || wait_limit_ns == 0 || wait_limit_ns > 2000000000ull) {
    set_error("kb_test_diff_attention_wait_limit: invalid arguments");
    return KB_E_INVALID;
  }
  return run(desc, q, k, v, lambda, nullptr, nullptr, nullptr, out, workspace, workspace_bytes, status,
             static_cast<uint32_t>(wait_limit_ns), stream);
}

extern "C" int kb_diff_lambda(const float* q1, const float* k1, const float* q2, const float* k2, int heads,
                              int head_dim, float lambda_init, float* lambda) {
  using namespace kb;
  if (!q1 || !k1 || !q2 || !k2 || !lambda || heads < 1 || head_dim < 1) {
    set_error("kb_diff_lambda: null pointer or empty shape");
    return KB_E_INVALID;
  }
  for (int h = 0; h < heads; ++h) {
    double s1 = 0.0, s2 = 0.0;
    for (int c = 0; c < head_dim; ++c) {
      const int64_t at = static_cast<int64_t>(h) * head_dim + c;
      s1 += static_cast<double>(q1[at]) * k1[at];
      s2 += static_cast<double>(q2[at]) * k2[at];
    }
    lambda[h] = static_cast<float>(exp(s1) - exp(s2) + lambda_init);
  }
  return KB_OK;
}
