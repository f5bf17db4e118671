// The norms around a block in one pass (kb_norm_residual):
//   r = res_scale * x + branch_scale * act(gate) * post_norm(y)
//   h = pre_norm(r) * (1 + mod_scale) + mod_shift
// x and y are read once, r and h written once, so HBM bounds it.  A group of
// threads (one warp, or one block for wide rows) holds a row in registers as
// fp32 from the first load to the last store; both norms reduce over the
// group.  Variances are taken from the centred values, not as E[v^2] - E[v]^2.
// h is computed from the unrounded r: rounding r first would add its error to h.
#include <stdint.h>

#include "kb_internal.h"
#include "kb_numeric.cuh"

namespace kb {
namespace {

struct NormArgs {
  kb_norm_residual_desc d;
  const void *x, *y;
  const float *post_gamma, *post_beta, *pre_gamma, *pre_beta;
  const void *gate, *mod_scale, *mod_shift;
  void *x_out, *h;
};

// Values of one row held by one thread: NC chunks of 8.  VEC: chunk c holds
// columns 8 (c TPR + i) .. + 7 (16- or 32-byte accesses); otherwise element e
// of chunk c is column (8 c + e) TPR + i, one element per access.
template <int NC, bool VEC>
__device__ __forceinline__ int column(int c, int e, int i, int tpr) {
  return VEC ? (c * tpr + i) * 8 + e : (c * 8 + e) * tpr + i;
}

__device__ __forceinline__ void unpack8(const uint4& w, bool f16, float* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = from16(static_cast<uint16_t>(u[i] & 0xffffu), f16);
    v[2 * i + 1] = from16(static_cast<uint16_t>(u[i] >> 16), f16);
  }
}

// Load the row piece of type `dtype` (KB_DT_*, uniform) at p.
template <int NC, bool VEC>
__device__ __forceinline__ void load_row(const void* p, int64_t offset, int dtype, int width, int i, int tpr,
                                         float (&v)[NC * 8]) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if constexpr (VEC) {
      const int col = (c * tpr + i) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c * 8 + e] = 0.0f;
      if (col < width) {
        if (dtype == KB_DT_F32) {
          const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + offset + col);
          *reinterpret_cast<float4*>(&v[c * 8]) = q[0];
          *reinterpret_cast<float4*>(&v[c * 8 + 4]) = q[1];
        } else {
          unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + offset + col), dtype == KB_DT_F16,
                  &v[c * 8]);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = (c * 8 + e) * tpr + i;
        v[c * 8 + e] = 0.0f;
        if (col < width) {
          if (dtype == KB_DT_F32) v[c * 8 + e] = static_cast<const float*>(p)[offset + col];
          else v[c * 8 + e] = from16(static_cast<const uint16_t*>(p)[offset + col], dtype == KB_DT_F16);
        }
      }
    }
  }
}

template <int NC, bool VEC>
__device__ __forceinline__ void store_row(void* p, int64_t offset, int dtype, int width, int i, int tpr,
                                          const float (&v)[NC * 8]) {
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if constexpr (VEC) {
      const int col = (c * tpr + i) * 8;
      if (col < width) {
        if (dtype == KB_DT_F32) {
          float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + offset + col);
          q[0] = make_float4(v[c * 8], v[c * 8 + 1], v[c * 8 + 2], v[c * 8 + 3]);
          q[1] = make_float4(v[c * 8 + 4], v[c * 8 + 5], v[c * 8 + 6], v[c * 8 + 7]);
        } else {
          const bool f16 = dtype == KB_DT_F16;
          uint4 w;
          w.x = pack16x2(make_float2(v[c * 8], v[c * 8 + 1]), f16);
          w.y = pack16x2(make_float2(v[c * 8 + 2], v[c * 8 + 3]), f16);
          w.z = pack16x2(make_float2(v[c * 8 + 4], v[c * 8 + 5]), f16);
          w.w = pack16x2(make_float2(v[c * 8 + 6], v[c * 8 + 7]), f16);
          *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + offset + col) = w;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = (c * 8 + e) * tpr + i;
        if (col < width) {
          if (dtype == KB_DT_F32) static_cast<float*>(p)[offset + col] = v[c * 8 + e];
          else static_cast<uint16_t*>(p)[offset + col] = bits16(v[c * 8 + e], dtype == KB_DT_F16);
        }
      }
    }
  }
}

// Sum over the row's threads; every thread gets it.  `red` holds one float per
// warp; it is free again after the call.
template <bool BLOCK>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (BLOCK) {
    const int warps = blockDim.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < warps; ++w) v += red[w];
  }
  return v;
}

// v = norm(v) * gamma + beta over the row; columns past `width` hold zeros.
template <int NC, bool VEC, bool BLOCK>
__device__ __forceinline__ void norm_row(float (&v)[NC * 8], int kind, const float* gamma, const float* beta, float eps,
                                         int width, int i, int tpr, float* red) {
  if (kind == KB_NORM_NONE) return;
  float mean = 0.0f;
  if (kind == KB_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < NC * 8; ++k) s += v[k];
    mean = row_sum<BLOCK>(s, red) / static_cast<float>(width);
  }
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = column<NC, VEC>(c, e, i, tpr) < width ? v[c * 8 + e] - mean : 0.0f;
      v[c * 8 + e] = t;
      s = fmaf(t, t, s);
    }
  const float rstd = 1.0f / sqrtf(row_sum<BLOCK>(s, red) / static_cast<float>(width) + eps);
  float g[NC * 8];
  if (gamma) load_row<NC, VEC>(gamma, 0, KB_DT_F32, width, i, tpr, g);
#pragma unroll
  for (int k = 0; k < NC * 8; ++k) v[k] = v[k] * rstd * (gamma ? g[k] : 1.0f);
  if (beta) {
    load_row<NC, VEC>(beta, 0, KB_DT_F32, width, i, tpr, g);
#pragma unroll
    for (int k = 0; k < NC * 8; ++k) v[k] += g[k];
  }
}

template <int NC, bool VEC, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) norm_residual_kernel(const NormArgs a) {
  __shared__ float red[32];
  const kb_norm_residual_desc& d = a.d;
  const int tpr = BLOCK ? blockDim.x : 32;
  const int i = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int64_t row = BLOCK ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= d.rows) return;  // whole warps, or the whole block
  const int w = d.width;
  float r[NC * 8];
  load_row<NC, VEC>(a.x, row * d.x_stride, d.stream_dtype, w, i, tpr, r);
  const int64_t cond = row / d.rows_per_cond * d.cond_stride;
  if (a.y) {
    float n[NC * 8];
    load_row<NC, VEC>(a.y, row * d.y_stride, d.branch_dtype, w, i, tpr, n);
    norm_row<NC, VEC, BLOCK>(n, d.post_norm, a.post_gamma, a.post_beta, d.eps, w, i, tpr, red);
    if (a.gate) {
      float g[NC * 8];
      load_row<NC, VEC>(a.gate, cond, d.branch_dtype, w, i, tpr, g);
#pragma unroll
      for (int k = 0; k < NC * 8; ++k) {
        float f = g[k];
        if (d.gate_act == KB_GATE_SIGMOID) f = 1.0f / (1.0f + expf(-f));
        else if (d.gate_act == KB_GATE_TANH) f = tanhf(f);
        n[k] *= f;
      }
    }
#pragma unroll
    for (int k = 0; k < NC * 8; ++k) r[k] = d.res_scale * r[k] + d.branch_scale * n[k];
  } else {
#pragma unroll
    for (int k = 0; k < NC * 8; ++k) r[k] *= d.res_scale;
  }
  if (a.x_out) store_row<NC, VEC>(a.x_out, row * d.x_out_stride, d.stream_dtype, w, i, tpr, r);
  if (a.h) {
    norm_row<NC, VEC, BLOCK>(r, d.pre_norm, a.pre_gamma, a.pre_beta, d.eps, w, i, tpr, red);
    float m[NC * 8];
    if (a.mod_scale) {
      load_row<NC, VEC>(a.mod_scale, cond, d.branch_dtype, w, i, tpr, m);
#pragma unroll
      for (int k = 0; k < NC * 8; ++k) r[k] *= 1.0f + m[k];
    }
    if (a.mod_shift) {
      load_row<NC, VEC>(a.mod_shift, cond, d.branch_dtype, w, i, tpr, m);
#pragma unroll
      for (int k = 0; k < NC * 8; ++k) r[k] += m[k];
    }
    store_row<NC, VEC>(a.h, row * d.h_stride, d.branch_dtype, w, i, tpr, r);
  }
}

template <bool VEC>
int launch(const NormArgs& a, cudaStream_t s) {
  const int chunks = (a.d.width + 7) / 8, rows = a.d.rows;
  // Rows of up to 1,024 columns take a warp each, wider ones a block with at
  // most 16 columns per thread.
  const int warps = rows < 8 * 148 ? 1 : 4;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(rows) + warps - 1) / warps);
  if (chunks <= 32) norm_residual_kernel<1, VEC, false><<<grid, 32 * warps, 0, s>>>(a);
  else if (chunks <= 64) norm_residual_kernel<2, VEC, false><<<grid, 32 * warps, 0, s>>>(a);
  else if (chunks <= 96) norm_residual_kernel<3, VEC, false><<<grid, 32 * warps, 0, s>>>(a);
  else if (chunks <= 128) norm_residual_kernel<4, VEC, false><<<grid, 32 * warps, 0, s>>>(a);
  else norm_residual_kernel<2, VEC, true><<<rows, ((chunks + 1) / 2 + 31) / 32 * 32, 0, s>>>(a);
  return check_cuda(cudaGetLastError(), "norm launch");
}

int bad(const char* what) {
  set_error(std::string("kb_norm_residual: ") + what);
  return KB_E_INVALID;
}

bool dtype_ok(int t) { return t == KB_DT_F32 || t == KB_DT_F16 || t == KB_DT_BF16; }

}  // namespace
}  // namespace kb

extern "C" int kb_norm_residual(const kb_norm_residual_desc* desc, const void* x, const void* y,
                                const float* post_gamma, const float* post_beta, const float* pre_gamma,
                                const float* pre_beta, const void* gate, const void* mod_scale, const void* mod_shift,
                                void* x_out, void* h, uintptr_t stream) {
  using namespace kb;
  if (!desc) return bad("null descriptor");
  const kb_norm_residual_desc& d = *desc;
  if (d.rows < 0 || d.width < 1 || d.width > 16384) return bad("rows >= 0 and width 1..16384 expected");
  if (!dtype_ok(d.stream_dtype) || !dtype_ok(d.branch_dtype)) return bad("dtypes must be KB_DT_*");
  for (int k : {d.post_norm, d.pre_norm})
    if (k < KB_NORM_NONE || k > KB_NORM_LAYER) return bad("norms must be KB_NORM_*");
  if (d.gate_act < KB_GATE_LINEAR || d.gate_act > KB_GATE_TANH) return bad("gate_act must be KB_GATE_*");
  if (!(d.eps >= 0.0f)) return bad("eps must not be negative");
  const bool cond = gate || mod_scale || mod_shift;
  if (cond && d.rows_per_cond < 1) return bad("rows_per_cond must be positive");
  if (d.rows == 0) return KB_OK;
  if (!x || (!x_out && !h)) return bad("x and one of x_out and h must be given");
  if (gate && !y) return bad("a gate needs y");
  for (int64_t st : {d.x_stride, y ? d.y_stride : 0, x_out ? d.x_out_stride : 0, h ? d.h_stride : 0,
                     cond ? d.cond_stride : 0})
    if (st < 0) return bad("strides must not be negative");
  if (d.rows > 1 && ((x_out && d.x_out_stride < d.width) || (h && d.h_stride < d.width)))
    return bad("output rows must not overlap");
  if ((x_out == x && d.x_out_stride != d.x_stride) || (h && h == y && d.h_stride != d.y_stride))
    return bad("in place needs equal strides");
  if (h && (h == x || h == x_out)) return bad("h must not be x or x_out");
  if (x_out && x_out == y) return bad("x_out must not be y");
  NormArgs a{d, x, y, post_gamma, post_beta, pre_gamma, pre_beta, gate, mod_scale, mod_shift, x_out, h};
  if (a.d.rows_per_cond < 1) a.d.rows_per_cond = 1;
  // Eight columns per access need whole groups and 16-byte rows; anything
  // else takes the kernel of single elements.
  bool vec = d.width % 8 == 0;
  for (const void* p : {x, y, static_cast<const void*>(post_gamma), static_cast<const void*>(post_beta),
                        static_cast<const void*>(pre_gamma), static_cast<const void*>(pre_beta), gate, mod_scale,
                        mod_shift, static_cast<const void*>(x_out), static_cast<const void*>(h)})
    vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  vec = vec && d.x_stride % 8 == 0 && (!y || d.y_stride % 8 == 0) && (!x_out || d.x_out_stride % 8 == 0) &&
        (!h || d.h_stride % 8 == 0) && (!cond || d.cond_stride % 8 == 0);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return vec ? launch<true>(a, s) : launch<false>(a, s);
}
