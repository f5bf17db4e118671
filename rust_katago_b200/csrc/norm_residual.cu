// The norms around a block in one pass (kb_norm_residual):
//   r = res_scale * x + branch_scale * act(gate) * post_norm(y)
//   h = pre_norm(r) * (1 + mod_scale) + mod_shift
// x and y are read once, r and h written once, so HBM bounds it.
//
// A group of threads (one warp, or one block for wide rows) walks a run of
// neighbouring rows and holds a row in registers as fp32 from the first load to
// the last store; the next row's x and y are loaded while this one is at work.
// What rows share is folded into at most four vectors in shared memory, built
// again only when the row of gate and modulation changes:
//   r = res_scale x + G n' + C   G = branch_scale gate gamma, C = branch_scale gate beta
//   h = A r' + B                 A = gamma' (1 + mod_scale),  B = beta' (1 + mod_scale) + mod_shift
// with n' and r' the normalised values.  (With the vectors applied one by one
// and the types chosen at run time, the instructions bounded it: 92,416 x 768
// took 317 us.)  Variances are taken from the centred values, not as E[v^2] -
// E[v]^2.  h is computed from the unrounded r: rounding r first would add its
// error to h.
// Measured: 92,416 x 768 bf16 with a gate row per 361 rows 99 us, 5.7 TB/s (0.88
// of the copy rate); 8,191 x 5,120, fp32 stream and bf16 branch, layer norms 100
// us, 5.0 TB/s (block-wide sums between loads); 20,000 rows of bf16 RMS norms by
// single elements, 1,001 columns 61 us (1,000 by eights 34), 4,099 columns 322.
#include <stdint.h>

#include <atomic>
#include <type_traits>

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

// Runs of rows per resident group (one leaves SMs idle at the end, 109 instead of
// 99 us for 92,416 x 768 with a gate per 361 rows; four build the shared vectors
// too often, 101 us, and 128 instead of 112 for 60,000 x 1,024 layer norms), and
// groups of one warp to plan for on an SM, by chunks per thread: they set the
// length of the runs, not what an SM holds (with four chunks and both shifts its
// shared memory has room for 13).  One and two chunks, 12 / 20 / 28: 92,416 x 512
// 76 / 66 / 67 us, 92,416 x 256 layer norms of fp32 61 / 58 / 58.  Three and four,
// 8 / 12 / 16 / 20: 92,416 x 768 RMS with gates 109 / 105 / 99 / 102, layer norms
// 131 / 99 / 104 / 110, 60,000 x 1,024 layer norms with gates 105 / 108 / 112 / 114.
constexpr int kRunsPerSlot = 2;
constexpr int kResident1 = 20, kResident2 = 20, kResident3 = 16;

// ------------------------------------------------------------------ typed kernels
// A thread holds NC chunks of eight columns.  VEC: chunk c is columns 8 (c TPR +
// i).. of the row, 16 or 32 bytes an access; otherwise element e of chunk c is
// column (8 c + e) TPR + i, an element an access, for rows of any width and
// alignment.

// Eight columns of type DT as fp32 pairs, and back.
template <int DT>
struct Raw8 {
  uint4 w[DT == KB_DT_F32 ? 2 : 1];
};

// A load that the compiler may move across the stores of other rows (which it
// cannot know to be other addresses), but not through the read-only path:
// outputs may be inputs.
__device__ __forceinline__ uint4 load_row16(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <int DT>
__device__ __forceinline__ Raw8<DT> load8(const void* p, int64_t at) {
  Raw8<DT> r;
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (DT == KB_DT_F32 ? 4 : 2));
  r.w[0] = load_row16(q);
  if constexpr (DT == KB_DT_F32) r.w[1] = load_row16(q + 1);
  return r;
}

// Eight single elements.
template <int DT>
struct Raw1 {
  std::conditional_t<DT == KB_DT_F32, float, uint16_t> e[8];
};

template <int DT>
__device__ __forceinline__ void load_one(const void* p, int64_t at, bool in, Raw1<DT>& r, int e) {
  if constexpr (DT == KB_DT_F32) {
    float v = 0.0f;
    if (in) asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(static_cast<const float*>(p) + at));
    r.e[e] = v;
  } else {
    uint16_t v = 0;
    if (in) asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(static_cast<const uint16_t*>(p) + at));
    r.e[e] = v;
  }
}

template <int DT>
__device__ __forceinline__ void open8(const Raw1<DT>& r, float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == KB_DT_F32) v[i] = make_float2(r.e[2 * i], r.e[2 * i + 1]);
    else v[i] = make_float2(from16(r.e[2 * i], DT == KB_DT_F16), from16(r.e[2 * i + 1], DT == KB_DT_F16));
  }
}

template <int DT>
__device__ __forceinline__ void open8(const Raw8<DT>& r, float2 (&v)[4]) {
  const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == KB_DT_F32) {
      const uint4& w = r.w[i >> 1];
      v[i] = i & 1 ? make_float2(__uint_as_float(w.z), __uint_as_float(w.w))
                   : make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    } else if constexpr (DT == KB_DT_F16) {
      v[i] = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    } else {
      v[i] = make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
    }
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t at, const float2 (&v)[4]) {
  if constexpr (DT == KB_DT_F32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    q[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    q[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) =
        make_uint4(pack16x2(v[0], DT == KB_DT_F16), pack16x2(v[1], DT == KB_DT_F16), pack16x2(v[2], DT == KB_DT_F16),
                   pack16x2(v[3], DT == KB_DT_F16));
  }
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Sum of v over the row's threads.  BLOCK: `red` holds two sets of one float
// per warp (zeros past the last) that successive sums alternate between, so
// each needs one barrier.
template <bool BLOCK>
__device__ __forceinline__ float group_sum(float2 v, float (*red)[16], int& turn) {
  float s = v.x + v.y;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if constexpr (BLOCK) {
    float* slot = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = s;
    __syncthreads();
    const float4* q = reinterpret_cast<const float4*>(slot);
    const float4 a = q[0], b = q[1], c = q[2], d = q[3];
    s = ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w)) + (((c.x + c.y) + (c.z + c.w)) + ((d.x + d.y) + (d.z + d.w)));
  }
  return s;
}

// v -> v centred (KB_NORM_LAYER); returns the factor 1 / sqrt(mean(v^2) + eps),
// or 1 without a norm.  Columns outside the row hold zeros.
template <int NC, bool BLOCK, bool VEC, typename In>
__device__ __forceinline__ float normalise(float2 (&v)[NC][4], int kind, float inv_width, float eps, const In& in,
                                           float (*red)[16], int& turn) {
  if (kind == KB_NORM_NONE) return 1.0f;
  if (kind == KB_NORM_LAYER) {
    float2 s = both(0.0f);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add2(s, v[c][i]);
    const float mean = group_sum<BLOCK>(s, red, turn) * inv_width;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (VEC && !in(c, 0)) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[c][i] = add2(v[c][i], both(-mean));
        if constexpr (!VEC) v[c][i] = make_float2(in(c, 2 * i) ? v[c][i].x : 0.0f, in(c, 2 * i + 1) ? v[c][i].y : 0.0f);
      }
    }
  }
  float2 s0 = both(0.0f), s1 = both(0.0f);
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      s0 = fma2(v[c][i], v[c][i], s0);
      s1 = fma2(v[c][i + 1], v[c][i + 1], s1);
    }
  return rsqrtf(group_sum<BLOCK>(add2(s0, s1), red, turn) * inv_width + eps);
}

__device__ __forceinline__ float gate_value(float v, int act) {
  if (act == KB_GATE_SIGMOID) return 1.0f / (1.0f + expf(-v));
  if (act == KB_GATE_TANH) return tanhf(v);
  return v;
}

// XT, YT: types of stream and branch.  SHIFT: 0 no shifts, 1 only B, 2 also C.
// THREADS: 32 (a warp per row) or the most that a block has.
template <int XT, int YT, int NC, int THREADS, int SHIFT, bool VEC>
__global__ void __launch_bounds__(THREADS, THREADS == 320 ? 2 : 1) norm_rows_kernel(const NormArgs a,
                                                                                   int rows_per_group) {
  constexpr bool BLOCK = THREADS > 32;
  __shared__ alignas(16) float red[2][16];
  extern __shared__ float4 shared_vectors[];  // [vector][chunk][half][thread]
  if constexpr (BLOCK) {
    if (threadIdx.x < 32) reinterpret_cast<float*>(red)[threadIdx.x] = 0.0f;
    __syncthreads();
  }
  const kb_norm_residual_desc& d = a.d;
  const int tpr = BLOCK ? blockDim.x : 32;
  const int i = threadIdx.x;
  int64_t row = static_cast<int64_t>(blockIdx.x) * rows_per_group;
  const int64_t end = min(row + rows_per_group, static_cast<int64_t>(d.rows));
  if (row >= end) return;
  const int col = i * 8, step = tpr * 8;
  int valid = 0;  // VEC: chunks of this thread inside the row
#pragma unroll
  for (int c = 0; c < NC; ++c) valid += col + c * step < d.width;
  auto column = [&](int c, int e) { return VEC ? col + c * step + e : (c * 8 + e) * tpr + i; };
  auto inside = [&](int c, int e) { return VEC ? c < valid : column(c, e) < d.width; };
  // Eight columns of a tensor of type DT at element `row_at` (VEC: of a chunk
  // inside the row; otherwise with zeros outside it).
  auto get = [&](auto dt, const void* p, int64_t row_at, int c) {
    constexpr int DT = decltype(dt)::value;
    if constexpr (VEC) {
      return load8<DT>(p, row_at + column(c, 0));
    } else {
      Raw1<DT> r;
#pragma unroll
      for (int e = 0; e < 8; ++e) load_one<DT>(p, row_at + column(c, e), inside(c, e), r, e);
      return r;
    }
  };
  auto put = [&](auto dt, void* p, int64_t row_at, int c, const float2 (&v)[4]) {
    constexpr int DT = decltype(dt)::value;
    if constexpr (VEC) {
      if (c < valid) store8<DT>(p, row_at + column(c, 0), v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!inside(c, e)) continue;
        const float f = e & 1 ? v[e / 2].y : v[e / 2].x;
        if constexpr (DT == KB_DT_F32) static_cast<float*>(p)[row_at + column(c, e)] = f;
        else static_cast<uint16_t*>(p)[row_at + column(c, e)] = bits16(f, DT == KB_DT_F16);
      }
    }
  };
  constexpr std::integral_constant<int, KB_DT_F32> kF32{};
  constexpr std::integral_constant<int, XT> kX{};
  constexpr std::integral_constant<int, YT> kY{};
  const float inv_width = 1.0f / static_cast<float>(d.width);
  int turn = 0;

  // The vectors G, A, B, C in shared memory, each thread's own columns (nothing
  // to synchronise).  In registers they cost half the warps: 118 us instead of
  // 99 for 92,416 x 768.
  auto keep = [&](int which, int c, const float2 (&v)[4]) {
    float4* at = shared_vectors + (which * NC + c) * 2 * tpr + i;
    at[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    at[tpr] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
  };
  auto vector = [&](int which, int c, float2 (&v)[4]) {
    const float4* at = shared_vectors + (which * NC + c) * 2 * tpr + i;
    const float4 p = at[0], q = at[tpr];
    v[0] = make_float2(p.x, p.y), v[1] = make_float2(p.z, p.w), v[2] = make_float2(q.x, q.y), v[3] = make_float2(q.z, q.w);
  };
  auto vectors = [&](int64_t cond) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float2 gv[4], av[4], cv[4], bv[4];
      float2 t[4], u[4];
      auto param = [&](const float* p, float otherwise, float2 (&v)[4]) {
        if (p && (!VEC || c < valid)) open8(get(kF32, p, 0, c), v);
        else
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = both(otherwise);
      };
      auto mod = [&](const void* p, float otherwise, float2 (&v)[4]) {
        if (p && (!VEC || c < valid)) open8(get(kY, p, cond * d.cond_stride, c), v);
        else
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] = both(otherwise);
      };
      mod(a.gate, 1.0f, t);
      param(d.post_norm == KB_NORM_NONE ? nullptr : a.post_gamma, 1.0f, gv);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (a.gate) t[k] = make_float2(gate_value(t[k].x, d.gate_act), gate_value(t[k].y, d.gate_act));
        t[k] = mul2(t[k], both(d.branch_scale));
        gv[k] = mul2(gv[k], t[k]);
      }
      if constexpr (SHIFT == 2) {
        param(d.post_norm == KB_NORM_NONE ? nullptr : a.post_beta, 0.0f, u);
#pragma unroll
        for (int k = 0; k < 4; ++k) cv[k] = mul2(u[k], t[k]);
      }
      mod(a.mod_scale, 0.0f, t);
      param(d.pre_norm == KB_NORM_NONE ? nullptr : a.pre_gamma, 1.0f, av);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        t[k] = add2(t[k], both(1.0f));
        av[k] = mul2(av[k], t[k]);
      }
      if constexpr (SHIFT) {
        param(d.pre_norm == KB_NORM_NONE ? nullptr : a.pre_beta, 0.0f, u);
        mod(a.mod_shift, 0.0f, bv);
#pragma unroll
        for (int k = 0; k < 4; ++k) bv[k] = fma2(u[k], t[k], bv[k]);
        keep(2, c, bv);
      }
      keep(0, c, gv);
      keep(1, c, av);
      if constexpr (SHIFT == 2) keep(3, c, cv);
    }
  };

  std::conditional_t<VEC, Raw8<XT>, Raw1<XT>> xr[NC];
  std::conditional_t<VEC, Raw8<YT>, Raw1<YT>> yr[NC];
  auto fetch = [&](int64_t at) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (VEC && c >= valid) continue;  // stays zero
      xr[c] = get(kX, a.x, at * d.x_stride, c);
      if (a.y) yr[c] = get(kY, a.y, at * d.y_stride, c);
    }
  };
#pragma unroll
  for (int c = 0; c < NC; ++c) xr[c] = {}, yr[c] = {};
  fetch(row);
  const bool conditioned = a.gate || a.mod_scale || a.mod_shift;
  int64_t cond = conditioned ? row / d.rows_per_cond : 0, next_cond = conditioned ? (cond + 1) * d.rows_per_cond : end;
  vectors(cond);
  for (; row < end; ++row) {
    if (row == next_cond) {
      vectors(++cond);
      next_cond += d.rows_per_cond;
    }
    float2 r[NC][4], n[NC][4];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      open8(xr[c], r[c]);
      open8(yr[c], n[c]);
    }
    if (row + 1 < end) fetch(row + 1);
    if (a.y) {
      const float2 f = both(normalise<NC, BLOCK, VEC>(n, d.post_norm, inv_width, d.eps, inside, red, turn));
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float2 gv[4], cv[4];
        vector(0, c, gv);
        if constexpr (SHIFT == 2) vector(3, c, cv);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float2 t = mul2(n[c][k], f);
          if constexpr (SHIFT == 2) t = fma2(t, gv[k], cv[k]);
          else t = mul2(t, gv[k]);
          r[c][k] = fma2(r[c][k], both(d.res_scale), t);
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k) r[c][k] = mul2(r[c][k], both(d.res_scale));
    }
    if (a.x_out)
#pragma unroll
      for (int c = 0; c < NC; ++c) put(kX, a.x_out, row * d.x_out_stride, c, r[c]);
    if (a.h) {
      const float2 f = both(normalise<NC, BLOCK, VEC>(r, d.pre_norm, inv_width, d.eps, inside, red, turn));
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (VEC && c >= valid) continue;
        float2 av[4], bv[4];
        vector(1, c, av);
        if constexpr (SHIFT) vector(2, c, bv);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 t = mul2(r[c][k], f);
          if constexpr (SHIFT) r[c][k] = fma2(t, av[k], bv[k]);
          else r[c][k] = mul2(t, av[k]);
        }
        put(kY, a.h, row * d.h_stride, c, r[c]);
      }
    }
  }
}

// Rows of up to 1,024 columns take a warp each (and a block of its own, which
// packs best at 90 to 190 registers a thread), wider ones a block of threads
// with 16 columns each; enough groups to fill the SMs, each with a run of
// neighbouring rows.
template <int XT, int YT, int NC, int THREADS, int SHIFT, bool VEC>
int launch_shift(const NormArgs& a, cudaStream_t s) {
  auto kern = norm_rows_kernel<XT, YT, NC, THREADS, SHIFT, VEC>;
  int dev = 0;
  cudaGetDevice(&dev);
  int threads = 32, resident = NC == 1 ? kResident1 : NC == 2 ? kResident2 : kResident3;
  if (THREADS > 32) {
    threads = ((a.d.width + 7) / 8 + NC * 32 - 1) / (NC * 32) * 32;
    resident = THREADS == 320 ? 2 : 1;
  }
  const int bytes = (2 + SHIFT) * NC * threads * 32;
  if (THREADS > 32) {
    if (bytes + static_cast<int>(sizeof(float)) * 32 > 48 * 1024) {  // with the static part
      static std::atomic<uint64_t> configured{0};
      const uint64_t bit = 1ull << (dev & 63);
      if (!(configured.load() & bit)) {
        const int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       (2 + SHIFT) * NC * THREADS * 32), "norm smem attribute");
        if (rc) return rc;
        configured.fetch_or(bit);
      }
    }
  }
  int64_t groups = static_cast<int64_t>(num_sms(dev)) * kRunsPerSlot * resident;
  const int64_t per = (a.d.rows + groups - 1) / groups;
  groups = (a.d.rows + per - 1) / per;
  kern<<<static_cast<unsigned>(groups), threads, bytes, s>>>(a, static_cast<int>(per));
  return check_cuda(cudaGetLastError(), "norm launch");
}

template <int XT, int YT, int NC, int THREADS, bool VEC>
int launch_rows(const NormArgs& a, cudaStream_t s) {
  if constexpr (VEC) {
    if (!a.post_beta && !a.pre_beta && !a.mod_shift) return launch_shift<XT, YT, NC, THREADS, 0, true>(a, s);
    if (!a.post_beta) return launch_shift<XT, YT, NC, THREADS, 1, true>(a, s);
  }
  return launch_shift<XT, YT, NC, THREADS, 2, VEC>(a, s);
}

constexpr int kTypedWidth = 8192;  // the widest row of the typed kernels

template <int XT, int YT, bool VEC>
int launch_width(const NormArgs& a, cudaStream_t s) {
  const int chunks = (a.d.width + 7) / 8;
  if (chunks <= 32) return launch_rows<XT, YT, 1, 32, VEC>(a, s);
  if (chunks <= 64) return launch_rows<XT, YT, 2, 32, VEC>(a, s);
  if (chunks <= 96) return launch_rows<XT, YT, 3, 32, VEC>(a, s);
  if (chunks <= 128) return launch_rows<XT, YT, 4, 32, VEC>(a, s);
  if (chunks <= 640) return launch_rows<XT, YT, 2, 320, VEC>(a, s);
  return launch_rows<XT, YT, 2, 512, VEC>(a, s);
}

template <int XT, int YT>
int launch_typed(const NormArgs& a, bool vec, cudaStream_t s) {
  return vec ? launch_width<XT, YT, true>(a, s) : launch_width<XT, YT, false>(a, s);
}

// ------------------------------------------------------------------ any types and width
// Values of one row held by one thread: element k is column k TPR + i, one
// element per access, types chosen at run time.

template <int N>
__device__ __forceinline__ void load_row(const void* p, int64_t offset, int dtype, int width, int i, int tpr,
                                         float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int col = k * tpr + i;
    v[k] = 0.0f;
    if (col < width) {
      if (dtype == KB_DT_F32) v[k] = static_cast<const float*>(p)[offset + col];
      else v[k] = from16(static_cast<const uint16_t*>(p)[offset + col], dtype == KB_DT_F16);
    }
  }
}

template <int N>
__device__ __forceinline__ void store_row(void* p, int64_t offset, int dtype, int width, int i, int tpr,
                                          const float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int col = k * tpr + i;
    if (col < width) {
      if (dtype == KB_DT_F32) static_cast<float*>(p)[offset + col] = v[k];
      else static_cast<uint16_t*>(p)[offset + col] = bits16(v[k], dtype == KB_DT_F16);
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
template <int N, bool BLOCK>
__device__ __forceinline__ void norm_row(float (&v)[N], int kind, const float* gamma, const float* beta, float eps,
                                         int width, int i, int tpr, float* red) {
  if (kind == KB_NORM_NONE) return;
  float mean = 0.0f;
  if (kind == KB_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) s += v[k];
    mean = row_sum<BLOCK>(s, red) / static_cast<float>(width);
  }
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    v[k] = k * tpr + i < width ? v[k] - mean : 0.0f;
    s = fmaf(v[k], v[k], s);
  }
  const float rstd = 1.0f / sqrtf(row_sum<BLOCK>(s, red) / static_cast<float>(width) + eps);
  float g[N];
  if (gamma) load_row(gamma, 0, KB_DT_F32, width, i, tpr, g);
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = v[k] * rstd * (gamma ? g[k] : 1.0f);
  if (beta) {
    load_row(beta, 0, KB_DT_F32, width, i, tpr, g);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += g[k];
  }
}

template <int N, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) norm_residual_kernel(const NormArgs a) {
  __shared__ float red[32];
  const kb_norm_residual_desc& d = a.d;
  const int tpr = BLOCK ? blockDim.x : 32;
  const int i = BLOCK ? threadIdx.x : threadIdx.x & 31;
  const int64_t row = BLOCK ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= d.rows) return;  // whole warps, or the whole block
  const int w = d.width;
  float r[N];
  load_row(a.x, row * d.x_stride, d.stream_dtype, w, i, tpr, r);
  const int64_t cond = row / d.rows_per_cond * d.cond_stride;
  if (a.y) {
    float n[N];
    load_row(a.y, row * d.y_stride, d.branch_dtype, w, i, tpr, n);
    norm_row<N, BLOCK>(n, d.post_norm, a.post_gamma, a.post_beta, d.eps, w, i, tpr, red);
    if (a.gate) {
      float g[N];
      load_row(a.gate, cond, d.branch_dtype, w, i, tpr, g);
#pragma unroll
      for (int k = 0; k < N; ++k) n[k] *= gate_value(g[k], d.gate_act);
    }
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] = d.res_scale * r[k] + d.branch_scale * n[k];
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) r[k] *= d.res_scale;
  }
  if (a.x_out) store_row(a.x_out, row * d.x_out_stride, d.stream_dtype, w, i, tpr, r);
  if (a.h) {
    norm_row<N, BLOCK>(r, d.pre_norm, a.pre_gamma, a.pre_beta, d.eps, w, i, tpr, red);
    float m[N];
    if (a.mod_scale) {
      load_row(a.mod_scale, cond, d.branch_dtype, w, i, tpr, m);
#pragma unroll
      for (int k = 0; k < N; ++k) r[k] *= 1.0f + m[k];
    }
    if (a.mod_shift) {
      load_row(a.mod_shift, cond, d.branch_dtype, w, i, tpr, m);
#pragma unroll
      for (int k = 0; k < N; ++k) r[k] += m[k];
    }
    store_row(a.h, row * d.h_stride, d.branch_dtype, w, i, tpr, r);
  }
}

int launch_any(const NormArgs& a, cudaStream_t s) {
  const int rows = a.d.rows, w = a.d.width;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(rows) + 3) / 4);
  if (w <= 256) norm_residual_kernel<8, false><<<grid, 128, 0, s>>>(a);
  else if (w <= 512) norm_residual_kernel<16, false><<<grid, 128, 0, s>>>(a);
  else if (w <= 1024) norm_residual_kernel<32, false><<<grid, 128, 0, s>>>(a);
  else norm_residual_kernel<16, true><<<rows, ((w + 15) / 16 + 31) / 32 * 32, 0, s>>>(a);
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
  // What rows share is read while other rows are written; a row of its own per
  // row is read before h's.
  for (const void* p : {static_cast<const void*>(post_gamma), static_cast<const void*>(post_beta),
                        static_cast<const void*>(pre_gamma), static_cast<const void*>(pre_beta), gate, mod_scale, mod_shift})
    if (p && (p == x_out || (p == h && (p == post_gamma || p == post_beta || p == pre_gamma || p == pre_beta ||
                                        (d.rows > 1 && (d.rows_per_cond != 1 || d.cond_stride != d.h_stride))))))
      return bad("x_out and h must not be a gamma, a beta, the gate or a modulation");
  auto off = [](const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == KB_DT_F32 ? 4 : 2) != 0; };
  for (const void* p : {x, static_cast<const void*>(x_out)})
    if (off(p, d.stream_dtype)) return bad("x and x_out must be aligned to their elements");
  for (const void* p : {y, gate, mod_scale, mod_shift, static_cast<const void*>(h)})
    if (off(p, d.branch_dtype)) return bad("y, gate, mod_scale, mod_shift and h must be aligned to their elements");
  for (const float* p : {post_gamma, post_beta, pre_gamma, pre_beta})
    if (off(p, KB_DT_F32)) return bad("gammas and betas must be aligned to their elements");
  NormArgs a{d, x, y, post_gamma, post_beta, pre_gamma, pre_beta, gate, mod_scale, mod_shift, x_out, h};
  if (a.d.rows_per_cond < 1) a.d.rows_per_cond = 1;
  // Eight columns per access need whole groups and 16-byte rows; type pairs that
  // no stream has and rows above kTypedWidth take the kernel of any types.
  bool vec = d.width % 8 == 0;
  for (const void* p : {x, y, static_cast<const void*>(post_gamma), static_cast<const void*>(post_beta),
                        static_cast<const void*>(pre_gamma), static_cast<const void*>(pre_beta), gate, mod_scale,
                        mod_shift, static_cast<const void*>(x_out), static_cast<const void*>(h)})
    vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  vec = vec && d.x_stride % 8 == 0 && (!y || d.y_stride % 8 == 0) && (!x_out || d.x_out_stride % 8 == 0) &&
        (!h || d.h_stride % 8 == 0) && (!cond || d.cond_stride % 8 == 0);
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (d.width <= kTypedWidth) {
    const int x_t = d.stream_dtype, y_t = d.branch_dtype;
    if (x_t == KB_DT_BF16 && y_t == KB_DT_BF16) return launch_typed<KB_DT_BF16, KB_DT_BF16>(a, vec, s);
    if (x_t == KB_DT_F16 && y_t == KB_DT_F16) return launch_typed<KB_DT_F16, KB_DT_F16>(a, vec, s);
    if (x_t == KB_DT_F32 && y_t == KB_DT_BF16) return launch_typed<KB_DT_F32, KB_DT_BF16>(a, vec, s);
    if (x_t == KB_DT_F32 && y_t == KB_DT_F16) return launch_typed<KB_DT_F32, KB_DT_F16>(a, vec, s);
    if (x_t == KB_DT_F32 && y_t == KB_DT_F32) return launch_typed<KB_DT_F32, KB_DT_F32>(a, vec, s);
  }
  return launch_any(a, s);
}
