// Rotary positions with several axes (kb_rope_axes).
//
// For token t, head h and pair p the angle is sum_a pos[a, t] * freq[h, p, a];
// the pair (u, v) becomes (u cos - v sin, u sin + v cos).
//
// The operator only has to read and write each element once, so HBM bounds it.
// Each thread owns one group of VE pairs of one head for many tokens: its
// frequencies stay in registers and nothing is shared between threads.
// Computing sine and cosine anew for every head costs less than a table would.
// Angles are fixed-point fractions of a turn, where whole turns drop out of
// integer arithmetic by themselves: a frequency is 64 bits of a turn, split into
// a high and a signed low word, and pos * high + mulhi(pos, low) is the angle to
// 2^-32 of a turn, exact for long positions where fp32 is not (position 30,000
// times a frequency of 1 costs fp32 1e-3).  (In fp64 the conversions bounded
// the kernel: 92,416 tokens of 36 x 64 bf16 took 195 us.)
// Measured: that case 160 us, 5.3 TB/s (0.81 of the copy rate), bound by the
// bytes that 480 threads of 126 registers keep in flight; 32,845 tokens of 12 x 32
// fp32, three axes, 25 us, 4.1 TB/s.
#include <math.h>
#include <stdint.h>

#include "kb_internal.h"
#include "kb_numeric.cuh"

namespace kb {
namespace {

struct RopeArgs {
  const void* x;
  const int32_t* positions;
  const float* freqs;
  const int64_t* slots;
  void* out;
  int64_t x_token, x_head, out_token, out_head, out_rows;
  int tokens, head_dim, pairs, rotary_heads, items, per_head, freq_head_stride, f16;
  int block_items, block_tokens, tokens_per_thread;
};

constexpr int kBlock = 256;  // most threads of a block
// Blocks per SM to aim for and the longest run of tokens per thread: fewer and
// longer runs leave SMs idle at the end of large calls (64 tokens: 180 us instead
// of 169 for 92,416), more and shorter ones convert frequencies too often (12
// blocks: 29 us instead of 24 for 32,845 fp32 tokens).
constexpr int kBlocksPerSm = 6, kMostTokens = 32;

constexpr double kInvTwoPi = 0.15915494309189533576888;
constexpr float kTwoPi = 6.28318530717958647692f;

// A frequency in 2^-64 of a turn per position: high word, signed low word.
struct Turns {
  int32_t high, low;
};

__device__ __forceinline__ Turns turns_of(float freq) {
  const double f = static_cast<double>(freq) * kInvTwoPi;
  const double part = f - rint(f);  // whole turns per position do not show
  const int64_t q = __double2ll_rn(part * 18446744073709551616.0);  // (+-1/2 saturates by one unit)
  const int32_t low = static_cast<int32_t>(q);
  return Turns{static_cast<int32_t>(static_cast<uint32_t>(q >> 32) + (low < 0)), low};
}

// cos and sin of angle * 2^-32 turns.  16-bit results: the special-function
// unit (absolute error about 2^-21 on [-pi, pi], far below their rounding);
// fp32 results: CUDA's sincospif.
template <bool WIDE>
__device__ __forceinline__ void cos_sin(int32_t angle, float& c, float& s) {
  if constexpr (WIDE) {
    sincospif(static_cast<float>(angle) * 0x1p-31f, &s, &c);
  } else {
    __sincosf(static_cast<float>(angle) * (kTwoPi * 0x1p-32f), &s, &c);
  }
}

// VE elements in one access: 16 bytes, or a single element.
template <typename T, int VE>
struct Raw;
template <>
struct Raw<uint16_t, 8> { using type = uint4; };
template <>
struct Raw<float, 4> { using type = uint4; };
template <>
struct Raw<uint16_t, 1> { using type = uint16_t; };
template <>
struct Raw<float, 1> { using type = float; };

template <typename T, int VE>
__device__ __forceinline__ void unpack(const typename Raw<T, VE>::type& raw, bool f16, float (&v)[VE]) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    if constexpr (sizeof(T) == 2) v[i] = from16(e[i], f16);
    else v[i] = e[i];
  }
}

template <typename T, int VE>
__device__ __forceinline__ typename Raw<T, VE>::type pack(const float (&v)[VE], bool f16) {
  typename Raw<T, VE>::type raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    if constexpr (sizeof(T) == 2) e[i] = bits16(v[i], f16);
    else e[i] = v[i];
  }
  return raw;
}

// Loads that stay where they are written, ahead of the work on the tokens before
// (the compiler otherwise moves them to their first use), and that see what an
// in-place call has written.
__device__ __forceinline__ uint4 load(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint16_t load(const uint16_t* p) { return *p; }
__device__ __forceinline__ float load(const float* p) { return *p; }

// Threads to compile for, which bounds the registers: 128 or 168 for the 16-byte
// kernels of 16-bit types with 3 or 4 axes (both words of 24 or 32 frequencies
// and the data of four tokens) and 64 for single elements with 3.  Left alone
// they take up to 216, 168 and 66, and an SM holds a block less (90,000 tokens of
// 36 x 64, halves: 192 instead of 179 us with 3 axes, 370 instead of 249 with 4;
// 30,000 tokens of 30 pairs in halves, 3 axes: 157 instead of 144).
template <typename T, int VE, bool HALVES, int AXES>
constexpr int most_threads() {
  if (VE == 1) return AXES == 3 ? 1024 : kBlock;
  return sizeof(T) == 4 || AXES < 3 ? kBlock : AXES == 3 ? 512 : 384;
}

// A thread's item: 2 VE elements of one head, VE of them at o0 and VE at o1.
// KB_ROPE_HALVES: u at o0 and v at o1 for pairs o0..; KB_ROPE_PAIRS: the pairs
// o0/2.. lie interleaved across both.  VE = 1 takes any alignment.
template <int VE, bool HALVES>
struct Item {
  int sub, head, c, o0, o1, rotated;  // sub: which of the block's tokens; rotated: pairs of this item that turn
  // The block's threads: its items of one token, then of the next.  False for those left over.
  __device__ __forceinline__ bool find(const RopeArgs& a) {
    sub = threadIdx.x / a.block_items;
    const int item = blockIdx.x * a.block_items + threadIdx.x - sub * a.block_items;
    if (sub >= a.block_tokens || item >= a.items) return false;
    head = item / a.per_head, c = item - head * a.per_head;
    o0 = 2 * VE * c, o1 = o0 + VE, rotated = 0;
    if (head < a.rotary_heads) {
      if constexpr (HALVES) {
        if (c * VE < a.pairs) {
          o0 = c * VE;
          o1 = a.pairs + o0;
          rotated = VE;
        }
      } else {
        rotated = max(0, min(VE, a.pairs - c * VE));
      }
    }
    return true;
  }
};

// The pairs of this thread's item that have a NaN or an infinity among their
// frequencies become NaN: no fixed-point angle stands for those.  A function of
// its own, after the loop over tokens and from nothing but the arguments, so that
// the loop carries one register for it (a check in the loop took up to 41 more).
template <typename T, int VE, bool HALVES, int AXES>
__device__ __noinline__ void break_pairs(const RopeArgs& a) {
  Item<VE, HALVES> it;
  if (!it.find(a)) return;
  const float* f = a.freqs + static_cast<int64_t>(it.head) * a.freq_head_stride + it.c * VE * AXES;
  T* dst = static_cast<T*>(a.out) + it.head * a.out_head;
  const int64_t run = static_cast<int64_t>(a.block_tokens) * a.tokens_per_thread;
  const int64_t end = min(static_cast<int64_t>(a.tokens), blockIdx.y * run + run);
  T nan;
  if constexpr (sizeof(T) == 2) nan = bits16(NAN, a.f16);
  else nan = NAN;
  for (int p = 0; p < it.rotated; ++p) {
    bool broken = false;
    for (int x = 0; x < AXES; ++x) broken |= !(fabsf(f[p * AXES + x]) < INFINITY);
    if (!broken) continue;
    for (int64_t t = blockIdx.y * run + it.sub; t < end; t += a.block_tokens) {
      const int64_t row = a.slots ? a.slots[t] : t;
      if (row < 0 || (a.slots && row >= a.out_rows)) continue;
      T* at = dst + row * a.out_token + it.o0 + (HALVES ? p : 2 * p);
      at[0] = nan, at[HALVES ? it.o1 - it.o0 : 1] = nan;
    }
  }
}

template <typename T, int VE, bool HALVES, int AXES>
__global__ void __launch_bounds__(most_threads<T, VE, HALVES, AXES>()) rope_axes_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kUnroll = 2;
  using R = typename Raw<T, VE>::type;
  Item<VE, HALVES> it;
  if (!it.find(a)) return;
  const int head = it.head, o0 = it.o0, o1 = it.o1, rotated = it.rotated;
  const bool f16 = a.f16;
  const T* src = static_cast<const T*>(a.x) + head * a.x_head;
  T* dst = static_cast<T*>(a.out) + head * a.out_head;
  const int step = a.block_tokens;
  const int64_t run = static_cast<int64_t>(step) * a.tokens_per_thread;
  int64_t t0 = blockIdx.y * run + it.sub;
  const int64_t end = min(static_cast<int64_t>(a.tokens), blockIdx.y * run + run);
  // kUnroll tokens at a time, the next ones loaded before these are at work (the
  // first before the frequencies are converted).
  R lo[kUnroll], hi[kUnroll];
  int pos[kUnroll][AXES];
  int64_t row[kUnroll];
  auto fetch = [&](int64_t from) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t t = from + u * step;
      row[u] = -1;
      if (t < end) {
        lo[u] = load(reinterpret_cast<const R*>(src + t * a.x_token + o0));
        hi[u] = load(reinterpret_cast<const R*>(src + t * a.x_token + o1));
#pragma unroll
        for (int x = 0; x < AXES; ++x) pos[u][x] = rotated ? a.positions[static_cast<int64_t>(x) * a.tokens + t] : 0;
        row[u] = t;
        if (a.slots) {
          row[u] = a.slots[t];
          if (row[u] >= a.out_rows) row[u] = -1;
        }
      }
    }
  };
  fetch(t0);
  Turns freq[VE][AXES];
  uint32_t worst = 0;  // the frequencies' largest magnitude, as bits
  if (rotated) {
    const float* f = a.freqs + static_cast<int64_t>(head) * a.freq_head_stride + it.c * VE * AXES;
#pragma unroll
    for (int p = 0; p < VE; ++p)
#pragma unroll
      for (int x = 0; x < AXES; ++x) {
        freq[p][x] = Turns{0, 0};
        if (p < rotated) {
          const float v = f[p * AXES + x];
          freq[p][x] = turns_of(v);
          worst = max(worst, __float_as_uint(v) << 1);
        }
      }
  }
  for (; t0 < end; t0 += kUnroll * step) {
    R now_lo[kUnroll], now_hi[kUnroll];
    int now_pos[kUnroll][AXES];
    int64_t now_row[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      now_lo[u] = lo[u], now_hi[u] = hi[u], now_row[u] = row[u];
#pragma unroll
      for (int x = 0; x < AXES; ++x) now_pos[u][x] = pos[u][x];
    }
    fetch(t0 + kUnroll * step);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (now_row[u] < 0) continue;
      R w0 = now_lo[u], w1 = now_hi[u];
      if (rotated) {
        float v0[VE], v1[VE];
        unpack<T, VE>(now_lo[u], f16, v0);
        unpack<T, VE>(now_hi[u], f16, v1);
#pragma unroll
        for (int p = 0; p < VE; ++p) {
          uint32_t angle = 0;
#pragma unroll
          for (int x = 0; x < AXES; ++x)
            angle += static_cast<uint32_t>(now_pos[u][x]) * static_cast<uint32_t>(freq[p][x].high) +
                     static_cast<uint32_t>(__mulhi(now_pos[u][x], freq[p][x].low));
          float cs, sn;
          cos_sin<sizeof(T) == 4>(static_cast<int32_t>(angle), cs, sn);
          // element indices of the pair (u, v) in the concatenation [v0 | v1]
          float* pu = HALVES || 2 * p < VE ? &v0[HALVES ? p : (2 * p) % VE] : &v1[(2 * p) % VE];
          float* pv = HALVES ? &v1[p] : 2 * p + 1 < VE ? &v0[(2 * p + 1) % VE] : &v1[(2 * p + 1) % VE];
          const float x0 = *pu, x1 = *pv;
          const bool turn = p < rotated;  // the rest is copied, NaN and infinities too
          *pu = turn ? x0 * cs - x1 * sn : x0;
          *pv = turn ? x0 * sn + x1 * cs : x1;
        }
        w0 = pack<T, VE>(v0, f16);
        w1 = pack<T, VE>(v1, f16);
      }
      *reinterpret_cast<R*>(dst + now_row[u] * a.out_token + o0) = w0;
      *reinterpret_cast<R*>(dst + now_row[u] * a.out_token + o1) = w1;
    }
  }
  if (worst >= 0xff000000u) break_pairs<T, VE, HALVES, AXES>(a);
}

template <typename T, int VE, bool HALVES>
int launch(RopeArgs a, int heads, int axes, cudaStream_t stream) {
  a.per_head = a.head_dim / (2 * VE);
  a.items = heads * a.per_head;
  int dev = 0;
  cudaGetDevice(&dev);
  const int nbx = (a.items + kBlock - 1) / kBlock;
  a.block_items = (a.items + nbx - 1) / nbx;
  a.block_tokens = kBlock / a.block_items;
  if (a.block_tokens > a.tokens) a.block_tokens = a.tokens;
  // Tokens per thread: enough to reuse its frequencies, few enough that every
  // SM gets several blocks.
  const int64_t groups = (static_cast<int64_t>(a.tokens) + a.block_tokens - 1) / a.block_tokens;
  int64_t tpt = groups * nbx / (kBlocksPerSm * num_sms(dev));
  tpt = tpt < 1 ? 1 : tpt > kMostTokens ? kMostTokens : tpt;
  int64_t gy = (groups + tpt - 1) / tpt;
  if (gy > 65535) {
    tpt = (groups + 65534) / 65535;
    gy = (groups + tpt - 1) / tpt;
  }
  a.tokens_per_thread = static_cast<int>(tpt);
  const dim3 grid(nbx, static_cast<unsigned>(gy)), block((a.block_items * a.block_tokens + 31) / 32 * 32);
  switch (axes) {
    case 1: rope_axes_kernel<T, VE, HALVES, 1><<<grid, block, 0, stream>>>(a); break;
    case 2: rope_axes_kernel<T, VE, HALVES, 2><<<grid, block, 0, stream>>>(a); break;
    case 3: rope_axes_kernel<T, VE, HALVES, 3><<<grid, block, 0, stream>>>(a); break;
    default: rope_axes_kernel<T, VE, HALVES, 4><<<grid, block, 0, stream>>>(a); break;
  }
  return check_cuda(cudaGetLastError(), "rope launch");
}

int bad(const char* what) {
  set_error(std::string("kb_rope_axes: ") + what);
  return KB_E_INVALID;
}

}  // namespace
}  // namespace kb

extern "C" int kb_rope_axes(const void* x, int dtype, int tokens, int heads, int head_dim, int64_t x_token,
                            int64_t x_head, const int32_t* positions, int axes, const float* freqs, int freq_heads,
                            int pairs, int rotary_heads, int layout, const int64_t* slots, int64_t out_rows, void* out,
                            int64_t out_token, int64_t out_head, uintptr_t stream) {
  using namespace kb;
  if (dtype != KB_DT_F32 && dtype != KB_DT_F16 && dtype != KB_DT_BF16) return bad("dtype must be KB_DT_*");
  if (tokens < 0 || heads < 1 || heads > 65536 || head_dim < 2 || head_dim % 2 || head_dim > 1024)
    return bad("tokens >= 0, heads 1..65536 and an even head_dim 2..1024 expected");
  if (axes < 1 || axes > 4) return bad("axes must be 1..4");
  if (pairs < 1 || 2 * pairs > head_dim) return bad("pairs must be 1..head_dim/2");
  if (rotary_heads < 0 || rotary_heads > heads) return bad("rotary_heads must be 0..heads");
  if (freq_heads != 1 && freq_heads != rotary_heads) return bad("freq_heads must be 1 or rotary_heads");
  if (layout != KB_ROPE_PAIRS && layout != KB_ROPE_HALVES) return bad("layout must be KB_ROPE_PAIRS or KB_ROPE_HALVES");
  if (x_token < 0 || x_head < 0 || out_token < 0 || out_head < 0 || (slots && out_rows < 0))
    return bad("strides and out_rows must not be negative");
  if (tokens == 0) return KB_OK;
  if (!x || !out || !positions || !freqs) return bad("null pointer");
  const int es = dtype == KB_DT_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(x) % es || reinterpret_cast<uintptr_t>(out) % es)
    return bad("x and out must be aligned to their elements");
  if (reinterpret_cast<uintptr_t>(positions) % 4 || reinterpret_cast<uintptr_t>(freqs) % 4 ||
      reinterpret_cast<uintptr_t>(slots) % 8)
    return bad("positions, freqs and slots must be aligned to their elements");
  // out's rows and heads must be disjoint, whichever of the two is outer
  const int64_t rows = slots ? out_rows : tokens, most = int64_t(1) << 40;
  if (x_token > most || x_head > most || out_token > most || out_head > most) return bad("strides above 2^40 elements");
  const int64_t head_span = (heads - 1) * out_head + head_dim;
  const bool token_outer = (heads == 1 || out_head >= head_dim) && (rows <= 1 || out_token >= head_span);
  const bool head_outer = (rows <= 1 || out_token >= head_dim) &&
                          (heads == 1 || (rows <= (int64_t(1) << 22) && out_head >= (rows - 1) * out_token + head_dim));
  if (!token_outer && !head_outer) return bad("out's rows and heads must not overlap");
  if (x == out && (slots || x_token != out_token || x_head != out_head))
    return bad("in place needs equal strides and no slots");
  RopeArgs a;
  a.x = x, a.positions = positions, a.freqs = freqs, a.slots = slots, a.out = out;
  a.x_token = x_token, a.x_head = x_head, a.out_token = out_token, a.out_head = out_head, a.out_rows = out_rows;
  a.tokens = tokens, a.head_dim = head_dim, a.pairs = pairs, a.rotary_heads = rotary_heads;
  a.freq_head_stride = freq_heads == 1 ? 0 : pairs * axes;
  a.f16 = dtype == KB_DT_F16;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // 16 bytes per access need such addresses and whole groups of 2 VE elements;
  // anything else takes the kernel of single elements.
  const int ve = 16 / es;
  const bool vec = head_dim % (2 * ve) == 0 && x_token % ve == 0 && x_head % ve == 0 && out_token % ve == 0 &&
                   out_head % ve == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(out) % 16 == 0 && (layout == KB_ROPE_PAIRS || pairs % ve == 0);
  const bool halves = layout == KB_ROPE_HALVES;
  if (es == 2) {
    if (vec) return halves ? launch<uint16_t, 8, true>(a, heads, axes, s) : launch<uint16_t, 8, false>(a, heads, axes, s);
    return halves ? launch<uint16_t, 1, true>(a, heads, axes, s) : launch<uint16_t, 1, false>(a, heads, axes, s);
  }
  if (vec) return halves ? launch<float, 4, true>(a, heads, axes, s) : launch<float, 4, false>(a, heads, axes, s);
  return halves ? launch<float, 1, true>(a, heads, axes, s) : launch<float, 1, false>(a, heads, axes, s);
}
