// Differential attention of many queries on the tcgen05 tensor cores.
//
// Per pair of a query and a key it does 12 D flop and 2 exponentials: at D = 64
// 0.094 clocks of an SM's tensor pipe against 0.125 of its special-function
// unit (16 exponentials a clock), at D = 32 0.047 against 0.125, so the
// softmax bounds it and the tensor cores have to be fed without holding it up.
//
// A block takes 128 queries of one head and walks the keys in tiles of 128.
// Each map has its own warpgroup of softmax (one query per thread) and its own
// S and O; one warp issues the products of both in strict turns, P V and the
// next S of map 0, then those of map 1, which keeps the maps half a step apart:
// while one is in the tensor cores the other is in its exponentials.
//   warps 0-3, 4-7   softmax of map 0, 1
//   warps 8-11       epilogue: the weighted difference, its norm, the output
//   warp 12          MMA issue
//   warp 13          TMA loads of Q, K and V
//   warp 14          limits of the keys' scores; clears the V rows of hidden keys
//   shared memory    Q of two items, a ring of K tiles (both maps) and one of
//                    V tiles (shared by the maps), swizzled as the MMAs read them
//   tensor memory    S of each map (128 columns, overwritten by P as packed
//                    16-bit pairs, the A operand of P V) and O of each map (2 D),
//                    for D = 32 of two items
// One pass over the keys with a running maximum and sum per map.  O is rescaled
// only when a row's maximum grows by more than 2^8 (then by the softmax
// warps, which at that point own it: S of a tile is issued after P V of the
// tile before is done).  P is rounded to the 16-bit type; sums are taken of the
// unrounded P in fp32.
// V rows of keys that kv_lens or key_mask hide are cleared in shared memory:
// their P is 0, but 0 * NaN is not.
// When items are too few for the SMs, the keys of an item are split over blocks
// and diff_combine joins the parts in a fixed order.
//
// Measured: 8,192-token causal prompt, 12 heads of 64 on 4 key/value heads, bf16:
// 350 to 360 us (0.87 PFLOP/s, 0.52 of the measured GEMM rate) at 970 to 990 W of the
// 1,000 W cap.  A tile of 128 keys of both maps takes about 3,400 clocks, of
// which its exponentials are 2,048 of the special-function unit and its products
// 1,536 of the tensor pipe.  What bounds it is the chain of one map: scores from
// tensor memory, maximum and exponentials 2,200 clocks, then 1,100 until the
// next scores, three hand-overs of about 300 and 384 of products.
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "kb_diff.cuh"
#include "kb_internal.h"
#include "kb_numeric.cuh"
#include "kb_ptx.cuh"

namespace kb {
namespace {

constexpr int kTile = 128;  // queries per item, keys per tile
// Keys of the first of the two parts of P (32 / 64 / 96: that prompt 361 / 347 /
// 355 us, 361 tokens on three 16,001-key caches 154 / 149 / 149: alike from 64 on).
constexpr int kFirst = 96;
constexpr int kThreads = 512;
constexpr int kEpiWarp = 8, kMmaWarp = 12, kLoadWarp = 13, kHiddenWarp = 14;
constexpr uint32_t kTmemCols = 512;
constexpr float kLazy = 8.0f;
// Registers of the softmax, epilogue and issuing warpgroups: together the
// 4 x 128 per thread that the block is launched with.
constexpr int kRegsLaunch = 128, kRegsSoft = 184, kRegsEpi = 88, kRegsRest = 56;
static_assert(2 * kRegsSoft + kRegsEpi + kRegsRest <= 4 * kRegsLaunch && kRegsLaunch * kThreads <= 65536,
              "register split");

template <int D>
struct Geo {
  static constexpr int kStages = D == 64 ? 2 : 4;
  static constexpr int kQk = kTile * D * 2;         // one map's Q or K tile
  static constexpr int kV = kTile * 2 * D * 2;      // V tile: 2 D / 64 columns of 128-byte rows
  static constexpr int kVCol = kTile * 128;
  static constexpr int kQOff = 0;                   // [2 items][2 maps]
  static constexpr int kKOff = 4 * kQk;             // [stage][2 maps]
  static constexpr int kVOff = kKOff + kStages * 2 * kQk;
  static constexpr int kBarOff = kVOff + kStages * kV;
  static constexpr int kBars = 512;
  // O of two items where tensor memory has room for it, so that the epilogue of
  // one runs beside the products of the next.
  static constexpr int kOBufs = D == 32 ? 2 : 1;
  static constexpr int kMlOff = kBarOff + kBars;    // [O buffer][2 maps][128] {m, l}
  static constexpr int kLimitOff = kMlOff + kOBufs * 2 * kTile * 8;  // [stage][128] limits of a key's scores
  static constexpr int kAllOff = kLimitOff + kStages * kTile * 4;        // [stage] whether all keys are seen
  static constexpr int kBytes = kAllOff + kStages * 4 + 1024;
  static constexpr uint32_t kO = 256, kDv = 2 * D;  // TMEM: S of map m at 128 m, O at kO + (2 buffer + m) kDv
  static_assert(kO + 2 * kOBufs * kDv <= kTmemCols, "tensor memory");
};

struct Items {
  int q_tiles, splits, count;
  uint32_t wait_limit_ns;
  FastDiv by_splits, by_tiles, by_heads;  // by_tiles: causal calls by batch x heads
};

// 0 for a dimension that the strides broadcast (its tensor map extent is 1), else 1.
struct Broadcast {
  int q_batch, q_head, q_map, k_batch, k_head, k_map, v_batch, v_head;
};

// Item `at`: (b, h, q tile, split).  Causal: the last query tiles, which see
// the most keys, first; otherwise the tiles of a head together, so that its K
// and V come from L2.
__device__ __forceinline__ void item_of(const DiffArgs& a, const Items& it, int at, int& b, int& h, int& qt, int& split) {
  uint32_t rest = it.by_splits.div(at);
  split = at - static_cast<int>(rest) * it.splits;
  const uint32_t outer = it.by_tiles.div(rest), inner = rest - outer * it.by_tiles.d;
  qt = a.d.causal ? it.q_tiles - 1 - static_cast<int>(outer) : static_cast<int>(inner);
  rest = a.d.causal ? inner : outer;
  b = static_cast<int>(it.by_heads.div(rest));
  h = static_cast<int>(rest) - b * a.d.heads;
}

// Key tiles [t0, t1) of an item.
__device__ __forceinline__ void tiles_of(const DiffArgs& a, const Items& it, int b, int qt, int split, int& n, int& off,
                                         int& t0, int& t1) {
  n = key_count(a, b, off);
  int first, last;
  key_range_n(a.d, n, off, qt * kTile, min(a.d.q_len, qt * kTile + kTile) - 1, first, last);
  const int lo = first / kTile, hi = last > first ? (last + kTile - 1) / kTile : lo;
  const int per = static_cast<int>(it.by_splits.div(hi - lo + it.splits - 1));
  t0 = min(hi, lo + split * per);
  t1 = min(hi, t0 + per);
}

// A block's items: one of each round of gridDim.x, from alternating ends, so
// that items in order of size add up alike in every block.
__device__ __forceinline__ int item_at(int round) {
  return round * static_cast<int>(gridDim.x) +
         static_cast<int>(round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// A walk over the tiles of a block's items, for the issuing warps.
struct Walk {
  int round, t, t0, t1;  // round of items, tile, its item's tiles
  int item, tile;        // items and tiles before this one
  bool valid;
  __device__ __forceinline__ void seek(const DiffArgs& a, const Items& it) {
    for (int at; (at = item_at(round)) < it.count; ++round) {
      int split, n, off, b, h, qt;
      item_of(a, it, at, b, h, qt, split);
      tiles_of(a, it, b, qt, split, n, off, t0, t1);
      if (t0 < t1) {
        t = t0;
        valid = true;
        return;
      }
    }
    valid = false;
  }
  __device__ __forceinline__ void start(const DiffArgs& a, const Items& it) {
    round = 0, item = 0, tile = 0;
    seek(a, it);
  }
  __device__ __forceinline__ bool begins_item() const { return t == t0; }
  __device__ __forceinline__ bool ends_item() const { return t == t1 - 1; }
  __device__ __forceinline__ void step(const DiffArgs& a, const Items& it) {
    ++tile;
    if (++t < t1) return;
    ++item;
    ++round;
    seek(a, it);
  }
};

template <int D>
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
  if constexpr (D == 64) return sw128_desc(saddr);
  else return sw64_desc(saddr);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}

// Bits [lo, hi) of a 32-bit word, lo and hi any integers.
__device__ __forceinline__ uint32_t bits_between(int lo, int hi) {
  const uint32_t below_hi = hi >= 32 ? 0xffffffffu : hi <= 0 ? 0u : (1u << hi) - 1u;
  const uint32_t below_lo = lo >= 32 ? 0xffffffffu : lo <= 0 ? 0u : (1u << lo) - 1u;
  return below_hi & ~below_lo;
}

// mbar_wait in few instructions (it is inlined some thirty times, and the
// kernel's loops have to stay in the instruction cache), without a hint of how
// long to suspend: the default wakes sooner.  The limit, two seconds or a test's
// shorter one, is measured on the timer's low word.
__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait_short(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t limit_ns) {
  if (try_wait(bar, parity)) return true;
  uint32_t t0, t1;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t0));
#pragma unroll 1
  while (!try_wait(bar, parity)) {
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t1));
    if (t1 - t0 > limit_ns) *abort_flag = 1;
    if (*abort_flag) return false;
  }
  return true;
}

// The same for a whole warp, all lanes of which return what one would.
#define KB_WARP_WAIT(bar, parity) __all_sync(0xffffffffu, wait_short(bar, parity, abort_flag, limit_ns))

// LIMITED: waits are limited to items.wait_limit_ns, for tests of what follows
// when one runs out (a limit read from an argument costs the product 1%).
template <int D, bool F16, bool LIMITED>
__global__ void __launch_bounds__(kThreads, 1) diff_tc_kernel(const __grid_constant__ CUtensorMap map_q,
                                                              const __grid_constant__ CUtensorMap map_k,
                                                              const __grid_constant__ CUtensorMap map_v,
                                                              const __grid_constant__ DiffArgs a, const Items items,
                                                              const Broadcast bc, unsigned* status) {
  using G = Geo<D>;
  constexpr int kS = G::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + G::kBarOff);
  uint64_t* q_full = bars;            // [2] Q of an item landed              (tx bytes)
  uint64_t* q_empty = bars + 2;       // [2] both maps' S MMAs read it        (commit)
  uint64_t* s_full = bars + 4;        // [map] S ready                        (commit)
  uint64_t* p_full = bars + 6;        // [map][part] part of P written        (128 arrivals)
  uint64_t* pv_done = bars + 10;      // [map] P V done: P consumed           (commit)
  uint64_t* o_full = bars + 12;       // [O buffer][map] O of an item complete (commit)
  uint64_t* o_empty = bars + 16;      // [O buffer] O, maxima and sums read   (128 arrivals)
  uint64_t* ml_full = bars + 18;      // [O buffer] maxima and sums written   (256 arrivals)
  uint64_t* drain = bars + 20;        // after an abort: issued MMAs done     (commit)
  uint64_t* k_full = bars + 21;       // [stage]                              (tx bytes)
  uint64_t* k_empty = k_full + kS;    // [stage]                              (commit)
  uint64_t* v_full = k_empty + kS;    // [stage]                              (tx bytes)
  uint64_t* v_empty = v_full + kS;    // [stage]                              (commit)
  uint64_t* v_ready = v_empty + kS;   // [stage] hidden rows cleared          (32 arrivals)
  uint64_t* limit_full = v_ready + kS; // [stage] limits written             (32 arrivals)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(limit_full + kS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((21 + 6 * kS) * 8 + 8 <= G::kBars, "barrier space");
  float2* ml = reinterpret_cast<float2*>(smem + G::kMlOff);
  // Keys that key_mask or kv_lens hide have the limit -inf, others +inf; the
  // smaller of score and limit hides a NaN too.
  float* limits = reinterpret_cast<float*>(smem + G::kLimitOff);
  int* all_seen = reinterpret_cast<int*>(smem + G::kAllOff);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], kTile);
      mbar_init(&p_full[2 * i + 1], kTile);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_full[2 * i], 1);
      mbar_init(&o_full[2 * i + 1], 1);
      mbar_init(&o_empty[i], kTile);
      mbar_init(&ml_full[i], 2 * kTile);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < kS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_ready[i], 32);
      mbar_init(&limit_full[i], 32);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const bool has_mask = a.key_mask != nullptr;
  const uint32_t limit_ns = LIMITED ? items.wait_limit_ns : static_cast<uint32_t>(kWaitLimitNs);

  if (warp < kEpiWarp) {
    // ------------------------------------------------------------ softmax
    set_regs<kRegsLaunch, kRegsSoft>();
    const int map = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    const float scale = a.scale_log2;
    const uint32_t s_addr = tmem + lanes + map * 128;
    int tile = 0, busy = 0;  // tiles and items with keys so far
    bool ok = true;
    for (int round = 0, at; ok && (at = item_at(round)) < items.count; ++round) {
      int b, h, qt, split, n, off, t0, t1;
      item_of(a, items, at, b, h, qt, split);
      tiles_of(a, items, b, qt, split, n, off, t0, t1);
      if (t0 >= t1) continue;
      int lo, hi, common_lo, common_hi, x0, x1;
      const int i0 = qt * kTile, i1 = min(a.d.q_len, i0 + kTile) - 1, i = min(i0 + row, i1);
      key_range_n(a.d, n, off, i, i, lo, hi);
      key_range_n(a.d, n, off, i1, i1, common_lo, x1);
      key_range_n(a.d, n, off, i0, i0, x0, common_hi);
      const int obuf = busy % G::kOBufs;
      const uint32_t o_addr = tmem + lanes + G::kO + (2 * obuf + map) * G::kDv;
      float m = -INFINITY, l = 0.0f;
      for (int t = t0; t < t1; ++t, ++tile) {
        const int stage = tile % kS;
        if (!KB_WARP_WAIT(&s_full[map], tile & 1) || (has_mask && !KB_WARP_WAIT(&limit_full[stage], (tile / kS) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[kTile];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait(*reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
        // Hidden keys to -inf: by their limits, then by the row's own bounds.
        if (has_mask && !all_seen[stage]) {
          const float4* limit = reinterpret_cast<const float4*>(limits + stage * kTile);
#pragma unroll
          for (int k = 0; k < kTile / 4; ++k) {
            const float4 w = limit[k];
            s[4 * k] = __float_as_uint(fminf(__uint_as_float(s[4 * k]), w.x));
            s[4 * k + 1] = __float_as_uint(fminf(__uint_as_float(s[4 * k + 1]), w.y));
            s[4 * k + 2] = __float_as_uint(fminf(__uint_as_float(s[4 * k + 2]), w.z));
            s[4 * k + 3] = __float_as_uint(fminf(__uint_as_float(s[4 * k + 3]), w.w));
          }
        }
        if (t * kTile < common_lo || (t + 1) * kTile > (has_mask && !a.d.causal ? INT_MAX : common_hi)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int base = t * kTile + 32 * c;
            const uint32_t see = bits_between(lo - base, hi - base);
            if (__all_sync(0xffffffffu, see == 0xffffffffu)) continue;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (!(see >> k & 1u)) s[32 * c + k] = 0xff800000u;
          }
        }
        float top[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          top[c] = __uint_as_float(s[c]);
#pragma unroll
          for (int k = 8 + c; k < kTile - 8; k += 16)
            top[c] = max3(top[c], __uint_as_float(s[k]), __uint_as_float(s[k + 8]));
          top[c] = max3(top[c], __uint_as_float(s[kTile - 8 + c]), -INFINITY);
        }
        const float now = max3(max3(top[0], top[1], top[2]), max3(top[3], top[4], top[5]), max3(top[6], top[7], -INFINITY)) * scale;
        // Raise the running maximum if some row of the warp is too far above it.
        if (__any_sync(0xffffffffu, now > m + kLazy || (m == -INFINITY && now > -INFINITY))) {
          const float next = fmaxf(m, now);
          const float f = m == -INFINITY ? 1.0f : ex2(m - next);  // sums are 0 before the first key
          m = next;
          l *= f;
          if (t > t0) {
#pragma unroll 1
            for (int c = 0; c < static_cast<int>(G::kDv) / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_addr + 16 * c, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
              tmem_st16(o_addr + 16 * c, o);
            }
          }
        }

        const float base = m == -INFINITY ? 0.0f : m;
        float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        // P of 32 keys at a time; P V of the first part starts while the second is at work.
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float2 x = fma2(make_float2(__uint_as_float(s[32 * c + 2 * k]), __uint_as_float(s[32 * c + 2 * k + 1])),
                                  make_float2(scale, scale), make_float2(-base, -base));
            const float2 p = make_float2(ex2(x.x), ex2(x.y));
            sum[k & 1] = add2(sum[k & 1], p);
            pk[k] = pack16x2(p, F16);
          }
          tmem_st16(s_addr + 16 * c, pk);
          if (32 * (c + 1) == kFirst || c == 3) {
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(&p_full[2 * map + (c == 3)]);
          }
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (!ok) break;
      // The epilogue has read the maxima and sums of the buffer's last item.
      if (busy >= G::kOBufs && !KB_WARP_WAIT(&o_empty[obuf], (busy / G::kOBufs - 1) & 1)) break;
      ml[(2 * obuf + map) * kTile + row] = make_float2(m, l);
      mbar_arrive(&ml_full[obuf]);
      ++busy;
    }
  } else if (warp < kMmaWarp) {
    // ------------------------------------------------------------ epilogue
    set_regs<kRegsLaunch, kRegsEpi>();
    const int row = threadIdx.x & (kTile - 1);
    int busy = 0;
    for (int round = 0, at; (at = item_at(round)) < items.count; ++round) {
      int b, h, qt, split, n, off, t0, t1;
      item_of(a, items, at, b, h, qt, split);
      tiles_of(a, items, b, qt, split, n, off, t0, t1);
      const int i = qt * kTile + row, obuf = busy % G::kOBufs;
      const uint32_t o_addr = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + G::kO + 2 * obuf * G::kDv;
      const bool live = i < a.d.q_len;
      const bool any = t0 < t1;
      const float lambda = a.lambda[h];
      float2 v0 = make_float2(-INFINITY, 0.0f), v1 = v0;
      if (any) {
        const uint32_t parity = (busy / G::kOBufs) & 1;
        if (!KB_WARP_WAIT(&ml_full[obuf], parity) || !KB_WARP_WAIT(&o_full[2 * obuf], parity) ||
            !KB_WARP_WAIT(&o_full[2 * obuf + 1], parity))
          break;
        tc_fence_after();
        v0 = ml[2 * obuf * kTile + row], v1 = ml[(2 * obuf + 1) * kTile + row];
      }
      // The last read of O: the products of a next item may overwrite it.
      auto release = [&]() {
        if (!any) return;
        tc_fence_before();
        mbar_arrive(&o_empty[obuf]);
        ++busy;
      };
      if (items.splits > 1) {
        const int64_t at2 = live ? (row_index(a, b, i, h) * items.splits + split) * 2 : 0;
        if (live) a.part_ml[at2] = v0, a.part_ml[at2 + 1] = v1;
        if (any) {
#pragma unroll 1
          for (int c = 0; c < 2 * static_cast<int>(G::kDv) / 32; ++c) {  // O of map 0, then of map 1
            uint32_t o[32];
            tmem_ld32(o_addr + 32 * c, o);
            tmem_ld_wait(o);
            if (live) {
              float4* dst = reinterpret_cast<float4*>(a.part_o + at2 * G::kDv + 32 * c);
#pragma unroll
              for (int k = 0; k < 8; ++k)
                dst[k] = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                     __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
            }
          }
        }
        release();
        continue;
      }
      const bool seen = v0.y != 0.0f || v1.y != 0.0f;  // a row without keys is zero whatever eps and gamma are
      const float w0 = v0.y == 0.0f ? 0.0f : 1.0f / v0.y;
      const float w1 = v1.y == 0.0f ? 0.0f : lambda / v1.y;
      uint16_t* out = a.out + b * a.d.out_batch + i * a.d.out_token + h * a.d.out_head;
      constexpr int kChunks = static_cast<int>(G::kDv) / 32;
      // 32 dims of the difference.
      auto difference = [&](int c, float2 (&r)[16]) {
        if (!any) {
#pragma unroll
          for (int k = 0; k < 16; ++k) r[k] = make_float2(0.0f, 0.0f);
          return;
        }
        uint32_t o0[32], o1[32];
        tmem_ld32(o_addr + 32 * c, o0);
        tmem_ld32(o_addr + G::kDv + 32 * c, o1);
        tmem_ld_wait(o0);
        tmem_ld_wait(o1);
#pragma unroll
        for (int k = 0; k < 16; ++k)
          r[k] = fma2(make_float2(__uint_as_float(o0[2 * k]), __uint_as_float(o0[2 * k + 1])), make_float2(w0, w0),
                      mul2(make_float2(__uint_as_float(o1[2 * k]), __uint_as_float(o1[2 * k + 1])), make_float2(-w1, -w1)));
      };
      // Two passes over O in tensor memory: the sum of squares, the output.
      float f = a.d.out_scale;
      float2 r[16];
      if (a.gamma) {
        float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
          difference(c, r);
#pragma unroll
          for (int k = 0; k < 16; ++k) ss = fma2(r[k], r[k], ss);
        }
        f *= rsqrtf((ss.x + ss.y) / static_cast<float>(G::kDv) + a.d.eps);
      }
#pragma unroll 1
      for (int c = 0; c < kChunks; ++c) {
        difference(c, r);
        if (c == kChunks - 1) release();
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 16; k += 2) {
          float4 g = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
          if (a.gamma) g = make_float4(a.gamma[32 * c + 2 * k], a.gamma[32 * c + 2 * k + 1], a.gamma[32 * c + 2 * k + 2], a.gamma[32 * c + 2 * k + 3]);
          w[k] = pack16x2(make_float2(r[k].x * f * g.x, r[k].y * f * g.y), F16);
          w[k + 1] = pack16x2(make_float2(r[k + 1].x * f * g.z, r[k + 1].y * f * g.w), F16);
        }
        if (live) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<uint4*>(out + 32 * c + 8 * k) =
                seen ? make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]) : make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else {
    set_regs<kRegsLaunch, kRegsRest>();
    constexpr uint32_t kFmt = F16 ? 0u : 1u;
    constexpr uint32_t kId = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (static_cast<uint32_t>(128 >> 4) << 24);
    constexpr uint32_t kIdS = kId | (static_cast<uint32_t>(kTile >> 3) << 17);
    constexpr uint32_t kIdV = kId | (1u << 16) /* B MN-major */ | (G::kDv >> 3 << 17);
    if (warp == kMmaWarp) {
      // ---------------------------------------------------------- MMA issue
      // The whole warp walks and waits; one lane issues.
      Walk ws, wp;  // the tiles whose S and whose P V come next
      ws.start(a, items);
      wp = ws;
      auto issue_s = [&](int map) -> bool {
        const int stage = ws.tile % kS;
        if (map == 0 && ((ws.begins_item() && !KB_WARP_WAIT(&q_full[ws.item & 1], (ws.item >> 1) & 1)) ||
                         !KB_WARP_WAIT(&k_full[stage], (ws.tile / kS) & 1)))
          return false;
        const uint64_t qdesc = tile_desc<D>(smem_u32(smem + G::kQOff + ((ws.item & 1) * 2 + map) * G::kQk));
        const uint64_t kdesc = tile_desc<D>(smem_u32(smem + G::kKOff + (stage * 2 + map) * G::kQk));
        // It overwrites the P of the tile before.
        if (ws.tile > 0 && !KB_WARP_WAIT(&pv_done[map], (ws.tile - 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_issue<kKindBF16>(tmem + map * 128, qdesc + 2 * k, kdesc + 2 * k, kIdS, k != 0, 0, 0);
          tc_commit(&s_full[map]);
          if (map == 1) {
            tc_commit(&k_empty[stage]);
            if (ws.ends_item()) tc_commit(&q_empty[ws.item & 1]);
          }
        }
        __syncwarp();
        if (map == 1) ws.step(a, items);
        return true;
      };
      auto issue_pv = [&](int map) -> bool {
        const int stage = wp.tile % kS;
        const uint64_t vdesc = sw128_mn_desc(smem_u32(smem + G::kVOff + stage * G::kV), G::kVCol);
        if (map == 0 && (!KB_WARP_WAIT(&v_ready[stage], (wp.tile / kS) & 1) ||
                         (wp.begins_item() && wp.item >= G::kOBufs &&
                          !KB_WARP_WAIT(&o_empty[wp.item % G::kOBufs], (wp.item / G::kOBufs - 1) & 1))))
          return false;
        const int obuf = wp.item % G::kOBufs;
        const uint32_t o_tmem = tmem + G::kO + (2 * obuf + map) * G::kDv;
        const uint32_t add = !wp.begins_item();
        if (!KB_WARP_WAIT(&p_full[2 * map], wp.tile & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kFirst / 16; ++k)
            mma_f16_ts(o_tmem, tmem + map * 128 + 8 * k,
                       vdesc + static_cast<uint64_t>(k * 16 * 128 >> 4), kIdV, k == 0 ? add : 1u);
        }
        __syncwarp();
        if (!KB_WARP_WAIT(&p_full[2 * map + 1], wp.tile & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = kFirst / 16; k < kTile / 16; ++k)
            mma_f16_ts(o_tmem, tmem + map * 128 + 8 * k,
                       vdesc + static_cast<uint64_t>(k * 16 * 128 >> 4), kIdV, 1u);
          tc_commit(&pv_done[map]);
          if (wp.ends_item()) tc_commit(&o_full[2 * obuf + map]);
          if (map == 1) tc_commit(&v_empty[stage]);
        }
        __syncwarp();
        if (map == 1) wp.step(a, items);
        return true;
      };
      bool ok = !ws.valid || (issue_s(0) && issue_s(1));
      while (ok && wp.valid) {
        const bool more = ws.valid;
        ok = issue_pv(0) && (!more || issue_s(0)) && issue_pv(1) && (!more || issue_s(1));
      }
      // Let the MMAs issued so far finish before tensor memory goes: whoever gives
      // up a wait may do so when this warp is already through (else they are done).
      if (elect_one()) {
        int none = 0;
        tc_commit(drain);
        mbar_wait(drain, 0, &none);
      }
    } else if (warp == kLoadWarp) {
      // ---------------------------------------------------------- TMA loads
      if (lane == 0) {
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
        const int share = a.d.heads / a.d.kv_heads;
        int tile = 0, tile_v = 0, busy = 0;  // K tiles, V tiles and items loaded
        bool ok = true;
        for (int round = 0, at; ok && (at = item_at(round)) < items.count; ++round) {
          int b, h, qt, split, n, off, t0, t1;
          item_of(a, items, at, b, h, qt, split);
          tiles_of(a, items, b, qt, split, n, off, t0, t1);
          if (t0 >= t1) continue;
          const int hk = h / share, qb = busy & 1;
          ok = wait_short(&q_empty[qb], ((busy >> 1) & 1) ^ 1, abort_flag, limit_ns);
          if (!ok) break;
          mbar_arrive_expect_tx(&q_full[qb], 2 * G::kQk);
          for (int m = 0; m < 2; ++m)
            tma_load_5d(smem + G::kQOff + (qb * 2 + m) * G::kQk, &map_q, &q_full[qb], 0, qt * kTile, h * bc.q_head,
                        m * bc.q_map, b * bc.q_batch);
          ++busy;
          for (int t = t0; t < t1; ++t) {
            const int stage = tile % kS;
            const uint32_t parity = ((tile / kS) & 1) ^ 1;
            ok = wait_short(&k_empty[stage], parity, abort_flag, limit_ns);
            if (!ok) break;
            mbar_arrive_expect_tx(&k_full[stage], 2 * G::kQk);
            for (int m = 0; m < 2; ++m)
              tma_load_5d(smem + G::kKOff + (stage * 2 + m) * G::kQk, &map_k, &k_full[stage], 0, t * kTile,
                          hk * bc.k_head, m * bc.k_map, b * bc.k_batch);
            ++tile;
            ok = wait_short(&v_empty[stage], parity, abort_flag, limit_ns);
            if (!ok) break;
            mbar_arrive_expect_tx(&v_full[stage], G::kV);
            for (int c = 0; c < static_cast<int>(G::kDv) / 64; ++c)
              tma_load_4d(smem + G::kVOff + stage * G::kV + c * G::kVCol, &map_v, &v_full[stage], 64 * c, t * kTile,
                          hk * bc.v_head, b * bc.v_batch);
            ++tile_v;
          }
        }
        // Let the copies issued so far land before shared memory goes, likewise.
        int none = 0;
        for (int u = busy > 2 ? busy - 2 : 0; u < busy; ++u) mbar_wait(&q_full[u & 1], (u >> 1) & 1, &none);
        for (int u = tile > kS ? tile - kS : 0; u < tile; ++u) mbar_wait(&k_full[u % kS], (u / kS) & 1, &none);
        for (int u = tile_v > kS ? tile_v - kS : 0; u < tile_v; ++u) mbar_wait(&v_full[u % kS], (u / kS) & 1, &none);
      }
    } else if (warp == kHiddenWarp) {
      // ---------------------------------------------------------- hidden keys
      int tile = 0;
      bool ok = true;
      for (int round = 0, at; ok && (at = item_at(round)) < items.count; ++round) {
        int b, h, qt, split, n, off, t0, t1;
        item_of(a, items, at, b, h, qt, split);
        tiles_of(a, items, b, qt, split, n, off, t0, t1);
        const uint8_t* mask = has_mask ? a.key_mask + b * a.d.mask_batch : nullptr;
        for (int t = t0; t < t1; ++t, ++tile) {
          const int stage = tile % kS;
          const uint32_t parity = (tile / kS) & 1;
          uint32_t see[4];
          if (!KB_WARP_WAIT(&v_empty[stage], parity ^ 1)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int key = t * kTile + 32 * c + lane;
            see[c] = __ballot_sync(0xffffffffu, key < n && (!has_mask || mask[key] != 0));
          }
          const bool all = (see[0] & see[1] & see[2] & see[3]) == 0xffffffffu;
          if (has_mask) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              limits[stage * kTile + 32 * c + lane] = see[c] >> lane & 1u ? INFINITY : -INFINITY;
            if (lane == 0) all_seen[stage] = all;
            mbar_arrive(&limit_full[stage]);
          }
          if (!KB_WARP_WAIT(&v_full[stage], parity)) {
            ok = false;
            break;
          }
          uint8_t* v = smem + G::kVOff + stage * G::kV;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (all || see[c] == 0xffffffffu) continue;
            // four rows at a time, 8 lanes a row; swizzling stays within a row
            for (int r = lane >> 3; r < 32; r += 4)
              if (!(see[c] >> r & 1u))
                for (int col = 0; col < static_cast<int>(G::kDv) / 64; ++col)
                  *reinterpret_cast<uint4*>(v + col * G::kVCol + (32 * c + r) * 128 + (lane & 7) * 16) =
                      make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          mbar_arrive(&v_ready[stage]);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && *abort_flag) record_status(status, KB_STATUS_TIMEOUT, KB_NO_LAYER);
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

#undef KB_WARP_WAIT

// Tensor map of 16-bit rows [.., token, `width`]: boxes of `box` columns by
// kTile tokens.  `strides` and `extents` of the dimensions after the token;
// broadcast ones collapse to extent 1 (flag 0).
int encode(CUtensorMap* map, const void* base, int width, int box, long tokens, int64_t token_stride, int more,
           const int64_t* strides, const long* extents, int* const* flags) {
  long dims[5] = {width, tokens, 1, 1, 1}, bytes[4];
  const int boxes[5] = {box, kTile, 1, 1, 1};
  bytes[0] = tokens > 1 ? token_stride * 2 : width * 2;
  for (int i = 0; i < more; ++i) {
    const bool steps = extents[i] > 1 && strides[i] != 0;
    *flags[i] = steps;
    dims[2 + i] = steps ? extents[i] : 1;
    bytes[1 + i] = steps ? strides[i] * 2 : width * 2;
  }
  const CUtensorMapSwizzle swz = box == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  return encode_nd(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, base, 2 + more, dims, bytes, boxes, swz);
}

template <int D, bool F16, bool LIMITED>
int launch(const DiffArgs& a, int splits, unsigned* status, uint32_t wait_limit_ns, cudaStream_t s) {
  auto kern = diff_tc_kernel<D, F16, LIMITED>;
  int dev = 0;
  cudaGetDevice(&dev);
  static std::atomic<uint64_t> configured{0};
  const uint64_t bit = 1ull << (dev & 63);
  if (!(configured.load() & bit)) {
    // The warpgroups trade registers: the launch has to hold all of them.
    cudaFuncAttributes attr;
    int rc = check_cuda(cudaFuncGetAttributes(&attr, kern), "differential attention attributes");
    if (rc) return rc;
    if (attr.numRegs != kRegsLaunch) {
      set_error("differential attention: the kernel was not built with the registers of its split");
      return KB_E_UNSUPPORTED;
    }
    rc = smem_opt_in(reinterpret_cast<const void*>(kern), Geo<D>::kBytes);
    if (rc) return rc;
    configured.fetch_or(bit);
  }
  const kb_diff_attention_desc& d = a.d;
  Broadcast bc;
  CUtensorMap mq, mk, mv;
  const int64_t qs[3] = {d.q_head, d.q_map, d.q_batch}, ks[3] = {d.k_head, d.k_map, d.k_batch},
                vs[2] = {d.v_head, d.v_batch};
  const long qe[3] = {d.heads, 2, d.batch}, ke[3] = {d.kv_heads, 2, d.batch}, ve[2] = {d.kv_heads, d.batch};
  int* const qf[3] = {&bc.q_head, &bc.q_map, &bc.q_batch};
  int* const kf[3] = {&bc.k_head, &bc.k_map, &bc.k_batch};
  int* const vf[2] = {&bc.v_head, &bc.v_batch};
  int rc = encode(&mq, a.q, D, D, d.q_len, d.q_token, 3, qs, qe, qf);
  if (!rc) rc = encode(&mk, a.k, D, D, d.kv_len, d.k_token, 3, ks, ke, kf);
  if (!rc) rc = encode(&mv, a.v, 2 * D, 64, d.kv_len, d.v_token, 2, vs, ve, vf);
  if (rc) return rc;
  Items it;
  it.q_tiles = (d.q_len + kTile - 1) / kTile;
  it.splits = splits;
  it.wait_limit_ns = wait_limit_ns;
  const int64_t count = static_cast<int64_t>(d.batch) * d.heads * it.q_tiles * splits;
  if (count > 0x7fffffff - 65536 || static_cast<int64_t>(d.batch) * d.heads > 0x3fffffff) {
    set_error("kb_diff_attention: too many query tiles");
    return KB_E_INVALID;
  }
  it.count = static_cast<int>(count);
  it.by_splits = FastDiv(splits);
  it.by_tiles = FastDiv(d.causal ? d.batch * d.heads : it.q_tiles);
  it.by_heads = FastDiv(d.heads);
  const int grid = it.count < num_sms(dev) ? it.count : num_sms(dev);
  kern<<<grid, kThreads, Geo<D>::kBytes, s>>>(mq, mk, mv, a, it, bc, status);
  return check_cuda(cudaGetLastError(), "differential attention launch");
}

}  // namespace

int diff_tc_launch(const DiffArgs& a, int splits, unsigned* status, uint32_t wait_limit_ns, cudaStream_t s) {
  const bool f16 = a.d.dtype == KB_DT_F16;
  auto run = [&](auto limited) {
    constexpr bool L = decltype(limited)::value;
    if (a.d.head_dim == 64)
      return f16 ? launch<64, true, L>(a, splits, status, wait_limit_ns, s) : launch<64, false, L>(a, splits, status, wait_limit_ns, s);
    return f16 ? launch<32, true, L>(a, splits, status, wait_limit_ns, s) : launch<32, false, L>(a, splits, status, wait_limit_ns, s);
  };
  return wait_limit_ns ? run(std::true_type{}) : run(std::false_type{});
}

}  // namespace kb
