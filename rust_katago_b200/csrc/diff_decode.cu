// Differential attention of few queries over many keys: single tokens, and
// short pieces whose queries and grouped heads fill at most a few tiles.
//
// Every key and value has to be read once, 8 D bytes per key and key/value
// head, for 12 D flop per query: HBM bounds it, so what counts is bytes in
// flight and no work between them.
//
// A warp takes 16 keys at a time with mma.sync in transposed form: S^T = K Q^T
// (16 keys x 8 rows) and O^T = V^T P^T (16 value dims x 8 rows), so a tile is 8
// rows wide (rows: queries x heads of the group) instead of the 16 that queries
// as the M side would pad to.  mma.sync and not tcgen05: a tcgen05 tile is 128
// rows of which one is used.  Fragments are 16-byte pieces of the K and V rows:
// the contraction over head dims uses the same permutation for Q, and value dims
// come out permuted, eight neighbours per thread.
// Each warp has a ring of steps of its own in shared memory, filled by
// asynchronous 16-byte copies kStages - 1 steps ahead, about 128 KB in flight
// per SM, with nothing to synchronise between warps.  (Loading the fragments
// straight into registers, one step ahead, kept half of that in flight and
// stopped at 4.3 TB/s.)
// P is rounded to the 16-bit type for the value product; sums are taken of the
// unrounded P in fp32.  The running maximum moves only when a score exceeds it
// by 2^8, so most steps skip the reduction over keys and the rescaling.
//
// Measured: one token each of 64 sequences on caches of 4,096 to 8,192 keys, 12
// heads of 64 on 4 key/value heads, bf16: 132 us in a graph, 6.1 TB/s (0.94 of the
// copy rate), 142 a call; one token on 1,083 keys, 6 heads: 8 us, launch and latency.
// Keys are split over blocks and within a block over its warps.  The warps'
// parts are joined in shared memory; the blocks' parts through distributed
// shared memory when the blocks of a tile form a cluster (up to eight: one
// launch, no workspace), else through the workspace by diff_combine.  Every join
// is in a fixed order: results do not depend on timing.
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kb_diff.cuh"
#include "kb_internal.h"
#include "kb_numeric.cuh"

namespace kb {
namespace {

constexpr int kWarps = 4;
// Steps of 16 keys in a warp's ring: 96 KB for a block of four warps.
template <int D>
constexpr int stages() { return D == 64 ? 3 : 6; }
constexpr float kLazy = 8.0f;  // log2 of how far a score may exceed the running maximum

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Transpose an 8 x 8 matrix of 16-bit values held as two per thread.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 16 bytes global -> shared without registers; zeros instead unless `in`.
__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Wait until at most N committed groups of this thread's copies are pending.
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 load16(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Four floats at the same shared-memory address in block `rank` of the cluster.
__device__ __forceinline__ float4 load_peer(const float* p, uint32_t rank) {
  uint32_t at;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// All threads of all blocks of the cluster.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// NR: 8-row tiles per warp.  (Two blocks per SM: three left 168 registers and
// spilled, 231 instead of 189 us for 64 tokens on 8,192 keys.)
template <int D, int NR, bool F16, bool CLUSTER>
__global__ void __launch_bounds__(32 * kWarps, 2) diff_decode_kernel(const DiffArgs a, int splits,
                                                                                      int row_tiles) {
  constexpr int kCh = D / 32;   // 16-byte pieces per thread of a K row, and of half a V row
  constexpr int kKs = D / 16;   // steps of the score product
  constexpr int kMt = D / 8;    // 16-dim tiles of the value product
  constexpr int kRows = 8 * NR, kDv = 2 * D;
  extern __shared__ __align__(128) float sm[];  // [warp][row][map]: kDv sums; then {m, l}
  const kb_diff_attention_desc& d = a.d;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int share = d.heads / d.kv_heads;
  const int split = blockIdx.x % splits, unit = blockIdx.x / splits;
  const int hk = unit / row_tiles, r0 = (unit % row_tiles) * kRows, b = blockIdx.y;
  const int rows = min(kRows, d.q_len * share - r0);  // valid rows of this tile

  // Keys of the tile, of this split, and of each row held by this thread.
  int off, first, last;
  const int n = key_count(a, b, off);
  key_range_n(d, n, off, r0 / share, (r0 + rows - 1) / share, first, last);
  const int steps = (max(0, last - first) + 15) / 16;
  const int per = (steps + splits - 1) / splits * 16;
  const int s0 = min(last, first + split * per), s1 = min(last, s0 + per);
  int common_lo = 0, common_hi = n;  // keys that every row sees
  if (d.causal) {
    common_hi = min(n, off + r0 / share + 1);
    if (d.window) common_lo = max(d.window, off + (r0 + rows - 1) / share + 1) - d.window;
  }
  int lo[NR][2], hi[NR][2];
#pragma unroll
  for (int t = 0; t < NR; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = r0 + 8 * t + 2 * c + u;
      key_range_n(d, n, off, r / share, r / share, lo[t][u], hi[t][u]);
    }
  const uint8_t* mask = a.key_mask ? a.key_mask + b * d.mask_batch : nullptr;

  // Q as the B operand: row g of each 8-row tile, dims permuted as K's are.
  uint32_t qf[2][NR][kKs][2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NR; ++t) {
      const int r = r0 + 8 * t + g;
      const bool ok = 8 * t + g < rows;
#pragma unroll
      for (int x = 0; x < kCh; ++x) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (ok) v = load16(a.q + b * d.q_batch + (r / share) * d.q_token + (hk * share + r % share) * d.q_head + m * d.q_map + x * 32 + c * 8);
        qf[m][t][2 * x][0] = v.x, qf[m][t][2 * x][1] = v.y, qf[m][t][2 * x + 1][0] = v.z, qf[m][t][2 * x + 1][1] = v.w;
      }
    }

  float mx[2][NR][2], l[2][NR][2], o[2][NR][kMt][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NR; ++t) {
#pragma unroll
      for (int u = 0; u < 2; ++u) mx[m][t][u] = -INFINITY, l[m][t][u] = 0.0f;
#pragma unroll
      for (int x = 0; x < kMt; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[m][t][x][e] = 0.0f;
    }

  // This warp's ring.  A step: K rows of 128 bytes (D = 64: map 0's 16 keys, then
  // map 1's; D = 32: both maps of a key side by side), then V rows of 128 bytes
  // (D = 64: the lower 64 dims of the keys, then the upper), 16-byte pieces
  // swizzled by the key.
  constexpr int kStages = stages<D>(), kKBytes = 16 * 4 * D, kStep = 2 * kKBytes;
  uint8_t* ring = reinterpret_cast<uint8_t*>(sm) + warp * kStages * kStep;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  constexpr int kRowPieces = D / 4;            // pieces of a key's K (both maps), and of its V
  constexpr int kKeysPer = 32 / kRowPieces;    // keys that 32 lanes copy at once
  const int my_key = lane / kRowPieces, piece = lane % kRowPieces;
  const uint16_t* kbase = a.k + b * d.k_batch + hk * d.k_head + (piece / (D / 8)) * d.k_map + piece % (D / 8) * 8;
  const uint16_t* vbase = a.v + b * d.v_batch + hk * d.v_head + piece * 8;
  auto fill = [&](int j, int stage) {
#pragma unroll
    for (int u = 0; u < 16 / kKeysPer; ++u) {
      const int key = my_key + u * kKeysPer;
      const bool in = j + key < s1;
      const int64_t row = in ? j + key : 0;
      const uint32_t at = ring_at + stage * kStep + ((piece >> 3) * 16 + key) * 128 + (((piece & 7) ^ (key & 7)) << 4);
      copy16(at, kbase + row * d.k_token, in);
      copy16(at + kKBytes, vbase + row * d.v_token, in);
    }
  };
  int next = s0 + 16 * warp, fill_stage = 0;
#pragma unroll
  for (int u = 0; u < kStages - 1; ++u, next += 16 * kWarps) {
    if (next < s1) fill(next, fill_stage);
    copies_commit();
    ++fill_stage;
  }
  int stage = 0;
  for (int j = s0 + 16 * warp; j < s1; j += 16 * kWarps) {
    copies_wait<kStages - 2>();
    __syncwarp();  // all lanes' copies of this step have landed, and all have left the step before
    if (next < s1) fill(next, fill_stage);
    copies_commit();
    next += 16 * kWarps;
    fill_stage = fill_stage + 1 == kStages ? 0 : fill_stage + 1;
    const uint8_t* kt = ring + stage * kStep;
    const uint8_t* vt = kt + kKBytes;
    stage = stage + 1 == kStages ? 0 : stage + 1;
    auto k_piece = [&](int m, int key, int x) -> uint4 {
      const int row = D == 64 ? m * 16 + key : key, p = D == 64 ? x * 4 + c : m * 4 + c;
      return *reinterpret_cast<const uint4*>(kt + row * 128 + ((p ^ (key & 7)) << 4));
    };
    float s[2][NR][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      uint4 kf[2][kCh];
#pragma unroll
      for (int x = 0; x < kCh; ++x) kf[0][x] = k_piece(m, g, x), kf[1][x] = k_piece(m, g + 8, x);
#pragma unroll
      for (int t = 0; t < NR; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[m][t][e] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          const uint4 &k0 = kf[0][ks / 2], &k1 = kf[1][ks / 2];
          const uint32_t af[4] = {word(k0, 2 * (ks & 1)), word(k1, 2 * (ks & 1)), word(k0, 2 * (ks & 1) + 1),
                                  word(k1, 2 * (ks & 1) + 1)};
          mma16816<F16>(s[m][t], af, qf[m][t][ks][0], qf[m][t][ks][1]);
        }
      }
    }
    // V: keys 2c, 2c + 1, 2c + 8, 2c + 9, dims 8g.. (and 64 + 8g.. for D = 64).
    uint4 vv[4][kCh];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int key = 2 * c + (y & 1) + 8 * (y >> 1);
#pragma unroll
      for (int x = 0; x < kCh; ++x)
        vv[y][x] = *reinterpret_cast<const uint4*>(vt + (x * 16 + key) * 128 + ((g ^ (key & 7)) << 4));
    }

    // Scores to log2 units, hidden ones to -inf; values of hidden keys to zero.
    const bool inside = j >= common_lo && j + 16 <= common_hi && mask == nullptr;
    bool see0 = true, see1 = true;
    if (!inside) {
      see0 = j + g < s1 && (mask == nullptr || mask[j + g]);
      see1 = j + g + 8 < s1 && (mask == nullptr || mask[j + g + 8]);
      if (mask) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int key = j + 2 * c + (y & 1) + 8 * (y >> 1);
          if (key < s1 && !mask[key])
#pragma unroll
            for (int x = 0; x < kCh; ++x) vv[y][x] = make_uint4(0, 0, 0, 0);
        }
      }
    }
    bool grow = false;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float x = s[m][t][e] * a.scale_log2;
          if (!inside) {
            const int key = j + g + 8 * (e >> 1);
            const bool see = (e >> 1 ? see1 : see0) && key >= lo[t][e & 1] && key < hi[t][e & 1];
            x = see ? x : -INFINITY;
          }
          s[m][t][e] = x;
          grow |= x > mx[m][t][e & 1] + kLazy || (mx[m][t][e & 1] == -INFINITY && x > -INFINITY);
        }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float v = fmaxf(mx[m][t][u], fmaxf(s[m][t][u], s[m][t][u + 2]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
            const float f = mx[m][t][u] == -INFINITY ? 1.0f : exp2_fast(mx[m][t][u] - v);  // sums are 0 before the first key
            mx[m][t][u] = v;
            l[m][t][u] *= f;
#pragma unroll
            for (int x = 0; x < kMt; ++x) o[m][t][x][u] *= f, o[m][t][x][u + 2] *= f;
          }
    }
    uint32_t pf[2][NR][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int t = 0; t < NR; ++t) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float base = mx[m][t][e & 1];
          p[e] = exp2_fast(s[m][t][e] - (base == -INFINITY ? 0.0f : base));
          l[m][t][e & 1] += p[e];
        }
        pf[m][t][0] = transpose8(pack16x2(make_float2(p[0], p[1]), F16));
        pf[m][t][1] = transpose8(pack16x2(make_float2(p[2], p[3]), F16));
      }
    // O^T += V^T P^T: tile x holds dims {lower: a0, a2; upper: a1, a3} of every g
#pragma unroll
    for (int x = 0; x < kMt; ++x) {
      uint32_t af[4];
      if constexpr (D == 64) {
        const int w = (x & 7) >> 1;
        const uint32_t sel = x & 1 ? 0x7632 : 0x5410;
        af[0] = __byte_perm(word(vv[0][0], w), word(vv[1][0], w), sel);
        af[1] = __byte_perm(word(vv[0][1], w), word(vv[1][1], w), sel);
        af[2] = __byte_perm(word(vv[2][0], w), word(vv[3][0], w), sel);
        af[3] = __byte_perm(word(vv[2][1], w), word(vv[3][1], w), sel);
      } else {  // 64 dims: tile x holds dims 8g + 2x (lower) and 8g + 2x + 1 (upper)
        af[0] = __byte_perm(word(vv[0][0], x), word(vv[1][0], x), 0x5410);
        af[1] = __byte_perm(word(vv[0][0], x), word(vv[1][0], x), 0x7632);
        af[2] = __byte_perm(word(vv[2][0], x), word(vv[3][0], x), 0x5410);
        af[3] = __byte_perm(word(vv[2][0], x), word(vv[3][0], x), 0x7632);
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < NR; ++t) mma16816<F16>(o[m][t][x], af, pf[m][t][0], pf[m][t][1]);
    }
  }
  copies_wait<0>();
  __syncthreads();  // the ring becomes the warps' parts

  // Sums over the keys of the warp's lanes, then the warps' parts to shared memory.
  float2* ml = reinterpret_cast<float2*>(sm + kWarps * kRows * 2 * kDv);
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float v = l[m][t][u];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        const int row = 8 * t + 2 * c + u;
        float* dst = sm + ((warp * kRows + row) * 2 + m) * kDv;
        if (g == 0) ml[(warp * kRows + row) * 2 + m] = make_float2(mx[m][t][u], v);
#pragma unroll
        for (int x = 0; x < kMt; ++x) {
          if constexpr (D == 64) {
            dst[8 * g + x] = o[m][t][x][u];
            dst[64 + 8 * g + x] = o[m][t][x][u + 2];
          } else {
            dst[8 * g + 2 * x] = o[m][t][x][u];
            dst[8 * g + 2 * x + 1] = o[m][t][x][u + 2];
          }
        }
      }
  __syncthreads();
  // One warp per row joins the warps' parts; lanes hold kDv / 32 dims.
  constexpr int kE = kDv / 32;
  // CLUSTER: this block's parts, {m, l} of both maps and the sums of each row.
  float* joined = reinterpret_cast<float*>(ml + kWarps * kRows * 2);
  float4* joined_ml = reinterpret_cast<float4*>(joined + kRows * 2 * kDv);
  for (int row = warp; row < rows; row += kWarps) {
    const int r = r0 + row, i = r / share, h = hk * share + r % share;
    float acc[2][kE], mm[2], ll[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      mm[m] = -INFINITY, ll[m] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm[m] = fmaxf(mm[m], ml[(w * kRows + row) * 2 + m].x);
#pragma unroll
      for (int e = 0; e < kE; ++e) acc[m][e] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 v = ml[(w * kRows + row) * 2 + m];
        const float f = v.x == -INFINITY ? 0.0f : exp2_fast(v.x - mm[m]);
        ll[m] += f * v.y;
        const float* src = sm + ((w * kRows + row) * 2 + m) * kDv + lane * kE;
#pragma unroll
        for (int e = 0; e < kE; ++e) acc[m][e] = fmaf(f, src[e], acc[m][e]);
      }
    }
    if constexpr (CLUSTER) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int e = 0; e < kE; ++e) joined[(row * 2 + m) * kDv + lane * kE + e] = acc[m][e];
      if (lane == 0) joined_ml[row] = make_float4(mm[0], ll[0], mm[1], ll[1]);
    } else if (splits == 1) {
      finish_row<kE>(a, b, i, h, lane, acc, ll);
    } else {
      write_partial<kE>(a, splits, split, b, i, h, lane, acc, mm, ll);
    }
  }
  if constexpr (CLUSTER) {
    // A warp of some block of the cluster joins each row: 16 lanes a map, kDv / 16
    // dims each, then the lanes of map 1 hand theirs over.
    cluster_sync();
    for (int row = split * kWarps + warp; row < rows; row += kWarps * splits) {
      const int r = r0 + row, i = r / share, h = hk * share + r % share;
      float acc[2][kE], ll[2];
      constexpr int kPer = kDv / 16;
      const int m = lane >> 4, at = (row * 2 + m) * kDv + (lane & 15) * kPer;
      float top = -INFINITY, sum = 0.0f, o[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] = 0.0f;
      for (int s = 0; s < splits; ++s) {
        const float4 v = load_peer(reinterpret_cast<const float*>(joined_ml + row), s);
        top = fmaxf(top, m ? v.z : v.x);
      }
      for (int s = 0; s < splits; ++s) {
        const float4 v = load_peer(reinterpret_cast<const float*>(joined_ml + row), s);
        const float ms = m ? v.z : v.x, ls = m ? v.w : v.y;
        const float f = ms == -INFINITY ? 0.0f : exp2_fast(ms - top);
        sum += f * ls;
#pragma unroll
        for (int e = 0; e < kPer; e += 4) {
          const float4 p = load_peer(joined + at + e, s);
          o[e] = fmaf(f, p.x, o[e]), o[e + 1] = fmaf(f, p.y, o[e + 1]);
          o[e + 2] = fmaf(f, p.z, o[e + 2]), o[e + 3] = fmaf(f, p.w, o[e + 3]);
        }
      }
      // to kE dims of both maps per lane: dims lane kE.. are half of lane / 2's
      ll[0] = __shfl_sync(0xffffffffu, sum, 0), ll[1] = __shfl_sync(0xffffffffu, sum, 16);
#pragma unroll
      for (int e = 0; e < kE; ++e) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float lower = __shfl_sync(0xffffffffu, o[e], 16 * t + (lane >> 1));
          const float upper = __shfl_sync(0xffffffffu, o[e + kE], 16 * t + (lane >> 1));
          acc[t][e] = lane & 1 ? upper : lower;
        }
      }
      finish_row<kE>(a, b, i, h, lane, acc, ll);
    }
    cluster_sync();  // nobody leaves while its shared memory is read
  }
}

template <int D, int NR, bool F16, bool CLUSTER>
int launch(const DiffArgs& a, int splits, cudaStream_t s) {
  constexpr int kRows = 8 * NR;
  constexpr int kJoin = kWarps * kRows * 2 * (2 * D * 4 + 8) + (CLUSTER ? kRows * (2 * 2 * D * 4 + 16) : 0);
  constexpr int kRing = kWarps * stages<D>() * 16 * 8 * D;
  constexpr int kBytes = kJoin > kRing ? kJoin : kRing;
  const int rows = a.d.q_len * (a.d.heads / a.d.kv_heads);
  const int row_tiles = (rows + kRows - 1) / kRows;
  auto kern = diff_decode_kernel<D, NR, F16, CLUSTER>;
  if constexpr (kBytes > 48 * 1024) {
    int dev = 0;
    cudaGetDevice(&dev);
    static std::atomic<uint64_t> configured{0};
    const uint64_t bit = 1ull << (dev & 63);
    if (!(configured.load() & bit)) {
      const int rc = smem_opt_in(reinterpret_cast<const void*>(kern), kBytes);
      if (rc) return rc;
      configured.fetch_or(bit);
    }
  }
  const int64_t grid = static_cast<int64_t>(splits) * a.d.kv_heads * row_tiles;
  if (grid > 0x7fffffff) {
    set_error("kb_diff_attention: too many queries");
    return KB_E_INVALID;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(grid), a.d.batch);
  config.blockDim = dim3(32 * kWarps);
  config.dynamicSmemBytes = kBytes;
  config.stream = s;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = splits, cluster.val.clusterDim.y = 1, cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = CLUSTER ? 1 : 0;
  return check_cuda(cudaLaunchKernelEx(&config, kern, a, splits, row_tiles),
                    "differential attention (few queries) launch");
}

template <int D, int NR, bool F16>
int launch(const DiffArgs& a, int splits, cudaStream_t s) {
  return splits > 1 && splits <= kMostCluster ? launch<D, NR, F16, true>(a, splits, s)
                                              : launch<D, NR, F16, false>(a, splits, s);
}

}  // namespace

int diff_decode_launch(const DiffArgs& a, int splits, cudaStream_t s) {
  const bool f16 = a.d.dtype == KB_DT_F16;
  const bool wide = a.d.q_len * (a.d.heads / a.d.kv_heads) > 8;
  if (a.d.head_dim == 64) {
    if (wide) return f16 ? launch<64, 2, true>(a, splits, s) : launch<64, 2, false>(a, splits, s);
    return f16 ? launch<64, 1, true>(a, splits, s) : launch<64, 1, false>(a, splits, s);
  }
  if (wide) return f16 ? launch<32, 2, true>(a, splits, s) : launch<32, 2, false>(a, splits, s);
  return f16 ? launch<32, 1, true>(a, splits, s) : launch<32, 1, false>(a, splits, s);
}

}  // namespace kb
