// Products of a few rows with 4-bit weights (layout: w4.cuh), bound by reading
// the weights: the dense product and the experts' gate/up (+ SwiGLU) and down
// projections.
//
//   D_g[f, r] = sum_{k in group g} (q[f, k] - z[f, g]) * x[r, k]
//   y[r, f]   = sum_g s[f, g] * D_g[f, r]
//
// Each warp streams its own weights (asynchronous copies into a ring of its own)
// -> registers -> integers q - z (exact in bf16) -> warp matrix instructions
// (m16n8k16: 16 weight rows, 8 rows of x), and adds a group's sum to fp32
// registers times its scale.  No barrier and no second warp is on the way of a
// weight, which is what a stream of 4-bit weights needs: at the copy rate an SM
// has 11 cycles for 512 codes, and decoding them takes 7 of each scheduler's.
// (tcgen05 wants the operand decoded by one warp, waited for by another and
// read back by a third; that pays from more than 16 rows on, w4_gemm_sm100.cu:
// 16 rows x [151552, 4096] take 97 us here and 107 there, 32 rows 220 and 107.)
//
// What bounds it: the loads of x beside the stream.  Without them it reads 4.7
// TB/s of weights (8 rows), without the products as well 6.1 with a ring of six.
// Not the instruction count (a variant that multiplies 128 + q and corrects by
// the sums of x, a fifth fewer, measured the same; one with shifts on the multiply
// pipe was slower), nor the depth of the ring (kDepth below).
// Measured (back to back, weights larger than L2): 1 row x [75776, 4096] 40.2 us
// = 3.98 TB/s of weights, 8 rows x [151552, 4096] 84.7 us = 3.78 TB/s, 16 rows
// 97.2 us = 3.29 TB/s; copy peak 6.5 TB/s.
//
// A warp owns 32 weight rows (a quarter of a tile): two 16-row operands, which
// in gate_up order are the gate and the up rows of the same 16 features, so the
// SwiGLU product needs no exchange.  Lane (g, t) = (lane / 4, lane % 4) reads
// 16 bytes of rows g, g + 8 of each operand: word c holds k = 32 c + 8 t ..
// + 7.  The order of k inside one instruction is free as long as both operands
// agree, so lane t feeds it its own eight k, and reads the same eight k of x.
//
// The blocks of k of an item are split over WK warps of the thread block where
// items are few, and summed through shared memory in a fixed order.
#pragma once

#include "w4.cuh"

namespace b200moe {
namespace w4s {

using w4::Shape;

enum Kind { kLinear = 0, kGateUp = 1, kDown = 2 };
constexpr int kWarps = 8;

struct Args {
  const uint8_t *w;
  Shape sh;
  int n_blocks;  // tiles per matrix
  int num_kb;
  int n_out;
  int k;
  int wk;  // warps that share an item's k
  int m;   // dense rows
  const void *x;  // bf16 rows of k values
  int64_t x_rows;
  const int32_t *mtiles;
  const int32_t *counters;
  int64_t max_mtiles;
  const int32_t *row_route;
  const __nv_bfloat16 *route_w;
  int64_t num_routes;
  int gather;  // x is the token matrix, rows through row_route
  int top_k;
  // Few routes: no packing, row tile m is route m alone (ids[m] its expert).
  const int64_t *ids;
  int num_experts;
  void *out;  // bf16 rows (linear, gate/up) or fp32 route rows (down)
};

__device__ __forceinline__ uint4 load_codes(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint32_t word(const uint4 &v, int c) {
  return c == 0 ? v.x : c == 1 ? v.y : c == 2 ? v.z : v.w;
}

// d = a b, or d += a b.
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                    uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Blocks on their way: each warp has a ring of its own in shared memory, filled
// by bulk copies (one per block and warp), so that six kilobytes per warp are
// in flight however few registers are left.  Measured at 8 rows x [151552,
// 4096]: depth 4 with two thread blocks per SM 86 us, depth 6 95, three or four
// thread blocks (whose rings leave less of the L1 to x) 94-108.
constexpr int kDepth = 4;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// Waits for a copy: bounded, and without a timer on the way of a satisfied wait.
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity) {
  if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
  int64_t start = 0;
  for (uint32_t tries = 1;; ++tries) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((tries & 1023u) == 0) {
      const int64_t now = clock64();
      if (start == 0) {
        start = now;
      } else if (now - start > 4000000000ll) {
        atomicOr(&g_status, kStatusTimeout);
        return false;
      }
    }
  }
}

// One block's share of a lane: 16 bytes of rows g, g + 8, ... (two per operand
// of 16 rows), and those rows' scales and zero points.
template <int GPB, bool ZEROS>
struct Block {
  uint4 codes[4];
  uint2 scale[GPB];    // four of 16 bits
  uint32_t zero[GPB];  // four of 8 bits

  __device__ __forceinline__ void read(uint32_t stage, int lane) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(codes[i].x), "=r"(codes[i].y), "=r"(codes[i].z), "=r"(codes[i].w)
                   : "r"(stage + (lane & 3) * 512 + (lane >> 2) * 16 + i * 128));
    const int g = lane >> 2;
#pragma unroll
    for (int j = 0; j < GPB; ++j)
      asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                   : "=r"(scale[j].x), "=r"(scale[j].y)
                   : "r"(stage + w4::kCodeBytes + j * 64 + g * 8));
    if (ZEROS) {
#pragma unroll
      for (int j = 0; j < GPB; ++j)
        asm volatile("ld.shared.u32 %0, [%1];"
                     : "=r"(zero[j])
                     : "r"(stage + w4::kCodeBytes + GPB * 64 + j * 32 + g * 4));
    }
  }
  // Scales of rows g, g + 8, g + 16, g + 24.
  __device__ __forceinline__ void scales(int j, bool half_scale, float (&s)[4]) const {
    if (__builtin_expect(half_scale, 0)) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&scale[j].x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&scale[j].y));
      s[0] = a.x, s[1] = a.y, s[2] = b.x, s[3] = b.y;
    } else {
      s[0] = __uint_as_float(scale[j].x << 16), s[1] = __uint_as_float(scale[j].x & 0xffff0000u);
      s[2] = __uint_as_float(scale[j].y << 16), s[3] = __uint_as_float(scale[j].y & 0xffff0000u);
    }
  }
  // Of row g + 8 i: the bytes z and 0x43 twice, 128 + z in both halves.
  __device__ __forceinline__ uint32_t zpair(int j, int i) const {
    return ZEROS ? __byte_perm(zero[j], 0x43434343u, 0x4040 | (i << 8) | i) : 0x43084308u;
  }
};

// In program order: the compiler would move a load that is asked for early to
// where it is used.
__device__ __forceinline__ uint4 load_row(const __nv_bfloat16 *p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// This lane's k of one block of its rows of x.  xp[n]: its eight k of chunk 0
// of row 8 n + g (of some other row where there are fewer; its sums are not
// stored).
template <int NB>
__device__ __forceinline__ void read_rows(uint4 (&xv)[4][NB], const __nv_bfloat16 *const (&xp)[NB],
                                          int k0, int k) {
  if (__builtin_expect(k0 + w4::kBlockK <= k, 1)) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < NB; ++n) xv[c][n] = load_row(xp[n] + k0 + 32 * c);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < NB; ++n)
        xv[c][n] = k0 + 32 * c < k ? load_row(xp[n] + k0 + 32 * c) : make_uint4(0, 0, 0, 0);
  }
}

// Adds one block to tot[operand][column tile][4].
template <int GPB, int NB, bool ZEROS>
__device__ __forceinline__ void add_block(const Block<GPB, ZEROS> &b, bool half_scale,
                                          const uint4 (&xv)[4][NB], float (&tot)[2][NB][4]) {
  constexpr int CPG = 4 / GPB;  // chunks per group
#pragma unroll
  for (int j = 0; j < GPB; ++j) {
    float s[4];
    b.scales(j, half_scale, s);
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float acc[NB][4];
      const uint32_t z0 = b.zpair(j, 2 * m), z1 = b.zpair(j, 2 * m + 1);
#pragma unroll
      for (int cc = 0; cc < CPG; ++cc) {
        const int c = j * CPG + cc;
        uint32_t lo[4], hi[4];
        w4::decode8(word(b.codes[2 * m], c), z0, lo);
        w4::decode8(word(b.codes[2 * m + 1], c), z1, hi);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if (cc == 0)
            mma_first(acc[n], lo[0], hi[0], lo[1], hi[1], xv[c][n].x, xv[c][n].y);
          else
            mma(acc[n], lo[0], hi[0], lo[1], hi[1], xv[c][n].x, xv[c][n].y);
          mma(acc[n], lo[2], hi[2], lo[3], hi[3], xv[c][n].z, xv[c][n].w);
        }
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        tot[m][n][0] = fmaf(s[2 * m], acc[n][0], tot[m][n][0]);
        tot[m][n][1] = fmaf(s[2 * m], acc[n][1], tot[m][n][1]);
        tot[m][n][2] = fmaf(s[2 * m + 1], acc[n][2], tot[m][n][2]);
        tot[m][n][3] = fmaf(s[2 * m + 1], acc[n][3], tot[m][n][3]);
      }
    }
  }
}

// A work item of a warp: a quarter of a tile, against the rows of one row tile.
struct Item {
  const uint8_t *w;  // its quarter of the tile's first block
  int rb, rows;
  int tile, quarter;
};

template <int KIND>
__device__ __forceinline__ Item item_of(const Args &a, int it) {
  const int per_tile = 4 * a.n_blocks;
  const int m = it / per_tile;
  const int rest = it - m * per_tile;
  Item r;
  r.tile = rest >> 2;
  r.quarter = rest & 3;
  int e = 0;
  if (KIND == kLinear) {
    r.rb = 0;
    r.rows = a.m;
  } else if (KIND == kGateUp && a.ids != nullptr) {
    const int64_t id = a.ids[m];
    const bool live = id >= 0 && id < a.num_experts;
    e = live ? static_cast<int>(id) : 0;
    r.rb = m;
    r.rows = live ? 1 : 0;
  } else {
    const int32_t *t = a.mtiles + m * B200MOE_MTILE_WORDS;
    e = t[0];
    r.rb = t[1];
    r.rows = t[2] - t[1];
  }
  r.w = a.w + (static_cast<int64_t>(e) * a.n_blocks + r.tile) * a.num_kb * a.sh.block_bytes() +
        r.quarter * a.sh.quarter_bytes();
  return r;
}

// The finished sums of one operand row pair, to memory.  f: feature row of the
// quarter's operand (g or g + 8 within 16), n: column.
template <int KIND>
__device__ __forceinline__ void store(const Args &a, const Item &it, int r0, int g, int n,
                                      float v0, float v1) {
  // v0: first operand (gate rows, or rows 0-15), v1: second (up, or 16-31).
  const int col = r0 + n;
  if (col >= it.rows) return;
  const int64_t row = it.rb + col;
  if constexpr (KIND == kGateUp) {
    const int f = it.tile * 64 + it.quarter * 16 + g;
    if (f < a.n_out)
      static_cast<__nv_bfloat16 *>(a.out)[row * a.n_out + f] =
          __float2bfloat16_rn(__fdividef(v0, 1.0f + __expf(-v0)) * v1);
  } else {
    const int f = it.tile * 128 + it.quarter * 32 + g;
    if constexpr (KIND == kDown) {
      const int32_t r = a.row_route[row];
      if (r < 0 || r >= a.num_routes) {
        atomicOr(&g_status, kStatusIndex);
        return;
      }
      const float w = __bfloat162float(a.route_w[r]);
      float *out = static_cast<float *>(a.out) + static_cast<int64_t>(r) * a.n_out + f;
      if (f < a.n_out) out[0] = v0 * w;
      if (f + 16 < a.n_out) out[16] = v1 * w;
    } else {
      __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(a.out) + row * a.n_out + f;
      if (f < a.n_out) out[0] = __float2bfloat16_rn(v0);
      if (f + 16 < a.n_out) out[16] = __float2bfloat16_rn(v1);
    }
  }
}

// NB * 8 rows of x at a time.
template <int GPB, int KIND, int NB, bool ZEROS>
__global__ void __launch_bounds__(32 * kWarps, 2) w4_stream_kernel(
    const __grid_constant__ Args a) {
  extern __shared__ __align__(16) uint8_t ring_smem[];  // [kWarps][kDepth] quarter blocks
  __shared__ float red[kWarps][2 * NB * 4][32];
  constexpr int kStage = w4::kCodeBytes + GPB * (ZEROS ? 96 : 64);
  __shared__ uint64_t bars[kWarps][kDepth];
  // Route by route, the next kernel reads the routes before it waits for this
  // one, so it may start only when they are there.
  const bool by_route = KIND == kGateUp && a.ids != nullptr;
  if (!by_route) pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wk = a.wk;
  const int wr = kWarps / wk;  // items of a thread block at a time
  const int part = warp / wr;
  const bool half_scale = a.sh.half_scale != 0;
  const uint32_t ring = smem_u32(ring_smem) + warp * (kDepth * kStage);
  const uint32_t full = smem_u32(bars[warp]);
  if (lane == 0) {
    for (int i = 0; i < kDepth; ++i) mbar_init(full + 8 * i, 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (KIND != kLinear) pdl_wait();
  if (by_route) pdl_trigger();
  const int mt = KIND == kLinear ? 1
                 : KIND == kGateUp && a.ids != nullptr
                     ? static_cast<int>(a.num_routes)
                     : static_cast<int>(min64(a.counters[B200MOE_CNT_MTILES], a.max_mtiles));
  const int items = mt * 4 * a.n_blocks;
  const int stride = gridDim.x * wr;
  const int begin = blockIdx.x * wr + warp % wr;

  // Where the copies are: they run kDepth - 1 blocks ahead of the products,
  // into the next items too.
  const uint8_t *src = nullptr, *src_next = nullptr;
  int src_item = begin, src_kb = a.num_kb, src_left = 0, src_stage = 0;
  auto copy_next = [&]() {
    if (__builtin_expect(src_kb >= a.num_kb, 0)) {  // the next pass over the item, or the next item
      while (src_left == 0 && src_item < items) {
        const Item n = item_of<KIND>(a, src_item);
        src_item += stride;
        src = n.w + static_cast<int64_t>(part) * (4 * kStage);
        src_left = (n.rows + 8 * NB - 1) / (8 * NB);
      }
      if (src_left == 0) return;
      --src_left;
      src_kb = part;
      src_next = src;
    }
    if (lane == 0) {
      mbar_arrive_expect_tx(full + 8 * src_stage, kStage);
      bulk_load(ring + src_stage * kStage, src_next, kStage, full + 8 * src_stage);
    }
    src_next += static_cast<int64_t>(wk) * (4 * kStage);
    src_kb += wk;
    src_stage = (src_stage + 1) % kDepth;
  };
#pragma unroll 1
  for (int i = 0; i < kDepth - 1; ++i) copy_next();
  if (KIND == kLinear) pdl_wait();  // codes are constant, x is not
  int stage = 0;
  uint32_t phase = 0;

  // All warps of a block take the same number of turns (they meet when k is
  // shared); a turn past the end does nothing.
  int cur = begin;
  for (int turn = blockIdx.x * wr; turn < items; turn += stride, cur += stride) {
    Item it = {};
    if (cur < items) it = item_of<KIND>(a, cur);
    const int rows = it.rows;
    for (int r0 = 0; r0 < rows || (r0 == 0 && wk > 1); r0 += 8 * NB) {
      float tot[2][NB][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) tot[m][n][j] = 0.f;
      if (rows > 0) {
        const __nv_bfloat16 *xp[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          const int col = r0 + 8 * n + g < rows ? r0 + 8 * n + g : 0;
          int64_t row = it.rb + col;
          if (KIND == kGateUp && a.gather)
            row = a.ids != nullptr ? row / a.top_k
                                   : gather_token(row, it.rb + it.rows, a.row_route, nullptr,
                                                  a.top_k, a.num_routes, a.x_rows);
          xp[n] = static_cast<const __nv_bfloat16 *>(a.x) + row * a.k + 8 * t;
        }
        // The rows of x come from L1 or L2 and are asked for one block ahead;
        // with two column tiles there is no room for that.
        uint4 xv[NB == 1 ? 2 : 1][4][NB];
        if (NB == 1) read_rows(xv[0], xp, part * w4::kBlockK, a.k);
        auto step = [&](int kb, uint4 (&now)[4][NB], uint4 (&next)[4][NB]) {
          const bool arrived = wait_copy(full + 8 * stage, phase);
          Block<GPB, ZEROS> b;
          b.read(ring + stage * kStage, lane);
          __syncwarp();  // every lane is done with the stage before, which is filled next
          copy_next();
          if (NB == 1) {
            if (kb + wk < a.num_kb) read_rows(next, xp, (kb + wk) * w4::kBlockK, a.k);
          } else {
            read_rows(now, xp, kb * w4::kBlockK, a.k);
          }
          stage = (stage + 1) % kDepth;
          phase ^= stage == 0 ? 1u : 0u;
          if (arrived) add_block<GPB, NB, ZEROS>(b, half_scale, now, tot);
        };
#pragma unroll 1
        for (int kb = part; kb < a.num_kb; kb += 2 * wk) {
          step(kb, xv[0], xv[NB == 1 ? 1 : 0]);
          if (kb + wk < a.num_kb) step(kb + wk, xv[NB == 1 ? 1 : 0], xv[0]);
        }
      }
      if (wk == 1) {
        if (rows > 0) {
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              store<KIND>(a, it, r0, g + (j >> 1) * 8, 8 * n + 2 * t + (j & 1), tot[0][n][j],
                          tot[1][n][j]);
        }
      } else {
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) red[warp][(m * NB + n) * 4 + j][lane] = tot[m][n][j];
        __syncthreads();
        // Warp `part` of the wk that share an item finishes every wk-th of its
        // values.
        for (int v = part; v < NB * 4; v += wk) {
          float v0 = 0.f, v1 = 0.f;
          for (int p = 0; p < wk; ++p) {
            v0 += red[p * wr + warp % wr][v][lane];
            v1 += red[p * wr + warp % wr][NB * 4 + v][lane];
          }
          const int n = v >> 2, j = v & 3;
          if (rows > 0)
            store<KIND>(a, it, r0, g + (j >> 1) * 8, 8 * n + 2 * t + (j & 1), v0, v1);
        }
      }
    }
  }
}

template <int GPB, int KIND, int NB, bool ZEROS>
int launch(const Args &a, int64_t blocks, cudaStream_t s) {
  constexpr int smem = kWarps * kDepth * (w4::kCodeBytes + GPB * (ZEROS ? 96 : 64));
  static bool done[64] = {false};
  const int dev = current_device();
  if (!(dev >= 0 && dev < 64 && done[dev])) {
    B200_CUDA(cudaFuncSetAttribute(w4_stream_kernel<GPB, KIND, NB, ZEROS>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  B200_LAUNCH_PDL(kPdlStream, w4_stream_kernel<GPB, KIND, NB, ZEROS>, dim3(static_cast<unsigned>(blocks)),
                  dim3(32 * kWarps), smem, s, a);
  B200_LAUNCHED();
  return B200MOE_OK;
}

template <int KIND, int NB>
int launch_tile(const Args &a, int64_t blocks, cudaStream_t s) {
  switch (a.sh.groups_per_block() * 2 + (a.sh.has_zero ? 1 : 0)) {
    case 2: return launch<1, KIND, NB, false>(a, blocks, s);
    case 3: return launch<1, KIND, NB, true>(a, blocks, s);
    case 4: return launch<2, KIND, NB, false>(a, blocks, s);
    case 5: return launch<2, KIND, NB, true>(a, blocks, s);
    case 8: return launch<4, KIND, NB, false>(a, blocks, s);
    default: return launch<4, KIND, NB, true>(a, blocks, s);
  }
}

// items: warp items (quarters of tiles) that the call is expected to work off;
// most: an upper bound.  rows: of a row tile.
template <int KIND>
int run(Args a, double items, int64_t most, int64_t rows, cudaStream_t s) {
  const int64_t slots = static_cast<int64_t>(sm_count()) * 2;  // resident blocks
  // Warps per item: as many as the machine has room for while there are few
  // items; else shared by two where a warp keeps at least eight blocks, so that
  // the warps of a block read one tile and the same rows of x.  Measured: 64
  // tokens through 128 experts, gate/up (16 blocks of k) 148 / 137 / 137 / 149 us
  // of the call with 1 / 2 / 4 / 8 warps, down (6 blocks) 148 / 152 / 160 with
  // 1 / 2 / 4.  The cost is rounds of items, each as long as its blocks and some
  // to begin and end.
  double best = 1e30;
  a.wk = 1;
  for (int wk = 1; wk <= kWarps && wk <= a.num_kb; wk *= 2) {
    if (wk > 1 && items * wk > static_cast<double>(slots) * kWarps && a.num_kb / wk < 8) break;
    const int64_t rounds = static_cast<int64_t>((items * wk + slots * kWarps - 1) /
                                                (slots * kWarps));
    const double time = static_cast<double>(rounds < 1 ? 1 : rounds) *
                        ((a.num_kb + wk - 1) / wk + (wk == 1 ? 2.0 : 1.0));
    if (time <= best) {
      best = time;
      a.wk = wk;
    }
  }
  const int wr = kWarps / a.wk;
  int64_t blocks = (most + wr - 1) / wr;
  if (blocks > slots) blocks = slots;
  if (blocks < 1) blocks = 1;
  return rows <= 8 ? launch_tile<KIND, 1>(a, blocks, s) : launch_tile<KIND, 2>(a, blocks, s);
}

}  // namespace w4s
}  // namespace b200moe
