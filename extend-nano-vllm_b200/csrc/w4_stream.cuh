// Products of a few rows with 4-bit weights (layout: w4.cuh), bound by reading
// the weights: the dense product and the experts' gate/up (+ SwiGLU) and down
// projections.
//
//   D_g[f, r] = sum_{k in group g} (q[f, k] - z[f, g]) * x[r, k]
//   y[r, f]   = sum_g s[f, g] * D_g[f, r]
//
// Each warp streams its own weights from memory into registers, one block ahead
// of its products -> integers q - z (exact in bf16) -> warp matrix instructions
// (m16n8k16: 16 weight rows, 8 rows of x), and adds a group's sum to fp32
// registers times its scale.  No barrier and no second warp is on the way of a
// weight, which is what a stream of 4-bit weights needs: at the copy rate an SM
// has 11 cycles for 512 codes, and decoding them takes 7 of each scheduler's.
// (tcgen05 wants the operand decoded by one warp, waited for by another and
// read back by a third; that pays from more than 16 rows on, w4_gemm_sm100.cu:
// x [151552, 4096], 16 rows take 92 us here, in a tcgen05 tile of their own they
// took 107; 32 rows 220 here in passes of 32 and 100 there.)
//
// Measured (back to back, weights larger than L2): 1 row x [75776, 4096] 34.4 us
// = 4.65 TB/s of weights, 8 rows x [151552, 4096] 67.0 us = 4.78 TB/s, 16 rows
// 92.1 us = 3.48 TB/s; 8 rows x [75776, 4096] with groups of 32 and zero points
// 49.3 us = 3.74 TB/s; copy peak 6.5 TB/s.  What bounds it: no one unit.  With 8
// rows (profiled on 75776 x 4096) the integer pipe works in 67 % of cycles and the
// schedulers issue in 60 % (297 instructions per 32 x 128 weights); warps wait for
// fixed latencies, for that pipe and for loads in turn (1.5, 1.2 and 1.0 of them an
// issue), at half of the DRAM's rate.  16 warps with a block in flight each are
// what the registers hold.  A row's four units lie
// side by side (w4.cuh): 512 bytes apart they took 34.2, 68, 97 and 50.6 us.
// A ring of asynchronous copies in shared memory per warp, four deep, in place
// of the registers took 42, 84 and 104 us for the first three: it fetches as far
// ahead as one likes, but every weight crosses shared memory once more and the
// ring takes L1 from x.
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

// One block's share of a lane: 16 bytes of rows g, g + 8, ... (two per operand
// of 16 rows), and those rows' scales and zero points.
template <int GPB, bool ZEROS>
struct Block {
  uint4 codes[4];
  // Of every group; of four groups that of lane t alone (the neighbours have the
  // others: fewer loads and registers, 8 rows x [75776, 4096] with groups of 32
  // and zero points 49.6 us against 54.0; of two groups shuffles cost more, the
  // experts of 16 tokens over 512 76 us against 70).
  static constexpr int kHeld = GPB < 4 ? GPB : 1;
  uint2 scale[kHeld];    // four of 16 bits: rows g, g + 8, g + 16, g + 24
  uint32_t zero[kHeld];  // four of 8 bits

  // q: the quarter's block.
  __device__ __forceinline__ void load(const uint8_t *q, int lane) {
    const int g = lane >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[i] = load_codes(q + w4::code_place(g, lane & 3) + i * 512);
    q += w4::kCodeBytes;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int j = kHeld == GPB ? h : lane & 3;
      asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];"
                   : "=r"(scale[h].x), "=r"(scale[h].y)
                   : "l"(q + j * 64 + g * 8));
      if (ZEROS)
        asm volatile("ld.global.nc.u32 %0, [%1];"
                     : "=r"(zero[h])
                     : "l"(q + GPB * 64 + j * 32 + g * 4));
    }
  }
  static __device__ __forceinline__ uint32_t from_lane(uint32_t v, int j) {
    return kHeld == GPB ? v : __shfl_sync(0xffffffffu, v, j, 4);
  }
  // Group j's scales of rows g, g + 8, g + 16, g + 24.
  __device__ __forceinline__ void scales(int j, bool half_scale, float (&s)[4]) const {
    const int h = kHeld == GPB ? j : 0;
    const uint32_t x = from_lane(scale[h].x, j), y = from_lane(scale[h].y, j);
    if (__builtin_expect(half_scale, 0)) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&y));
      s[0] = a.x, s[1] = a.y, s[2] = b.x, s[3] = b.y;
    } else {
      s[0] = __uint_as_float(x << 16), s[1] = __uint_as_float(x & 0xffff0000u);
      s[2] = __uint_as_float(y << 16), s[3] = __uint_as_float(y & 0xffff0000u);
    }
  }
  // Per row g + 8 i: the bytes z and 0x43 twice, 128 + z in both halves.
  __device__ __forceinline__ void zpairs(int j, uint32_t (&z)[4]) const {
    const uint32_t v = ZEROS ? from_lane(zero[kHeld == GPB ? j : 0], j) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      z[i] = ZEROS ? __byte_perm(v, 0x43434343u, 0x4040 | (i << 8) | i) : 0x43084308u;
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

// This lane's chunks of one block of its rows of x.  xp[n]: its eight k of chunk
// 0 of row 8 n + g (of some other row where there are fewer; its sums are not
// stored).  One column tile has the registers for all four chunks at once, two
// column tiles for two: 16 rows x [151552, 4096] 92.6 us, with four 96.6, one 157.
template <int NB>
struct Rows {
  static constexpr int kAhead = NB == 1 ? 4 : 2;
  uint4 v[4][NB];

  __device__ __forceinline__ void read(int c, const __nv_bfloat16 *const (&xp)[NB], int k0, int k) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
      v[c][n] = k0 + 32 * c < k ? load_row(xp[n] + k0 + 32 * c) : make_uint4(0, 0, 0, 0);
  }
};

// Adds one block to tot[operand][column tile][4].  x: its first chunks are read.
template <int GPB, int NB, bool ZEROS>
__device__ __forceinline__ void add_block(const Block<GPB, ZEROS> &b, bool half_scale, Rows<NB> &x,
                                          const __nv_bfloat16 *const (&xp)[NB], int k0, int k,
                                          float (&tot)[2][NB][4]) {
  constexpr int CPG = 4 / GPB;  // chunks per group
#pragma unroll
  for (int j = 0; j < GPB; ++j) {
    float acc[2][NB][4];
    uint32_t z[4];
    b.zpairs(j, z);
#pragma unroll
    for (int cc = 0; cc < CPG; ++cc) {
      const int c = j * CPG + cc;
      if (c > 0 && c + x.kAhead - 1 < 4) x.read(c + x.kAhead - 1, xp, k0, k);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        uint32_t lo[4], hi[4];
        w4::decode8(word(b.codes[2 * m], c), z[2 * m], lo);
        w4::decode8(word(b.codes[2 * m + 1], c), z[2 * m + 1], hi);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if (cc == 0)
            mma_first(acc[m][n], lo[0], hi[0], lo[1], hi[1], x.v[c][n].x, x.v[c][n].y);
          else
            mma(acc[m][n], lo[0], hi[0], lo[1], hi[1], x.v[c][n].x, x.v[c][n].y);
          mma(acc[m][n], lo[2], hi[2], lo[3], hi[3], x.v[c][n].z, x.v[c][n].w);
        }
      }
    }
    float s[4];
    b.scales(j, half_scale, s);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        tot[m][n][0] = fmaf(s[2 * m], acc[m][n][0], tot[m][n][0]);
        tot[m][n][1] = fmaf(s[2 * m], acc[m][n][1], tot[m][n][1]);
        tot[m][n][2] = fmaf(s[2 * m + 1], acc[m][n][2], tot[m][n][2]);
        tot[m][n][3] = fmaf(s[2 * m + 1], acc[m][n][3], tot[m][n][3]);
      }
  }
}

// Adds an item's share of a warp, the blocks part, part + wk, ... of the quarter
// at w.  The block after the one at work is on its way meanwhile.  (Asking for the
// next item's first block too costs more in the loop than it gains: 8 rows 78 us
// against 68, 64 tokens through 128 experts 126 against 118.)
template <int GPB, int NB, bool ZEROS>
__device__ __forceinline__ void add_item(const Args &a, const uint8_t *w, int part,
                                         const __nv_bfloat16 *const (&xp)[NB], int lane,
                                         float (&tot)[2][NB][4]) {
  const bool half_scale = a.sh.half_scale != 0;
  const int wk = a.wk;
  constexpr int kBlock = 4 * (w4::kCodeBytes + GPB * (ZEROS ? 96 : 64));
  w += static_cast<int64_t>(part) * kBlock;
  const int64_t hop = static_cast<int64_t>(wk) * kBlock;
  Block<GPB, ZEROS> even, odd;
  even.load(w, lane);
  auto step = [&](int kb, const Block<GPB, ZEROS> &now, Block<GPB, ZEROS> &next) {
    Rows<NB> x;
#pragma unroll
    for (int c = 0; c < x.kAhead; ++c) x.read(c, xp, kb * w4::kBlockK, a.k);
    w += hop;
    if (kb + wk < a.num_kb) next.load(w, lane);
    add_block<GPB, NB, ZEROS>(now, half_scale, x, xp, kb * w4::kBlockK, a.k, tot);
  };
#pragma unroll 1
  for (int kb = part; kb < a.num_kb; kb += 2 * wk) {
    step(kb, even, odd);
    if (kb + wk < a.num_kb) step(kb + wk, odd, even);
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
  __shared__ float red[kWarps][2 * NB * 4][32];
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
  // Before the codes too: the kernel before may be the one that packs or updates
  // them, and only this wait promises that its writes are seen.
  pdl_wait();
  if (by_route) pdl_trigger();
  const int mt = KIND == kLinear ? 1
                 : KIND == kGateUp && a.ids != nullptr
                     ? static_cast<int>(a.num_routes)
                     : static_cast<int>(min64(a.counters[B200MOE_CNT_MTILES], a.max_mtiles));
  const int items = mt * 4 * a.n_blocks;
  const int stride = gridDim.x * wr;
  const int begin = blockIdx.x * wr + warp % wr;

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
        add_item<GPB, NB, ZEROS>(a, it.w, part, xp, lane, tot);
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
  B200_LAUNCH_PDL(kPdlStream, w4_stream_kernel<GPB, KIND, NB, ZEROS>, dim3(static_cast<unsigned>(blocks)),
                  dim3(32 * kWarps), 0, s, a);
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
// most: an upper bound.  cols: rows of x of a pass, 8 or 16.
template <int KIND>
int run(Args a, double items, int64_t most, int cols, cudaStream_t s) {
  const int64_t slots = static_cast<int64_t>(sm_count()) * 2;  // resident blocks
  // Warps per item: as many as the machine has room for while there are few
  // items; else shared by two where a warp keeps at least eight blocks, so that
  // the warps of a block read one tile and the same rows of x.  Measured, us of the
  // call with 1 / 2 / 4 / 8 warps: 64 tokens through 128 experts, gate/up (16 blocks
  // of k) 123 / 115 / 113 / 120, down (6 blocks) 115 / 118 / 131; down of 16 tokens
  // through 16 experts (50 blocks) 191 / 180 / 180 / 179; two rows x [8192, 4096]
  // 19.6 / 12.0 / 9.6 / 6.5, x [37888, 4096] 23.0 / 18.8 / 19.3 / 20.9.  The cost is
  // rounds of items, each as long as its blocks and some to begin and end.
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
  return cols <= 8 ? launch_tile<KIND, 1>(a, blocks, s) : launch_tile<KIND, 2>(a, blocks, s);
}

}  // namespace w4s
}  // namespace b200moe
