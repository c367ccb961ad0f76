// Products with 4-bit weights on tcgen05: the dense product and the experts'
// gate/up (+ SwiGLU) and down projections, for more rows than the streaming
// kernels (w4_stream.cuh) take.
//
//   D_g[f, r] = sum_{k in group g} (q[f, k] - z[f, g]) * x[r, k]
//   y[r, f]   = sum_g s[f, g] * D_g[f, r]
//
// The weight rows are the M = 128 side of the matrix instruction and the rows
// of x its N side.  The A operand is the integer q - z, exact in bf16, written
// to TMEM by the warps that decode it (lane = weight row); shared memory then
// carries only packed codes and x.  A group's sum is its own accumulator, which
// the promoting warps read and add to fp32 registers times the group's scale:
// lane = weight row, so the scale is one register.  No weight is ever rounded.
//
// Work item = (rows of one tile, 128 weight rows), split over the k blocks of a
// cluster of S CTAs where items are few; the first CTA adds the others' sums,
// in rank order, from its shared memory.
//
// Warps of a CTA: 0 codes (one bulk copy per block of 128 k), 1 rows of x
// (TMA boxes, or four-row gathers), 2 TMEM allocation and matrix instructions,
// then decoding (groups of four, alternate blocks), then promoting and epilogue
// (groups of four, alternate column chunks).
// Every wait is bounded; on expiry the CTA records a status bit and leaves.
//
// What bounds it: at 128 rows the turns that matrix instructions, promoting and
// decoding take.  A block of 128 x 128 weights takes some 1050 cycles (profiled,
// 4096 rows x [4096, 4096]), the tensor pipe works in 49 % of them: TMEM holds two
// accumulators beside the operand stages.  Decoding and promoting take 64 % of the
// issue slots (the integer pipe 51 %) and wait for TMEM most.  With groups of 32 a
// block takes some 1940 cycles, the tensor pipe 26 %: four accumulators to promote
// instead of one.
// Neither fewer reads of x (a pair of SMs: slower, its hand-overs cross the
// pair) nor more decoding warps or fewer, larger promoting warps helped.
// Measured (back to back): 32 rows x [75776, 4096] 54 us = 2.95 TB/s of weights,
// 64 rows 60 us, 128 rows 84 us; 4096 rows x [4096, 4096] 133 us = 1.03 PFLOP/s
// (cuBLAS bf16 burst 1.64).  Groups of 32 with zero points: 64 rows 93 us, 128 rows
// 141 us; 4096 rows x [4096, 4096] 240 us, groups of 64 157 us.
#include <cudaTypedefs.h>

#include <type_traits>

#include "w4.cuh"

namespace b200moe {
namespace tcg {
int make_map(CUtensorMap *map, const void *base, int rank, const uint64_t *dims,
             const uint64_t *strides_bytes, const uint32_t *box);
}  // namespace tcg

namespace w4g {

using w4::Shape;

enum Kind { kLinear = 0, kGateUp = 1, kDown = 2 };

constexpr int MAX_WS = 16;
constexpr int SMEM_LIMIT = 226 * 1024;
constexpr int TAIL_BYTES = 1024;  // barriers

// Operand stages; the down projection's largest tile leaves one to the staging
// of its fp32 rows.
constexpr int operand_stages_of(int kind, int nt) { return kind == kDown && nt == 128 ? 3 : 4; }

// Whether the first CTA of a cluster has room for the others' sums of nt rows.
constexpr bool split_ok(int split, int nt) {
  return split >= 1 && (split & (split - 1)) == 0 && (split - 1) * nt <= 112;
}

// NT: rows of x per tile (the N side); GPB: groups per block of 128 k.
template <int NT, int GPB, int KIND>
struct Cfg {
  // TMEM: accumulators in the lower half, operand stages of 64 columns (128 k
  // in bf16 pairs) in the upper.  The operand stages and those of the x rows
  // advance together, so one completion frees both.
  static constexpr int D_COLS = 256;
  // A unit: the accumulators of U groups, handed over at once.  As many groups
  // as leave room for two units, because each hand-over costs its latency.
  static constexpr int U = GPB < 128 / NT ? GPB : 128 / NT;
  static constexpr int UPB = GPB / U;                               // units per block
  static constexpr int ND = 256 / (U * NT) < 4 ? 256 / (U * NT) : 4;  // units in TMEM
  static constexpr int BS = operand_stages_of(KIND, NT);
  static constexpr bool LOCKSTEP = UPB == 1 && ND == BS;  // the two rings are one
  static constexpr int B_BYTES = NT * 256;                // 128 k of NT rows
  static constexpr int C = NT == 128 ? 8 : 16;              // columns per chunk
  static constexpr int DG = 2;                              // decoding groups
  static constexpr int PG = NT == 128 ? 4 : 2;              // promoting groups
  static constexpr int NCH = NT / C / PG;                   // chunks per promoting group
  static constexpr int UNROLL = NT == 128 ? 1 : 2;          // blocks per loop turn
  static constexpr int PROMOTE0 = 3 + 4 * DG;               // first promoting warp
  static constexpr int PROMOTERS = 4 * PG;
  static constexpr int THREADS = 32 * (PROMOTE0 + PROMOTERS);
  // Finished rows of a tile on their way out: [NT][128] (gate/up: 64) values.
  static constexpr int OUT_ROW = KIND == kDown ? 512 : KIND == kLinear ? 256 : 128;  // bytes
  static constexpr int OUT_BYTES = NT * OUT_ROW;
  // Scales as fp32, by block: [SCALES][GPB][128].  The decoding warps are at
  // most seven blocks ahead of the promoting ones (four operand stages, four
  // accumulators), so eight places need no barrier of their own.
  static constexpr int SCALES = 8;
  static constexpr int SCALE_BYTES = SCALES * GPB * 512;
  // Routes and weights of a tile's rows, of two tiles: [2][2][NT].
  static constexpr int ROUTE_BYTES = KIND == kDown ? 16 * NT : 0;
  // Shared memory beside the stages of codes.
  __host__ __device__ static constexpr int fixed_bytes(int split) {
    return BS * B_BYTES + OUT_BYTES + SCALE_BYTES + ROUTE_BYTES + (split - 1) * NT * 512 +
           TAIL_BYTES;
  }
  // Stages of codes: as many as there is room for.  The decoding groups take
  // alternate blocks, and a wait goes by the parity of a stage's use: the group
  // that asks for use u has to know that use u - 1 has landed.  With DG | stages
  // that was a block of its own; else it knows of the blocks up to b - DG - BS,
  // whose products ended before it took the operand stage of block b - DG, and use
  // u - 1 is among them with BS + DG stages or more.  Five stages of codes beside
  // four of operands become four.
  __host__ __device__ static constexpr int code_stages(int block_bytes, int split) {
    const int room = (SMEM_LIMIT - fixed_bytes(split)) / block_bytes;
    const int ws = room > MAX_WS ? MAX_WS : room;
    return ws < BS + DG ? ws / DG * DG : ws;
  }
};

struct Args {
  const uint8_t *w;
  Shape sh;
  int n_blocks;  // weight tiles per matrix
  int num_kb;
  int n_out;     // features written per row
  int ws;        // stages of codes
  int split;     // CTAs per cluster
  int staged;    // output rows allow 16-byte copies
  // dense rows
  int64_t m;
  // experts
  const int32_t *mtiles;
  const int32_t *counters;
  int64_t max_mtiles;
  const int32_t *row_route;
  const __nv_bfloat16 *route_w;
  int64_t num_routes;
  int gather;
  int top_k;
  int64_t x_rows;
  void *out;  // bf16 rows (linear, gate/up) or fp32 route rows (down)
};

struct Tile {
  int e, rb, rows;
};

template <int NT, int KIND>
__device__ __forceinline__ Tile tile_of(const Args &a, int m) {
  if (KIND == kLinear) {
    const int64_t rb = static_cast<int64_t>(m) * NT;
    return Tile{0, static_cast<int>(rb), static_cast<int>(min64(NT, a.m - rb))};
  }
  const int32_t *t = a.mtiles + m * B200MOE_MTILE_WORDS;
  return Tile{t[0], t[1], t[2] - t[1]};
}

// The items of a CTA in order; the record of the next tile is read while the
// current one is worked off.
template <int NT, int KIND>
struct Items {
  const Args &a;
  int it, items, step;
  Tile t, next;
  __device__ __forceinline__ Items(const Args &args, int first, int count, int by)
      : a(args), it(first), items(count), step(by), t{0, 0, 0}, next{0, 0, 0} {
    if (it < items) next = tile_of<NT, KIND>(a, it / a.n_blocks);
  }
  // Makes item `it` current; false at the end.
  __device__ __forceinline__ bool take() {
    if (it >= items) return false;
    t = next;
    if (it + step < items) next = tile_of<NT, KIND>(a, (it + step) / a.n_blocks);
    return true;
  }
  __device__ __forceinline__ int block() const { return it % a.n_blocks; }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[smem]^T.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
      "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr));
}

// Two fp32 values in one register pair, and acc += s * (lo, hi) on both.
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void fma2(uint64_t &acc, uint64_t s, uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm volatile("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(s), "l"(v));
}

__device__ __forceinline__ void st_shared(uint32_t addr, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t addr, __nv_bfloat16 v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(__bfloat16_as_ushort(v)) : "memory");
}
// ---- cluster helpers ------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
               : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// The rest of a wait that the first try did not satisfy.  No timer is read on
// the way; gives up after about two seconds of cycles, or when another role did.
template <bool kCluster>
__device__ __forceinline__ bool wait_more(uint32_t bar, uint32_t parity, volatile int *abort) {
  int64_t start = 0;
  for (uint32_t tries = 1;; ++tries) {
    if (kCluster ? try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if ((tries & 1023u) == 0) {
      if (*abort) return false;
      const int64_t now = clock64();
      if (start == 0) {
        start = now;
      } else if (now - start > 4000000000ll) {
        *abort = 1;
        atomicOr(&g_status, kStatusTimeout);
        return false;
      }
    }
  }
}

// One try in line, the loop out of the way: a taken branch costs a lone warp
// about 70-140 cycles here (measured), as much as a whole step of a role.
template <bool kCluster = false>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int *abort) {
  const bool now = kCluster ? try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity);
  if (__builtin_expect(now, 1)) return true;
  return wait_more<kCluster>(bar, parity, abort);
}

// One lane of the warp, in a form that tells the compiler so: matrix
// instructions issued under it take uniform registers (37 cycles each, measured at
// N = 16, against 128 under a test of the lane number).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// x * sigmoid(x); the fast exp and division are good to a few units in 2^-23,
// far below the bf16 store of the result.
__device__ __forceinline__ float silu_fast(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// A ring position: stage and the parity of its current use.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n, int by = 1) {
    stage += by;
    const bool wrap = stage >= n;
    stage -= wrap ? n : 0;
    phase ^= wrap ? 1u : 0u;
  }
};

// What every role of a CTA knows (shared-memory addresses, this CTA's share).
struct Ctx {
  uint32_t s_b, s_w, s_red;
  uint32_t w_full, w_empty, b_full, a_full, ab_empty, d_full, d_empty, red_full, red_empty;
  uint32_t s_out, s_scale, s_route, out_free, out_full;
  uint32_t tmem;
  volatile int *abort;
  int wbytes, qbytes, scale_off, zero_off;
  int items, first, step, kb0, kb1;
  int rank, split;
};

// Codes: one bulk copy per block of 128 k.  One lane.
template <int NT, int KIND>
__device__ __forceinline__ void load_codes(const Args &args, const Ctx &c) {
  Ring w;
  for (Items<NT, KIND> item(args, c.first, c.items, c.step); item.take(); item.it += c.step) {
    const Tile t = item.t;
    const uint8_t *src = args.w + (static_cast<int64_t>(t.e) * args.n_blocks + item.block()) *
                                      args.num_kb * c.wbytes;
    for (int r0 = 0; r0 < t.rows; r0 += NT)
#pragma unroll 4
      for (int kb = c.kb0; kb < c.kb1; ++kb) {
        if (!wait(c.w_empty + 8 * w.stage, w.phase ^ 1, c.abort)) return;
        const uint32_t bar = c.w_full + 8 * w.stage;
        mbar_arrive_expect_tx(bar, c.wbytes);
        bulk_load(c.s_w + w.stage * c.wbytes, src + static_cast<int64_t>(kb) * c.wbytes, c.wbytes,
                  bar);
        w.next(args.ws);
      }
  }
}

// Rows of x.  Dense rows and nearly full tiles come as one box of NT rows per
// 64 k (rows past the tile are multiplied with nothing), those of other tiles as
// boxes of 16, gathered rows four at a time (lane l loads the l-th four).  A
// whole warp.
template <int NT, int GPB, int KIND>
__device__ __forceinline__ void load_rows(const Args &args, const Ctx &c, const CUtensorMap *tm,
                                          const CUtensorMap *tm_whole) {
  using C = Cfg<NT, GPB, KIND>;
  const int lane = threadIdx.x & 31;
  const bool gather = KIND == kGateUp && args.gather != 0;
  Ring b;
  for (Items<NT, KIND> item(args, c.first, c.items, c.step); item.take(); item.it += c.step) {
    const Tile t = item.t;
    for (int r0 = 0; r0 < t.rows; r0 += NT) {
      const int rows = min(NT, t.rows - r0);
      const int nbox = (rows + 15) >> 4;
      // One box of NT rows, unless at least half of it would be wasted.
      const bool whole = !gather && (KIND == kLinear || nbox * 32 > NT);
      const bool mine = gather && lane < nbox * 4;
      const uint32_t bytes = whole ? C::B_BYTES : nbox * 16 * 256;
      int tok[4] = {0, 0, 0, 0};
      if (gather && mine) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          tok[j] = gather_token(t.rb + r0 + 4 * lane + j, t.rb + t.rows, args.row_route, nullptr,
                                args.top_k, args.num_routes, args.x_rows);
      }
#pragma unroll 2
      for (int kb = c.kb0; kb < c.kb1; ++kb) {
        if (!wait(c.ab_empty + 8 * b.stage, b.phase ^ 1, c.abort)) return;
        const uint32_t bar = c.b_full + 8 * b.stage;
        const uint32_t dst = c.s_b + b.stage * C::B_BYTES;
        const int c0 = kb * w4::kBlockK;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar, bytes);
          if (whole) {
            tma_load_2d(dst, tm_whole, bar, c0, t.rb + r0);
            tma_load_2d(dst + NT * 128, tm_whole, bar, c0 + 64, t.rb + r0);
          } else if (!gather) {
            for (int i = 0; i < nbox; ++i) {
              tma_load_2d(dst + i * 2048, tm, bar, c0, t.rb + r0 + i * 16);
              tma_load_2d(dst + NT * 128 + i * 2048, tm, bar, c0 + 64, t.rb + r0 + i * 16);
            }
          }
        }
        __syncwarp();
        if (mine) {
          tma_gather4(dst + lane * 512, tm, bar, c0, tok[0], tok[1], tok[2], tok[3]);
          tma_gather4(dst + NT * 128 + lane * 512, tm, bar, c0 + 64, tok[0], tok[1], tok[2],
                      tok[3]);
        }
        __syncwarp();
        b.next(C::BS);
      }
    }
  }
}

// Matrix instructions.  One lane.
template <int NT, int GPB, int KIND>
__device__ __forceinline__ void issue_mma(const Args &args, const Ctx &c) {
  using C = Cfg<NT, GPB, KIND>;
  constexpr int KK = 8 / GPB;  // instructions of 16 k per group
  Ring b, d;
  // Descriptor of stage 0; the start address field counts 16 bytes.
  const uint64_t desc0 = sw128_kmajor_desc(c.s_b);
  for (Items<NT, KIND> item(args, c.first, c.items, c.step); item.take(); item.it += c.step) {
    const Tile t = item.t;
    for (int r0 = 0; r0 < t.rows; r0 += NT) {
      const int n_mma = (min(NT, t.rows - r0) + 15) & ~15;
      const uint32_t idesc = idesc_bf16_f32(128, n_mma);
#pragma unroll 4
      for (int kb = c.kb0; kb < c.kb1; ++kb) {
        // Tried together: each alone costs its latency.
        const uint32_t b_full = c.b_full + 8 * b.stage, a_full = c.a_full + 8 * b.stage;
        const uint32_t d_empty = c.d_empty + 8 * d.stage;
        const bool b_ready = mbar_try_wait(b_full, b.phase);
        const bool a_ready = mbar_try_wait(a_full, b.phase);
        const bool d_ready = mbar_try_wait(d_empty, d.phase ^ 1);
        if (__builtin_expect(!(b_ready && a_ready && d_ready), 0)) {
          if (!wait_more<false>(b_full, b.phase, c.abort)) return;
          if (!wait_more<false>(a_full, b.phase, c.abort)) return;
          if (!wait_more<false>(d_empty, d.phase ^ 1, c.abort)) return;
        }
        const uint64_t desc = desc0 + static_cast<uint32_t>(b.stage * (C::B_BYTES >> 4));
        const uint32_t ta = c.tmem + C::D_COLS + b.stage * 64;
#pragma unroll
        for (int u = 0; u < C::UPB; ++u) {
          if (u > 0 && !wait(c.d_empty + 8 * d.stage, d.phase ^ 1, c.abort)) return;
          tc_fence_after();
#pragma unroll
          for (int g = 0; g < C::U; ++g) {
            const uint32_t td = c.tmem + (d.stage * C::U + g) * NT;
#pragma unroll
            for (int j = 0; j < KK; ++j) {
              const int kk = (u * C::U + g) * KK + j;
              mma_ts(td, ta + kk * 8, desc + ((kk >> 2) * (NT * 8) + (kk & 3) * 2), idesc, j != 0);
            }
          }
          // Accumulators in step with the operand stages: one completion
          // serves both.
          if (!C::LOCKSTEP) tc_commit(c.d_full + 8 * d.stage);
          d.next(C::ND);
        }
        tc_commit(c.ab_empty + 8 * b.stage);
        b.next(C::BS);
      }
    }
  }
}

// Decoding: the codes of a block -> q - z as bf16 in the operand stage.  Group
// `grp` of DG takes every DG-th block.  Four warps, one weight row per thread.
template <int NT, int GPB, int KIND>
__device__ __forceinline__ void decode(const Args &args, const Ctx &c, int grp, int q) {
  using C = Cfg<NT, GPB, KIND>;
  const int lane = threadIdx.x & 31;
  const int place = w4::scale_place(lane);
  const bool zeros = args.sh.has_zero != 0;
  const uint32_t tq = c.tmem + C::D_COLS + (static_cast<uint32_t>(q * 32) << 16);
  Ring w, a;
  w.next(args.ws, grp);
  a.next(C::BS, grp);
  int skip = grp;   // blocks until this group's next one
  int block = grp;  // of all this CTA's blocks
  for (Items<NT, KIND> item(args, c.first, c.items, c.step); item.take(); item.it += c.step) {
    const Tile t = item.t;
    for (int r0 = 0; r0 < t.rows; r0 += NT) {
      int kb = c.kb0 + skip;
#pragma unroll C::UNROLL
      for (; kb < c.kb1; kb += C::DG) {
        if (!wait(c.w_full + 8 * w.stage, w.phase, c.abort)) return;
        const uint32_t st = c.s_w + w.stage * c.wbytes + q * c.qbytes;
        uint32_t code[16];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(code[4 * i]), "=r"(code[4 * i + 1]), "=r"(code[4 * i + 2]),
                         "=r"(code[4 * i + 3])
                       : "r"(st + w4::code_place(lane, i)));
        uint32_t zp[GPB];
#pragma unroll
        for (int g = 0; g < GPB; ++g) {
          uint32_t z = 8;
          if (zeros)
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(z) : "r"(st + c.zero_off + g * 32 + place));
          zp[g] = w4::zero_pair(z);
        }
        uint16_t scale[GPB];
#pragma unroll
        for (int g = 0; g < GPB; ++g)
          asm volatile("ld.shared.u16 %0, [%1];"
                       : "=h"(scale[g])
                       : "r"(st + c.scale_off + g * 64 + place * 2));
        if (!wait(c.ab_empty + 8 * a.stage, a.phase ^ 1, c.abort)) return;
        tc_fence_after();
        const uint32_t ta = tq + a.stage * 64;
        const uint32_t ss = c.s_scale + (block & (C::SCALES - 1)) * (GPB * 512) + (q * 32 + lane) * 4;
#pragma unroll
        for (int g = 0; g < GPB; ++g)
          st_shared(ss + g * 512, w4::scale_f32(scale[g], args.sh.half_scale));
        block += C::DG;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int ch = 2 * h + (j >> 2), u = j & 3;  // chunk of 32 k, unit
            uint32_t o[4];
            w4::decode8(code[4 * u + ch], zp[ch * GPB / 4], o);
#pragma unroll
            for (int i = 0; i < 4; ++i) r[4 * j + i] = o[i];
          }
          tmem_st32(ta + h * 32, r);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(c.a_full + 8 * a.stage);
          mbar_arrive(c.w_empty + 8 * w.stage);
        }
        w.next(args.ws, C::DG);
        a.next(C::BS, C::DG);
      }
      skip = kb - c.kb1;
    }
  }
}

// Promoting and epilogue.  PG groups of four warps (alternate column chunks), one
// weight row per thread.
template <int NT, int GPB, int KIND>
__device__ __forceinline__ void promote(const Args &args, const Ctx &c, int half, int q) {
  using C = Cfg<NT, GPB, KIND>;
  const int lane = threadIdx.x & 31;
  const int row = q * 32 + lane;
  const uint32_t tq = c.tmem + (static_cast<uint32_t>(q * 32) << 16);
  Ring d;
  int block = 0;
  uint32_t red_phase = 0, out_phase = 0;
  const int mine = (half * 4 + q) * 32 + lane;  // of a tile's rows
  int32_t next_route = -1;
  bool ahead = false;
  for (Items<NT, KIND> item(args, c.first, c.items, c.step); item.take(); item.it += c.step) {
    const Tile t = item.t;
    const int fb = item.block();
    for (int r0 = 0; r0 < t.rows; r0 += NT) {
      const int rows = min(NT, t.rows - r0);
      const int n_mma = (rows + 15) & ~15;
      // Route and weight of row `mine`: the route was asked for one item ago (of
      // a tile's first rows), the weight is asked for before the products.
      int32_t route = -1;
      __nv_bfloat16 weight = __float2bfloat16_rn(0.f);
      if (KIND == kDown) {
        if (mine < rows) {
          route = r0 == 0 && ahead ? next_route : args.row_route[t.rb + r0 + mine];
          if (route < 0 || route >= args.num_routes) {
            atomicOr(&g_status, kStatusIndex);
            route = -1;
          } else {
            weight = args.route_w[route];
          }
        }
        if (r0 == 0) {
          ahead = item.it + item.step < item.items;
          if (ahead && mine < item.next.rows) next_route = args.row_route[item.next.rb + mine];
        }
      }
      uint64_t acc2[C::NCH][C::C / 2];  // pairs of neighbouring columns
#pragma unroll
      for (int i = 0; i < C::NCH; ++i)
#pragma unroll
        for (int j = 0; j < C::C / 2; ++j) acc2[i][j] = 0;
#pragma unroll C::UNROLL
      for (int kb = c.kb0; kb < c.kb1; ++kb) {
        const uint32_t scales =
            c.s_scale + (block & (C::SCALES - 1)) * (GPB * 512) + row * 4;
        ++block;
#pragma unroll
        for (int u = 0; u < C::UPB; ++u) {
          // A finished product implies its scales: the decoding warps wrote
          // them before they signalled the operand.
          if (!wait((C::LOCKSTEP ? c.ab_empty : c.d_full) + 8 * d.stage, d.phase, c.abort)) return;
          tc_fence_after();
          const uint32_t td = tq + d.stage * (C::U * NT) + half * C::C;
          // Piece l = (group, chunk): the next one loads while this one is
          // added.  Columns beyond n_mma hold old sums; they are never stored.
          uint32_t v[2][C::C];
          tmem_ld(td, v[0]);
          uint64_t s2[C::U];
#pragma unroll
          for (int g = 0; g < C::U; ++g) {
            float s;
            asm volatile("ld.shared.f32 %0, [%1];"
                         : "=f"(s)
                         : "r"(scales + (u * C::U + g) * 512));
            s2[g] = pack2(s, s);
          }
#pragma unroll
          for (int l = 0; l < C::U * C::NCH; ++l) {
            const int g = l / C::NCH, i = l % C::NCH;
            tmem_ld_wait();
            if (l + 1 < C::U * C::NCH)
              tmem_ld(td + ((l + 1) / C::NCH) * NT + ((l + 1) % C::NCH) * C::PG * C::C, v[(l + 1) & 1]);
#pragma unroll
            for (int j = 0; j < C::C / 2; ++j)
              fma2(acc2[i][j], s2[g], v[l & 1][2 * j], v[l & 1][2 * j + 1]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(c.d_empty + 8 * d.stage);
          d.next(C::ND);
        }
      }
      float acc[C::NCH][C::C];
#pragma unroll
      for (int i = 0; i < C::NCH; ++i)
#pragma unroll
        for (int j = 0; j < C::C / 2; ++j)
          asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[i][2 * j]), "=f"(acc[i][2 * j + 1]) : "l"(acc2[i][j]));
      if (c.split > 1) {
        if (c.rank != 0) {
          // This CTA's sums into the first one's shared memory.
          if (!wait<true>(c.red_empty, red_phase ^ 1, c.abort)) return;
          const uint32_t dst = map_rank(c.s_red + ((c.rank - 1) * NT * 128 + row) * 4, 0);
#pragma unroll
          for (int i = 0; i < C::NCH; ++i) {
            const int col = (C::PG * i + half) * C::C;
            if (col < n_mma) {
#pragma unroll
              for (int j = 0; j < C::C; ++j) st_cluster(dst + (col + j) * 512, acc[i][j]);
            }
          }
          __syncwarp();
          if (lane == 0) arrive_cluster(map_rank(c.red_full, 0));
          red_phase ^= 1;
          continue;
        }
        if (!wait<true>(c.red_full, red_phase, c.abort)) return;
        red_phase ^= 1;
        for (int p = 0; p < c.split - 1; ++p) {
#pragma unroll
          for (int i = 0; i < C::NCH; ++i) {
            const int col = (C::PG * i + half) * C::C;
            if (col < n_mma) {
#pragma unroll
              for (int j = 0; j < C::C; ++j) {
                float v;
                asm volatile("ld.shared.f32 %0, [%1];"
                             : "=f"(v)
                             : "r"(c.s_red + ((p * NT + col + j) * 128 + row) * 4));
                acc[i][j] += v;
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0)
          for (int p = 1; p < c.split; ++p) arrive_cluster(map_rank(c.red_empty, p));
      }
      const int64_t row0 = static_cast<int64_t>(t.rb) + r0;
      // Finished values go to shared memory as whole output rows and leave in
      // 16-byte pieces, a row at a time.  (Stored from the registers, one
      // column of 32 features per store, a tile took longer than its six
      // blocks of products; a bulk copy per row, issued lane by lane, too.)
      const bool staged = args.staged != 0;
      const uint32_t s_route = c.s_route + out_phase * (8 * NT);
      if (staged) {
        if (KIND == kDown && mine < rows) {
          asm volatile("st.shared.s32 [%0], %1;" ::"r"(s_route + mine * 4), "r"(route) : "memory");
          st_shared(s_route + (NT + mine) * 4, __bfloat162float(weight));
        }
        // The rows of the item before have been read, by every warp.
        __syncwarp();
        if (lane == 0) mbar_arrive(c.out_free);
        if (!wait(c.out_free, out_phase, c.abort)) return;
      }
      if constexpr (KIND == kGateUp) {
        // Lanes 0-15 hold gate rows, 16-31 the up rows of the same features:
        // of each pair of columns the lower half finishes the first, the upper
        // half the second.
        const int f = fb * 64 + q * 16 + (lane & 15);
        const bool up = lane >= 16;
        const int odd = up ? 1 : 0;
        const int last = f < args.n_out ? rows : 0;
#pragma unroll
        for (int i = 0; i < C::NCH; ++i) {
          const int col = (C::PG * i + half) * C::C;
          if (col < n_mma) {
            auto *out = static_cast<__nv_bfloat16 *>(args.out) + (row0 + col + odd) * args.n_out + f;
            const uint32_t so = c.s_out + (col + odd) * C::OUT_ROW + (q * 16 + (lane & 15)) * 2;
#pragma unroll
            for (int j = 0; j < C::C; j += 2) {
              const float other =
                  __shfl_xor_sync(0xffffffffu, up ? acc[i][j] : acc[i][j + 1], 16);
              const float gv = up ? other : acc[i][j];
              const float uv = up ? acc[i][j + 1] : other;
              const __nv_bfloat16 v = __float2bfloat16_rn(silu_fast(gv) * uv);
              if (staged) {
                st_shared(so + j * C::OUT_ROW, v);
              } else {
                if (col + j + odd < last) *out = v;
                out += 2 * static_cast<int64_t>(args.n_out);
              }
            }
          }
        }
      } else if constexpr (KIND == kDown) {
        // Route rows are multiples of 128 bytes: always staged.
#pragma unroll
        for (int i = 0; i < C::NCH; ++i) {
          const int col = (C::PG * i + half) * C::C;
          if (col < n_mma) {
#pragma unroll
            for (int j = 0; j < C::C; ++j)
              st_shared(c.s_out + (col + j) * C::OUT_ROW + row * 4, acc[i][j]);
          }
        }
      } else {
        const int f = fb * 128 + row;
        const int last = f < args.n_out ? rows : 0;
#pragma unroll
        for (int i = 0; i < C::NCH; ++i) {
          const int col = (C::PG * i + half) * C::C;
          if (col < n_mma) {
            auto *out = static_cast<__nv_bfloat16 *>(args.out) + (row0 + col) * args.n_out + f;
            const uint32_t so = c.s_out + col * C::OUT_ROW + row * 2;
#pragma unroll
            for (int j = 0; j < C::C; ++j) {
              const __nv_bfloat16 v = __float2bfloat16_rn(acc[i][j]);
              if (staged) {
                st_shared(so + j * C::OUT_ROW, v);
              } else {
                if (col + j < last) *out = v;
                out += args.n_out;
              }
            }
          }
        }
      }
      if (staged) {
        __syncwarp();
        if (lane == 0) mbar_arrive(c.out_full);
        if (!wait(c.out_full, out_phase, c.abort)) return;
        out_phase ^= 1;
        constexpr int PER = KIND == kGateUp ? 64 : 128;  // features of an item
        constexpr int SIZE = KIND == kDown ? 4 : 2;
        constexpr int LANES = C::OUT_ROW / 16;  // of a row
        constexpr int STEP = C::PROMOTERS * (32 / LANES);
        const int bytes = min(PER, args.n_out - fb * PER) * SIZE;
        const bool mine = (lane % LANES) * 16 < bytes;
        char *out = static_cast<char *>(args.out) + static_cast<int64_t>(fb) * (PER * SIZE) +
                    (lane % LANES) * 16;
        const int n0 = (half * 4 + q) * (32 / LANES) + lane / LANES;
#pragma unroll
        for (int i = 0; i < (NT + STEP - 1) / STEP; ++i) {
          const int n = n0 + i * STEP;
          if (n < rows && mine) {
            int64_t to = row0 + n;
            if (KIND == kDown) {
              int32_t r;
              asm volatile("ld.shared.s32 %0, [%1];" : "=r"(r) : "r"(s_route + n * 4));
              if (r < 0) continue;
              to = r;
            }
            uint4 v;
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(c.s_out + n * C::OUT_ROW + (lane % LANES) * 16));
            if (KIND == kDown) {
              float w;
              asm volatile("ld.shared.f32 %0, [%1];" : "=f"(w) : "r"(s_route + (NT + n) * 4));
              v.x = __float_as_uint(__uint_as_float(v.x) * w);
              v.y = __float_as_uint(__uint_as_float(v.y) * w);
              v.z = __float_as_uint(__uint_as_float(v.z) * w);
              v.w = __float_as_uint(__uint_as_float(v.w) * w);
            }
            *reinterpret_cast<uint4 *>(out + to * (static_cast<int64_t>(args.n_out) * SIZE)) = v;
          }
        }
      }
    }
  }
}

// NT: rows of x per tile; GPB: groups per block of 128 k.
template <int NT, int GPB, int KIND>
__global__ void __launch_bounds__(Cfg<NT, GPB, KIND>::THREADS, 1)
    w4_gemm_kernel(const __grid_constant__ CUtensorMap tmX,
                   const __grid_constant__ CUtensorMap tmWhole, const __grid_constant__ Args args) {
  using C = Cfg<NT, GPB, KIND>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  const int split = args.split;
  Ctx c;
  c.wbytes = args.sh.block_bytes();
  c.qbytes = args.sh.quarter_bytes();
  c.scale_off = args.sh.scale_off();
  c.zero_off = args.sh.zero_off();
  uint8_t *s_w = smem + C::BS * C::B_BYTES;
  uint8_t *s_red = s_w + args.ws * c.wbytes;  // [split - 1][NT][128] fp32
  uint8_t *s_out = s_red + (split - 1) * NT * 512;  // [NT] output rows
  uint8_t *s_scale = s_out + C::OUT_BYTES;
  uint64_t *bars = reinterpret_cast<uint64_t *>(s_scale + C::SCALE_BYTES + C::ROUTE_BYTES);
  c.s_scale = smem_u32(s_scale);
  c.s_route = c.s_scale + C::SCALE_BYTES;
  c.s_out = smem_u32(s_out);
  c.s_b = smem_u32(smem);
  c.s_w = smem_u32(s_w);
  c.s_red = smem_u32(s_red);
  c.w_full = smem_u32(bars);
  c.w_empty = c.w_full + 8 * MAX_WS;
  c.b_full = c.w_empty + 8 * MAX_WS;
  c.a_full = c.b_full + 8 * C::BS;
  c.ab_empty = c.a_full + 8 * C::BS;
  c.d_full = c.ab_empty + 8 * C::BS;
  c.d_empty = c.d_full + 8 * C::ND;
  c.red_full = c.d_empty + 8 * C::ND;
  c.red_empty = c.red_full + 8;
  c.out_free = c.red_empty + 8;
  c.out_full = c.out_free + 8;
  uint32_t *tmem_holder =
      reinterpret_cast<uint32_t *>(bars + 2 * MAX_WS + 3 * C::BS + 2 * C::ND + 4);
  c.abort = reinterpret_cast<volatile int *>(tmem_holder + 1);

  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  c.split = split;
  c.rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.ws; ++s) {
      mbar_init(c.w_full + 8 * s, 1);
      mbar_init(c.w_empty + 8 * s, 4);  // a decoding group
    }
    for (int s = 0; s < C::BS; ++s) {
      mbar_init(c.b_full + 8 * s, 1);
      mbar_init(c.a_full + 8 * s, 4);
      mbar_init(c.ab_empty + 8 * s, 1);
    }
    for (int s = 0; s < C::ND; ++s) {
      mbar_init(c.d_full + 8 * s, 1);
      mbar_init(c.d_empty + 8 * s, C::PROMOTERS);
    }
    mbar_init(c.red_full, C::PROMOTERS * (split > 1 ? split - 1 : 1));
    mbar_init(c.red_empty, C::PROMOTERS);
    mbar_init(c.out_free, C::PROMOTERS);
    mbar_init(c.out_full, C::PROMOTERS);
    *c.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1 && lane == 0) {
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmWhole);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (split > 1) cluster_sync();  // the peers' barriers are ready
  c.tmem = *tmem_holder;
  // Every role, that of the codes too: the kernel before may be the one that packs
  // or updates them, and only this wait promises that its writes are seen.
  pdl_wait();
  const int mt = KIND == kLinear
                     ? static_cast<int>((args.m + NT - 1) / NT)
                     : static_cast<int>(min64(args.counters[B200MOE_CNT_MTILES], args.max_mtiles));
  c.items = mt * args.n_blocks;
  c.first = blockIdx.x / split;
  c.step = gridDim.x / split;
  c.kb0 = c.rank * args.num_kb / split;
  c.kb1 = (c.rank + 1) * args.num_kb / split;

  if (warp == 0) {
    if (elect_one()) load_codes<NT, KIND>(args, c);
  } else if (warp == 1) {
    load_rows<NT, GPB, KIND>(args, c, &tmX, &tmWhole);
  } else if (warp == 2) {
    if (elect_one()) issue_mma<NT, GPB, KIND>(args, c);
  } else if (warp >= C::PROMOTE0) {
    promote<NT, GPB, KIND>(args, c, (warp - C::PROMOTE0) >> 2, warp & 3);
  } else if (warp >= 3) {
    decode<NT, GPB, KIND>(args, c, (warp - 3) >> 2, warp & 3);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*c.abort) {
    // A wait ran out: give copies in flight time to land before leaving.
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < 2000000ull) {
    }
    __syncthreads();
  }
  if (split > 1) cluster_sync();  // nobody leaves while a peer may write here
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(c.tmem, 512);
  }
}

template <int NT, int GPB, int KIND>
int launch(const CUtensorMap &mx, const CUtensorMap &mwhole, Args a, double items,
           cudaStream_t s) {
  using C = Cfg<NT, GPB, KIND>;
  static_assert((2 * MAX_WS + 3 * C::BS + 2 * C::ND + 4) * 8 + 16 <= TAIL_BYTES,
                "shared memory tail");
  static bool done[64] = {false};
  const int dev = current_device();
  if (!(dev >= 0 && dev < 64 && done[dev])) {
    B200_CUDA(cudaFuncSetAttribute(w4_gemm_kernel<NT, GPB, KIND>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT + 1024));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  // CTAs per cluster: the split whose rounds of items, each as long as its k
  // blocks and two more for filling and the epilogue, end first.
  const int sms = sm_count();
  int best = 1;
  double best_time = 1e30;
  for (int sp = 1; split_ok(sp, NT) && sp <= a.num_kb; sp *= 2) {
    const double rounds = static_cast<double>(
        static_cast<int64_t>((items + sms / sp - 1) / (sms / sp)));
    const double time = rounds * ((a.num_kb + sp - 1) / sp + 2.0 + (sp > 1 ? 1.0 : 0.0));
    if (time < best_time - 1e-9) {
      best_time = time;
      best = sp;
    }
  }
  a.split = best;
  a.ws = C::code_stages(a.sh.block_bytes(), a.split);
  int clusters = sms / a.split;
  const int64_t most = (KIND == kLinear ? (a.m + NT - 1) / NT : a.max_mtiles) * a.n_blocks;
  if (most < clusters) clusters = static_cast<int>(most < 1 ? 1 : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * a.split);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes =
      1024 + static_cast<size_t>(C::fixed_bytes(a.split)) + static_cast<size_t>(a.ws) * a.sh.block_bytes();
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (a.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.split;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled(kPdlTcgen05)) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  B200_CUDA(cudaLaunchKernelEx(&cfg, w4_gemm_kernel<NT, GPB, KIND>, mx, mwhole, a));
  B200_LAUNCHED();
  return B200MOE_OK;
}

template <int NT, int KIND>
int launch_nt(const CUtensorMap &mx, const CUtensorMap &mwhole, const Args &a, double items,
              cudaStream_t s) {
  switch (a.sh.groups_per_block()) {
    case 1: return launch<NT, 1, KIND>(mx, mwhole, a, items, s);
    case 2: return launch<NT, 2, KIND>(mx, mwhole, a, items, s);
    default: return launch<NT, 4, KIND>(mx, mwhole, a, items, s);
  }
}

int rows_map(CUtensorMap *map, const void *base, int64_t rows, int k, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(k) * 2};
  const uint32_t box[2] = {64, static_cast<uint32_t>(box_rows)};
  return tcg::make_map(map, base, 2, dims, strides, box);
}

template <int KIND>
int stages_of(int nt, const Shape &sh, int split) {
  auto of = [&](auto rows, auto gpb) {
    return Cfg<decltype(rows)::value, decltype(gpb)::value, KIND>::code_stages(sh.block_bytes(),
                                                                               split);
  };
  auto by_group = [&](auto rows) {
    switch (sh.groups_per_block()) {
      case 1: return of(rows, std::integral_constant<int, 1>{});
      case 2: return of(rows, std::integral_constant<int, 2>{});
      default: return of(rows, std::integral_constant<int, 4>{});
    }
  };
  switch (nt) {
    case 32: return by_group(std::integral_constant<int, 32>{});
    case 64: return by_group(std::integral_constant<int, 64>{});
    default: return by_group(std::integral_constant<int, 128>{});
  }
}

// The smallest tile that holds `rows` rows, or the largest.  Sixteen rows and fewer
// are streamed (w4_stream.cuh).
int tile_of_rows(int64_t rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

// x: [rows, k]; gathered four rows at a time, or in boxes of 16 and nt rows.
template <int KIND>
int launch_any(const void *x, int64_t rows, int k, const Args &a, int nt, double items,
               cudaStream_t s) {
  CUtensorMap mx, mwhole;
  int rc = rows_map(&mx, x, rows, k, a.gather ? 1 : 16);
  if (rc) return rc;
  rc = a.gather ? B200MOE_OK : rows_map(&mwhole, x, rows, k, nt);
  if (rc) return rc;
  if (a.gather) mwhole = mx;
  switch (nt) {
    case 32: return launch_nt<32, KIND>(mx, mwhole, a, items, s);
    case 64: return launch_nt<64, KIND>(mx, mwhole, a, items, s);
    default: return launch_nt<128, KIND>(mx, mwhole, a, items, s);
  }
}

}  // namespace w4g

int w4_linear_tc(const void *x, int64_t m, int n, int k, const void *w, const w4::Shape &sh,
                 void *out, cudaStream_t s) {
  using namespace w4g;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w);
  a.sh = sh;
  a.n_blocks = (n + 127) / 128;
  a.num_kb = static_cast<int>(w4::blocks_of(k));
  a.n_out = n;
  a.staged = n % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  a.m = m;
  a.out = out;
  const int nt = tile_of_rows(m);
  return launch_any<kLinear>(x, m, k, a, nt, static_cast<double>((m + nt - 1) / nt) * a.n_blocks, s);
}

// `tiles`: how many row tiles the routes are expected to fill; `rows`: rows of
// the fullest tile to expect (tiles with more are worked off in turns).
int w4_gate_up_tc(const RowSource &src, int hidden, int inter, const void *w13,
                  const w4::Shape &sh, int64_t row_capacity, const int32_t *mtiles,
                  int64_t max_mtiles, const int32_t *counters, double tiles, int64_t rows,
                  void *act, cudaStream_t s) {
  using namespace w4g;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w13);
  a.sh = sh;
  a.n_blocks = (inter + 63) / 64;
  a.num_kb = static_cast<int>(w4::blocks_of(hidden));
  a.n_out = inter;
  a.staged = 1;
  a.mtiles = mtiles;
  a.counters = counters;
  a.max_mtiles = max_mtiles;
  a.row_route = src.row_route;
  a.num_routes = src.num_routes;
  a.gather = src.x_packed == nullptr ? 1 : 0;
  a.top_k = src.top_k;
  a.x_rows = src.x_rows;
  a.out = act;
  return a.gather
             ? launch_any<kGateUp>(src.x, src.x_rows, hidden, a, tile_of_rows(rows), tiles * a.n_blocks, s)
             : launch_any<kGateUp>(src.x_packed, row_capacity, hidden, a, tile_of_rows(rows),
                          tiles * a.n_blocks, s);
}

int w4_down_tc(const void *act, int hidden, int inter, const void *w2, const w4::Shape &sh,
               const int32_t *row_route, const void *route_weights, int64_t num_routes,
               int64_t row_capacity, const int32_t *mtiles, int64_t max_mtiles,
               const int32_t *counters, double tiles, int64_t rows, float *y, cudaStream_t s) {
  using namespace w4g;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w2);
  a.sh = sh;
  a.n_blocks = (hidden + 127) / 128;
  a.num_kb = static_cast<int>(w4::blocks_of(inter));
  a.n_out = hidden;
  a.staged = 1;
  a.mtiles = mtiles;
  a.counters = counters;
  a.max_mtiles = max_mtiles;
  a.row_route = row_route;
  a.route_w = static_cast<const __nv_bfloat16 *>(route_weights);
  a.num_routes = num_routes;
  a.out = y;
  return launch_any<kDown>(act, row_capacity, inter, a, tile_of_rows(rows), tiles * a.n_blocks, s);
}

}  // namespace b200moe

extern "C" int b200moe_w4_ring_stages(int product, int tile_rows, int group, int flags, int split,
                                      int *code_stages, int *operand_stages) {
  using namespace b200moe;
  using namespace b200moe::w4g;
  B200_ARG(product >= kLinear && product <= kDown, "unknown product code %d", product);
  B200_ARG(tile_rows == 32 || tile_rows == 64 || tile_rows == 128,
           "no tile of %d rows", tile_rows);
  B200_ARG(w4::group_ok(group), "group size %d must be 32, 64 or 128", group);
  B200_ARG(split_ok(split, tile_rows), "no clusters of %d CTAs with %d rows", split, tile_rows);
  B200_ARG(code_stages && operand_stages, "null pointer argument");
  const w4::Shape sh = w4::shape_of(group, flags);
  *code_stages = product == kLinear   ? stages_of<kLinear>(tile_rows, sh, split)
                 : product == kGateUp ? stages_of<kGateUp>(tile_rows, sh, split)
                                      : stages_of<kDown>(tile_rows, sh, split);
  *operand_stages = operand_stages_of(product, tile_rows);
  return B200MOE_OK;
}
