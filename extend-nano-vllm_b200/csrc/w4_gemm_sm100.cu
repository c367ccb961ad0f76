// Products with 4-bit weights on tcgen05: the dense product and the experts'
// gate/up (+ SwiGLU) and down projections, for more rows than the CUDA-core
// kernels (w4_gemv.cu) take.
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
// (TMA boxes, or four-row gathers), 2 matrix instructions, 3 TMEM allocation,
// then decoding (groups of four, alternate blocks), then promoting and epilogue
// (two groups of four, alternate column chunks).
// Every wait is bounded; on expiry the CTA records a status bit and leaves.
#include <cudaTypedefs.h>

#include "w4.cuh"

namespace b200moe {
namespace tcg {
int make_map(CUtensorMap *map, const void *base, int rank, const uint64_t *dims,
             const uint64_t *strides_bytes, const uint32_t *box);
}  // namespace tcg

namespace w4g {

using w4::Shape;

enum Kind { kLinear = 0, kGateUp = 1, kDown = 2 };

constexpr int A_STAGES = 4;   // of 64 TMEM columns: 128 k in bf16 pairs
constexpr int A_COL0 = 256;   // accumulators below, operand stages above
constexpr int MAX_WS = 16;
constexpr int SMEM_LIMIT = 226 * 1024;
constexpr int TAIL_BYTES = 1024;  // barriers

template <int NT>
struct Cfg {
  static constexpr int BS = NT == 128 ? 4 : NT == 64 ? 6 : 8;  // stages of x rows
  static constexpr int B_BYTES = NT * 256;                     // 128 k of NT rows
  static constexpr int ND = 256 / NT > 8 ? 8 : 256 / NT;       // accumulators
  static constexpr int C = NT == 16 ? 8 : 16;                  // columns per chunk
  static constexpr int NCH = NT / C / 2;                       // chunks per promoting group
  // Decoding groups: one keeps up with 128-row tiles (512 cycles of matrix
  // instructions per block) and leaves the 64 sums per promoting thread room
  // in the register file; smaller tiles are bound by the code stream.
  static constexpr int DG = NT == 128 ? 1 : 2;
  static constexpr int PROMOTE0 = 4 + 4 * DG;  // first promoting warp
  static constexpr int THREADS = 32 * (PROMOTE0 + 8);
};

struct Args {
  const uint8_t *w;
  Shape sh;
  int kind;
  int n_blocks;  // weight tiles per matrix
  int num_kb;
  int n_out;     // features written per row
  int ws;        // stages of codes
  int split;     // CTAs per cluster
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

template <int NT>
__device__ __forceinline__ Tile tile_of(const Args &a, int m) {
  if (a.kind == kLinear) {
    const int64_t rb = static_cast<int64_t>(m) * NT;
    return Tile{0, static_cast<int>(rb), static_cast<int>(min64(NT, a.m - rb))};
  }
  const int32_t *t = a.mtiles + m * B200MOE_MTILE_WORDS;
  return Tile{t[0], t[1], t[2] - t[1]};
}

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

__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[16]) { tmem_ld16(taddr, v); }
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
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
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int *abort) {
  const uint64_t start = global_timer_ns();
  for (uint32_t spins = 0;; ++spins) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((spins & 63u) == 63u) {
      if (*abort) return false;
      if (global_timer_ns() - start > 2000000000ull) {
        *abort = 1;
        atomicOr(&g_status, kStatusTimeout);
        return false;
      }
    }
  }
}

// x * sigmoid(x); the fast exp and division are good to a few units in 2^-23,
// far below the bf16 store of the result.
__device__ __forceinline__ float silu_fast(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// A ring position: stage and the parity of its current use.
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++stage == n) {
      stage = 0;
      phase ^= 1;
    }
  }
};

template <int NT>
__global__ void __launch_bounds__(Cfg<NT>::THREADS, 1)
    w4_gemm_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ Args args) {
  using C = Cfg<NT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~static_cast<uintptr_t>(1023));
  const int wbytes = args.sh.block_bytes();
  uint8_t *s_b = smem;
  uint8_t *s_w = smem + C::BS * C::B_BYTES;
  float *s_red = reinterpret_cast<float *>(s_w + args.ws * wbytes);  // [split - 1][NT][128]
  uint64_t *bars = reinterpret_cast<uint64_t *>(s_red + (args.split - 1) * NT * 128);
  uint64_t *w_full = bars;
  uint64_t *w_empty = w_full + MAX_WS;
  uint64_t *b_full = w_empty + MAX_WS;
  uint64_t *b_empty = b_full + C::BS;
  uint64_t *a_full = b_empty + C::BS;
  uint64_t *a_empty = a_full + A_STAGES;
  uint64_t *d_full = a_empty + A_STAGES;
  uint64_t *d_empty = d_full + C::ND;
  uint64_t *red_full = d_empty + C::ND;
  uint64_t *red_empty = red_full + 1;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(red_empty + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = args.split;
  const int rank = split > 1 ? static_cast<int>(cluster_rank()) : 0;
  pdl_trigger();

  if (threadIdx.x == 0) {
    for (int s = 0; s < args.ws; ++s) {
      mbar_init(smem_u32(&w_full[s]), 1);
      mbar_init(smem_u32(&w_empty[s]), 12);  // four decoding and eight promoting warps
    }
    for (int s = 0; s < C::BS; ++s) {
      mbar_init(smem_u32(&b_full[s]), 1);
      mbar_init(smem_u32(&b_empty[s]), 1);
    }
    for (int s = 0; s < A_STAGES; ++s) {
      mbar_init(smem_u32(&a_full[s]), 4);
      mbar_init(smem_u32(&a_empty[s]), 1);
    }
    for (int s = 0; s < C::ND; ++s) {
      mbar_init(smem_u32(&d_full[s]), 1);
      mbar_init(smem_u32(&d_empty[s]), 8);
    }
    mbar_init(smem_u32(red_full), 8 * (split > 1 ? split - 1 : 1));
    mbar_init(smem_u32(red_empty), 8);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1 && lane == 0) prefetch_tmap(&tmX);
  if (warp == 3) {
    tmem_alloc(smem_u32(tmem_holder), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (split > 1) cluster_sync();  // the peers' barriers are ready
  const uint32_t tmem = *tmem_holder;
  // Codes are constant; a dense call's items are known too, so its first
  // blocks are fetched while the previous kernel still runs.
  if (!(args.kind == kLinear && warp == 0)) pdl_wait();
  const int mt = args.kind == kLinear
                     ? static_cast<int>((args.m + NT - 1) / NT)
                     : static_cast<int>(min64(args.counters[B200MOE_CNT_MTILES], args.max_mtiles));
  const int items = mt * args.n_blocks;
  const int first = blockIdx.x / split;
  const int step = gridDim.x / split;
  const int kb0 = rank * args.num_kb / split;
  const int kb1 = (rank + 1) * args.num_kb / split;
  const int gpb = args.sh.groups_per_block();

  if (warp < 4) {
    if (warp == 0) {
      // ---------------- codes ----------------
      if (lane == 0) {
        Ring w;
        bool ok = true;
        for (int it = first; it < items && ok; it += step) {
          const Tile t = tile_of<NT>(args, it / args.n_blocks);
          const uint8_t *src = args.w + (static_cast<int64_t>(t.e) * args.n_blocks +
                                         it % args.n_blocks) * args.num_kb * wbytes;
          for (int r0 = 0; r0 < t.rows && ok; r0 += NT)
            for (int kb = kb0; kb < kb1; ++kb) {
              if (!mbar_wait_bounded(smem_u32(&w_empty[w.stage]), w.phase ^ 1, abort_flag)) {
                ok = false;
                break;
              }
              const uint32_t bar = smem_u32(&w_full[w.stage]);
              mbar_arrive_expect_tx(bar, wbytes);
              bulk_load(smem_u32(s_w + w.stage * wbytes), src + static_cast<int64_t>(kb) * wbytes,
                        wbytes, bar);
              w.next(args.ws);
            }
        }
      }
    } else if (warp == 1) {
      // ---------------- rows of x ----------------
      // Lane b loads the b-th 16 rows (or, gathering, the b-th four rows).
      const bool gather = args.gather != 0;
      Ring b;
      bool ok = true;
      for (int it = first; it < items && ok; it += step) {
        const Tile t = tile_of<NT>(args, it / args.n_blocks);
        for (int r0 = 0; r0 < t.rows && ok; r0 += NT) {
          const int rows = min(NT, t.rows - r0);
          const int nbox = (rows + 15) >> 4;
          const bool mine = lane < (gather ? nbox * 4 : nbox);
          int tok[4] = {0, 0, 0, 0};
          if (gather && mine) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              tok[j] = gather_token(t.rb + r0 + 4 * lane + j, t.rb + t.rows, args.row_route,
                                    nullptr, args.top_k, args.num_routes, args.x_rows);
          }
          for (int kb = kb0; kb < kb1; ++kb) {
            bool got = true;
            if (lane == 0)
              got = mbar_wait_bounded(smem_u32(&b_empty[b.stage]), b.phase ^ 1, abort_flag);
            if (!__shfl_sync(0xffffffffu, got ? 1 : 0, 0)) {
              ok = false;
              break;
            }
            const uint32_t bar = smem_u32(&b_full[b.stage]);
            const uint32_t dst = smem_u32(s_b + b.stage * C::B_BYTES);
            if (lane == 0) mbar_arrive_expect_tx(bar, nbox * 16 * 256);
            __syncwarp();
            if (mine) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t half = dst + h * NT * 128;
                const int c0 = kb * w4::kBlockK + h * 64;
                if (gather)
                  tma_gather4(half + lane * 512, &tmX, bar, c0, tok[0], tok[1], tok[2], tok[3]);
                else
                  tma_load_2d(half + lane * 2048, &tmX, bar, c0, t.rb + r0 + lane * 16);
              }
            }
            b.next(C::BS);
          }
        }
      }
    } else if (warp == 2) {
      // ---------------- matrix instructions ----------------
      if (lane == 0) {
        Ring b, a, d;
        bool ok = true;
        const int kk_per_group = args.sh.group / 16;
        for (int it = first; it < items && ok; it += step) {
          const Tile t = tile_of<NT>(args, it / args.n_blocks);
          for (int r0 = 0; r0 < t.rows && ok; r0 += NT) {
            const int n_mma = (min(NT, t.rows - r0) + 15) & ~15;
            const uint32_t idesc = idesc_bf16_f32(128, n_mma);
            for (int kb = kb0; kb < kb1 && ok; ++kb) {
              ok = mbar_wait_bounded(smem_u32(&b_full[b.stage]), b.phase, abort_flag) &&
                   mbar_wait_bounded(smem_u32(&a_full[a.stage]), a.phase, abort_flag);
              if (!ok) break;
              const uint32_t sb = smem_u32(s_b + b.stage * C::B_BYTES);
              const uint32_t ta = tmem + A_COL0 + a.stage * 64;
              int kk = 0;
              for (int g = 0; g < gpb; ++g) {
                if (!mbar_wait_bounded(smem_u32(&d_empty[d.stage]), d.phase ^ 1, abort_flag)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                const uint32_t td = tmem + d.stage * NT;
                for (int j = 0; j < kk_per_group; ++j, ++kk)
                  mma_ts(td, ta + kk * 8,
                         sw128_kmajor_desc(sb + (kk >> 2) * NT * 128 + (kk & 3) * 32), idesc,
                         j != 0);
                tc_commit(smem_u32(&d_full[d.stage]));
                d.next(C::ND);
              }
              if (!ok) break;
              tc_commit(smem_u32(&a_empty[a.stage]));
              tc_commit(smem_u32(&b_empty[b.stage]));
              a.next(A_STAGES);
              b.next(C::BS);
            }
          }
        }
      }
    }
  } else if (warp < C::PROMOTE0) {
    // ---------------- decoding: codes -> q - z in TMEM ----------------
    const int q = warp & 3;
    const int row = q * 32 + lane;
    const int grp = (warp - 4) >> 2;
    const int gshift = args.sh.group == 32 ? 0 : args.sh.group == 64 ? 1 : 2;
    Ring w, a;
    int turn = 0;
    bool ok = true;
    for (int it = first; it < items && ok; it += step) {
      const Tile t = tile_of<NT>(args, it / args.n_blocks);
      for (int r0 = 0; r0 < t.rows && ok; r0 += NT)
        for (int kb = kb0; kb < kb1; ++kb) {
          if (turn == grp) {
            if (!mbar_wait_bounded(smem_u32(&w_full[w.stage]), w.phase, abort_flag)) {
              ok = false;
              break;
            }
            const uint8_t *st = s_w + w.stage * wbytes;
            uint4 codes[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
              codes[c] = *reinterpret_cast<const uint4 *>(st + c * 2048 + row * 16);
            uint32_t zp[4] = {0x43084308u, 0x43084308u, 0x43084308u, 0x43084308u};
            if (args.sh.has_zero) {
#pragma unroll
              for (int c = 0; c < 4; ++c)
                zp[c] = w4::zero_pair(st[args.sh.zero_off() + (c >> gshift) * 128 + row]);
            }
            if (!mbar_wait_bounded(smem_u32(&a_empty[a.stage]), a.phase ^ 1, abort_flag)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t ta =
                tmem + A_COL0 + a.stage * 64 + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t r[32];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint4 v = codes[2 * h + c];
                const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  uint32_t o[4];
                  w4::decode8(word[j], zp[2 * h + c], o);
#pragma unroll
                  for (int i = 0; i < 4; ++i) r[c * 16 + j * 4 + i] = o[i];
                }
              }
              tmem_st32(ta + h * 32, r);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(smem_u32(&a_full[a.stage]));
              mbar_arrive(smem_u32(&w_empty[w.stage]));
            }
          }
          if (++turn == C::DG) turn = 0;
          w.next(args.ws);
          a.next(A_STAGES);
        }
    }
  } else {
    // ---------------- promoting and epilogue ----------------
    const int q = warp & 3;
    const int row = q * 32 + lane;
    const int half = (warp - C::PROMOTE0) >> 2;
    const uint32_t tq = tmem + (static_cast<uint32_t>(q * 32) << 16);
    Ring w, d;
    uint32_t red_phase = 0;
    bool ok = true;
    for (int it = first; it < items && ok; it += step) {
      const Tile t = tile_of<NT>(args, it / args.n_blocks);
      const int fb = it % args.n_blocks;
      for (int r0 = 0; r0 < t.rows && ok; r0 += NT) {
        const int rows = min(NT, t.rows - r0);
        const int n_mma = (rows + 15) & ~15;
        float acc[C::NCH][C::C];
#pragma unroll
        for (int i = 0; i < C::NCH; ++i)
#pragma unroll
          for (int j = 0; j < C::C; ++j) acc[i][j] = 0.f;
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          // The copy that wrote this stage is long complete (the decoding
          // warps waited for it); this wait makes its writes visible here.
          ok = mbar_wait_bounded(smem_u32(&w_full[w.stage]), w.phase, abort_flag);
          if (!ok) break;
          const uint16_t *scales = reinterpret_cast<const uint16_t *>(
              s_w + w.stage * wbytes + args.sh.scale_off());
          for (int g = 0; g < gpb; ++g) {
            const float s = w4::scale_f32(scales[g * 128 + row], args.sh.half_scale);
            ok = mbar_wait_bounded(smem_u32(&d_full[d.stage]), d.phase, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t td = tq + d.stage * NT;
#pragma unroll
            for (int i = 0; i < C::NCH; i += 2) {
              float v0[C::C], v1[C::C];
              const int c0 = (2 * i + half) * C::C;
              const int c1 = c0 + 2 * C::C;
              if (c0 < n_mma) {
                tmem_ld(td + c0, v0);
                if (i + 1 < C::NCH && c1 < n_mma) tmem_ld(td + c1, v1);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < C::C; ++j) acc[i][j] = fmaf(s, v0[j], acc[i][j]);
                if (i + 1 < C::NCH && c1 < n_mma) {
#pragma unroll
                  for (int j = 0; j < C::C; ++j)
                    acc[i + 1 < C::NCH ? i + 1 : i][j] =
                        fmaf(s, v1[j], acc[i + 1 < C::NCH ? i + 1 : i][j]);
                }
              }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&d_empty[d.stage]));
            d.next(C::ND);
          }
          if (!ok) break;
          if (lane == 0) mbar_arrive(smem_u32(&w_empty[w.stage]));
          w.next(args.ws);
        }
        if (!ok) break;
        if (split > 1) {
          if (rank != 0) {
            // This CTA's sums into the first one's shared memory.
            ok = wait_cluster(smem_u32(red_empty), red_phase ^ 1, abort_flag);
            if (!ok) break;
            const uint32_t dst =
                map_rank(smem_u32(s_red + (rank - 1) * NT * 128 + row), 0);
#pragma unroll
            for (int i = 0; i < C::NCH; ++i) {
              const int c = (2 * i + half) * C::C;
              if (c < n_mma) {
#pragma unroll
                for (int j = 0; j < C::C; ++j) st_cluster(dst + (c + j) * 512, acc[i][j]);
              }
            }
            __syncwarp();
            if (lane == 0) arrive_cluster(map_rank(smem_u32(red_full), 0));
            red_phase ^= 1;
            continue;
          }
          ok = wait_cluster(smem_u32(red_full), red_phase, abort_flag);
          if (!ok) break;
          red_phase ^= 1;
          for (int p = 0; p < split - 1; ++p) {
#pragma unroll
            for (int i = 0; i < C::NCH; ++i) {
              const int c = (2 * i + half) * C::C;
              if (c < n_mma) {
#pragma unroll
                for (int j = 0; j < C::C; ++j) acc[i][j] += s_red[(p * NT + c + j) * 128 + row];
              }
            }
          }
          __syncwarp();
          if (lane == 0)
            for (int p = 1; p < split; ++p) arrive_cluster(map_rank(smem_u32(red_empty), p));
        }
        const int64_t row0 = static_cast<int64_t>(t.rb) + r0;
        if (args.kind == kGateUp) {
          // Lanes 0-15 hold gate rows, 16-31 the up rows of the same features:
          // of each pair of columns the lower half finishes the first, the
          // upper half the second.
          auto *out = static_cast<__nv_bfloat16 *>(args.out);
          const int f = fb * 64 + q * 16 + (lane & 15);
          const bool up = lane >= 16;
#pragma unroll
          for (int i = 0; i < C::NCH; ++i) {
            const int c = (2 * i + half) * C::C;
            if (c < n_mma) {
#pragma unroll
              for (int j = 0; j < C::C; j += 2) {
                const float other =
                    __shfl_xor_sync(0xffffffffu, up ? acc[i][j] : acc[i][j + 1], 16);
                const float gv = up ? other : acc[i][j];
                const float uv = up ? acc[i][j + 1] : other;
                const int n = c + j + (up ? 1 : 0);
                if (f < args.n_out && n < rows)
                  out[(row0 + n) * args.n_out + f] = __float2bfloat16_rn(silu_fast(gv) * uv);
              }
            }
          }
        } else {
          const int f = fb * 128 + row;
#pragma unroll
          for (int i = 0; i < C::NCH; ++i) {
            const int c = (2 * i + half) * C::C;
            if (c < n_mma) {
              // Lane j knows the route and the weight of column c + j.
              int32_t route = -1;
              float weight = 0.f;
              if (args.kind == kDown && lane < C::C && c + lane < rows) {
                route = args.row_route[row0 + c + lane];
                if (route < 0 || route >= args.num_routes) {
                  atomicOr(&g_status, kStatusIndex);
                  route = -1;
                } else {
                  weight = __bfloat162float(args.route_w[route]);
                }
              }
#pragma unroll
              for (int j = 0; j < C::C; ++j) {
                const int n = c + j;
                const int32_t r = __shfl_sync(0xffffffffu, route, j);
                const float wgt = __shfl_sync(0xffffffffu, weight, j);
                if (f < args.n_out && n < rows) {
                  if (args.kind == kDown) {
                    if (r >= 0)
                      static_cast<float *>(args.out)[static_cast<int64_t>(r) * args.n_out + f] =
                          acc[i][j] * wgt;
                  } else {
                    static_cast<__nv_bfloat16 *>(args.out)[(row0 + n) * args.n_out + f] =
                        __float2bfloat16_rn(acc[i][j]);
                  }
                }
              }
            }
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // A wait ran out: give copies in flight time to land before leaving.
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < 2000000ull) {
    }
    __syncthreads();
  }
  if (split > 1) cluster_sync();  // nobody leaves while a peer may write here
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int NT>
size_t smem_bytes(const Args &a) {
  return 1024 + static_cast<size_t>(Cfg<NT>::BS) * Cfg<NT>::B_BYTES +
         static_cast<size_t>(a.ws) * a.sh.block_bytes() +
         static_cast<size_t>(a.split - 1) * NT * 512 + TAIL_BYTES;
}

template <int NT>
int launch(const CUtensorMap &mx, Args a, double items, cudaStream_t s) {
  static_assert((2 * MAX_WS + 2 * Cfg<NT>::BS + 2 * A_STAGES + 2 * Cfg<NT>::ND + 2) * 8 + 16 <=
                    TAIL_BYTES,
                "shared memory tail");
  static bool done[64] = {false};
  const int dev = current_device();
  if (!(dev >= 0 && dev < 64 && done[dev])) {
    B200_CUDA(cudaFuncSetAttribute(w4_gemm_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   SMEM_LIMIT + 1024));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  // CTAs per cluster: the split whose rounds of items, each as long as its k
  // blocks and two more for filling and the epilogue, end first.
  const int sms = sm_count();
  int best = 1;
  double best_time = 1e30;
  for (int sp = 1; sp <= 8 && sp <= a.num_kb; sp *= 2) {
    if ((sp - 1) * NT > 112) break;
    const double rounds = static_cast<double>(
        static_cast<int64_t>((items + sms / sp - 1) / (sms / sp)));
    const double time = rounds * ((a.num_kb + sp - 1) / sp + 2.0 + (sp > 1 ? 1.0 : 0.0));
    if (time < best_time - 1e-9) {
      best_time = time;
      best = sp;
    }
  }
  a.split = best;
  a.ws = static_cast<int>((SMEM_LIMIT - static_cast<int64_t>(Cfg<NT>::BS) * Cfg<NT>::B_BYTES -
                           static_cast<int64_t>(a.split - 1) * NT * 512 - TAIL_BYTES) /
                          a.sh.block_bytes());
  if (a.ws > MAX_WS) a.ws = MAX_WS;
  int clusters = sms / a.split;
  const int64_t most = (a.kind == kLinear ? (a.m + NT - 1) / NT : a.max_mtiles) * a.n_blocks;
  if (most < clusters) clusters = static_cast<int>(most < 1 ? 1 : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(clusters * a.split);
  cfg.blockDim = dim3(Cfg<NT>::THREADS);
  cfg.dynamicSmemBytes = smem_bytes<NT>(a);
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
  B200_CUDA(cudaLaunchKernelEx(&cfg, w4_gemm_kernel<NT>, mx, a));
  B200_LAUNCHED();
  return B200MOE_OK;
}

int launch_any(const CUtensorMap &mx, const Args &a, int nt, double items, cudaStream_t s) {
  switch (nt) {
    case 16: return launch<16>(mx, a, items, s);
    case 32: return launch<32>(mx, a, items, s);
    case 64: return launch<64>(mx, a, items, s);
    default: return launch<128>(mx, a, items, s);
  }
}

int rows_map(CUtensorMap *map, const void *base, int64_t rows, int k, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(k), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(k) * 2};
  const uint32_t box[2] = {64, static_cast<uint32_t>(box_rows)};
  return tcg::make_map(map, base, 2, dims, strides, box);
}

// The smallest tile that holds `rows` rows.
int tile_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

}  // namespace w4g

int w4_linear_tc(const void *x, int64_t m, int n, int k, const void *w, const w4::Shape &sh,
                 void *out, cudaStream_t s) {
  using namespace w4g;
  CUtensorMap mx;
  const int rc = rows_map(&mx, x, m, k, 16);
  if (rc) return rc;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w);
  a.sh = sh;
  a.kind = kLinear;
  a.n_blocks = (n + 127) / 128;
  a.num_kb = static_cast<int>(w4::blocks_of(k));
  a.n_out = n;
  a.m = m;
  a.out = out;
  const int nt = tile_rows(m);
  return launch_any(mx, a, nt, static_cast<double>((m + nt - 1) / nt) * a.n_blocks, s);
}

// `tiles`: how many row tiles the routes are expected to fill; `rows`: rows of
// the fullest tile to expect (tiles with more are worked off in turns).
int w4_gate_up_tc(const RowSource &src, int hidden, int inter, const void *w13,
                  const w4::Shape &sh, int64_t row_capacity, const int32_t *mtiles,
                  int64_t max_mtiles, const int32_t *counters, double tiles, int64_t rows,
                  void *act, cudaStream_t s) {
  using namespace w4g;
  CUtensorMap mx;
  const bool gather = src.x_packed == nullptr;
  const int rc = rows_map(&mx, gather ? src.x : src.x_packed, gather ? src.x_rows : row_capacity,
                          hidden, gather ? 1 : 16);
  if (rc) return rc;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w13);
  a.sh = sh;
  a.kind = kGateUp;
  a.n_blocks = (inter + 63) / 64;
  a.num_kb = static_cast<int>(w4::blocks_of(hidden));
  a.n_out = inter;
  a.mtiles = mtiles;
  a.counters = counters;
  a.max_mtiles = max_mtiles;
  a.row_route = src.row_route;
  a.num_routes = src.num_routes;
  a.gather = gather ? 1 : 0;
  a.top_k = src.top_k;
  a.x_rows = src.x_rows;
  a.out = act;
  return launch_any(mx, a, tile_rows(rows), tiles * a.n_blocks, s);
}

int w4_down_tc(const void *act, int hidden, int inter, const void *w2, const w4::Shape &sh,
               const int32_t *row_route, const void *route_weights, int64_t num_routes,
               int64_t row_capacity, const int32_t *mtiles, int64_t max_mtiles,
               const int32_t *counters, double tiles, int64_t rows, float *y, cudaStream_t s) {
  using namespace w4g;
  CUtensorMap mx;
  const int rc = rows_map(&mx, act, row_capacity, inter, 16);
  if (rc) return rc;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w2);
  a.sh = sh;
  a.kind = kDown;
  a.n_blocks = (hidden + 127) / 128;
  a.num_kb = static_cast<int>(w4::blocks_of(inter));
  a.n_out = hidden;
  a.mtiles = mtiles;
  a.counters = counters;
  a.max_mtiles = max_mtiles;
  a.row_route = row_route;
  a.route_w = static_cast<const __nv_bfloat16 *>(route_weights);
  a.num_routes = num_routes;
  a.out = y;
  return launch_any(mx, a, tile_rows(rows), tiles * a.n_blocks, s);
}

}  // namespace b200moe
