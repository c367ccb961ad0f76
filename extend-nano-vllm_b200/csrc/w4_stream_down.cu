// The experts' down projection of a few rows with 4-bit weights.
#include "w4_stream.cuh"

namespace b200moe {
namespace w4s {

// Few routes: out[t, f] = sum_s weight[t, s] * (D_e act[t, s])[f] in slot order.
// grid (16-row slabs, tokens); warp w takes slots w, w + 8, ...
template <int GPB>
__global__ void __launch_bounds__(32 * kWarps) w4_down_slots_kernel(
    const __nv_bfloat16 *act, int hidden, int inter, const int64_t *ids,
    const __nv_bfloat16 *weights, int top_k, int num_experts, const uint8_t *w2, const Shape sh,
    int tiles, int num_kb, __nv_bfloat16 *__restrict__ out) {
  constexpr int BATCH = GPB == 4 ? 4 : 6;  // blocks in flight
  __shared__ float part[32][16];
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x >> 3, quarter = (blockIdx.x >> 1) & 3, op = blockIdx.x & 1;
  const int64_t token = blockIdx.y;
  const bool zeros = sh.has_zero != 0;
  const int bytes = sh.block_bytes();
  // Only w4_route_gate_up comes before this kernel, and each of its blocks lets it
  // start after its own wait: every kernel before that one has ended and its writes
  // are seen, so the routes and the codes are there, and the first blocks are
  // fetched while gate/up still computes act.
  bool act_ready = false;
  for (int s = warp; s < top_k; s += kWarps) {
    const int64_t route = token * top_k + s;
    const int64_t e = ids[route];
    const bool live = e >= 0 && e < num_experts;
    float tot[4] = {0.f, 0.f, 0.f, 0.f};
    if (live) {
      const uint8_t *w = w2 + (e * tiles + tile) * num_kb * bytes + quarter * sh.quarter_bytes();
      const __nv_bfloat16 *x = act + route * inter + 8 * t;
      for (int kb0 = 0; kb0 < num_kb; kb0 += BATCH) {
        uint4 codes[BATCH][2];
        uint32_t scale[BATCH][GPB];
        uint32_t zero[BATCH][GPB];
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
          if (kb0 + b < num_kb) {
            const uint8_t *block = w + static_cast<int64_t>(kb0 + b) * bytes;
            const uint8_t *c = block + w4::code_place(op * 16 + g, t);
            codes[b][0] = load_codes(c);
            codes[b][1] = load_codes(c + 512);
            const uint8_t *sc = block + w4::kCodeBytes + (4 * g + 2 * op) * 2;
#pragma unroll
            for (int j = 0; j < GPB; ++j) {
              scale[b][j] = __ldg(reinterpret_cast<const uint32_t *>(sc + j * 64));
              if (zeros)
                zero[b][j] = __ldg(reinterpret_cast<const uint16_t *>(
                    block + w4::kCodeBytes + GPB * 64 + j * 32 + 4 * g + 2 * op));
            }
          }
        if (!act_ready) {
          pdl_wait();
          act_ready = true;
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
          if (kb0 + b < num_kb) {
#pragma unroll
            for (int j = 0; j < GPB; ++j) {
              float acc[4] = {0.f, 0.f, 0.f, 0.f};
              const uint32_t z0 = w4::zero_pair(zeros ? zero[b][j] & 15u : 8u);
              const uint32_t z1 = w4::zero_pair(zeros ? (zero[b][j] >> 8) & 15u : 8u);
#pragma unroll
              for (int cc = 0; cc < 4 / GPB; ++cc) {
                const int c = j * (4 / GPB) + cc;
                const int at = (kb0 + b) * w4::kBlockK + 32 * c;
                // Column 0 is the act row, the other columns are zero.
                const uint4 xv = g == 0 && at < inter ? *reinterpret_cast<const uint4 *>(x + at)
                                                      : make_uint4(0, 0, 0, 0);
                uint32_t lo[4], hi[4];
                w4::decode8(word(codes[b][0], c), z0, lo);
                w4::decode8(word(codes[b][1], c), z1, hi);
                mma(acc, lo[0], hi[0], lo[1], hi[1], xv.x, xv.y);
                mma(acc, lo[2], hi[2], lo[3], hi[3], xv.z, xv.w);
              }
              const float s0 = w4::scale_f32(scale[b][j] & 0xffffu, sh.half_scale);
              const float s1 = w4::scale_f32(scale[b][j] >> 16, sh.half_scale);
              tot[0] = fmaf(s0, acc[0], tot[0]);
              tot[2] = fmaf(s1, acc[2], tot[2]);
            }
          }
      }
    }
    if (t == 0) {
      const float w = live ? __bfloat162float(weights[route]) : 0.f;
      part[s][g] = live ? tot[0] * w : 0.f;
      part[s][g + 8] = live ? tot[2] * w : 0.f;
    }
  }
  if (!act_ready) pdl_wait();
  __syncthreads();
  const int f = tile * w4::kTileRows + quarter * 32 + op * 16 + threadIdx.x;
  if (threadIdx.x < 16 && f < hidden) {
    float v = 0.f;
    for (int s = 0; s < top_k; ++s) v += part[s][threadIdx.x];
    out[token * hidden + f] = __float2bfloat16_rn(v);
  }
}

}  // namespace w4s

int w4_down_stream(const void *act, int hidden, int inter, const void *w2, const w4::Shape &sh,
                   const int32_t *row_route, const void *route_weights, int64_t num_routes,
                   const int32_t *mtiles, int64_t max_mtiles, const int32_t *counters,
                   double tiles, int cols, float *y, cudaStream_t s) {
  using namespace w4s;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w2);
  a.sh = sh;
  a.n_blocks = (hidden + 127) / 128;
  a.num_kb = static_cast<int>(w4::blocks_of(inter));
  a.n_out = hidden;
  a.k = inter;
  a.x = act;
  a.mtiles = mtiles;
  a.counters = counters;
  a.max_mtiles = max_mtiles;
  a.row_route = row_route;
  a.route_w = static_cast<const __nv_bfloat16 *>(route_weights);
  a.num_routes = num_routes;
  a.out = y;
  return run<kDown>(a, 4.0 * tiles * a.n_blocks, 4 * max_mtiles * a.n_blocks, cols, s);
}

// Few routes: down projection of act [tokens * top_k, inter] and the sum over a
// token's slots in one launch.
int w4_route_down(const void *act, int64_t tokens, int hidden, int inter, const int64_t *ids,
                  const void *weights, int top_k, int num_experts, const void *w2,
                  const w4::Shape &sh2, void *out, cudaStream_t s) {
  using namespace w4s;
  const int tiles = (hidden + 127) / 128;
  const dim3 grid(8 * tiles, static_cast<unsigned>(tokens));
  auto down = [&](auto kernel) {
    return launch_pdl(kPdlTiny, kernel, grid, dim3(32 * kWarps), 0, s,
                      static_cast<const __nv_bfloat16 *>(act), hidden, inter, ids,
                      static_cast<const __nv_bfloat16 *>(weights), top_k, num_experts,
                      static_cast<const uint8_t *>(w2), sh2, tiles,
                      static_cast<int>(w4::blocks_of(inter)), static_cast<__nv_bfloat16 *>(out));
  };
  switch (sh2.groups_per_block()) {
    case 1: B200_CUDA(down(w4_down_slots_kernel<1>)); break;
    case 2: B200_CUDA(down(w4_down_slots_kernel<2>)); break;
    default: B200_CUDA(down(w4_down_slots_kernel<4>)); break;
  }
  B200_LAUNCHED();
  return B200MOE_OK;
}

}  // namespace b200moe
