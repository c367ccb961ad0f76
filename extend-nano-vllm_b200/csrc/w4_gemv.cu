// Matrix-vector products with 4-bit weights (layout: w4.cuh) on the CUDA
// cores, for calls of a few rows: the dense product and the experts' pair
// (gate/up + SwiGLU, then down + route-order sum).
//
//   y[n] = sum_g s[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * x[k]
//
// The inner sum is over integers times bf16 values in fp32; a weight itself is
// never rounded.  Lane l of a warp owns one row; a chunk is 32 k of 32 rows
// (512 consecutive bytes).  The chunks of a row are split over the warps of the
// block (and over half-warps where rows are few), which are summed in a fixed
// order, so results repeat bit for bit.
#include "w4.cuh"

namespace b200moe {
namespace {

using w4::Shape;

constexpr int kWarps = 8;
constexpr int kSegK = 4096;  // k of x staged at a time, as fp32

// acc += a * b on two fp32 values at once.
__device__ __forceinline__ void fma2(float2 &acc, float2 a, float2 b) {
  uint64_t d, x, y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(acc.x), "f"(acc.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(x), "l"(y));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(acc.x), "=f"(acc.y) : "l"(d));
}

__device__ __forceinline__ uint4 load_codes(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// Sum over the 32 k of one chunk for R rows of x (fp32 in shared memory,
// row r at xs + r * stride).
template <int R>
__device__ __forceinline__ void chunk_dot(const uint4 &codes, uint32_t zpair, const float *xs,
                                          int stride, float2 (&sum)[R]) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int r = 0; r < R; ++r) sum[r] = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t d[4];
    w4::decode8(w[j], zpair, d);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float2 a = make_float2(__uint_as_float(d[i] << 16),
                                   __uint_as_float(d[i] & 0xffff0000u));
      const float2 b = make_float2(__uint_as_float(d[i + 1] << 16),
                                   __uint_as_float(d[i + 1] & 0xffff0000u));
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float4 x = *reinterpret_cast<const float4 *>(xs + r * stride + 8 * j + 2 * i);
        fma2(sum[r], a, make_float2(x.x, x.y));
        fma2(sum[r], b, make_float2(x.z, x.w));
      }
    }
  }
}

// One row's sum over chunks first, first + step, ... < last of a tile, for R
// rows of x whose k from 32 * base on are staged at xs.
template <int R, int BATCH>
__device__ __forceinline__ void row_dot(const uint8_t *tile, const Shape &sh, int row, int first,
                                        int last, int step, int base, const float *xs, int stride,
                                        float (&acc)[R]) {
  const int block_bytes = sh.block_bytes();
  const int shift = sh.group == 32 ? 0 : sh.group == 64 ? 1 : 2;  // chunks per group, log2
  for (int c0 = first; c0 < last; c0 += BATCH * step) {
    uint4 codes[BATCH];
    uint16_t scale[BATCH];
    uint32_t zero[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int c = c0 + b * step;
      if (c < last) {
        const uint8_t *block = tile + static_cast<int64_t>(c >> 2) * block_bytes;
        const int g = (c & 3) >> shift;
        codes[b] = load_codes(block + (c & 3) * 2048 + row * 16);
        scale[b] = __ldg(reinterpret_cast<const uint16_t *>(block + sh.scale_off()) +
                         g * w4::kTileRows + row);
        zero[b] = sh.has_zero ? __ldg(block + sh.zero_off() + g * w4::kTileRows + row) : 8u;
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int c = c0 + b * step;
      if (c < last) {
        float2 sum[R];
        chunk_dot<R>(codes[b], w4::zero_pair(zero[b]), xs + (c - base) * 32, stride, sum);
        const float s = w4::scale_f32(scale[b], sh.half_scale);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = fmaf(s, sum[r].x + sum[r].y, acc[r]);
      }
    }
  }
}

// Stages k [k0, k0 + n) of a bf16 row as fp32; zeros from `valid` on.
__device__ __forceinline__ void stage_bf16(float *xs, const __nv_bfloat16 *x, int k0, int n,
                                           int valid) {
  for (int i = threadIdx.x * 8; i < n; i += blockDim.x * 8) {
    float v[8];
    if (k0 + i + 8 <= valid) {
      const uint4 raw = *reinterpret_cast<const uint4 *>(x + k0 + i);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {  // valid is a multiple of 32
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
    *reinterpret_cast<float4 *>(xs + i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(xs + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}

__device__ __forceinline__ void stage_f32(float *xs, const float *x, int k0, int n, int valid) {
  for (int i = threadIdx.x * 4; i < n; i += blockDim.x * 4)
    *reinterpret_cast<float4 *>(xs + i) =
        k0 + i < valid ? __ldcg(reinterpret_cast<const float4 *>(x + k0 + i))
                       : make_float4(0.f, 0.f, 0.f, 0.f);
}

// ---------------------------------------------------------------------------
// Dense: out[m, n] for R rows of x per block; grid (32-row slabs, row groups).
// ---------------------------------------------------------------------------
template <int R>
__global__ void __launch_bounds__(32 * kWarps) w4_linear_gemv_kernel(
    const __nv_bfloat16 *x, int64_t m, int n_out, int k, const uint8_t *w, Shape sh,
    __nv_bfloat16 *__restrict__ out) {
  constexpr int SEG = kSegK / R;
  __shared__ __align__(16) float xs[R * SEG];
  __shared__ float red[kWarps][R][32];
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int tile = blockIdx.x >> 2;
  const int row = (blockIdx.x & 3) * 32 + lane;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * R;
  const int blocks = static_cast<int>(w4::blocks_of(k));
  const uint8_t *wt = w + static_cast<int64_t>(tile) * blocks * sh.block_bytes();
  float acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.f;
  pdl_wait();
  for (int k0 = 0; k0 < k; k0 += SEG) {
    const int kpad = blocks * w4::kBlockK;
    const int n = min(SEG, kpad - k0);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (m0 + r < m) stage_bf16(xs + r * SEG, x + (m0 + r) * k, k0, n, k);
    __syncthreads();
    row_dot<R, 8>(wt, sh, row, k0 / 32 + warp, (k0 + n) / 32, kWarps, k0 / 32, xs, SEG, acc);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) red[warp][r][lane] = acc[r];
  __syncthreads();
  for (int i = threadIdx.x; i < R * 32; i += blockDim.x) {
    const int r = i >> 5, l = i & 31;
    const int f = tile * w4::kTileRows + (blockIdx.x & 3) * 32 + l;
    if (m0 + r < m && f < n_out) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) v += red[q][r][l];
      out[(m0 + r) * n_out + f] = __float2bfloat16_rn(v);
    }
  }
}

// ---------------------------------------------------------------------------
// Experts, one route at a time: act[r, :] = silu(W1 x_t) * (W3 x_t) in fp32
// for route r = (t, s).  grid (16-feature slabs, routes).
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(32 * kWarps) w4_route_gate_up_kernel(
    const __nv_bfloat16 *x, int hidden, int inter, const int64_t *ids, int top_k, int num_experts,
    const uint8_t *w13, Shape sh, int tiles, float *__restrict__ act) {
  __shared__ __align__(16) float xs[kSegK];
  __shared__ float red[kWarps][32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t route = blockIdx.y;
  const int64_t e = ids[route];
  if (e < 0 || e >= num_experts) return;  // a dropped route
  const int tile = blockIdx.x >> 2;
  const int quarter = blockIdx.x & 3;
  const int blocks = static_cast<int>(w4::blocks_of(hidden));
  const uint8_t *wt = w13 + (e * tiles + tile) * blocks * sh.block_bytes();
  const __nv_bfloat16 *xr = x + route / top_k * hidden;
  float acc[1] = {0.f};
  for (int k0 = 0; k0 < hidden; k0 += kSegK) {
    const int n = min(kSegK, blocks * w4::kBlockK - k0);
    __syncthreads();
    stage_bf16(xs, xr, k0, n, hidden);
    __syncthreads();
    row_dot<1, 8>(wt, sh, quarter * 32 + lane, k0 / 32 + warp, (k0 + n) / 32, kWarps, k0 / 32, xs,
                  0, acc);
  }
  red[warp][lane] = acc[0];
  __syncthreads();
  if (warp == 0) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) v += red[q][lane];
    const float up = __shfl_down_sync(0xffffffffu, v, 16);
    const int f = tile * 64 + quarter * 16 + lane;
    if (lane < 16 && f < inter) act[route * inter + f] = silu_f32(v) * up;
  }
}

// out[t, n] = sum_s weight[t, s] * (W2 act[t, s])[n], in slot order.
// grid (16-row slabs, tokens); warp w takes slots w, w + 8, ...; the halves of
// a warp take the even and the odd chunks.
__global__ void __launch_bounds__(32 * kWarps) w4_route_down_kernel(
    const float *act, int hidden, int inter, const int64_t *ids, const __nv_bfloat16 *weights,
    int top_k, int num_experts, const uint8_t *w2, Shape sh, int tiles,
    __nv_bfloat16 *__restrict__ out) {
  extern __shared__ __align__(16) float down_smem[];  // [top_k][16], then act rows
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t token = blockIdx.y;
  const int blocks = static_cast<int>(w4::blocks_of(inter));
  const int kpad = blocks * w4::kBlockK;
  float *part = down_smem;
  float *xs = down_smem + top_k * 16;
  const int row = (blockIdx.x & 7) * 16 + (lane & 15);
  const int tile = blockIdx.x >> 3;
  // As many act rows at a time as there are warps.
  for (int s0 = 0; s0 < top_k; s0 += kWarps) {
    __syncthreads();
    for (int s = s0; s < min(s0 + kWarps, top_k); ++s)
      stage_f32(xs + (s - s0) * kpad, act + (token * top_k + s) * inter, 0, kpad, inter);
    __syncthreads();
    const int s = s0 + warp;
    if (s < top_k) {
      const int64_t e = ids[token * top_k + s];
      float acc[1] = {0.f};
      const bool live = e >= 0 && e < num_experts;
      if (live) {
        const uint8_t *wt = w2 + (e * tiles + tile) * blocks * sh.block_bytes();
        row_dot<1, 6>(wt, sh, row, lane >> 4, kpad / 32, 2, 0, xs + warp * kpad, 0, acc);
      }
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 16);
      const float wgt = __bfloat162float(weights[token * top_k + s]);
      if (lane < 16) part[s * 16 + lane] = live ? acc[0] * wgt : 0.f;
    }
  }
  __syncthreads();
  if (threadIdx.x < 16) {
    float v = 0.f;
    for (int s = 0; s < top_k; ++s) v += part[s * 16 + threadIdx.x];
    const int f = tile * w4::kTileRows + (blockIdx.x & 7) * 16 + threadIdx.x;
    if (f < hidden) out[token * hidden + f] = __float2bfloat16_rn(v);
  }
}

}  // namespace

int w4_linear_gemv(const void *x, int64_t m, int n, int k, const void *w, const Shape &sh,
                   void *out, cudaStream_t s) {
  const int tiles = (n + w4::kTileRows - 1) / w4::kTileRows;
  const auto *xp = static_cast<const __nv_bfloat16 *>(x);
  const auto *wp = static_cast<const uint8_t *>(w);
  auto *op = static_cast<__nv_bfloat16 *>(out);
#define B200_W4_GEMV(R)                                                                       \
  B200_LAUNCH_PDL(kPdlStream, w4_linear_gemv_kernel<R>,                                       \
                  dim3(4 * tiles, static_cast<unsigned>((m + R - 1) / R)), dim3(32 * kWarps), \
                  0, s, xp, m, n, k, wp, sh, op);
  if (m == 1) {
    B200_W4_GEMV(1)
  } else if (m == 2) {
    B200_W4_GEMV(2)
  } else {
    B200_W4_GEMV(4)
  }
#undef B200_W4_GEMV
  B200_LAUNCHED();
  return B200MOE_OK;
}

int w4_route_experts(const void *x, int64_t tokens, int hidden, int inter, const int64_t *ids,
                     const void *weights, int top_k, int num_experts, const void *w13,
                     const Shape &sh13, const void *w2, const Shape &sh2, float *act, void *out,
                     cudaStream_t s) {
  const int t13 = (inter + 63) / 64;
  const int t2 = (hidden + w4::kTileRows - 1) / w4::kTileRows;
  const int64_t routes = tokens * top_k;
  B200_LAUNCH_PDL(kPdlTiny, w4_route_gate_up_kernel, dim3(4 * t13, static_cast<unsigned>(routes)),
                  dim3(32 * kWarps), 0, s, static_cast<const __nv_bfloat16 *>(x), hidden, inter,
                  ids, top_k, num_experts, static_cast<const uint8_t *>(w13), sh13, t13, act);
  const int rows = top_k < kWarps ? top_k : kWarps;
  const size_t smem = static_cast<size_t>(top_k) * 64 +
                      static_cast<size_t>(rows) * w4::blocks_of(inter) * w4::kBlockK * 4;
  B200_UNSUPPORTED(smem <= 200 * 1024, "intermediate size %d is too large for the routed product",
                   inter);
  if (smem > 48 * 1024)
    B200_CUDA(cudaFuncSetAttribute(w4_route_down_kernel,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(smem)));
  B200_LAUNCH_PDL(kPdlTiny, w4_route_down_kernel, dim3(8 * t2, static_cast<unsigned>(tokens)),
                  dim3(32 * kWarps), smem, s, static_cast<const float *>(act), hidden, inter, ids,
                  static_cast<const __nv_bfloat16 *>(weights), top_k, num_experts,
                  static_cast<const uint8_t *>(w2), sh2, t2, static_cast<__nv_bfloat16 *>(out));
  B200_LAUNCHED();
  return B200MOE_OK;
}

}  // namespace b200moe
