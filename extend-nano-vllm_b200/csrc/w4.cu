// C entry points of the products with 4-bit weights: argument checks, workspace
// layout and the choice of kernel.
#include <math.h>

#include "w4.cuh"

namespace b200moe {
int w4_linear_stream(const void *x, int64_t m, int n, int k, const void *w, const w4::Shape &sh,
                     void *out, cudaStream_t s);
int w4_gate_up_stream(const RowSource &src, int hidden, int inter, const void *w13,
                      const w4::Shape &sh, const int32_t *mtiles, int64_t max_mtiles,
                      const int32_t *counters, double tiles, int cols, void *act,
                      cudaStream_t s);
int w4_down_stream(const void *act, int hidden, int inter, const void *w2, const w4::Shape &sh,
                   const int32_t *row_route, const void *route_weights, int64_t num_routes,
                   const int32_t *mtiles, int64_t max_mtiles, const int32_t *counters,
                   double tiles, int cols, float *y, cudaStream_t s);
int w4_route_gate_up(const void *x, int64_t tokens, int hidden, int inter, const int64_t *ids,
                     int top_k, int num_experts, const void *w13, const w4::Shape &sh, void *act,
                     cudaStream_t s);
int w4_route_down(const void *act, int64_t tokens, int hidden, int inter, const int64_t *ids,
                  const void *weights, int top_k, int num_experts, const void *w2,
                  const w4::Shape &sh2, void *out, cudaStream_t s);
int w4_linear_tc(const void *x, int64_t m, int n, int k, const void *w, const w4::Shape &sh,
                 void *out, cudaStream_t s);
int w4_gate_up_tc(const RowSource &src, int hidden, int inter, const void *w13,
                  const w4::Shape &sh, int64_t row_capacity, const int32_t *mtiles,
                  int64_t max_mtiles, const int32_t *counters, double tiles, int64_t rows,
                  void *act, cudaStream_t s);
int w4_down_tc(const void *act, int hidden, int inter, const void *w2, const w4::Shape &sh,
               const int32_t *row_route, const void *route_weights, int64_t num_routes,
               int64_t row_capacity, const int32_t *mtiles, int64_t max_mtiles,
               const int32_t *counters, double tiles, int64_t rows, float *y, cudaStream_t s);

namespace {
bool aligned(const void *p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(bytes - 1)) == 0;
}
bool aligned16(const void *p) { return aligned(p, 16); }

// Rows of x up to which the weights of a dense product are streamed
// (w4_stream.cuh); with more, tcgen05 (w4_gemm_sm100.cu).
constexpr int64_t kStreamRows = 16;

// The same for experts, from the rows that an expert has on average.  A streamed
// expert is passed over once per eight rows (or sixteen, stream_cols), a tile of
// tcgen05 costs the same for one row as for many.  Small experts with small groups
// have the dearest passes.  Measured, the whole call in us, streamed against tcgen05:
//   128 experts of 768 x 2048, top-8, 64 / 80 / 96 / 112 tokens (4 / 5 / 6 / 7 rows):
//     g 128  110 142 154 175 against 176 154 161 164
//     g 64   121 157 173 194 against 170 152 160 169
//     g 32   144 186 208 231 against 181 167 175 186
//   16 experts of 6400 x 4096, top-4, 24 tokens (6 rows): g 128, 64, 32
//     202 232 287 against 327 332 358
bool stream_experts(int64_t tokens, double mean, int inter, const w4::Shape &sh13,
                    const w4::Shape &sh2) {
  if (tokens <= kStreamRows) return true;
  const bool large_groups = sh13.groups_per_block() == 1 && sh2.groups_per_block() == 1;
  return mean <= (large_groups || inter >= 2048 ? 6.0 : 4.5);
}

// Rows that a pass over a streamed expert takes.  Measured with 8 and with 16: 64
// tokens through 128 experts of 768 x 2048 (4 rows) 115 and 118 us, 16 tokens
// through 16 of 6400 x 4096 (4 rows) 181 and 239, through 8 of 14336 x 4096, top-8
// (16 rows) 349 and 264.
int stream_cols(int64_t tokens, double mean) { return tokens <= 8 || mean <= 6.0 ? 8 : 16; }

// Routes up to which the experts run route by route, without packing.
constexpr int64_t kRouteRoutes = 16;
// Routes up to which the gate/up product gathers its rows in its own loads
// instead of reading a packed copy.
constexpr int64_t kGatherRoutes = 512;

// Rows of the tiles that an expert product is cut into, from the rows to expect
// of a fuller expert (`rows`: half as many again as the mean, and eight).  A tile
// that is too small costs passes over the weights, one that is too large costs
// time only by the hand-over of each group's accumulators, so that large groups
// want large tiles.  Measured with 128 experts, top-8, the whole call in us with
// tiles of 32 / 64 / 128 rows:
//   g 128: 64 tokens 165 / 177 / 171, 96 162 / 168 / 160, 256 207 / 197 / 175,
//          509 276 / 225 / 197
//   g 64:  96 tokens 161 / 190 / 188, 192 196 / 199 / 196, 256 214 / 217 / 203,
//          509 288 / 256 / 229
//   g 32:  96 tokens 177 / 240 / 281, 384 282 / 307 / 331, 509 323 / 317 / 346,
//          768 438 / 388 / 377
int64_t tile_rows(int64_t rows, const w4::Shape &sh) {
  switch (sh.groups_per_block()) {
    case 1: return 128;
    case 2: return rows <= 26 ? 32 : 128;
    default: return rows <= 50 ? 32 : rows <= 64 ? 64 : 128;
  }
}

// Pieces of the workspace, each on a 256-byte boundary.
struct Workspace {
  int64_t bytes = 0;
  char *base = nullptr;
  template <typename T>
  T *take(int64_t count) {
    T *p = reinterpret_cast<T *>(base + bytes);
    bytes += (count * static_cast<int64_t>(sizeof(T)) + 255) / 256 * 256;
    return p;
  }
};

// Packing in one block: routes and experts it takes.
constexpr int64_t kPackRoutes = 8192;
constexpr int kPackExperts = 4096;

struct ExpertBuffers {
  int64_t row_capacity = 0, max_mtiles = 0, scratch_bytes = 0;
  int32_t *row_route = nullptr, *route_row = nullptr, *combine_rows = nullptr,
          *tile_expert = nullptr, *offsets = nullptr, *counts = nullptr, *mtiles = nullptr,
          *counters = nullptr, *scratch = nullptr;
  __nv_bfloat16 *x_packed = nullptr;  // above kGatherRoutes routes
  // [row_capacity, inter], packed order (few routes: route order).  bf16, the type
  // of the down product's operand: the call's error against 64 bits is 0.0023 of
  // the result with it and would be 0.0017 (the last store's) without; the bf16
  // experts round here too.
  __nv_bfloat16 *act = nullptr;
  // [routes, hidden], route order.  fp32: in bf16 the rows would be half of the
  // traffic (8192 tokens, top-8, 2048 wide: 537 MB written and read) and the error 0.0029.
  float *y = nullptr;
};

ExpertBuffers expert_buffers(Workspace &ws, int64_t tokens, int hidden, int inter, int top_k,
                             int num_experts) {
  ExpertBuffers b;
  const int64_t routes = tokens * top_k;
  if (routes <= kRouteRoutes) {
    b.act = ws.take<__nv_bfloat16>(routes * inter);
    return b;
  }
  b.row_capacity = b200moe_pack_row_capacity(routes, num_experts);
  b.max_mtiles = b200moe_pack_max_mtiles(routes, num_experts);
  b.scratch_bytes = static_cast<int64_t>(b200moe_pack_scratch_bytes(routes, num_experts));
  b.row_route = ws.take<int32_t>(b.row_capacity);
  b.mtiles = ws.take<int32_t>(b.max_mtiles * B200MOE_MTILE_WORDS);
  b.counters = ws.take<int32_t>(B200MOE_NUM_COUNTERS);
  if (routes > kPackRoutes || num_experts > kPackExperts) {
    b.route_row = ws.take<int32_t>(routes);
    b.combine_rows = ws.take<int32_t>(routes);
    b.tile_expert = ws.take<int32_t>(b.row_capacity / B200MOE_BLOCK_ROWS);
    b.offsets = ws.take<int32_t>(num_experts + 1);
    b.counts = ws.take<int32_t>(num_experts);
    b.scratch = ws.take<int32_t>(b.scratch_bytes / 4);
  }
  if (routes > kGatherRoutes) b.x_packed = ws.take<__nv_bfloat16>(b.row_capacity * hidden);
  b.act = ws.take<__nv_bfloat16>(b.row_capacity * inter);
  b.y = ws.take<float>(routes * hidden);
  return b;
}

// Packing for up to kPackRoutes routes in one block: rows by expert, every
// expert's rows on a 16-row boundary, row tiles of 128.  The place of a route
// among its expert's rows is whichever came first: a row's product does not
// depend on its place, so results are the same whatever the order.
constexpr int kPackThreads = 1024;

__global__ void __launch_bounds__(kPackThreads) w4_pack_routes_kernel(
    const int64_t *ids, int num_routes, int num_experts, int32_t *row_route, int32_t *mtiles,
    int32_t *counters) {
  extern __shared__ int32_t pack_smem[];  // count[E], first row[E]
  __shared__ int32_t warp_rows[32], warp_tiles[32];
  pdl_trigger();
  pdl_wait();
  int32_t *count = pack_smem, *row0 = count + num_experts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int e = tid; e < num_experts; e += kPackThreads) count[e] = 0;
  __syncthreads();
  constexpr int kMost = kPackRoutes / kPackThreads;
  int expert[kMost], place[kMost];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int r = tid + i * kPackThreads;
    expert[i] = -1;
    if (r < num_routes) {
      const int64_t e = ids[r];
      if (e >= 0 && e < num_experts) {
        expert[i] = static_cast<int>(e);
        place[i] = atomicAdd(&count[e], 1);
      }
    }
  }
  __syncthreads();
  // Rows and tiles before each expert; thread t takes `per` experts in a row.
  const int per = (num_experts + kPackThreads - 1) / kPackThreads;
  int rows = 0, tiles = 0;
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e < num_experts) {
      rows += (count[e] + 15) & ~15;
      tiles += (count[e] + B200MOE_MTILE_ROWS - 1) / B200MOE_MTILE_ROWS;
    }
  }
  int rows_in = rows, tiles_in = tiles;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int r = __shfl_up_sync(0xffffffffu, rows_in, off);
    const int t = __shfl_up_sync(0xffffffffu, tiles_in, off);
    if (lane >= off) {
      rows_in += r;
      tiles_in += t;
    }
  }
  if (lane == 31) {
    warp_rows[warp] = rows_in;
    warp_tiles[warp] = tiles_in;
  }
  __syncthreads();
  int row = rows_in - rows, tile = tiles_in - tiles;
  for (int w = 0; w < warp; ++w) {
    row += warp_rows[w];
    tile += warp_tiles[w];
  }
  if (tid == kPackThreads - 1) {
    counters[B200MOE_CNT_PADDED_ROWS] = row + rows;
    counters[B200MOE_CNT_MTILES] = tile + tiles;
  }
  for (int i = 0; i < per; ++i) {
    const int e = tid * per + i;
    if (e < num_experts) {
      const int n = count[e];
      row0[e] = row;
      for (int r = 0; r < n; r += B200MOE_MTILE_ROWS, ++tile) {
        mtiles[tile * B200MOE_MTILE_WORDS + 0] = e;
        mtiles[tile * B200MOE_MTILE_WORDS + 1] = row + r;
        mtiles[tile * B200MOE_MTILE_WORDS + 2] = row + min(n, r + B200MOE_MTILE_ROWS);
      }
      // The rows that fill an expert's last sixteen belong to no route.
      for (int r = n; r < ((n + 15) & ~15); ++r) row_route[row + r] = num_routes;
      row += (n + 15) & ~15;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMost; ++i)
    if (expert[i] >= 0) row_route[row0[expert[i]] + place[i]] = tid + i * kPackThreads;
}

// out[t, :] = sum over slots, in slot order, of the fp32 route rows y (rows of
// routes whose id is no expert are not read).  One thread per 4 columns; B slots'
// ids and rows are in flight together: eight where few tokens leave the machine
// waiting, four where many fill it (8192 tokens: 91 us against 141).
template <int B>
__global__ void __launch_bounds__(256) w4_combine_kernel(const float *y, const int64_t *ids,
                                                         int num_experts, int64_t tokens,
                                                         int top_k, int hidden,
                                                         __nv_bfloat16 *__restrict__ out) {
  pdl_trigger();
  pdl_wait();
  const int vecs = hidden / 4;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t token = idx / vecs;
  const int col = static_cast<int>(idx - token * vecs) * 4;
  if (token >= tokens) return;
  const float *row = y + token * top_k * hidden + col;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < top_k; s0 += B) {
    bool live[B];
    float4 v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const int64_t id = s0 + j < top_k ? ids[token * top_k + s0 + j] : -1;
      live[j] = id >= 0 && id < num_experts;
    }
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (live[j])
        v[j] = *reinterpret_cast<const float4 *>(row + (s0 + j) * static_cast<int64_t>(hidden));
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (live[j]) {
        acc.x += v[j].x;
        acc.y += v[j].y;
        acc.z += v[j].z;
        acc.w += v[j].w;
      }
  }
  uint2 o;
  __nv_bfloat162 *op = reinterpret_cast<__nv_bfloat162 *>(&o);
  op[0] = __floats2bfloat162_rn(acc.x, acc.y);
  op[1] = __floats2bfloat162_rn(acc.z, acc.w);
  *reinterpret_cast<uint2 *>(out + token * hidden + col) = o;
}

}  // namespace
}  // namespace b200moe

extern "C" {

int b200moe_w4_linear(const void *x, int64_t m, int n, int k, const void *w, int group, int flags,
                      void *out, void *stream) {
  using namespace b200moe;
  B200_ARG(m >= 0 && n >= 1 && k >= 1, "bad shape");
  B200_ARG(w4::group_ok(group), "group size %d must be 32, 64 or 128", group);
  B200_ARG(k % group == 0, "k (%d) must be a multiple of the group size %d", k, group);
  B200_ARG(!(flags & B200MOE_W4_GATE_UP), "the dense product takes plain row order");
  if (m == 0) return B200MOE_OK;
  B200_ARG(x && w && out, "null pointer argument");
  B200_ARG(aligned16(x) && aligned16(w), "x and w must be 16-byte aligned");
  B200_ARG(aligned(out, 2), "out must be aligned to its type");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const w4::Shape sh = w4::shape_of(group, flags);
  B200_UNSUPPORTED(m < (int64_t)0x7fffffff &&
                       (m + 15) / 16 * ((n + 127) / 128) < (int64_t)0x7fffffff,
                   "too many rows");
  return m <= kStreamRows ? w4_linear_stream(x, m, n, k, w, sh, out, s)
                          : w4_linear_tc(x, m, n, k, w, sh, out, s);
}

int64_t b200moe_w4_experts_workspace(int64_t tokens, int hidden, int inter, int top_k,
                                     int num_experts) {
  if (tokens < 0 || hidden < 1 || inter < 1 || top_k < 1 || num_experts < 1) return -1;
  b200moe::Workspace ws;
  b200moe::expert_buffers(ws, tokens, hidden, inter, top_k, num_experts);
  return ws.bytes;
}

int b200moe_w4_experts_launches(int64_t tokens, int top_k, int num_experts) {
  using namespace b200moe;
  const int64_t routes = tokens * top_k;
  if (routes <= 0) return 0;
  if (routes <= kRouteRoutes) return 2;
  return (routes <= kPackRoutes && num_experts <= kPackExperts ? 1 : 2) +
         (routes > kGatherRoutes ? 1 : 0) + 3;
}

int b200moe_w4_experts(const void *x, int64_t tokens, int hidden, int inter,
                       const int64_t *expert_ids, const void *weights, int top_k, int num_experts,
                       const void *w13, int group13, int flags13, const void *w2, int group2,
                       int flags2, void *workspace, int64_t workspace_bytes, void *out,
                       void *stream) {
  using namespace b200moe;
  B200_ARG(tokens >= 0 && hidden >= 1 && inter >= 1, "bad shape");
  B200_ARG(top_k >= 1 && num_experts >= 1, "top_k and num_experts must be >= 1");
  B200_ARG(w4::group_ok(group13) && w4::group_ok(group2),
           "group sizes %d and %d must be 32, 64 or 128", group13, group2);
  B200_ARG(hidden % group13 == 0 && inter % group2 == 0,
           "hidden (%d) and intermediate (%d) sizes must be multiples of the group sizes", hidden,
           inter);
  B200_ARG((flags13 & B200MOE_W4_GATE_UP) && !(flags2 & B200MOE_W4_GATE_UP),
           "w13 needs the gate_up row order and w2 plain rows");
  B200_ARG(tokens < (int64_t)0x7fffffff / top_k, "too many routes");
  if (tokens == 0) return B200MOE_OK;
  B200_ARG(x && expert_ids && weights && w13 && w2 && workspace && out, "null pointer argument");
  B200_ARG(aligned16(x) && aligned16(w13) && aligned16(w2) && aligned16(workspace) &&
               aligned16(out),
           "x, w13, w2, workspace and out must be 16-byte aligned");
  B200_ARG(aligned(expert_ids, 8) && aligned(weights, 2),
           "expert_ids and weights must be aligned to their types");
  const int64_t need = b200moe_w4_experts_workspace(tokens, hidden, inter, top_k, num_experts);
  B200_ARG(workspace_bytes >= need, "workspace needs %lld bytes", (long long)need);
  // Work items are counted in 32 bits.
  B200_UNSUPPORTED(b200moe_pack_max_mtiles(tokens * top_k, num_experts) * 4 *
                           ((hidden > inter ? hidden : inter) / 64 + 1) <
                       (int64_t)0x7fffffff,
                   "too many routes");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const w4::Shape sh13 = w4::shape_of(group13, flags13), sh2 = w4::shape_of(group2, flags2);
  const int64_t routes = tokens * top_k;
  Workspace ws;
  ws.base = static_cast<char *>(workspace);
  const ExpertBuffers b = expert_buffers(ws, tokens, hidden, inter, top_k, num_experts);
  int rc;
  if (routes <= kRouteRoutes) {
    rc = w4_route_gate_up(x, tokens, hidden, inter, expert_ids, top_k, num_experts, w13, sh13,
                          b.act, s);
    return rc ? rc
              : w4_route_down(b.act, tokens, hidden, inter, expert_ids, weights, top_k,
                              num_experts, w2, sh2, out, s);
  }
  if (b.scratch == nullptr) {
    const size_t smem = static_cast<size_t>(num_experts) * 8;  // 32 KB at most
    B200_LAUNCH_PDL(kPdlPack, w4_pack_routes_kernel, dim3(1), dim3(kPackThreads), smem, s,
                    expert_ids, static_cast<int>(routes), num_experts, b.row_route, b.mtiles,
                    b.counters);
    B200_LAUNCHED();
  } else {
    // Without a capacity the packing call writes neither ids nor weights.
    rc = b200moe_pack_routes(const_cast<int64_t *>(expert_ids), nullptr, routes, num_experts,
                             nullptr, 0, num_experts, nullptr, -1, b.row_capacity, b.row_route,
                             b.route_row, b.combine_rows, b.tile_expert, b.offsets, b.counts,
                             b.mtiles, b.max_mtiles, nullptr, b.counters, nullptr, b.scratch,
                             static_cast<size_t>(b.scratch_bytes), stream);
    if (rc) return rc;
  }
  RowSource src = {};
  src.x = x;
  src.x_rows = tokens;
  src.x_packed = b.x_packed;
  src.row_route = b.row_route;
  src.top_k = top_k;
  src.num_routes = routes;
  if (b.x_packed) {
    rc = b200moe_gather_rows(x, tokens, hidden, b.row_route, nullptr, top_k, routes,
                             b.row_capacity, b.counters, b.x_packed, stream);
    if (rc) return rc;
  }
  // Row tiles to expect when routes fall evenly, and rows of a full one.
  const double mean = static_cast<double>(routes) / num_experts;
  const double tiles = num_experts * (1.0 - exp(-mean)) + static_cast<double>(routes) / 128;
  const int64_t rows = min64(tokens, static_cast<int64_t>(1.5 * mean + 8.0));
  const bool stream_w = stream_experts(tokens, mean, inter, sh13, sh2);
  const int cols = stream_cols(tokens, mean);
  rc = stream_w ? w4_gate_up_stream(src, hidden, inter, w13, sh13, b.mtiles, b.max_mtiles,
                                    b.counters, tiles, cols, b.act, s)
                : w4_gate_up_tc(src, hidden, inter, w13, sh13, b.row_capacity, b.mtiles,
                                b.max_mtiles, b.counters, tiles,
                                min64(tokens, tile_rows(rows, sh13)), b.act, s);
  if (rc) return rc;
  rc = stream_w ? w4_down_stream(b.act, hidden, inter, w2, sh2, b.row_route, weights, routes,
                                b.mtiles, b.max_mtiles, b.counters, tiles, cols, b.y, s)
               : w4_down_tc(b.act, hidden, inter, w2, sh2, b.row_route, weights, routes,
                            b.row_capacity, b.mtiles, b.max_mtiles, b.counters, tiles,
                            min64(tokens, tile_rows(rows, sh2)), b.y, s);
  if (rc) return rc;
  const int64_t threads = tokens * (hidden / 4);
  B200_LAUNCH_PDL(kPdlCombine, tokens <= 256 ? w4_combine_kernel<8> : w4_combine_kernel<4>,
                  dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, s, b.y, expert_ids,
                  num_experts, tokens, top_k, hidden, static_cast<__nv_bfloat16 *>(out));
  B200_LAUNCHED();
  return B200MOE_OK;
}

}  // extern "C"
