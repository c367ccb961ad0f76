// The experts' gate/up projection and SwiGLU of a few rows with 4-bit weights.
#include "w4_stream.cuh"

namespace b200moe {

int w4_gate_up_stream(const RowSource &src, int hidden, int inter, const void *w13,
                      const w4::Shape &sh, const int32_t *mtiles, int64_t max_mtiles,
                      const int32_t *counters, double tiles, int cols, void *act,
                      cudaStream_t s) {
  using namespace w4s;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w13);
  a.sh = sh;
  a.n_blocks = (inter + 63) / 64;
  a.num_kb = static_cast<int>(w4::blocks_of(hidden));
  a.n_out = inter;
  a.k = hidden;
  a.gather = src.x_packed == nullptr ? 1 : 0;
  a.x = a.gather ? src.x : src.x_packed;
  a.x_rows = src.x_rows;
  a.mtiles = mtiles;
  a.counters = counters;
  a.max_mtiles = max_mtiles;
  a.row_route = src.row_route;
  a.num_routes = src.num_routes;
  a.top_k = src.top_k;
  a.out = act;
  return run<kGateUp>(a, 4.0 * tiles * a.n_blocks, 4 * max_mtiles * a.n_blocks, cols, s);
}

// Route by route, without packing: act[r] for route r = (t, s), expert ids[r].
int w4_route_gate_up(const void *x, int64_t tokens, int hidden, int inter, const int64_t *ids,
                     int top_k, int num_experts, const void *w13, const w4::Shape &sh, void *act,
                     cudaStream_t s) {
  using namespace w4s;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w13);
  a.sh = sh;
  a.n_blocks = (inter + 63) / 64;
  a.num_kb = static_cast<int>(w4::blocks_of(hidden));
  a.n_out = inter;
  a.k = hidden;
  a.gather = 1;
  a.x = x;
  a.x_rows = tokens;
  a.num_routes = tokens * top_k;
  a.top_k = top_k;
  a.ids = ids;
  a.num_experts = num_experts;
  a.out = act;
  const int64_t items = 4 * a.num_routes * a.n_blocks;
  return run<kGateUp>(a, static_cast<double>(items), items, 8, s);
}

}  // namespace b200moe
