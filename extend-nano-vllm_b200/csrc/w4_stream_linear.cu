// The dense product of a few rows with 4-bit weights.
#include "w4_stream.cuh"

namespace b200moe {

int w4_linear_stream(const void *x, int64_t m, int n, int k, const void *w, const w4::Shape &sh,
                     void *out, cudaStream_t s) {
  using namespace w4s;
  Args a = {};
  a.w = static_cast<const uint8_t *>(w);
  a.sh = sh;
  a.n_blocks = (n + 127) / 128;
  a.num_kb = static_cast<int>(w4::blocks_of(k));
  a.n_out = n;
  a.k = k;
  a.m = static_cast<int>(m);
  a.x = x;
  a.x_rows = m;
  a.out = out;
  return run<kLinear>(a, 4.0 * a.n_blocks, 4ll * a.n_blocks, m <= 8 ? 8 : 16, s);
}

}  // namespace b200moe
