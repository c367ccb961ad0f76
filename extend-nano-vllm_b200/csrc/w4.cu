// C entry points of the products with 4-bit weights: argument checks, workspace
// layout and the choice of kernel.
#include "w4.cuh"

namespace b200moe {
int w4_linear_gemv(const void *x, int64_t m, int n, int k, const void *w, const w4::Shape &sh,
                   void *out, cudaStream_t s);
int w4_route_experts(const void *x, int64_t tokens, int hidden, int inter, const int64_t *ids,
                     const void *weights, int top_k, int num_experts, const void *w13,
                     const w4::Shape &sh13, const void *w2, const w4::Shape &sh2, float *act,
                     void *out, cudaStream_t s);

namespace {
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const w4::Shape sh = w4::shape_of(group, flags);
  constexpr int64_t kRows = 65535 * 4;
  for (int64_t m0 = 0; m0 < m; m0 += kRows) {
    const int rc = w4_linear_gemv(static_cast<const char *>(x) + m0 * k * 2,
                                  min64(kRows, m - m0), n, k, w, sh,
                                  static_cast<char *>(out) + m0 * n * 2, s);
    if (rc) return rc;
  }
  return B200MOE_OK;
}

int64_t b200moe_w4_experts_workspace(int64_t tokens, int hidden, int inter, int top_k,
                                     int num_experts) {
  if (tokens < 0 || hidden < 1 || inter < 1 || top_k < 1 || num_experts < 1) return -1;
  return tokens * top_k * inter * 4;
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
  B200_ARG(aligned16(x) && aligned16(w13) && aligned16(w2) && aligned16(workspace),
           "x, w13, w2 and workspace must be 16-byte aligned");
  const int64_t need = b200moe_w4_experts_workspace(tokens, hidden, inter, top_k, num_experts);
  B200_ARG(workspace_bytes >= need, "workspace needs %lld bytes", (long long)need);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const w4::Shape sh13 = w4::shape_of(group13, flags13), sh2 = w4::shape_of(group2, flags2);
  const int64_t most = 65535 / top_k;
  B200_UNSUPPORTED(most >= 1, "top_k too large");
  for (int64_t t = 0; t < tokens; t += most) {
    const int rc = w4_route_experts(
        static_cast<const char *>(x) + t * hidden * 2, min64(most, tokens - t), hidden, inter,
        expert_ids + t * top_k, static_cast<const char *>(weights) + t * top_k * 2, top_k,
        num_experts, w13, sh13, w2, sh2, static_cast<float *>(workspace) + t * top_k * inter,
        static_cast<char *>(out) + t * hidden * 2, s);
    if (rc) return rc;
  }
  return B200MOE_OK;
}

}  // extern "C"
