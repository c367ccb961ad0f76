// Scored routing: sigmoid or softmax scores, a selection bias, expert groups,
// top-k, renormalised weights.  One warp routes one token.
//
//   s_e = 1 / (1 + exp(-l_e))  or  exp(l_e - max l) / sum exp(l - max l)
//   c_e = s_e + b_e                                    (what the choice goes by)
//   v_g = max or sum of the two largest c of group g (+inf where the largest is
//         +inf, whatever the other); the topk_groups groups with the largest v
//         stay (lowest index first among equals)
//   ids = the top_k experts with the largest c in them (lowest id first)
//   w   = s_ids / sum(s_ids) * scale                   (the bias is not in it)
//
// Scores, sums and the choice are fp32; the weights are rounded to bf16 once,
// at the end, because the expert kernels take bf16 route weights.  A NaN logit
// counts as -inf, a NaN choice likewise; a row without a finite score has
// weights 0.
//
// One warp a token, because the choice is a chain of top_k rounds and a token's
// scores fit one warp's registers; no two warps ever meet.  What bounds it: at few
// tokens that chain (1 token of 256 experts, 8 groups: 4.6 us on the GPU, 64 of
// 128: 3.2); at many the issue of its instructions.  8192 tokens of 256 experts
// take 16-17 us, of which 1570 instructions a token are 11 us of all schedulers'
// issue (profiled: 70 % of the cycles issue, the integer pipe 73 %); their 8.4 MB
// would take 1.4.
#include "common.cuh"

namespace b200moe {
namespace {

constexpr int kWarps = 4;  // tokens per thread block

struct ScoredArgs {
  const float *bias;
  int64_t num_tokens;
  int num_experts;
  int top_k;
  int sigmoid;
  int groups;
  int topk_groups;
  int group_size;   // num_experts / groups
  int group_lanes;  // largest power of two <= 32 / groups
  uint32_t group_mul;  // expert * group_mul >> 20 is its group
  int group_pad;    // places between groups in shared memory
  int top2;
  int renormalize;
  float scale;
  __nv_bfloat16 *weights;
  int64_t *ids;
};

// Unsigned key in the order of the float (NaN never gets here); > 0 for every
// float, so 0 marks an expert that is taken or not on offer.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 becomes +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename T, int VPL>
__global__ void __launch_bounds__(32 * kWarps) route_scored_kernel(const T *logits,
                                                                   const ScoredArgs a) {
  // With groups: [kWarps] choice values, each group group_pad places after the
  // one before, so that the lanes that look through the groups side by side
  // meet different banks.
  extern __shared__ float s_choice[];
  __shared__ float s_sel[kWarps][32];
  __shared__ int s_id[kWarps][32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  if (token >= a.num_tokens) return;
  const T *row = logits + token * a.num_experts;
  float s[VPL], bias[VPL];
  bool live[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    live[i] = e < a.num_experts;
    const float v = live[i] ? to_f32(row[e]) : -INFINITY;
    bias[i] = live[i] && a.bias ? a.bias[e] : 0.f;
    s[i] = v == v ? v : -INFINITY;
  }
  const int stretch = a.num_experts + a.groups * a.group_pad;
  float *choice = s_choice + warp * stretch;
  if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) s[i] = 1.0f / (1.0f + expf(-s[i]));
  } else {
    float m = s[0];
#pragma unroll
    for (int i = 1; i < VPL; ++i) m = fmaxf(m, s[i]);
    m = warp_max(m);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      // The largest logit itself gives 1 even where it is infinite.
      s[i] = s[i] == m ? (m == -INFINITY ? 0.f : 1.f) : expf(s[i] - m);
      sum += live[i] ? s[i] : 0.f;
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < VPL; ++i) s[i] = sum > 0.f ? s[i] / sum : 0.f;
  }
  uint32_t key[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    float c = live[i] ? s[i] + bias[i] : -INFINITY;
    c = c == c ? c : -INFINITY;
    key[i] = live[i] ? order_key(c) : 0u;
    if (a.groups > 1 && live[i])
      choice[e + static_cast<int>((e * a.group_mul) >> 20) * a.group_pad] = c;
  }
  if (a.groups > 1) {
    // group_lanes lanes look through one group, then merge their two largest.
    __syncwarp();
    const int width = a.group_lanes;
    const int group = lane / width;
    const int size = a.group_size;
    float best = -INFINITY, second = -INFINITY;
    if (group < a.groups) {
      const float *c = choice + group * (size + a.group_pad);
      for (int i = lane % width; i < size; i += width) {
        const float v = c[i];
        second = fmaxf(second, fminf(best, v));
        best = fmaxf(best, v);
      }
    }
    for (int off = width >> 1; off > 0; off >>= 1) {
      const float b = __shfl_xor_sync(0xffffffffu, best, off);
      const float d = __shfl_xor_sync(0xffffffffu, second, off);
      second = fmaxf(fminf(best, b), fmaxf(second, d));
      best = fmaxf(best, b);
    }
    // A choice of +inf (a forced expert) beside others of -inf has no sum: its
    // group counts as +inf.
    const float value = a.top2 && size > 1 && best < INFINITY ? best + second : best;
    // Rank of each group: how many come before it.
    const uint32_t mine = group < a.groups ? order_key(value) : 0u;
    int before = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t other = __shfl_sync(0xffffffffu, mine, g * width);
      before += other > mine || (other == mine && g < group);
    }
    const bool kept = group < a.groups && before < a.topk_groups;
    const unsigned mask = __ballot_sync(0xffffffffu, kept && lane % width == 0);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      if (live[i] && !((mask >> (((e * a.group_mul) >> 20) * width)) & 1u)) key[i] = 0u;
    }
  }
  // top_k rounds: the largest key of the warp; among lanes that hold it, the
  // lowest expert.  Its lane notes the choice and looks for its next best.
  uint32_t bk = 0u;
  int bi = 0;
  float bs = 0.f;
  auto best_of_lane = [&]() {
    bk = 0u;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if (key[i] > bk) {
        bk = key[i];
        bi = i;
        bs = s[i];
      }
    }
  };
  best_of_lane();
  for (int slot = 0; slot < a.top_k; ++slot) {
    const uint32_t kmax = __reduce_max_sync(0xffffffffu, bk);
    const unsigned who = __ballot_sync(0xffffffffu, bk == kmax);
    bool mine = bk == kmax;
    if (who & (who - 1)) {
      const uint32_t id = mine ? static_cast<uint32_t>(lane + 32 * bi) : 0xffffffffu;
      mine = __reduce_min_sync(0xffffffffu, id) == static_cast<uint32_t>(lane + 32 * bi) && mine;
    }
    if (mine) {
      s_sel[warp][slot] = bs;
      s_id[warp][slot] = lane + 32 * bi;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (i == bi) key[i] = 0u;
      best_of_lane();
    }
    __syncwarp();
  }
  const float sel = lane < a.top_k ? s_sel[warp][lane] : 0.f;
  if (lane < a.top_k) {
    const int64_t at = token * a.top_k + lane;
    a.ids[at] = s_id[warp][lane];
  }
  const float total = warp_sum(sel);
  if (lane < a.top_k) {
    const float w = a.renormalize ? (total > 0.f ? sel / total : 0.f) : sel;
    a.weights[token * a.top_k + lane] = __float2bfloat16_rn(w * a.scale);
  }
}

template <typename T>
int launch_scored(const void *logits, const ScoredArgs &a, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((a.num_tokens + kWarps - 1) / kWarps));
  const size_t smem = a.groups > 1 ? static_cast<size_t>(kWarps) * (a.num_experts + a.groups * a.group_pad) * 4
                                    : 0;
  const int vpl = (a.num_experts + 31) / 32;
#define B200_SCORED_CASE(V)                                                                  \
  if (vpl <= V) {                                                                            \
    B200_LAUNCH_PDL(kPdlRoute, route_scored_kernel<T, V>, grid, dim3(32 * kWarps), smem,     \
                    stream, static_cast<const T *>(logits), a);                              \
    B200_LAUNCHED();                                                                         \
    return B200MOE_OK;                                                                       \
  }
  B200_SCORED_CASE(2)
  B200_SCORED_CASE(4)
  B200_SCORED_CASE(8)
  B200_SCORED_CASE(16)
  B200_SCORED_CASE(32)
#undef B200_SCORED_CASE
  set_error("num_experts %d exceeds 1024", a.num_experts);
  return B200MOE_EUNSUPPORTED;
}

}  // namespace
}  // namespace b200moe

extern "C" int b200moe_route_scored_topk(const void *logits, int logits_dtype, int64_t num_tokens,
                                         int num_experts, int top_k, int score, const float *bias,
                                         int num_groups, int topk_groups, int group_score,
                                         int renormalize, float scale, void *weights,
                                         int64_t *expert_ids, void *stream) {
  using namespace b200moe;
  B200_ARG(num_tokens >= 0, "num_tokens must be >= 0");
  B200_ARG(num_experts >= 1, "num_experts must be >= 1");
  B200_ARG(top_k >= 1 && top_k <= num_experts, "top_k must be between 1 and num_experts");
  B200_ARG(score == B200MOE_SCORE_SOFTMAX || score == B200MOE_SCORE_SIGMOID,
           "unknown score function code %d", score);
  B200_ARG(group_score == B200MOE_GROUP_MAX || group_score == B200MOE_GROUP_TOP2,
           "unknown group score code %d", group_score);
  B200_ARG(num_groups >= 1 && num_experts % num_groups == 0,
           "num_groups must divide the number of experts");
  B200_ARG(topk_groups >= 1 && topk_groups <= num_groups,
           "topk_groups must be between 1 and num_groups");
  B200_ARG(top_k <= topk_groups * (num_experts / num_groups),
           "top_k exceeds the experts of topk_groups groups");
  B200_UNSUPPORTED(top_k <= 32, "top_k %d > 32 is not supported", top_k);
  B200_UNSUPPORTED(num_experts <= 1024, "num_experts %d > 1024 is not supported", num_experts);
  B200_UNSUPPORTED(num_groups <= 32, "num_groups %d > 32 is not supported", num_groups);
  B200_UNSUPPORTED(num_tokens < (1ll << 32), "too many tokens");
  B200_ARG(logits_dtype == B200MOE_F32 || logits_dtype == B200MOE_BF16 ||
               logits_dtype == B200MOE_F16,
           "unsupported logits dtype code %d", logits_dtype);
  if (num_tokens == 0) return B200MOE_OK;
  B200_ARG(logits && weights && expert_ids, "null pointer argument");
  ScoredArgs a;
  a.bias = bias;
  a.num_tokens = num_tokens;
  a.num_experts = num_experts;
  a.top_k = top_k;
  a.sigmoid = score == B200MOE_SCORE_SIGMOID;
  a.groups = num_groups;
  a.topk_groups = topk_groups;
  a.group_size = num_experts / num_groups;
  a.group_lanes = 32;
  while (a.group_lanes * num_groups > 32) a.group_lanes >>= 1;
  // Exact for e * group_size < 2^20.
  a.group_mul = (1u << 20) / static_cast<uint32_t>(a.group_size) + 1u;
  a.group_pad = ((a.group_lanes - a.group_size) % 32 + 32) % 32;
  a.top2 = group_score == B200MOE_GROUP_TOP2;
  a.renormalize = renormalize;
  a.scale = scale;
  a.weights = static_cast<__nv_bfloat16 *>(weights);
  a.ids = expert_ids;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (logits_dtype) {
    case B200MOE_F32: return launch_scored<float>(logits, a, s);
    case B200MOE_BF16: return launch_scored<__nv_bfloat16>(logits, a, s);
    default: return launch_scored<__half>(logits, a, s);
  }
}
