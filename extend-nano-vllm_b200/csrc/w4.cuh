// 4-bit weights with group scales: the layout that the kernels read, and the
// conversion of codes to operands.
//
//   W[n, k] = scale[n, k / g] * (q[n, k] - zero[n, k / g]),  q in 0..15,
//   g in {32, 64, 128}, zero = 8 where no zero points are given.
//
// A matrix [rows, k] is laid out once as tiles of 128 rows; a tile is a run of
// blocks of 128 k, a block four quarters of 32 rows, and a quarter one
// contiguous piece of memory (what one copy brings):
//   codes  32 rows x 4 units x 16 bytes: word c of unit u holds the eight k
//          32 c + 8 u .. + 7 of a row.  In a warp matrix instruction lane t of a
//          row reads unit t, so that eight lanes read one line; a thread that
//          owns a row reads its four units in turn, and their exchange within the
//          row (code_place) spreads eight such threads over all banks;
//   scales [128 / g][32] of 16 bits (bf16 or fp16), row r at place
//          4 (r % 8) + r / 8 (scale_place): the four rows r, r + 8, r + 16,
//          r + 24 that one lane needs are neighbours;
//   zeros  [128 / g][32] of 8 bits in the same order, only with zero points.
// In each word k = 2 i sits at bit 4 i and k = 2 i + 1 at bit 16 + 4 i:
// (word >> 4 i) & 0x000f000f is a pair of neighbouring k in the halves of a
// register, which is how the matrix instructions want them.  Rows and k beyond
// the matrix have scale 0.
//
// "gate_up" order: a tile holds 64 features of a SwiGLU pair [2 I, k] (gate
// rows first); each quarter of 32 rows is 16 gate rows, then the 16 up rows of
// the same features, so one warp owns both factors of its products.
#pragma once

#include "common.cuh"

namespace b200moe {
namespace w4 {

constexpr int kTileRows = 128;
constexpr int kBlockK = 128;
constexpr int kQuarterRows = 32;
constexpr int kCodeBytes = kQuarterRows * kBlockK / 2;  // 2048 per quarter

struct Shape {
  int group;       // k per scale: 32, 64 or 128
  int has_zero;    // zero points follow the scales
  int half_scale;  // scales are fp16 (else bf16)
  __host__ __device__ int groups_per_block() const { return kBlockK / group; }
  // Within a quarter.
  __host__ __device__ int scale_off() const { return kCodeBytes; }
  __host__ __device__ int zero_off() const { return kCodeBytes + groups_per_block() * 64; }
  __host__ __device__ int quarter_bytes() const {
    return kCodeBytes + groups_per_block() * (has_zero ? 96 : 64);
  }
  __host__ __device__ int block_bytes() const { return 4 * quarter_bytes(); }
};

inline Shape shape_of(int group, int flags) {
  return Shape{group, (flags & B200MOE_W4_ZEROS) != 0, (flags & B200MOE_W4_F16_SCALES) != 0};
}
inline bool group_ok(int group) { return group == 32 || group == 64 || group == 128; }
__host__ __device__ inline int64_t blocks_of(int64_t k) { return (k + kBlockK - 1) / kBlockK; }

// Place of unit u of a quarter's row among its codes, in bytes.
__host__ __device__ __forceinline__ int code_place(int row, int u) {
  return row * 64 + ((u ^ ((row >> 1) & 3)) << 4);
}

// Place of a quarter's row among its scales.
__host__ __device__ __forceinline__ int scale_place(int row) {
  return ((row & 7) << 2) | ((row >> 3) & 3);
}

__device__ __forceinline__ float scale_f32(uint16_t bits, int half_scale) {
  return half_scale ? __half2float(__ushort_as_half(bits))
                    : __uint_as_float(static_cast<uint32_t>(bits) << 16);
}

// (128 + z) in both halves, as bf16 (exact: bf16 has steps of 1 from 128 to 256).
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) { return 0x43004300u | z | (z << 16); }

// Eight codes -> four pairs q - z in bf16.  The code goes into the low bits
// of 128.0 (0x4300), which reads as 128 + q; subtracting 128 + z leaves the
// integer q - z, exact in bf16.
__device__ __forceinline__ void decode8(uint32_t word, uint32_t zpair, uint32_t (&out)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t v;  // (shifted & 0x000f000f) | 0x43004300 in one instruction
    asm("lop3.b32 %0, %1, %2, %3, 0xea;"
        : "=r"(v)
        : "r"(word >> (4 * i)), "r"(0x000f000fu), "r"(0x43004300u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(out[i]) : "r"(v), "r"(zpair));
  }
}

}  // namespace w4
}  // namespace b200moe
