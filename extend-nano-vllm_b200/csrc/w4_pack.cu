// Lays 4-bit weights out for the kernels (w4.cuh), once per weight: codes (one
// per byte, [matrices, rows, k]), scales and optional zero points
// [matrices, rows, k / group] -> tiles of 128 rows, blocks of 128 k.
#include "w4.cuh"

namespace b200moe {
namespace {

// One block of the layout per thread block, one row per thread.  A code or zero
// point above 15 has no place in the layout: its low four bits are taken, and the
// status word says that it was there.
__global__ void __launch_bounds__(w4::kTileRows) w4_pack_kernel(
    const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros, int64_t rows, int64_t k,
    w4::Shape sh, int gate_up, uint8_t *out) {
  const int row = threadIdx.x;
  const int64_t kb = blockIdx.x, tile = blockIdx.y, mat = blockIdx.z;
  uint8_t *block = out + ((mat * gridDim.y + tile) * gridDim.x + kb) * sh.block_bytes();
  int64_t src;
  bool valid;
  if (gate_up) {
    const int64_t inter = rows / 2;
    const int64_t f = tile * 64 + (row >> 5) * 16 + (row & 15);
    src = (row & 16) ? inter + f : f;
    valid = f < inter;
  } else {
    src = tile * w4::kTileRows + row;
    valid = src < rows;
  }
  const int64_t groups = k / sh.group;
  const int place = w4::scale_place(row & 31);
  uint8_t *quarter = block + (row >> 5) * sh.quarter_bytes();
  const uint8_t *crow = codes + (mat * rows + src) * k;
  uint32_t word[4][4];  // [unit][chunk of 32 k]
  uint32_t high = 0;    // bits of codes and zero points above the lowest four
#pragma unroll
  for (int c = 0; c < 4; ++c) {
#pragma unroll
    for (int u = 0; u < 4; ++u) word[u][c] = 0u;
    const int64_t k0 = kb * w4::kBlockK + c * 32;
    if (valid && k0 < k) {  // k is a multiple of 32
      uint32_t in[8];
      *reinterpret_cast<uint4 *>(in) = *reinterpret_cast<const uint4 *>(crow + k0);
      *reinterpret_cast<uint4 *>(in + 4) = *reinterpret_cast<const uint4 *>(crow + k0 + 16);
#pragma unroll
      for (int i = 0; i < 8; ++i) high |= in[i] & 0xf0f0f0f0u;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t q = (in[2 * u + i / 4] >> (8 * (i & 3))) & 15u;
          word[u][c] |= q << ((i & 1) * 16 + (i >> 1) * 4);
        }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    *reinterpret_cast<uint4 *>(quarter + w4::code_place(row & 31, u)) =
        make_uint4(word[u][0], word[u][1], word[u][2], word[u][3]);
  for (int g = 0; g < sh.groups_per_block(); ++g) {
    const int64_t gi = kb * sh.groups_per_block() + g;
    const bool in = valid && gi < groups;
    const int64_t at = (mat * rows + src) * groups + gi;
    reinterpret_cast<uint16_t *>(quarter + sh.scale_off())[g * 32 + place] =
        in ? scales[at] : static_cast<uint16_t>(0);
    if (sh.has_zero) {
      const uint32_t z = in ? zeros[at] : 0u;
      high |= z & 0xf0u;
      quarter[sh.zero_off() + g * 32 + place] = static_cast<uint8_t>(z & 15u);
    }
  }
  if (high) atomicOr(&g_status, kStatusIndex);
}

}  // namespace
}  // namespace b200moe

extern "C" {

int64_t b200moe_w4_bytes(int64_t matrices, int64_t rows, int64_t k, int group, int flags) {
  using namespace b200moe;
  if (matrices < 1 || rows < 1 || k < 1 || !w4::group_ok(group) || k % group != 0) return -1;
  if ((flags & B200MOE_W4_GATE_UP) && rows % 2 != 0) return -1;
  const int64_t per_tile = (flags & B200MOE_W4_GATE_UP) ? 64 : 128;
  const int64_t feats = (flags & B200MOE_W4_GATE_UP) ? rows / 2 : rows;
  const int64_t tiles = (feats + per_tile - 1) / per_tile;
  return matrices * tiles * w4::blocks_of(k) * w4::shape_of(group, flags).block_bytes();
}

int b200moe_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros,
                    int64_t matrices, int64_t rows, int64_t k, int group, int flags, void *out,
                    void *stream) {
  using namespace b200moe;
  B200_ARG(matrices >= 1 && rows >= 1 && k >= 1, "bad shape");
  B200_ARG(w4::group_ok(group), "group size %d must be 32, 64 or 128", group);
  B200_ARG(k % group == 0, "k (%lld) must be a multiple of the group size %d", (long long)k, group);
  B200_ARG(!(flags & B200MOE_W4_GATE_UP) || rows % 2 == 0,
           "a gate/up weight has an even number of rows");
  B200_ARG(codes && scales && out, "null pointer argument");
  B200_ARG(((flags & B200MOE_W4_ZEROS) != 0) == (zeros != nullptr),
           "zero points and the zeros flag go together");
  B200_ARG((reinterpret_cast<uintptr_t>(codes) & 15u) == 0 &&
               (reinterpret_cast<uintptr_t>(out) & 15u) == 0,
           "codes and out must be 16-byte aligned");
  const bool gate_up = (flags & B200MOE_W4_GATE_UP) != 0;
  const int64_t feats = gate_up ? rows / 2 : rows;
  const int64_t per_tile = gate_up ? 64 : 128;
  const int64_t tiles = (feats + per_tile - 1) / per_tile;
  B200_UNSUPPORTED(tiles <= 65535 && matrices <= 65535 && w4::blocks_of(k) < (1 << 30),
                   "weight too large");
  w4_pack_kernel<<<dim3(static_cast<unsigned>(w4::blocks_of(k)), static_cast<unsigned>(tiles),
                        static_cast<unsigned>(matrices)),
                   w4::kTileRows, 0, static_cast<cudaStream_t>(stream)>>>(
      codes, static_cast<const uint16_t *>(scales), zeros, rows, k, w4::shape_of(group, flags),
      gate_up ? 1 : 0, static_cast<uint8_t *>(out));
  B200_LAUNCHED();
  return B200MOE_OK;
}

}  // extern "C"
