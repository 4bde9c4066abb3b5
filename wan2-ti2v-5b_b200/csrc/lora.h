// Low-rank adapters beside a projection: what lora.cu (the down-projection) hands to the GEMM
// (gemm.cu), which adds the up-projection to its accumulators.
#pragma once

#include "internal.h"

namespace wanb200 {

// The adapters' columns (adapter a, rank index i -> column a * rank + i) are handled in steps of 16,
// the K of one tcgen05.mma, and loaded in chunks of 64, one 128-byte swizzle row.
constexpr int LORA_STEP = 16, LORA_CHUNK = 64, LORA_MAX_COLS = 4096;
constexpr int LORA_RUN = 8;  // ring stages (of 64 K values) of one run of sums beside an fp32 output
constexpr int LORA_F32_PLANES = 3;  // bf16 planes of h beside an fp32 output
constexpr int LORA_MASK_WORDS = LORA_MAX_COLS / LORA_STEP / 32;  // 8 words of step bits per row tile

// Workspace of one call: [row tiles][8] step bits | [row tiles] mixed | h planes.
struct LoraPlan {
  const uint32_t* step_mask;  // steps that some row of the tile uses
  const int* mixed;           // the tile's steps hold columns of an adapter that not all its rows use, or h has planes
  const __nv_bfloat16* h;     // [planes][rows_pad][cols]: scale * (x . down^T) in bf16 planes that add up
  const __nv_bfloat16* up;    // [N][adapters * rank]
  const int32_t* ids;
  int adapters, rank, cols, planes;
  int64_t rows_pad;
  int bn, ksplit, grid;  // the GEMM's tile width, blocks that share a tile's K (a cluster), blocks
};

}  // namespace wanb200
