// moe_w4.cuh -- integer 4-bit matrices with a scale (and a zero) per group of
// consecutive values of a row: value = scale * (code - zero), zero 8 where the
// matrix has none.
//
// Laid out once (w4_pack_kernel) as the tensor cores' fragments want them: a tile is
// 16 rows x 64 values, 512 bytes, 16 bytes per lane of a warp. Word i of lane
// 4 g + t feeds MMA i of the tile: bits 4 j..4 j + 3 and 16 + 4 j..16 + 4 j + 3 hold
// values 32 (i >> 1) + 8 t + 4 (i & 1) + 2 (j >> 1) and + 1 of row g + 8 (j & 1). The
// order of the values along K is the kernel's own: x is read from shared memory in
// the same order, 16 consecutive bytes of a lane for the two MMAs of a half of the tile.
//
//   codes   [E][RT][KS][512]              RT = ceil(rows / 16), KS = ceil(K / 64)
//   scales  [E][RT][G][8] words           word g: rows g (low half) and g + 8, 16 bits each
//   zeros   [E][RT][G][4] words           word g / 2: bytes of rows g, g + 8, g + 1, g + 9 (g even)
#pragma once
#include "moe_common.cuh"

namespace moe {

constexpr int W4_M = 16;          // rows of a tile
constexpr int W4_KT = 64;         // values of a tile along K
constexpr int W4_TILE = W4_M * W4_KT / 2;
constexpr int W4_DIRECT = 64;     // picks up to which every CTA groups them by itself
constexpr int W4_MAX_ZERO = 127;  // 128 + zero is exact in bf16

enum : int { W4_F16 = 1, W4_BF16 = 2 };   // types of the scales (as MX_F16, MX_BF16)

struct W4Matrix {
    const uint8_t *codes, *scales, *zeros;   // zeros null: 8
};

struct W4Args {
    W4Matrix w[2];                   // the product's; with a gate [0] is the gate's and [1] the product's
    const float *bias[2];            // [E][rows] or null, in the same order
    int32_t mats;                    // 1, or 2 with a gate
    int32_t n_experts, rows, K, RT, KS, G;
    int32_t gshift;                  // group of 64-value step s: s >> gshift (groups of 32: 2 s and 2 s + 1)
    int32_t scale_type, glu_op;
    float glu_limit;
    const void *x;
    int64_t x_stride;                // elements
    int32_t x_type, x_vec;           // MX_*; whether rows may be read 16 bytes at a time
    int32_t per_pick, k, n_entries;
    const int32_t *ids;              // null: one matrix, every entry's
    int64_t ids_stride;
    const int32_t *entries;          // grouped by launch_mmq_group, null: by the kernel itself
    const int4 *chunks;              // {expert, first entry, count, -}
    const int32_t *n_chunks;
    float *dst;                      // [entry][rows]
    int *err;
    // plan (launch_w4)
    int32_t planes, nc;              // MMA columns of an entry; entries of a chunk
    int32_t wk_shift, tiles;         // 1 << wk_shift warps share a row's K; row blocks of 16 << (3 - wk_shift)
    int32_t passes, sp, seg;         // K passes of sp steps; row blocks whose sums are kept over the passes
    uint32_t x_off, red_off, acc_off;
};

}  // namespace moe
