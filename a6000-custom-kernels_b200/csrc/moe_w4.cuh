// moe_w4.cuh -- integer 4-bit matrices with a scale (and a zero) per group of
// consecutive values of a row: value = scale * (code - zero), zero 8 where the
// matrix has none.
//
// Laid out once (w4_pack_kernel) as a warp reads it: [E][RT][KS] stages of 16 rows x 256 values
// (RT = ceil(rows / 16), KS = ceil(K / 256)), each
//   codes   4 tiles of 16 x 64 values, 512 bytes, 16 bytes per lane
//   scales  [groups of the stage][8] words: rows g (low half) and g + 8, 16 bits each
//   zeros   [groups of the stage][4] words: bytes of rows g, g + 8, g + 1, g + 9 (g even)
// Word i of lane 4 g + t feeds MMA i of its tile: the four bits from 4 j + 2 and from 4 j + 18 on (bit 32 is bit 0)
// hold values 32 (i >> 1) + 8 t + 4 (i & 1) + 2 (j >> 1) and + 1 of row g + 8 (j & 1).
// The order of the values along K is the kernel's own: x is read from shared memory in
// the same order, 16 consecutive bytes of a lane for the two MMAs of a half of the tile.
// (A group longer than a stage has its scale in each of them.)
#pragma once
#include "moe_common.cuh"

namespace moe {

constexpr int W4_M = 16;            // rows of a tile
constexpr int W4_KT = 64;           // values of a tile along K
constexpr int W4_TILE = W4_M * W4_KT / 2;
constexpr int W4_KS = 256;          // values of a stage
constexpr int W4_CODES = W4_TILE * W4_KS / W4_KT;
constexpr int W4_DIRECT = 1024;     // picks up to which every CTA groups them by itself
constexpr int W4_MAX_EXPERTS = 1024;
constexpr int W4_MAX_ZERO = 127;

__host__ __device__ constexpr int w4_stage_bytes(int groups, bool zeros) { return W4_CODES + groups * (zeros ? 48 : 32); }

struct W4Args {
    const uint8_t *w[2];             // the product's matrices; with a gate [0] is the gate's and [1] the product's
    const float *bias[2];            // [E][rows] or null, in the same order
    int32_t mats;                    // 1, or 2 with a gate
    int32_t n_experts, rows, K, RT, KS;
    int32_t groups;                  // of a stage: 8, 4, 2 or 1
    int32_t zeros;                   // whether stages hold zeros
    int32_t scale_type, glu_op;      // MX_F16 or MX_BF16
    float glu_limit;
    const void *x;
    int64_t x_stride;                // elements
    int32_t x_type, x_vec;           // MX_*; whether rows may be read 16 bytes at a time
    const uint8_t *staged;           // x in the products' form (w4_stage_kernel), `unit` bytes for 256 values; null: not yet
    int32_t unit;
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
    int32_t split_shift, wk_shift;   // 1 << split_shift CTAs of a cluster, and 1 << wk_shift warps of each, share a row's K
    int32_t wm;                      // row tiles of a block, a CTA's at a time (for experts: at most)
    float deep, per_block;           // a warp's stages for a block, and what a block costs besides (w4_plan)
    int32_t passes, sp;              // K passes of sp stages (of the whole cluster)
    int32_t x_shift;                 // 1 << x_shift warps bring an entry's x
    int32_t dst_vec;                 // whether four rows of dst may be written at once
    int32_t seg;                     // blocks of a run, whose sums are held over passes or for the cluster
    uint32_t x_off, red_off, acc_off, tab_off;
};

}  // namespace moe
