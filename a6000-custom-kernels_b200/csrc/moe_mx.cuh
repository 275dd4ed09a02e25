// moe_mx.cuh -- MXFP4 (microscaled 4-bit floating point) on sm_100a: the
// quantiser and its read-back, the layout of expert matrices for the tensor
// cores, and the grouped product of tokens with the experts they picked.
//
// Format (ggml's block_mxfp4, 17 bytes per 32 values): one power-of-two scale
// 2^(byte - 127) (byte 255: NaN), then 16 bytes of e2m1 codes (magnitudes 0,
// 0.5, 1, 1.5, 2, 3, 4, 6; bit 3 the sign), value j in the low nibble of byte
// j and value j + 16 in its high nibble.
//
// The tensor cores take both operands in this form (tcgen05.mma kind::mxf4:
// e2m1 x e2m1, one scale per 32 values along K, f32 accumulators), so a
// weight never passes through a register: the 16 code bytes of a block are
// one 16-byte chunk of the MMA's shared-memory layout as they are. Within a
// block both operands keep ggml's value order, so each product meets its
// partner whatever order the hardware reads a chunk's nibbles in.
#pragma once
#include "moe_common.cuh"

namespace moe {

constexpr int MX_M = 128;                          // weight rows per tile (TMEM lanes)
constexpr int MX_KT = 128;                         // values along K per tile (4 blocks, two K = 64 MMAs)
constexpr uint32_t MX_CODES = MX_M * MX_KT / 2;    // code bytes of a weight tile
constexpr uint32_t MX_SF = MX_M * MX_KT / 32;      // scale bytes of a tile
constexpr uint32_t MX_TILE = MX_CODES + MX_SF;
constexpr int MX_MAX_PLANES = 2;
constexpr int MX_MAX_STAGES = 16;
constexpr int64_t MX_DIRECT_VALUES = 24 * 1024;    // of a chunk's rows, in the direct form
constexpr int MX_DIRECT = 64;                      // entries up to which the product groups and quantises by itself

enum : int { MX_F32 = 0, MX_F16 = 1, MX_BF16 = 2 };   // element types of x and of the read-back

struct MxArgs {
    const uint8_t *w, *gate;         // laid-out matrices (mx_pack_kernel); gate null: no GLU
    uint64_t expert_bytes;           // RT * KT * MX_TILE
    const float *bias, *gate_bias;   // [E][rows] or null
    int32_t n_experts, rows, RT, KT;
    int32_t glu_op;
    float glu_limit;
    const uint8_t *images;           // quantised rows, per chunk (mx_images_kernel); direct form:
    const void *x;                   // the rows themselves
    int64_t x_stride;
    int32_t x_type, x_vec, nb;       // MX_*, whether groups of 4 values are aligned, blocks of a row
    int32_t planes, k, n_entries, per_pick;
    const int32_t *ids;              // direct form: [tok * ids_stride + pick]
    int64_t ids_stride;
    const int32_t *entries;          // chunked form: entries grouped by expert,
    int2 *where;                     // scratch of the grouping: per entry,
    int4 *experts;                   // and per expert;
    const int4 *chunks;              // {expert, first entry, count, -},
    const int32_t *n_chunks;         // and their number on the device
    float *dst;                      // [entry][rows]
    int32_t split, stages, acc;      // CTAs of a cluster that share K; ring stages; accumulator sets
    uint32_t tmem_cols;
    int *err;
    uint64_t timeout_ns;
};

}  // namespace moe
