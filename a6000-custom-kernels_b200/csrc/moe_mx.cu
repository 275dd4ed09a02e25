// moe_mx.cu -- MXFP4 kernels (see moe_mx.cuh): quantise, read back, lay out,
// and the grouped product on tcgen05.
#include "moe_aux.h"
#include "moe_mmq.cuh"
#include "moe_mx.cuh"

#include <cuda_bf16.h>

namespace moe {

namespace {

// ---------------------------------------------------------------------------
// One block of 32 values by 4 lanes: lane i holds values 4 i .. 4 i + 3 (v[0..3])
// and 16 + 4 i .. 16 + 4 i + 3 (v[4..7]), so its 4 code bytes pair them as the
// format does. scale byte = max(floor(log2 amax) - 2, -127) + 127, read off
// amax's exponent field; codes are the nearest magnitudes of v 2^-e, ties to the
// even code, saturating at 6 (the scaled values lie below 8). An infinity or a
// NaN makes the block's scale NaN.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], float inv) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %5, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %6, %2;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %7, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %4;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w)
        : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv),
          "f"(v[6] * inv), "f"(v[7] * inv));
    return w;
}

// the 8 magnitudes with signs that 4 code bytes hold: v[0..3] their low
// nibbles, v[4..7] their high ones (unscaled)
__device__ __forceinline__ void mx_values(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
        v[j] = f.x;
        v[4 + j] = f.y;
    }
}

__device__ __forceinline__ float mx_scale(uint32_t byte) {   // 2^(byte - 127); 255: NaN
    return __uint_as_float(byte == 255u ? 0x7FFFFFFFu : byte == 0u ? 0x00400000u : byte << 23);
}

__device__ __forceinline__ uint32_t mx_quant_block(const float (&v)[8], uint32_t &byte) {
    uint32_t top = 0;   // magnitudes compare as integers; a NaN above infinity above every number
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t ex = top >> 23;
    if (ex == 255u) {
        byte = 255u;
        return 0u;
    }
    byte = ex > 2u ? ex - 2u : 0u;
    return mx_codes(v, __uint_as_float((254u - byte) << 23));   // 2^(127 - byte), exact
}

// what the block's codes leave of v (exact: a multiple of v's last place, no larger than v's block)
__device__ __forceinline__ void mx_residual(float (&v)[8], uint32_t codes, uint32_t byte) {
    float q[8];
    mx_values(codes, q);
    const float s = mx_scale(byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] -= q[j] * s;
}

template <int XT> struct MxElem;
template <> struct MxElem<MX_F32> { using T = float; };
template <> struct MxElem<MX_F16> { using T = __half; };
template <> struct MxElem<MX_BF16> { using T = __nv_bfloat16; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// 4 consecutive elements at p (VEC: aligned to their total size)
template <int XT, bool VEC>
__device__ __forceinline__ void mx_load4(const typename MxElem<XT>::T *p, float *v) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_f32(p[j]);
    } else if constexpr (XT == MX_F32) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p));
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
        const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p));
        const typename MxElem<XT>::T *e = reinterpret_cast<const typename MxElem<XT>::T *>(&a);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = to_f32(e[j]);
    }
}

// ---------------------------------------------------------------------------
// quantise into ggml blocks: y [planes][rows][nb] blocks. A CTA makes MXQ_BLK
// consecutive blocks of the rows' concatenation; the 17-byte blocks are put
// together in shared memory and leave as whole words.
// ---------------------------------------------------------------------------
constexpr int MXQ_BLK = 128;                    // blocks per CTA (512 threads, 4 lanes each)
constexpr int MXQ_BYTES = MXQ_BLK * 17;         // a multiple of 16

template <int XT, bool VEC>
__global__ void __launch_bounds__(4 * MXQ_BLK) mx_quantize_kernel(const typename MxElem<XT>::T *__restrict__ x,
                                                                  int64_t stride, int64_t n_blocks, int nb, int planes,
                                                                  uint8_t *__restrict__ y) {
    __shared__ __align__(16) uint8_t buf[MX_MAX_PLANES][MXQ_BYTES];
    const int lb = threadIdx.x >> 2, i = threadIdx.x & 3;
    const int64_t b0 = static_cast<int64_t>(blockIdx.x) * MXQ_BLK;
    const int64_t g = b0 + lb;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (g < n_blocks) {
        const int64_t row = g / nb;
        const typename MxElem<XT>::T *p = x + row * stride + (g - row * nb) * 32 + 4 * i;
        mx_load4<XT, VEC>(p, v);
        mx_load4<XT, VEC>(p + 16, v + 4);
    }
    for (int pl = 0; pl < planes; ++pl) {
        uint32_t byte;
        const uint32_t w = mx_quant_block(v, byte);
        uint8_t *o = buf[pl] + lb * 17;
        if (i == 0) o[0] = static_cast<uint8_t>(byte);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[1 + 4 * i + j] = static_cast<uint8_t>(w >> (8 * j));
        if (pl + 1 < planes) mx_residual(v, w, byte);
    }
    __syncthreads();
    const int64_t left = (n_blocks - b0) * 17;
    const int bytes = left < MXQ_BYTES ? static_cast<int>(left) : MXQ_BYTES;
    for (int pl = 0; pl < planes; ++pl) {
        uint8_t *o = y + pl * n_blocks * 17 + b0 * 17;
        if ((reinterpret_cast<uintptr_t>(o) & 15u) == 0) {
            for (int t = threadIdx.x; t < bytes / 16; t += blockDim.x)
                reinterpret_cast<uint4 *>(o)[t] = reinterpret_cast<const uint4 *>(buf[pl])[t];
            for (int t = (bytes & ~15) + threadIdx.x; t < bytes; t += blockDim.x) o[t] = buf[pl][t];
        } else {
            for (int t = threadIdx.x; t < bytes; t += blockDim.x) o[t] = buf[pl][t];
        }
    }
}

// ---------------------------------------------------------------------------
// read back: out [rows][K] = the planes' values added, rounded once to OT
// ---------------------------------------------------------------------------
template <int OT, bool VEC>
__global__ void __launch_bounds__(4 * MXQ_BLK) mx_dequantize_kernel(const uint8_t *__restrict__ y, int64_t n_blocks,
                                                                    int nb, int planes, int64_t stride,
                                                                    typename MxElem<OT>::T *__restrict__ out) {
    using T = typename MxElem<OT>::T;
    __shared__ __align__(16) uint8_t buf[MX_MAX_PLANES][MXQ_BYTES];
    const int lb = threadIdx.x >> 2, i = threadIdx.x & 3;
    const int64_t b0 = static_cast<int64_t>(blockIdx.x) * MXQ_BLK;
    const int64_t left = (n_blocks - b0) * 17;
    const int bytes = left < MXQ_BYTES ? static_cast<int>(left) : MXQ_BYTES;
    for (int pl = 0; pl < planes; ++pl) {
        const uint8_t *o = y + pl * n_blocks * 17 + b0 * 17;
        if ((reinterpret_cast<uintptr_t>(o) & 15u) == 0) {
            for (int t = threadIdx.x; t < bytes / 16; t += blockDim.x)
                reinterpret_cast<uint4 *>(buf[pl])[t] = __ldg(reinterpret_cast<const uint4 *>(o) + t);
            for (int t = (bytes & ~15) + threadIdx.x; t < bytes; t += blockDim.x) buf[pl][t] = o[t];
        } else {
            for (int t = threadIdx.x; t < bytes; t += blockDim.x) buf[pl][t] = o[t];
        }
    }
    __syncthreads();
    const int64_t g = b0 + lb;
    if (g >= n_blocks) return;
    float v[8];
    for (int pl = 0; pl < planes; ++pl) {
        const uint8_t *o = buf[pl] + lb * 17;
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w |= static_cast<uint32_t>(o[1 + 4 * i + j]) << (8 * j);
        const float s = mx_scale(o[0]);
        float q[8];
        mx_values(w, q);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = pl == 0 ? q[j] * s : v[j] + q[j] * s;
    }
    const int64_t row = g / nb;
    T *p = out + row * stride + (g - row * nb) * 32 + 4 * i;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        T e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (OT == MX_F32) e[j] = v[4 * h + j];
            else if constexpr (OT == MX_F16) e[j] = __float2half_rn(v[4 * h + j]);
            else e[j] = __float2bfloat16_rn(v[4 * h + j]);
        }
        if constexpr (!VEC) {
#pragma unroll
            for (int j = 0; j < 4; ++j) p[16 * h + j] = e[j];
        } else if constexpr (OT == MX_F32) {
            *reinterpret_cast<float4 *>(p + 16 * h) = make_float4(e[0], e[1], e[2], e[3]);
        } else {
            *reinterpret_cast<uint2 *>(p + 16 * h) = *reinterpret_cast<const uint2 *>(e);
        }
    }
}

// ---------------------------------------------------------------------------
// lay out: ggml blocks [E][rows][nb] -> per expert [row tile][K tile] of
// MX_TILE bytes: the codes in the MMA's K-major layout (16-byte chunk c of row
// r at c * 16 * 128 + r * 16: 8-row groups 128 bytes apart, chunks 2 KB), then
// the scales as the tensor memory wants them (block c of row r at
// (r % 32) * 16 + (r / 32) * 4 + c). Rows and blocks past the matrix are zero.
// One thread per block; done once per tensor.
// ---------------------------------------------------------------------------
__global__ void mx_pack_kernel(const uint8_t *__restrict__ src, int rows, int nb, int RT, int KT, int64_t total,
                               uint8_t *__restrict__ dst) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;   // (expert, row, block), padded
    if (i >= total) return;
    const int b = static_cast<int>(i % (KT * 4));
    const int64_t er = i / (KT * 4);
    const int r = static_cast<int>(er % (RT * MX_M));
    const int64_t e = er / (RT * MX_M);
    uint8_t q[16] = {}, s = 0;
    if (r < rows && b < nb) {
        const uint8_t *p = src + ((e * rows + r) * nb + b) * 17;
        s = p[0];
#pragma unroll
        for (int j = 0; j < 16; ++j) q[j] = p[1 + j];
    }
    uint8_t *t = dst + ((e * RT + r / MX_M) * KT + b / 4) * static_cast<int64_t>(MX_TILE);
    const int rr = r % MX_M, c = b % 4;
    *reinterpret_cast<uint4 *>(t + c * (16 * MX_M) + rr * 16) = *reinterpret_cast<const uint4 *>(q);
    t[MX_CODES + (rr % 32) * 16 + (rr / 32) * 4 + c] = s;
}

// ---------------------------------------------------------------------------
// quantise the product's activations: per x row, K tile and plane 64 bytes of
// codes and 4 scale bytes, K padded to whole tiles with zeros
// ---------------------------------------------------------------------------
template <int XT, bool VEC>
__global__ void __launch_bounds__(256) mx_quantize_x_kernel(const typename MxElem<XT>::T *__restrict__ x,
                                                            int64_t stride, int64_t n_rows, int nb, int KT, int planes,
                                                            uint8_t *__restrict__ xq, uint8_t *__restrict__ xs) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t g = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 2;   // (row, block), K padded
    const int i = threadIdx.x & 3;
    const int64_t row = g / (KT * 4);
    const int b = static_cast<int>(g - row * (KT * 4));
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < n_rows && b < nb) {
        const typename MxElem<XT>::T *p = x + row * stride + static_cast<int64_t>(b) * 32 + 4 * i;
        mx_load4<XT, VEC>(p, v);
        mx_load4<XT, VEC>(p + 16, v + 4);
    }
    for (int pl = 0; pl < planes; ++pl) {
        uint32_t byte;
        const uint32_t w = mx_quant_block(v, byte);
        if (row < n_rows) {
            const int64_t at = (row * KT + b / 4) * planes + pl;
            *reinterpret_cast<uint32_t *>(xq + at * 64 + (b % 4) * 16 + 4 * i) = w;
            if (i == 0) xs[at * 4 + b % 4] = static_cast<uint8_t>(byte);
        }
        if (pl + 1 < planes) mx_residual(v, w, byte);
    }
}

// ---------------------------------------------------------------------------
// The grouped product
// ---------------------------------------------------------------------------
constexpr int MXP_THREADS = 192;   // warp 0: weights, warp 1: MMA, warps 2-5: activations, then the epilogue

// Instruction descriptor of kind::mxf4: e2m1 A and B (K-major), UE8M0 scales,
// M = 128, N; `half` picks the pair of scale bytes of the tile's K = 64 half.
__device__ __forceinline__ uint32_t mx_idesc(int N, int half) {
    return (static_cast<uint32_t>(2 * half) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
           (1u << 23) | (static_cast<uint32_t>(MX_M >> 4) << 24) | (static_cast<uint32_t>(2 * half) << 29);
}

__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// 512 scale bytes (32 rows of 16) from shared memory to 4 TMEM columns of all four lane quarters
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint32_t saddr) {
    const uint64_t desc = umma_desc(saddr, 0u, 128u);
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

template <int NT>
struct MxCtl {
    uint64_t a_full[MX_MAX_STAGES], b_full[MX_MAX_STAGES], empty[MX_MAX_STAGES], done;
    uint32_t tmem;
    int32_t abort, expert, count;
    int32_t entry[NT];
};

template <int NT>
__host__ __device__ constexpr uint32_t mx_lbo() { return 16u * NT + 16u; }   // 16 bytes past a power of two: no bank conflicts
template <int NT>
__host__ __device__ constexpr uint32_t mx_b_bytes() { return (4u * mx_lbo<NT>() + MX_SF + 127u) / 128u * 128u; }
template <int NT>
__host__ __device__ constexpr uint32_t mx_stage_bytes(int mats, int planes) {
    return mats * MX_TILE + planes * mx_b_bytes<NT>();
}

template <int NT>
__device__ __forceinline__ bool mx_wait(MxCtl<NT> &C, uint64_t *bar, uint32_t parity, const MxArgs &a) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = clock64(), lim = timeout_cycles(a.timeout_ns);
    for (;;) {
        if (mbar_try_wait_hint(bar, parity, 2000u)) return true;
        if (*reinterpret_cast<volatile int32_t *>(&C.abort)) return false;
        if (static_cast<uint64_t>(clock64()) - t0 > lim) {
            *reinterpret_cast<volatile int32_t *>(&C.abort) = 1;
            set_error(a.err, DERR_TIMEOUT_FULL);
            return false;
        }
    }
}

// One CTA: 128 weight rows (of w, and of gate with GLU) x the up to NT entries
// of one chunk x this cluster rank's share of K.
//   warp 0    one lane streams the weight tiles, one bulk copy each (a tile is
//             contiguous and already in the MMA's layout);
//   warp 1    one lane copies each tile's scales to tensor memory and issues
//             the MMAs, D += A B_plane over the planes;
//   warps 2-5 bring the entries' quantised rows (cp.async, 16-byte chunks),
//             then read the accumulators (thread = weight row) and store.
// With split > 1 the ranks' partial sums meet in shared memory and are added
// in rank order, so results do not depend on timing.
template <int NT, bool GLU, bool DIRECT>
__global__ void __launch_bounds__(MXP_THREADS) mx_product_kernel(const MxArgs a) {
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ MxCtl<NT> C;
    constexpr int MATS = GLU ? 2 : 1;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = a.split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int unit = blockIdx.x / a.split;
    const int rt = unit % a.RT, chunk = unit / a.RT;

    // ids and the chunk table are complete before the launch of the quantiser
    // that this one overlaps with; only the quantised rows wait for its end
    if (!DIRECT) {
        const bool have = chunk < *a.n_chunks;   // (the grid covers the largest possible table)
        if (tid < NT) {
            const int4 ch = have ? a.chunks[chunk] : make_int4(0, 0, 0, 0);
            if (tid == 0) { C.expert = ch.x; C.count = ch.z; }
            if (tid < ch.z) C.entry[tid] = a.entries[ch.y + tid];
        }
    } else if (warp == 0) {
        // entry `chunk` leads a chunk when it is number 0, NT, 2 NT, ... of its expert's entries
        auto id_of = [&](int i) {
            return i < a.n_entries ? a.ids[(i / a.k) * a.ids_stride + i % a.k] : -2;
        };
        const int x0 = id_of(lane), x1 = id_of(lane + 32);
        const int e = __shfl_sync(0xffffffffu, chunk < 32 ? x0 : x1, chunk & 31);
        const uint64_t same = __ballot_sync(0xffffffffu, x0 == e) |
                              (static_cast<uint64_t>(__ballot_sync(0xffffffffu, x1 == e)) << 32);
        const auto before = [&](int i) { return __popcll(same & ((1ull << i) - 1ull)); };
        const int pos = before(chunk);
        const bool ok = e >= 0 && e < a.n_experts;
        const int count = ok && pos % NT == 0 ? min(__popcll(same) - pos, NT) : 0;
        if (!ok && e != -1 && lane == 0) set_error(a.err, DERR_BAD_ID);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = lane + 32 * h, n = before(i) - pos;
            if (((same >> i) & 1ull) && n >= 0 && n < count) C.entry[n] = i;
        }
        if (lane == 0) { C.expert = e; C.count = count; }
    }
    if (tid == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&C.a_full[s], 1);
            mbar_init(&C.b_full[s], 4);
            mbar_init(&C.empty[s], 1);
        }
        mbar_init(&C.done, 1);
        C.abort = 0;
        fence_mbar_init();
    }
    __syncthreads();
    const int count = C.count, expert = C.expert;
    if (count == 0) {   // the same for every rank of the cluster
        asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&C.tmem)),
                     "r"(a.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int kt0 = a.KT * rank / a.split, n_it = a.KT * (rank + 1) / a.split - kt0;
    const int planes = a.planes, stages = a.stages;
    const uint32_t stage_bytes = mx_stage_bytes<NT>(MATS, planes);
    const uint32_t ring0 = smem_u32(ring);

    int fills = 0;   // weight copies issued by this thread
    auto fill = [&](int until) {
        // weights depend on nothing that the launches before write: stream at once
        const uint64_t pol = l2_evict_first_policy();
        const uint64_t at = static_cast<uint64_t>(expert) * a.expert_bytes +
                            (static_cast<uint64_t>(rt) * a.KT + kt0) * MX_TILE;
        for (; fills < until; ++fills) {
            const int i = fills, s = i % stages;
            if (i >= stages && !mx_wait(C, &C.empty[s], ((i / stages) - 1) & 1, a)) return;
            mbar_arrive_expect_tx(&C.a_full[s], MATS * MX_TILE);
            uint8_t *dst = ring + s * stage_bytes;
            bulk_g2s(dst, a.w + at + static_cast<uint64_t>(i) * MX_TILE, MX_TILE, &C.a_full[s], pol);
            if (GLU) bulk_g2s(dst + MX_TILE, a.gate + at + static_cast<uint64_t>(i) * MX_TILE, MX_TILE, &C.a_full[s], pol);
        }
    };
    if (warp == 0 && lane == 0) fill(n_it < stages ? n_it : stages);   // what the ring holds, before anything else
    tc_fence_before();
    __syncthreads();   // the tensor memory's address
    tc_fence_after();
    const uint32_t tmem = C.tmem;
    const int N = (count + 15) / 16 * 16;
    const uint32_t sf0 = tmem + MATS * NT;                                     // scale columns, a slot per stage
    const uint32_t sf_slot = 4u * (MATS + planes);

    if (warp == 0 && lane == 0) {
        fill(n_it);
    } else if (warp == 1 && lane == 0) {
        bool ok = true;
        for (int i = 0; i < n_it && ok; ++i) {
            const int s = i % stages;
            const uint32_t ph = (i / stages) & 1;
            ok = mx_wait(C, &C.a_full[s], ph, a) && mx_wait(C, &C.b_full[s], ph, a);
            if (!ok) break;
            tc_fence_after();
            const uint32_t A = ring0 + s * stage_bytes, B = A + MATS * MX_TILE, sf = sf0 + s * sf_slot;
#pragma unroll
            for (int m = 0; m < MATS; ++m) tmem_cp_scales(sf + 4 * m, A + m * MX_TILE + MX_CODES);
            for (int p = 0; p < planes; ++p) tmem_cp_scales(sf + 4 * (MATS + p), B + p * mx_b_bytes<NT>() + 4 * mx_lbo<NT>());
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t idesc = mx_idesc(N, h);
                for (int p = 0; p < planes; ++p) {
                    const uint64_t bd = umma_desc(B + p * mx_b_bytes<NT>() + 2 * h * mx_lbo<NT>(), mx_lbo<NT>(), 128u);
#pragma unroll
                    for (int m = 0; m < MATS; ++m) {
                        const uint64_t ad = umma_desc(A + m * MX_TILE + 2 * h * (16 * MX_M), 16 * MX_M, 128u);
                        umma_mxf4(tmem + m * NT, ad, bd, idesc, sf + 4 * m, sf + 4 * (MATS + p),
                                  (i | h | p) != 0 ? 1u : 0u);
                    }
                }
            }
            umma_commit(&C.empty[s]);
        }
        umma_commit(&C.done);
    } else if (warp >= 2) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        // the rows' quantised tiles: piece = 16 bytes of codes, planes * 4 pieces per row, then the scale words
        constexpr int LAG = 2;
        const int t = tid - 64, per = 4 * planes;
        auto arrive = [&](int i) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&C.b_full[i % stages]);
        };
        bool ok = true;
        int issued = 0;
        for (int i = 0; i < n_it; ++i) {
            const int s = i % stages;
            if (i >= stages) ok = mx_wait(C, &C.empty[s], ((i / stages) - 1) & 1, a);
            if (!__all_sync(0xffffffffu, ok)) break;
            const uint32_t B = ring0 + s * stage_bytes + MATS * MX_TILE;
            for (int q = t; q < count * per; q += 128) {
                const int j = q / per, c = q - j * per, p = c >> 2;
                const int64_t row = a.per_pick ? C.entry[j] : C.entry[j] / a.k;
                const uint8_t *src = a.xq + ((row * a.KT + kt0 + i) * planes) * 64 + c * 16;
                cp_async16(B + p * mx_b_bytes<NT>() + (c & 3) * mx_lbo<NT>() + (j >> 3) * 128 + (j & 7) * 16, src);
            }
            for (int q = t; q < count * planes; q += 128) {
                const int j = q / planes, p = q - j * planes;
                const int64_t row = a.per_pick ? C.entry[j] : C.entry[j] / a.k;
                cp_async4(B + p * mx_b_bytes<NT>() + 4 * mx_lbo<NT>() + (j & 31) * 16 + (j >> 5) * 4,
                          a.xs + (row * a.KT + kt0 + i) * planes + p);
            }
            cp_async_commit();
            ++issued;
            if (i >= LAG) {
                cp_async_wait<LAG>();
                arrive(i - LAG);
            }
        }
        cp_async_wait<0>();
        for (int i = issued > LAG ? issued - LAG : 0; i < issued; ++i) arrive(i);
    }

    // ---- epilogue ----------------------------------------------------------
    __syncwarp();   // (the lanes that had no role wait here, not at the barrier)
    const bool fine = __all_sync(0xffffffffu, mx_wait(C, &C.done, 0, a) &&
                                                  *reinterpret_cast<volatile int32_t *>(&C.abort) == 0);
    tc_fence_after();
    const int quarter = warp & 3;                 // TMEM lanes this warp may read
    const int r = 32 * quarter + lane;            // weight row of the tile
    const int row = rt * MX_M + r;
    const bool row_ok = row < a.rows;
    const float bu = a.bias && row_ok ? a.bias[static_cast<int64_t>(expert) * a.rows + row] : 0.f;
    const float bg = GLU && a.gate_bias && row_ok ? a.gate_bias[static_cast<int64_t>(expert) * a.rows + row] : 0.f;
    auto finish = [&](int j, float u, float gt) {
        u += bu;
        if (GLU) u = glu_apply(a.glu_op, gt + bg, u, a.glu_limit);
        if (row_ok) a.dst[static_cast<int64_t>(C.entry[j]) * a.rows + row] = u;
    };
    if (warp >= 2 && fine) {
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * quarter) << 16);
        for (int n0 = 0; n0 < N; n0 += 16) {
            uint32_t u[16], gt[16];
            tmem_ld16(lanes + n0, u);
            if (GLU) tmem_ld16(lanes + NT + n0, gt);
            tmem_wait_ld();
            if (a.split == 1) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (n0 + j < count) finish(n0 + j, __uint_as_float(u[j]), GLU ? __uint_as_float(gt[j]) : 0.f);
            } else {
                float *part = reinterpret_cast<float *>(ring);
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    part[(n0 + j) * MX_M + r] = __uint_as_float(u[j]);
                    if (GLU) part[(NT + n0 + j) * MX_M + r] = __uint_as_float(gt[j]);
                }
            }
        }
    }
    if (a.split > 1) {
        cluster_sync();
        if (warp >= 2 && fine) {
            for (int j = rank; j < count; j += a.split) {
                float u = 0.f, gt = 0.f;
                for (int q = 0; q < a.split; ++q) {
                    u += ld_cluster_f32(ring0 + 4 * (j * MX_M + r), q);
                    if (GLU) gt += ld_cluster_f32(ring0 + 4 * ((NT + j) * MX_M + r), q);
                }
                finish(j, u, gt);
            }
        }
        cluster_sync();   // the partial sums stay until every rank has read them
    }
    if (!fine && lane == 0) {
        // a wait ran out: let the weight copies and MMAs in flight end before the memory they use goes
        const uint64_t lim = drain_limit_ns(a.timeout_ns);
        if (warp == 0)
            for (int i = fills > stages ? fills - stages : 0; i < fills; ++i)
                if (!mbar_wait_bounded(&C.a_full[i % stages], (i / stages) & 1, lim)) set_error(a.err, DERR_DRAIN);
        if (warp == 1 && !mbar_wait_bounded(&C.done, 0, lim)) set_error(a.err, DERR_DRAIN);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}


template <int XT>
bool mx_vec_ok(const void *p, int64_t stride) {
    constexpr int64_t need = 4 * sizeof(typename MxElem<XT>::T);
    return reinterpret_cast<uintptr_t>(p) % need == 0 && (stride * static_cast<int64_t>(sizeof(typename MxElem<XT>::T))) % need == 0;
}

template <int XT>
void quantize_t(const void *x, int64_t stride, int64_t n_blocks, int nb, int planes, uint8_t *y, cudaStream_t st) {
    using T = typename MxElem<XT>::T;
    const unsigned grid = static_cast<unsigned>((n_blocks + MXQ_BLK - 1) / MXQ_BLK);
    if (mx_vec_ok<XT>(x, stride))
        mx_quantize_kernel<XT, true><<<grid, 4 * MXQ_BLK, 0, st>>>(static_cast<const T *>(x), stride, n_blocks, nb, planes, y);
    else
        mx_quantize_kernel<XT, false><<<grid, 4 * MXQ_BLK, 0, st>>>(static_cast<const T *>(x), stride, n_blocks, nb, planes, y);
}

template <int OT>
void dequantize_t(const uint8_t *y, int64_t n_blocks, int nb, int planes, void *out, int64_t stride, cudaStream_t st) {
    using T = typename MxElem<OT>::T;
    const unsigned grid = static_cast<unsigned>((n_blocks + MXQ_BLK - 1) / MXQ_BLK);
    if (mx_vec_ok<OT>(out, stride))
        mx_dequantize_kernel<OT, true><<<grid, 4 * MXQ_BLK, 0, st>>>(y, n_blocks, nb, planes, stride, static_cast<T *>(out));
    else
        mx_dequantize_kernel<OT, false><<<grid, 4 * MXQ_BLK, 0, st>>>(y, n_blocks, nb, planes, stride, static_cast<T *>(out));
}

template <int XT>
void quantize_x_t(const void *x, int64_t stride, int64_t n_rows, int nb, int KT, int planes, uint8_t *xq, uint8_t *xs,
                  cudaStream_t st) {
    using T = typename MxElem<XT>::T;
    const unsigned grid = static_cast<unsigned>((n_rows * KT * 16 + 255) / 256);
    if (mx_vec_ok<XT>(x, stride))
        mx_quantize_x_kernel<XT, true><<<grid, 256, 0, st>>>(static_cast<const T *>(x), stride, n_rows, nb, KT, planes, xq, xs);
    else
        mx_quantize_x_kernel<XT, false><<<grid, 256, 0, st>>>(static_cast<const T *>(x), stride, n_rows, nb, KT, planes, xq, xs);
}

constexpr uint32_t kSmemMax = 227u * 1024u;

template <int NT, bool GLU, bool DIRECT>
cudaError_t product_t(MxArgs &a, int64_t units, cudaStream_t st) {
    constexpr int MATS = GLU ? 2 : 1;
    auto kern = mx_product_kernel<NT, GLU, DIRECT>;
    constexpr uint32_t fixed = (sizeof(MxCtl<NT>) + 127u) / 128u * 128u + 1024u;   // static part and the system's 1 KB
    const uint32_t sb = mx_stage_bytes<NT>(MATS, a.planes);
    const int per = (a.KT + a.split - 1) / a.split;
    const uint32_t part = a.split > 1 ? MATS * NT * MX_M * 4u : 0u;
    // two CTAs per SM where their accumulators and scales fit in half the tensor memory each
    uint32_t budget = kSmemMax / 2 - fixed;
    auto cols_of = [&](int stages) {
        const uint32_t need = MATS * NT + stages * 4u * (MATS + a.planes);
        uint32_t c = 32;
        while (c < need) c *= 2;
        return c;
    };
    int stages = static_cast<int>(budget / sb);
    if (stages > per) stages = per;
    if (stages < 2 || cols_of(stages) > 256u) {
        budget = kSmemMax - fixed;
        stages = static_cast<int>(budget / sb);
        if (stages > per) stages = per;
    }
    if (stages > MX_MAX_STAGES) stages = MX_MAX_STAGES;
    while (stages > 1 && cols_of(stages) > 512u) --stages;
    a.stages = stages;
    a.tmem_cols = cols_of(stages);
    // shared memory in proportion to the tensor memory: CTAs that fit an SM together never wait for
    // columns, so ranks of a cluster cannot wait for one another through them
    uint32_t smem = stages * sb > part ? stages * sb : part;
    const uint32_t fair = static_cast<uint32_t>((static_cast<uint64_t>(kSmemMax) * a.tmem_cols + 511) / 512);
    if (smem + fixed < fair) smem = (fair - fixed + 127u) / 128u * 128u;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(kSmemMax - fixed + 1024u));
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(units * a.RT * a.split));
    cfg.blockDim = dim3(MXP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(a.split);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int NT>
cudaError_t product_n(MxArgs &a, bool glu, bool direct, int64_t units, cudaStream_t st) {
    if (glu) return direct ? product_t<NT, true, true>(a, units, st) : product_t<NT, true, false>(a, units, st);
    return direct ? product_t<NT, false, true>(a, units, st) : product_t<NT, false, false>(a, units, st);
}

}  // namespace

cudaError_t launch_mx_quantize(const void *x, int xt, int64_t stride, int64_t n_rows, int64_t n_cols, int planes,
                               uint8_t *y, cudaStream_t st) {
    const int nb = static_cast<int>(n_cols / 32);
    const int64_t n = n_rows * nb;
    if (n == 0) return cudaSuccess;
    if (xt == MX_F32) quantize_t<MX_F32>(x, stride, n, nb, planes, y, st);
    else if (xt == MX_F16) quantize_t<MX_F16>(x, stride, n, nb, planes, y, st);
    else quantize_t<MX_BF16>(x, stride, n, nb, planes, y, st);
    return cudaGetLastError();
}

cudaError_t launch_mx_dequantize(const uint8_t *y, int64_t n_rows, int64_t n_cols, int planes, void *out, int ot,
                                 int64_t stride, cudaStream_t st) {
    const int nb = static_cast<int>(n_cols / 32);
    const int64_t n = n_rows * nb;
    if (n == 0) return cudaSuccess;
    if (ot == MX_F32) dequantize_t<MX_F32>(y, n, nb, planes, out, stride, st);
    else if (ot == MX_F16) dequantize_t<MX_F16>(y, n, nb, planes, out, stride, st);
    else dequantize_t<MX_BF16>(y, n, nb, planes, out, stride, st);
    return cudaGetLastError();
}

cudaError_t launch_mx_pack(const uint8_t *src, int64_t E, int64_t rows, int64_t K, uint8_t *dst, cudaStream_t st) {
    const int RT = static_cast<int>((rows + MX_M - 1) / MX_M), KT = static_cast<int>((K + MX_KT - 1) / MX_KT);
    const int64_t total = E * RT * MX_M * KT * 4;
    if (total == 0) return cudaSuccess;
    mx_pack_kernel<<<static_cast<unsigned>((total + 255) / 256), 256, 0, st>>>(src, static_cast<int>(rows),
                                                                              static_cast<int>(K / 32), RT, KT, total, dst);
    return cudaGetLastError();
}

cudaError_t launch_mx_quantize_x(const void *x, int xt, int64_t stride, int64_t n_rows, int64_t K, int planes,
                                 uint8_t *xq, uint32_t *xs, cudaStream_t st) {
    const int nb = static_cast<int>(K / 32), KT = static_cast<int>((K + MX_KT - 1) / MX_KT);
    uint8_t *s = reinterpret_cast<uint8_t *>(xs);
    if (xt == MX_F32) quantize_x_t<MX_F32>(x, stride, n_rows, nb, KT, planes, xq, s, st);
    else if (xt == MX_F16) quantize_x_t<MX_F16>(x, stride, n_rows, nb, KT, planes, xq, s, st);
    else quantize_x_t<MX_BF16>(x, stride, n_rows, nb, KT, planes, xq, s, st);
    return cudaGetLastError();
}

int mx_chunk_tokens(int64_t n_tok, int64_t k, int64_t n_experts) {
    const int64_t n = n_tok * k;
    if (n <= MX_DIRECT) return n_tok <= 16 ? 16 : 64;
    const int64_t per = n / (n < n_experts ? n : n_experts);   // entries of an expert, on average
    return per <= 12 ? 16 : per <= 48 ? 64 : 128;
}

bool mx_direct(int64_t n_tok, int64_t k) { return n_tok * k <= MX_DIRECT; }

cudaError_t launch_mx_product(MxArgs &a, int NT, int64_t units, cudaStream_t st) {
    const bool glu = a.gate != nullptr, direct = a.chunks == nullptr;
    int split = 1;
    if (NT <= 64)
        while (split < 8 && units * a.RT * split < 296 && a.KT / (2 * split) >= 2) split *= 2;
    a.split = split;
    if (NT == 16) return product_n<16>(a, glu, direct, units, st);
    if (NT == 64) return product_n<64>(a, glu, direct, units, st);
    return glu ? product_t<128, true, false>(a, units, st) : product_t<128, false, false>(a, units, st);
}

}  // namespace moe
