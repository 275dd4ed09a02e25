// moe_mx.cu -- MXFP4 kernels (see moe_mx.cuh): quantise, read back, lay out,
// and the grouped product on tcgen05.
#include "moe_aux.h"
#include "moe_mmq.cuh"
#include "moe_mx.cuh"

#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>

namespace moe {

namespace {

// ---------------------------------------------------------------------------
// One block of 32 values by 4 lanes: lane i holds values 4 i .. 4 i + 3 and
// 16 + 4 i .. 16 + 4 i + 3, the pairs that share its 4 code bytes.
// scale byte = max(floor(log2 amax) - 2, -127) + 127, read off amax's exponent
// field; codes are the nearest magnitudes of v 2^-e, ties to the even code,
// saturating at 6 (the scaled values lie below 8). An infinity or a NaN makes
// the block's scale NaN.
// ---------------------------------------------------------------------------
template <int XT> struct MxElem;
template <> struct MxElem<MX_F32> { using T = float; };
template <> struct MxElem<MX_F16> { using T = __half; };
template <> struct MxElem<MX_BF16> { using T = __nv_bfloat16; };

// a lane's 8 values of the block at p (VEC: groups of 4 aligned to their size), as loaded
template <int XT> struct MxRaw { uint32_t w[XT == MX_F32 ? 8 : 4]; };
template <int XT, bool VEC>
__device__ __forceinline__ MxRaw<XT> mx_load(const typename MxElem<XT>::T *p, int i) {
    MxRaw<XT> r;
    p += 4 * i;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (XT == MX_F32 && VEC) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p + 16 * h));
            r.w[4 * h] = a.x; r.w[4 * h + 1] = a.y; r.w[4 * h + 2] = a.z; r.w[4 * h + 3] = a.w;
        } else if constexpr (XT == MX_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * h + j] = reinterpret_cast<const uint32_t *>(p + 16 * h)[j];
        } else if constexpr (VEC) {
            const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p + 16 * h));
            r.w[2 * h] = a.x; r.w[2 * h + 1] = a.y;
        } else {
            const uint16_t *q = reinterpret_cast<const uint16_t *>(p + 16 * h);
            r.w[2 * h] = q[0] | static_cast<uint32_t>(q[1]) << 16;
            r.w[2 * h + 1] = q[2] | static_cast<uint32_t>(q[3]) << 16;
        }
    }
    return r;
}
template <int XT>
__device__ __forceinline__ MxRaw<XT> mx_zero() {
    MxRaw<XT> r;
#pragma unroll
    for (uint32_t &w : r.w) w = 0u;
    return r;
}
// rows whose groups of 4 values are aligned to their size
template <int XT>
__host__ __device__ __forceinline__ bool mx_vec_ok(const void *p, int64_t stride) {
    constexpr int64_t need = 4 * sizeof(typename MxElem<XT>::T);
    return reinterpret_cast<uintptr_t>(p) % need == 0 && (stride * static_cast<int64_t>(sizeof(typename MxElem<XT>::T))) % need == 0;
}
template <int XT> struct MxPair;
template <> struct MxPair<MX_F16> {
    using T = __half2;
    static __device__ __forceinline__ T abs(uint32_t w) { w &= 0x7FFF7FFFu; return *reinterpret_cast<T *>(&w); }
};
template <> struct MxPair<MX_BF16> {
    using T = __nv_bfloat162;
    static __device__ __forceinline__ T abs(uint32_t w) { w &= 0x7FFF7FFFu; return *reinterpret_cast<T *>(&w); }
};
// the largest magnitude's f32 bits, a NaN's where there is one
__device__ __forceinline__ float mx_max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(fabsf(a)), "f"(fabsf(b)));
    return c;
}
__device__ __forceinline__ uint32_t mx_top(const float (&v)[8]) {
    const float a = mx_max_nan(v[0], v[1]), b = mx_max_nan(v[2], v[3]), c = mx_max_nan(v[4], v[5]), d = mx_max_nan(v[6], v[7]);
    return __float_as_uint(mx_max_nan(mx_max_nan(a, b), mx_max_nan(c, d)));
}
// the values, and their largest magnitude's bits
template <int XT>
__device__ __forceinline__ uint32_t mx_floats(const MxRaw<XT> &r, float (&v)[8]) {
    if constexpr (XT == MX_F32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(r.w[j]);
        return mx_top(v);
    } else {
        // two at a time; the .NaN maximum keeps a NaN
        typename MxPair<XT>::T two = MxPair<XT>::abs(r.w[0]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > 0) two = __hmax2_nan(two, MxPair<XT>::abs(r.w[j]));
            if constexpr (XT == MX_BF16) {
                v[2 * j] = __uint_as_float(r.w[j] << 16);
                v[2 * j + 1] = __uint_as_float(r.w[j] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[j]));
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
        const uint32_t both = *reinterpret_cast<const uint32_t *>(&two), one = max(both & 0xFFFFu, both >> 16);
        if constexpr (XT == MX_BF16) return one << 16;
        else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(one)))) & 0x7FFFFFFFu;
    }
}
// byte j: the code of a[j] in its low nibble, of b[j] in its high one (scaled by inv first)
__device__ __forceinline__ uint32_t mx_codes(const float (&a)[4], const float (&b)[4], float inv) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %5, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %6, %2;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %7, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %4;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w)
        : "f"(a[0] * inv), "f"(a[1] * inv), "f"(a[2] * inv), "f"(a[3] * inv), "f"(b[0] * inv), "f"(b[1] * inv),
          "f"(b[2] * inv), "f"(b[3] * inv));
    return w;
}

// the signed magnitudes (unscaled) that 4 code bytes hold, of the low nibbles and the high ones
__device__ __forceinline__ void mx_values(uint32_t w, float (&lo)[4], float (&hi)[4]) {
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
        lo[j] = f.x;
        hi[j] = f.y;
    }
}

__device__ __forceinline__ float mx_scale(uint32_t byte) {   // 2^(byte - 127); 255: NaN
    return __uint_as_float(byte == 255u ? 0x7FFFFFFFu : byte == 0u ? 0x00400000u : byte << 23);
}

// The block's scale byte and this lane's 4 code bytes, from its values and the
// lane's largest magnitude
__device__ __forceinline__ uint32_t mx_quant_block(const float (&v)[8], uint32_t top, uint32_t &byte) {
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t ex = top >> 23;
    byte = ex == 255u ? 255u : ex > 2u ? ex - 2u : 0u;
    const float inv = __uint_as_float((254u - min(byte, 252u)) << 23);   // 2^(127 - byte), exact
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    return byte == 255u ? 0u : mx_codes(a, b, inv);
}
// what the codes leave of v (exact: a multiple of v's last place, no larger than the block's largest value)
__device__ __forceinline__ void mx_residual(float (&v)[8], uint32_t codes, uint32_t byte) {
    float a[4], b[4];
    mx_values(codes, a, b);
    const float s = mx_scale(byte);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] -= a[j] * s; v[4 + j] -= b[j] * s; }
}

// ---------------------------------------------------------------------------
// The 17-byte blocks as a stream of words: 4 consecutive blocks are 17 words.
// 16 lanes hold them, lane 4 q + i code bytes 4 i .. 4 i + 3 of block q, which
// begin q + 1 bytes past a word; so lane l's word l is its own code word and
// the bytes before it (the lane before's, and the scale where i = 0) shifted
// together, and word 16 is lane 15's code word as it is. Reading goes the other
// way. Words leave and arrive straight from registers; y may have any
// alignment (bytes then), and past `end` nothing is touched.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void mx_put(uint8_t *y, int64_t at, int64_t end, bool words, uint32_t w) {
    if (words && at + 4 <= end) {
        *reinterpret_cast<uint32_t *>(y + at) = w;
    } else {
        for (int j = 0; j < 4; ++j)
            if (at + j < end) y[at + j] = static_cast<uint8_t>(w >> (8 * j));
    }
}
__device__ __forceinline__ uint32_t mx_get(const uint8_t *y, int64_t at, int64_t end, bool words) {
    if (words && at + 4 <= end) return __ldg(reinterpret_cast<const uint32_t *>(y + at));
    uint32_t w = 0;
    for (int j = 0; j < 4; ++j)
        if (at + j < end) w |= static_cast<uint32_t>(y[at + j]) << (8 * j);
    return w;
}
// the stream word that a lane writes (lane 15 of 16 also writes its codes behind it)
__device__ __forceinline__ uint32_t mx_stream_word(uint32_t codes, uint32_t byte, int lane) {
    const uint32_t before = __shfl_up_sync(0xffffffffu, codes, 1);
    const uint32_t pre = (lane & 3) == 0 ? before >> 8 | byte << 24 : before;
    return __funnelshift_lc(pre, codes, 8 * (((lane >> 2) & 3) + 1));
}
struct MxWords { uint32_t own, extra; };   // word l, and lane 15's word 16
__device__ __forceinline__ MxWords mx_get_words(const uint8_t *y, int64_t group, int64_t n_blocks, bool words, int lane) {
    const int l = lane & 15;
    const int64_t at = group * 17, end = n_blocks * 17;
    return {mx_get(y, at + 4 * l, end, words), l == 15 ? mx_get(y, at + 64, end, words) : 0u};
}
__device__ __forceinline__ uint32_t mx_take_block(const MxWords &m, int lane, uint32_t &byte) {
    const int q = (lane >> 2) & 3;
    const uint32_t next = __shfl_down_sync(0xffffffffu, m.own, 1);
    byte = __shfl_sync(0xffffffffu, m.own, lane & ~3) >> (8 * q) & 255u;
    return __funnelshift_rc(m.own, (lane & 15) == 15 ? m.extra : next, 8 * (q + 1));
}

// ---------------------------------------------------------------------------
// quantise into ggml blocks, y [planes][rows][nb], and read back: out [rows][K]
// = the planes' values added, rounded once to OT. 4 blocks per lane quad with
// all their loads in flight at once (one per quad left the memory waiting:
// 2.4 TB/s); byte stores through shared memory cost a quarter of the time.
// 16384 x 4096 bf16, one plane: 35.5 us (4.8 TB/s, bound by issue) and 28.1 us (6.0 TB/s, bound by HBM).
// ---------------------------------------------------------------------------
constexpr int MXQ_THREADS = 256;
constexpr int MXQ_PER = 4;                                // blocks per lane quad
constexpr int MXQ_STEP = MXQ_THREADS / 4;
constexpr int MXQ_BLK = MXQ_STEP * MXQ_PER;               // blocks per CTA

// a CTA whose blocks are all there, in dense rows, every plane's stream on word boundaries
__device__ __forceinline__ bool mx_whole(const void *y, int64_t stride, int64_t n_blocks, int nb, int planes) {
    return (static_cast<int64_t>(blockIdx.x) + 1) * MXQ_BLK <= n_blocks && stride == static_cast<int64_t>(nb) * 32 &&
           (reinterpret_cast<uintptr_t>(y) & 3u) == 0 && (planes == 1 || n_blocks % 4 == 0);
}
// row of block g: 32-bit division where the number of blocks allows
__device__ __forceinline__ int64_t mx_row_of(int64_t g, int nb, bool small) {
    return small ? static_cast<int64_t>(static_cast<uint32_t>(g) / static_cast<uint32_t>(nb)) : g / nb;
}
// element offset of block g; dense rows follow one another
__device__ __forceinline__ int64_t mx_block_at(int64_t g, int nb, int64_t stride, bool dense, bool small) {
    if (dense) return g * 32;
    const int64_t row = mx_row_of(g, nb, small);
    return row * stride + (g - row * nb) * 32;
}

// FAST: dense rows, aligned words and a whole CTA of blocks -- addresses are one
// base and constants (with 64-bit offsets and tests per word the kernel was
// bound by its 140 instructions per 8 values)
template <int XT, bool VEC, bool FAST>
__device__ __forceinline__ void mx_quantize_blocks(const typename MxElem<XT>::T *__restrict__ x, int64_t stride,
                                                   int64_t n_blocks, int nb, int planes, uint8_t *__restrict__ y) {
    const int lane = threadIdx.x & 31, quad = threadIdx.x >> 2, i = threadIdx.x & 3;
    const int64_t b0 = static_cast<int64_t>(blockIdx.x) * MXQ_BLK;
    const bool dense = stride == static_cast<int64_t>(nb) * 32, small = n_blocks < (int64_t{1} << 31);
    const typename MxElem<XT>::T *const x0 = x + (b0 + quad) * 32;
    uint8_t *const y0 = y + (b0 + (quad & ~3)) * 17 + 4 * (lane & 15);
    MxRaw<XT> raw[MXQ_PER];
#pragma unroll
    for (int u = 0; u < MXQ_PER; ++u) {
        if constexpr (FAST) {
            raw[u] = mx_load<XT, VEC>(x0 + u * (MXQ_STEP * 32), i);
        } else {
            const int64_t g = b0 + u * MXQ_STEP + quad;
            raw[u] = mx_zero<XT>();
            if (g < n_blocks) raw[u] = mx_load<XT, VEC>(x + mx_block_at(g, nb, stride, dense, small), i);
        }
    }
#pragma unroll
    for (int u = 0; u < MXQ_PER; ++u) {
        float v[8];
        uint32_t top = mx_floats<XT>(raw[u], v);
        for (int pl = 0;; ++pl) {
            uint32_t byte;
            const uint32_t w = mx_quant_block(v, top, byte);
            const int64_t plane = pl * n_blocks * 17;
            if constexpr (FAST) {
                uint8_t *o = y0 + plane + u * (MXQ_STEP * 17);
                *reinterpret_cast<uint32_t *>(o) = mx_stream_word(w, byte, lane);
                if ((lane & 15) == 15) *reinterpret_cast<uint32_t *>(o + 4) = w;
            } else {
                uint8_t *o = y + plane;
                const int64_t at = (b0 + u * MXQ_STEP + (quad & ~3)) * 17, end = n_blocks * 17;
                const bool words = (reinterpret_cast<uintptr_t>(o) & 3u) == 0;
                mx_put(o, at + 4 * (lane & 15), end, words, mx_stream_word(w, byte, lane));
                if ((lane & 15) == 15) mx_put(o, at + 64, end, words, w);
            }
            if (pl + 1 == planes) break;
            mx_residual(v, w, byte);
            top = mx_top(v);
        }
    }
}

template <int XT, bool VEC>
__global__ void __launch_bounds__(MXQ_THREADS) mx_quantize_kernel(const typename MxElem<XT>::T *__restrict__ x,
                                                                  int64_t stride, int64_t n_blocks, int nb, int planes,
                                                                  uint8_t *__restrict__ y) {
    if (VEC && mx_whole(y, stride, n_blocks, nb, planes)) mx_quantize_blocks<XT, VEC, VEC>(x, stride, n_blocks, nb, planes, y);
    else mx_quantize_blocks<XT, VEC, false>(x, stride, n_blocks, nb, planes, y);
}

template <int OT, bool VEC, bool FAST>
__device__ __forceinline__ void mx_dequantize_blocks(const uint8_t *__restrict__ y, int64_t n_blocks, int nb, int planes,
                                                     int64_t stride, typename MxElem<OT>::T *__restrict__ out) {
    using T = typename MxElem<OT>::T;
    const int lane = threadIdx.x & 31, quad = threadIdx.x >> 2, i = threadIdx.x & 3;
    const int64_t b0 = static_cast<int64_t>(blockIdx.x) * MXQ_BLK;
    const bool dense = stride == static_cast<int64_t>(nb) * 32, small = n_blocks < (int64_t{1} << 31);
    const uint8_t *const y0 = y + (b0 + (quad & ~3)) * 17 + 4 * (lane & 15);
    T *const out0 = out + (b0 + quad) * 32 + 4 * i;
    MxWords m[MX_MAX_PLANES][MXQ_PER];
#pragma unroll
    for (int pl = 0; pl < MX_MAX_PLANES; ++pl) {
        if (pl >= planes) break;
        const int64_t plane = pl * n_blocks * 17;
#pragma unroll
        for (int u = 0; u < MXQ_PER; ++u) {
            if constexpr (FAST) {
                const uint32_t *o = reinterpret_cast<const uint32_t *>(y0 + plane + u * (MXQ_STEP * 17));
                m[pl][u].own = __ldg(o);
                m[pl][u].extra = (lane & 15) == 15 ? __ldg(o + 1) : 0u;
            } else {
                const uint8_t *o = y + plane;
                m[pl][u] = mx_get_words(o, b0 + u * MXQ_STEP + (quad & ~3), n_blocks, (reinterpret_cast<uintptr_t>(o) & 3u) == 0, lane);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < MXQ_PER; ++u) {
        const int64_t g = b0 + u * MXQ_STEP + quad;
        float v[8];
#pragma unroll
        for (int pl = 0; pl < MX_MAX_PLANES; ++pl) {
            if (pl >= planes) break;
            uint32_t byte;
            float lo[4], hi[4];
            mx_values(mx_take_block(m[pl][u], lane, byte), lo, hi);
            const float s = mx_scale(byte);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = pl == 0 ? lo[j] * s : __fadd_rn(v[j], __fmul_rn(lo[j], s));   // (each value as it stands in 32 bits)
                v[4 + j] = pl == 0 ? hi[j] * s : __fadd_rn(v[4 + j], __fmul_rn(hi[j], s));
            }
        }
        if (!FAST && g >= n_blocks) continue;
        T *p = FAST ? out0 + u * (MXQ_STEP * 32) : out + mx_block_at(g, nb, stride, dense, small) + 4 * i;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            __align__(16) T e[4];
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
}

template <int OT, bool VEC>
__global__ void __launch_bounds__(MXQ_THREADS) mx_dequantize_kernel(const uint8_t *__restrict__ y, int64_t n_blocks,
                                                                    int nb, int planes, int64_t stride,
                                                                    typename MxElem<OT>::T *__restrict__ out) {
    if (VEC && mx_whole(y, stride, n_blocks, nb, planes)) mx_dequantize_blocks<OT, VEC, VEC>(y, n_blocks, nb, planes, stride, out);
    else mx_dequantize_blocks<OT, VEC, false>(y, n_blocks, nb, planes, stride, out);
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
// The grouped product
// ---------------------------------------------------------------------------
// Per chunk width NT (entries = MMA N): groups of 4 epilogue warps (behind warp
// 0, copies, and warp 1, MMA)
template <int NT> __host__ __device__ constexpr int mxp_epi() { return NT >= 64 ? 2 : 1; }
template <int NT> __host__ __device__ constexpr int mxp_threads() { return 64 + 128 * mxp_epi<NT>(); }
// K tiles per ring stage: two halve what a stage costs the two issuing warps; a
// tile of the widest chunk keeps the tensor cores busy long enough by itself
template <int NT> __host__ __device__ constexpr int mxp_tps() { return NT >= 192 ? 1 : 2; }
// The widest chunks: 384 TMEM columns hold one matrix's accumulators, or gate's
// and up's, twice. Shared memory bounds them (the MMAs' operand reads and the
// copies' writes share its 128 bytes a cycle), so the product is fastest where
// an operand byte meets the most others: 128 x 192, and 256 x 96 with the gate.
constexpr int MXP_WIDE = 192, MXP_WIDE_GLU = 96;

// Instruction descriptor of kind::mxf4: e2m1 A and B (K-major), UE8M0 scales,
// M = 128, N; `half` picks the pair of scale bytes of the tile's K = 64 half.
__device__ __forceinline__ uint32_t mx_idesc(int N, int half) {
    return (static_cast<uint32_t>(2 * half) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
           (1u << 23) | (static_cast<uint32_t>(MX_M >> 4) << 24) | (static_cast<uint32_t>(2 * half) << 29);
}

// Shared-memory descriptors (K-major, no swizzle, 8-row groups 128 bytes apart)
// as their two words: the low one holds the address and the distance of the
// 16-byte chunks along K, the high one is the same for every operand here.
constexpr uint32_t MX_DESC_HI = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t mx_desc_lo(uint32_t saddr, uint32_t lbo) {
    return ((saddr >> 4) & 0x3FFFu) | ((lbo >> 4) << 16);   // (in a cluster the address also holds the CTA's rank)
}

// The tcgen05 instructions below are issued by the lane whose `on` is set, all
// lanes of the warp calling: with a predicate instead of a branch the control
// flow stays uniform, and the operands -- which the hardware takes from uniform
// registers -- are computed there instead of being moved one by one.
__device__ __forceinline__ void umma_mxf4(uint32_t on, uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %6, 0;\n\tsetp.ne.b32 q, %8, 0;\n\t"
        "mov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], da, db, %3, [%4], [%5], p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(MX_DESC_HI), "r"(on)
        : "memory");
}

// 512 scale bytes (32 rows of 16) from shared memory to 4 TMEM columns of all four lane quarters
__device__ __forceinline__ void tmem_cp_scales(uint32_t on, uint32_t taddr, uint32_t lo) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b64 d;\n\tsetp.ne.b32 q, %3, 0;\n\tmov.b64 d, {%1, %2};\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(taddr), "r"(lo), "r"(MX_DESC_HI), "r"(on)
        : "memory");
}
// bulk copy global -> shared, and the barrier's arrival that announces its bytes
__device__ __forceinline__ void bulk_g2s_if(uint32_t on, uint32_t dst, const void *src, uint32_t bytes, uint32_t bar,
                                            uint64_t policy) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;\n\t}"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy), "r"(on)
        : "memory");
}
__device__ __forceinline__ void mbar_expect_if(uint32_t on, uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes), "r"(on)
        : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t on, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(on)
        : "memory");
}

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

// ---------------------------------------------------------------------------
// What the product needs first: its entries grouped into chunks (up to NT
// entries of one expert), and per chunk the entries' quantised rows as the MMA
// reads them -- an image: per K tile and plane, with N = the chunk's entries
// rounded up to 16, 16-byte chunk c of entry j at c * 16 N + j * 16, then per 128
// entries 512 bytes of scales (block c of entry j at j / 128 * 512 + (j % 32) * 16
// + j % 128 / 32 * 4 + c). A tile's planes are contiguous, so the product
// fetches them with one bulk copy; a row that k experts picked is quantised once and written k times.
// (Gathering rows inside the product, 16 bytes at a time by four warps, cost
// about 1,000 cycles per tile against the 250 that its MMAs take.)
//
// Up to MX_DIRECT entries nothing is grouped beforehand (mx_direct): every CTA works the
// chunks out for itself and quantises their rows; there are no images.
// ---------------------------------------------------------------------------
constexpr int MXG_CTAS = 8;         // CTAs (one cluster) that group
constexpr int MXG_THREADS = 1024;   // at most
constexpr int MXG_MAX_EXPERTS = 4096;

__host__ __device__ constexpr int mx_round16(int n) { return (n + 15) / 16 * 16; }
// bytes of one tile's plane: codes, then 512 bytes of scales for every 128 entries begun
__host__ __device__ constexpr uint32_t mx_image_plane(int N) { return 64u * N + (N > 128 ? 2u : 1u) * MX_SF; }
__host__ __device__ constexpr uint64_t mx_image_bytes(int NT, int KT, int planes) {               // between chunks
    return static_cast<uint64_t>(KT) * planes * mx_image_plane(NT);
}

struct MxPrep {
    const void *x;
    int64_t stride, n_rows;
    int32_t nb, KT, planes, per_pick;
    uint8_t *images;
    const int32_t *ids;
    int64_t ids_stride;
    int32_t n_entries, k, n_experts, NT;
    // chunked form: of each entry its expert (-1: left out) and its number among the expert's entries; of
    // each expert {first chunk, entries, first entry, -}
    int32_t *entries, *n_chunks;
    int2 *where;
    int4 *experts, *chunks;
    int *err;
};

__host__ __device__ constexpr int mx_group_sets(int E) { return E <= 512 ? 8 : 1; }

// Grouping by one cluster of MXG_CTAS: each CTA counts its share of the entries
// per expert in shared memory, reads the other CTAs' counts, and places its
// entries behind theirs. Chunks of an expert are consecutive. Order inside an
// expert changes no result. Id -1: left out. What an entry's number means -- its
// chunk, its place in the image -- is worked out by the kernel behind this one,
// on every SM: done here, on 8 of them, it took twice as long. Latency bound: 3.5 us for 64 entries, 8.7 for 32768.
__global__ void __cluster_dims__(MXG_CTAS, 1, 1) __launch_bounds__(MXG_THREADS) mx_group_kernel(const MxPrep a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ int group_smem[];
    __shared__ int scratch[64];
    // counts of several sets of warps: a popular expert's counter, one for all, took 20 cycles an entry
    const int sets = mx_group_sets(a.n_experts);
    int *sum = group_smem, *cur = sum + a.n_experts, *kept = cur + a.n_experts, *cnt = kept + a.n_experts;   // cnt: [sets][n_experts]
    const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, E = a.n_experts, N = a.n_entries;
    int *const mine = cnt + warp % sets * E;
    for (int e = tid; e < sets * E; e += nth) cnt[e] = 0;
    __syncthreads();
    auto id_of = [&](int i) {
        if (i >= N) return -1;
        const int t = i / a.k;
        const int x = a.ids[static_cast<int64_t>(t) * a.ids_stride + (i - t * a.k)];
        if (x >= 0 && x < E) return x;
        if (x != -1) set_error(a.err, DERR_BAD_ID);
        return -1;
    };
    // shared-memory atomics; one per warp where all its entries are of one expert (a token's picks
    // differ, so otherwise at most 32 / k lanes meet)
    auto add = [&](int *c, int x) {
        const int x0 = __shfl_sync(0xffffffffu, x, 0);
        if (__all_sync(0xffffffffu, x == x0)) {
            int base = 0;
            if (x0 >= 0 && lane == 0) base = atomicAdd(&c[x0], 32);
            return __shfl_sync(0xffffffffu, base, 0) + lane;
        }
        return x >= 0 ? atomicAdd(&c[x], 1) : 0;
    };
    constexpr int KEEP = 4;   // ids kept in registers, and their places among the CTA's
    int x[KEEP], at_cta[KEEP];
#pragma unroll
    for (int m = 0; m < KEEP; ++m) x[m] = id_of((m * MXG_CTAS + rank) * nth + tid);
#pragma unroll
    for (int m = 0; m < KEEP; ++m) {
        at_cta[m] = 0;
        if ((m * MXG_CTAS + rank) * nth < N) at_cta[m] = add(mine, x[m]);
    }
    __syncthreads();
    for (int e = tid; e < E; e += nth) {   // each set's first place
        int run = 0;
        for (int c = 0; c < sets; ++c) {
            const int n = cnt[c * E + e];
            cnt[c * E + e] = run;
            run += n;
        }
        sum[e] = kept[e] = run;
    }
    __syncthreads();
    const bool more = static_cast<int64_t>(KEEP * MXG_CTAS) * nth < N;   // entries past the registers: counted here, placed below
    if (more)
        for (int64_t i0 = static_cast<int64_t>(KEEP * MXG_CTAS + rank) * nth; i0 < N; i0 += MXG_CTAS * nth)
            add(sum, id_of(static_cast<int>(i0) + tid));
    __syncthreads();
    cluster_sync();
    int carry_e = 0, carry_c = 0;
    for (int base = 0; base < E; base += nth) {
        const int e = base + tid;
        int total = 0, before = 0;
        if (e < E)
#pragma unroll
            for (int c = 0; c < MXG_CTAS; ++c) {
                const int v = __float_as_int(ld_cluster_f32(smem_u32(&sum[e]), c));
                if (c < rank) before += v;
                total += v;
            }
        const int nc = (total + a.NT - 1) / a.NT;
        int se = total, sc = nc;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int oe = __shfl_up_sync(0xffffffffu, se, off), oc = __shfl_up_sync(0xffffffffu, sc, off);
            if (lane >= off) { se += oe; sc += oc; }
        }
        if (lane == 31) { scratch[warp] = se; scratch[32 + warp] = sc; }
        __syncthreads();
        // every warp scans the warps' sums
        int we = lane < nth / 32 ? scratch[lane] : 0, wc = lane < nth / 32 ? scratch[32 + lane] : 0;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int oe = __shfl_up_sync(0xffffffffu, we, off), oc = __shfl_up_sync(0xffffffffu, wc, off);
            if (lane >= off) { we += oe; wc += oc; }
        }
        const int pe = carry_e + (warp ? __shfl_sync(0xffffffffu, we, (warp - 1) & 31) : 0);
        const int pc = carry_c + (warp ? __shfl_sync(0xffffffffu, wc, (warp - 1) & 31) : 0);
        carry_e += __shfl_sync(0xffffffffu, we, 31);
        carry_c += __shfl_sync(0xffffffffu, wc, 31);
        __syncthreads();
        if (e < E) {
            const int first = pe + se - total, c0 = pc + sc - nc;
            cur[e] = before;
            if (rank == 0) a.experts[e] = make_int4(c0, total, first, 0);
            for (int q = rank; q < nc; q += MXG_CTAS)
                a.chunks[c0 + q] = make_int4(e, first + q * a.NT, min(a.NT, total - q * a.NT), 0);
        }
    }
    if (rank == 0 && tid == 0) *a.n_chunks = carry_c;
    __syncthreads();
#pragma unroll
    for (int m = 0; m < KEEP; ++m) {
        const int i = (m * MXG_CTAS + rank) * nth + tid;
        if (i < N) a.where[i] = make_int2(x[m], x[m] >= 0 ? cur[x[m]] + mine[x[m]] + at_cta[m] : 0);
    }
    if (more) {
        __syncthreads();
        for (int e = tid; e < E; e += nth) cur[e] += kept[e];
        __syncthreads();
        for (int64_t i0 = static_cast<int64_t>(KEEP * MXG_CTAS + rank) * nth; i0 < N; i0 += MXG_CTAS * nth) {
            const int i = static_cast<int>(i0) + tid, xi = id_of(i), at = add(cur, xi);
            if (i < N) a.where[i] = make_int2(xi, at);
        }
    }
    cluster_sync();   // the counts stay until every CTA has read them
}

// The direct form groups its entries by itself: bit j of `same` says that entry j has an entry's expert.
__device__ __forceinline__ int mx_before(uint64_t same, int i) { return __popcll(same & ((1ull << i) - 1ull)); }
__device__ __forceinline__ int mx_id(const int32_t *ids, int64_t stride, int n_entries, int k, int i) {
    return i < n_entries ? ids[(i / k) * stride + i % k] : -2;
}

// Quantise x and write the images: 4 lanes per block, 16 per K tile of a row, RUN
// tiles in turn: what finds a row's places serves them all, and their loads are
// in flight together (1 / 2 / 4 / 6 of them: 27.3, 24.3, 28.4 and 28.0 us). 16384 f32 rows of K = 768, two planes:
// 22.2 to 24.2 us, bound by issue (69 % of the slots) and the last wave; 2.4 TB/s.
template <int XT, bool VEC, int RUN>
__global__ void __launch_bounds__(256, 4) mx_images_kernel(const MxPrep a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const int64_t g = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4;   // (row, run of RUN tiles)
    const int i = threadIdx.x & 3, b = (threadIdx.x >> 2) & 3;                           // block b of a tile
    const int runs = (a.KT + RUN - 1) / RUN;
    const int64_t row = mx_row_of(g, runs, a.n_rows * runs < (int64_t{1} << 31));
    const int t0 = static_cast<int>(g - row * runs) * RUN;
    const bool row_ok = row < a.n_rows;
    const typename MxElem<XT>::T *x = static_cast<const typename MxElem<XT>::T *>(a.x) + row * a.stride + (t0 * 4 + b) * 32;
    MxRaw<XT> raw[RUN];
#pragma unroll
    for (int u = 0; u < RUN; ++u) {   // K padded to whole tiles with zeros
        raw[u] = mx_zero<XT>();
        if (row_ok && (t0 + u) * 4 + b < a.nb) raw[u] = mx_load<XT, VEC>(x + 128 * u, i);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the grouping
    // The row's destinations: lane i of the 4 serves number i, i + 4, ... Two of them are looked up
    // here, while x is on its way: behind the arithmetic the look-ups were most of the kernel's time.
    const int n_dst = row_ok ? (a.per_pick ? 1 : a.k) : 0;
    const int64_t en0 = row * (a.per_pick ? 1 : a.k);
    struct Place { int chunk, j, N; };
    auto place_of = [&](int64_t en) {
        Place d;
        const int2 w = a.where[en];
        const int4 ex = a.experts[max(w.x, 0)];
        const int c = w.y / a.NT;
        d.chunk = w.x < 0 ? -1 : ex.x + c;
        d.j = w.y - c * a.NT;
        d.N = mx_round16(min(a.NT, ex.y - c * a.NT));
        if (t0 == 0 && b == 0 && w.x >= 0) a.entries[ex.z + w.y] = static_cast<int32_t>(en);
        return d;
    };
    const uint64_t image = mx_image_bytes(a.NT, a.KT, a.planes);
    // where tile t0 of a destination's image keeps this block's codes and the tile's scales, and the step to the next tile
    struct Spot { uint8_t *codes; uint32_t scales, plane; };
    auto spot_of = [&](const Place &d) {
        Spot o;
        o.plane = mx_image_plane(d.N);
        uint8_t *t = a.images + static_cast<uint64_t>(d.chunk) * image + static_cast<uint64_t>(t0 * a.planes) * o.plane;
        o.codes = d.chunk < 0 ? nullptr : t + b * 16 * d.N + d.j * 16;
        o.scales = 64 * d.N + (d.j >> 7) * MX_SF + (d.j & 31) * 16 + ((d.j >> 5) & 3) * 4 - (b * 16 * d.N + d.j * 16);
        return o;
    };
    constexpr int AHEAD = 2;
    Spot ahead[AHEAD];
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) {
        ahead[p].codes = nullptr;
        ahead[p].plane = ahead[p].scales = 0;
        if (i + 4 * p < n_dst) ahead[p] = spot_of(place_of(en0 + i + 4 * p));
    }

#pragma unroll
    for (int u = 0; u < RUN; ++u) {
        // a tile past K is quantised too (zeros) and written nowhere: half a warp may be at its row's
        // last, shorter run, and the shuffles below name all 32 lanes
        const bool tile_ok = t0 + u < a.KT;
        float v[8];
        uint32_t top = mx_floats<XT>(raw[u], v);
        uint32_t w[MX_MAX_PLANES][4], sc[MX_MAX_PLANES];
#pragma unroll
        for (int pl = 0; pl < MX_MAX_PLANES; ++pl) {
            if (pl >= a.planes) break;
            uint32_t byte;
            const uint32_t mine = mx_quant_block(v, top, byte);
            if (pl + 1 < a.planes) {
                mx_residual(v, mine, byte);
                top = mx_top(v);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) w[pl][j] = __shfl_sync(0xffffffffu, mine, (lane & ~3) + j);   // the block's 16 bytes
            uint32_t word = byte << (8 * b);                                                          // the tile's 4 scales
            word |= __shfl_xor_sync(0xffffffffu, word, 4);
            word |= __shfl_xor_sync(0xffffffffu, word, 8);
            sc[pl] = word;
        }
        auto put = [&](uint8_t *codes, const Spot &o) {
#pragma unroll
            for (int pl = 0; pl < MX_MAX_PLANES; ++pl)
                if (pl < a.planes) {
                    uint8_t *c = codes + pl * o.plane;
                    *reinterpret_cast<uint4 *>(c) = make_uint4(w[pl][0], w[pl][1], w[pl][2], w[pl][3]);
                    if (b == 0) *reinterpret_cast<uint32_t *>(c + static_cast<int32_t>(o.scales)) = sc[pl];
                }
        };
#pragma unroll
        for (int p = 0; p < AHEAD; ++p)
            if (tile_ok && ahead[p].codes) {
                put(ahead[p].codes, ahead[p]);
                ahead[p].codes += a.planes * ahead[p].plane;
            }
        for (int q = i + 4 * AHEAD; tile_ok && q < n_dst; q += 4) {
            const Spot o = spot_of(place_of(en0 + q));
            if (o.codes) put(o.codes + static_cast<uint64_t>(u * a.planes) * o.plane, o);
        }
    }
}

// One lane of the converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
    return p != 0;
}

template <int ENTRIES>
struct MxCtl {
    uint64_t full[MX_MAX_STAGES], empty[MX_MAX_STAGES], acc_full[2], acc_empty[2], drain;
    uint64_t rows[MX_MAX_STAGES];   // a stage's image, where the CTA quantises it
    uint32_t tmem;
    int32_t abort, n_chunks;
    int32_t entry[ENTRIES];     // direct form: the entries grouped by expert
    int4 chunk[ENTRIES];        // {expert, first entry, count, -}
};

template <int NT>
__host__ __device__ constexpr uint32_t mx_stage_bytes(int mats, int planes) {
    return mxp_tps<NT>() * (mats * MX_TILE + planes * mx_image_plane(NT));
}

template <int ENTRIES>
__device__ __forceinline__ bool mx_wait(MxCtl<ENTRIES> &C, uint64_t *bar, uint32_t parity, const MxArgs &a) {
    // limits below 20 us poll (try_wait may suspend for longer), so that a tiny limit gives up at once
    const bool poll = a.timeout_ns < 20000u;
    if (poll ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = clock64(), lim = timeout_cycles(a.timeout_ns);
    for (;;) {
        if (poll ? mbar_test_wait(bar, parity) : mbar_try_wait_hint(bar, parity, 2000u)) return true;
        if (*reinterpret_cast<volatile int32_t *>(&C.abort)) return false;
        if (static_cast<uint64_t>(clock64()) - t0 > lim) {
            *reinterpret_cast<volatile int32_t *>(&C.abort) = 1;
            set_error(a.err, DERR_TIMEOUT_FULL);
            return false;
        }
    }
}
// the same for a whole warp: the lanes agree
template <int NT>
__device__ __forceinline__ bool mx_wait_warp(MxCtl<NT> &C, uint64_t *bar, uint32_t parity, const MxArgs &a) {
    return __all_sync(0xffffffffu, mx_wait(C, bar, parity, a)) != 0;
}

// The direct form's chunks, by one warp from the ids of up to 64 entries: lane l
// looks at entries l and l + 32. Experts follow one another as they first appear.
template <int NT>
__device__ __forceinline__ void mx_direct_table(MxCtl<MX_DIRECT> &C, const MxArgs &a, int lane) {
    int x[2];
    uint64_t same[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        x[h] = mx_id(a.ids, a.ids_stride, a.n_entries, a.k, lane + 32 * h);
        if (lane + 32 * h < a.n_entries && x[h] != -1 && (x[h] < 0 || x[h] >= a.n_experts)) {
            set_error(a.err, DERR_BAD_ID);
            x[h] = -1;
        }
    }
    if (a.n_entries <= 32) {
        same[0] = __match_any_sync(0xffffffffu, x[0]);
        same[1] = 0;
    } else {
        same[0] = same[1] = 0;
#pragma unroll 8
        for (int j = 0; j < MX_DIRECT; ++j) {
            const int y = __shfl_sync(0xffffffffu, x[j >> 5], j & 31);
            same[0] |= static_cast<uint64_t>(x[0] == y) << j;
            same[1] |= static_cast<uint64_t>(x[1] == y) << j;
        }
    }
    // (entries, chunks) of the experts that appear before: a scan over each expert's first entry
    int before[2], carry = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int cnt = __popcll(same[h]);
        const bool leads = x[h] >= 0 && mx_before(same[h], lane + 32 * h) == 0;
        const int mine = leads ? cnt | ((cnt + NT - 1) / NT) << 16 : 0;
        int sum = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += o;
        }
        before[h] = carry + sum - mine;
        carry += __shfl_sync(0xffffffffu, sum, 31);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h, pos = mx_before(same[h], i), lead = same[h] ? __ffsll(static_cast<long long>(same[h])) - 1 : 0;
        const int lo = __shfl_sync(0xffffffffu, before[0], lead & 31), hi = __shfl_sync(0xffffffffu, before[1], lead & 31);
        const int at = lead < 32 ? lo : hi, first = at & 0xFFFF;
        if (x[h] >= 0) {
            C.entry[first + pos] = i;
            if (pos % NT == 0)
                C.chunk[(at >> 16) + pos / NT] = make_int4(x[h], first + pos, min(NT, __popcll(same[h]) - pos), 0);
        }
    }
    if (lane == 0) C.n_chunks = carry >> 16;
}

// A chunk's rows into the ring's images, by the warps behind the first two: one
// row of one stage (8 blocks, 4 lanes each) per warp and step, the next step's
// values on their way meanwhile.
struct MxRing { int s, ph, fills; };   // the ring's next stage, the parity of its use, stages used so far
template <int NT, int PLANES, int MATS>
__device__ __forceinline__ void mx_rows(MxCtl<MX_DIRECT> &C, const MxArgs &a, int first, int count, int kt0, int n_it,
                                        MxRing &at, int warp, int lane, uint8_t *ring) {
    static_assert(mxp_tps<NT>() * MX_KT == 8 * 32, "a warp takes a row of a stage");
    constexpr int WARPS = 4 * mxp_epi<NT>(), TPS = mxp_tps<NT>();
    constexpr uint32_t PLANE = mx_image_plane(NT);
    using Raw = MxRaw<MX_F32>;                                     // of any type: f16 and bf16 fill half of it
    const int i4 = lane & 3, b = (lane >> 2) & 3, t = lane >> 4;   // block b of tile t
    const int steps = n_it * count;
    auto load = [&](int p) {
        const int i = p / count, en = C.entry[first + p - i * count], blk = (kt0 + i * TPS) * 4 + (lane >> 2);
        const int64_t from = static_cast<int64_t>(a.per_pick ? en : en / a.k) * a.x_stride + blk * 32;
        Raw r = mx_zero<MX_F32>();
        if (p >= steps || blk >= a.nb) return r;                   // K padded to whole tiles with zeros
        if (a.x_type == MX_F32) {
            const float *x = static_cast<const float *>(a.x) + from;
            r = a.x_vec ? mx_load<MX_F32, true>(x, i4) : mx_load<MX_F32, false>(x, i4);
        } else {
            const __half *x = static_cast<const __half *>(a.x) + from;   // (16 bits each; what they mean comes later)
            const MxRaw<MX_F16> h = a.x_vec ? mx_load<MX_F16, true>(x, i4) : mx_load<MX_F16, false>(x, i4);
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[j] = h.w[j];
        }
        return r;
    };
    auto floats = [&](const Raw &r, float (&v)[8]) {
        if (a.x_type == MX_F32) return mx_floats<MX_F32>(r, v);
        const MxRaw<MX_F16> f{{r.w[0], r.w[1], r.w[2], r.w[3]}};
        const MxRaw<MX_BF16> g{{r.w[0], r.w[1], r.w[2], r.w[3]}};
        return a.x_type == MX_F16 ? mx_floats<MX_F16>(f, v) : mx_floats<MX_BF16>(g, v);
    };
    int p = warp;
    Raw next = load(p);
    for (int i = 0; i < n_it; ++i) {
        if (at.fills >= a.stages && !mx_wait_warp(C, &C.empty[at.s], at.ph ^ 1, a)) return;
        uint8_t *const image = ring + at.s * mx_stage_bytes<NT>(MATS, PLANES) + TPS * MATS * MX_TILE + t * (PLANES * PLANE);
        for (; p < (i + 1) * count; p += WARPS) {
            const int j = p - i * count;
            float v[8];
            uint32_t top = floats(next, v);
            next = load(p + WARPS);
#pragma unroll
            for (int pl = 0; pl < PLANES; ++pl) {
                uint32_t byte;
                const uint32_t w = mx_quant_block(v, top, byte);
                uint8_t *const o = image + pl * PLANE;
                *reinterpret_cast<uint32_t *>(o + b * (16 * NT) + j * 16 + 4 * i4) = w;
                if (i4 == 0) o[64 * NT + j * 16 + b] = static_cast<uint8_t>(byte);
                if (pl + 1 < PLANES) {
                    mx_residual(v, w, byte);
                    top = mx_top(v);
                }
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&C.rows[at.s]);
        ++at.fills;
        if (++at.s == a.stages) { at.s = 0; at.ph ^= 1; }
    }
}

// Work item: 128 weight rows (of w, and of gate with GLU) x the up to NT
// entries of one chunk x this cluster rank's share of K. A CTA walks items
// blockIdx / split, + gridDim / split, ... with its roles running ahead of one
// another through the ring and the accumulators:
//   warp 0    streams tiles by bulk copies: the weights' (contiguous and already
//             in the MMA's layout, as is the chunk's image);
//   warp 1    copies each tile's scales to tensor memory and issues the MMAs,
//             D += A B_plane over the planes;
//   the rest  in groups of 4 warps that take 16 columns in turn, read the
//             accumulators (thread = weight row), add biases, apply the GLU and
//             store, while the next item multiplies.
// In the direct form (NT = 16) the last warps first quantise the chunk's rows
// straight into the ring: every tile of weight rows does it again, but a
// few rows are done before their weights arrive, and the call is one launch
// without a workspace (a launch more cost 3 us of 17 for one token).
// 32768 entries of 64 experts (K = 2048, 1024 rows, gate and up, one plane): 99 us, 2.8 PFLOP/s; 16384 of 32
// (K = 768, 2048 rows, two planes): 40 us. Bound by shared memory, then by the stores of the results.
// The direct form keeps its chunks in shared memory (a CTA for each possible
// chunk instead, most of them empty, took 10 us for 1024 CTAs by itself).
// With split > 1 a cluster's CTAs have one item each; their partial sums meet in
// shared memory and are added in rank order, so results do not depend on timing.
template <int NT, bool GLU, bool DIRECT, int PLANES>
__global__ void __launch_bounds__(mxp_threads<NT>()) mx_product_kernel(const MxArgs a) {
    extern __shared__ __align__(128) uint8_t ring[];
    constexpr int MATS = GLU ? 2 : 1, MXP_EPI = mxp_epi<NT>(), MXP_TPS = mxp_tps<NT>();
    __shared__ MxCtl<DIRECT ? MX_DIRECT : 1> C;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int rank = a.split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int item0 = blockIdx.x / a.split, item_step = gridDim.x / a.split;

    if constexpr (DIRECT)
        if (warp == 0) mx_direct_table<NT>(C, a, lane);
    if (tid == 32) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.empty[s], 1);
            if (DIRECT) mbar_init(&C.rows[s], 4 * MXP_EPI);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&C.acc_full[s], 1);
            mbar_init(&C.acc_empty[s], 4 * MXP_EPI);
        }
        mbar_init(&C.drain, 1);
        C.abort = 0;
        fence_mbar_init();
    }
    __syncthreads();
    int n_items = 0;
    if (DIRECT) {
        n_items = C.n_chunks * a.RT;
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        n_items = *a.n_chunks * a.RT;
    }
    if (item0 >= n_items) return;   // nothing here; the same for every rank of the cluster
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&C.tmem)),
                     "r"(a.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const int kt0 = a.KT * rank / a.split, n_kt = a.KT * (rank + 1) / a.split - kt0;   // this rank's K tiles,
    const int n_it = (n_kt + MXP_TPS - 1) / MXP_TPS;                                   // MXP_TPS to a stage
    constexpr int planes = PLANES;
    const int stages = a.stages, acc = a.acc;
    constexpr uint32_t stage_bytes = mx_stage_bytes<NT>(MATS, planes);
    const uint32_t ring0 = smem_u32(ring);
    struct Item { int rt, chunk, expert, count, first; };
    auto item_at = [&](int item) {
        Item I;
        I.chunk = item / a.RT;
        I.rt = item - I.chunk * a.RT;
        const int4 ch = DIRECT ? C.chunk[I.chunk] : a.chunks[I.chunk];
        I.expert = ch.x; I.first = ch.y; I.count = ch.z;
        return I;
    };
    auto entry_of = [&](const Item &I, int j) { return DIRECT ? C.entry[I.first + j] : a.entries[I.first + j]; };

    // warp 0: stages issued so far, and the ring's next stage
    int fills = 0;
    uint32_t w_stage = 0, w_phase = 0;
    const uint32_t full0 = smem_u32(C.full);
    auto tiles_of = [&](int i) { return min(MXP_TPS, n_kt - i * MXP_TPS); };
    // stage: the weight tiles, the gate's, then the image's
    auto fill_weights = [&](uint32_t on, uint64_t at, int i, uint32_t image_tile, uint64_t pol) {
        const uint32_t n = tiles_of(i), dst = ring0 + w_stage * stage_bytes, bar = full0 + 8 * w_stage;
        at += static_cast<uint64_t>(i) * (MXP_TPS * MX_TILE);
        mbar_expect_if(on, bar, n * (MATS * MX_TILE + image_tile));
        bulk_g2s_if(on, dst, a.w + at, n * MX_TILE, bar, pol);
        if (GLU) bulk_g2s_if(on, dst + MXP_TPS * MX_TILE, a.gate + at, n * MX_TILE, bar, pol);
    };
    auto weights_at = [&](const Item &I) {
        return static_cast<uint64_t>(I.expert) * a.expert_bytes + (static_cast<uint64_t>(I.rt) * a.KT + kt0) * MX_TILE;
    };
    const uint32_t on = elect_one() ? 1u : 0u;   // the lane that issues for its warp
    int early = 0;
    if (DIRECT && warp == 0) {   // what the ring holds, at once
        const Item I = item_at(item0);
        early = n_it < stages ? n_it : stages;
        const uint64_t pol = l2_evict_first_policy();
        for (w_stage = 0; static_cast<int>(w_stage) < early; ++w_stage)
            fill_weights(on, weights_at(I), w_stage, 0u, pol);
        w_stage = 0;
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();   // the tensor memory's address
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, C.tmem, 0);

    if (warp == 0) {
        const uint64_t pol_w = l2_evict_first_policy(), pol_x = l2_evict_last_policy();
        bool ok = true;
        for (int item = item0; item < n_items && ok; item += item_step) {
            const Item I = item_at(item);
            const uint32_t tile = DIRECT ? 0u : __shfl_sync(0xffffffffu, planes * mx_image_plane(mx_round16(I.count)), 0);
            const uint64_t wat = weights_at(I);
            const uint8_t *image = a.images + static_cast<uint64_t>(I.chunk) * mx_image_bytes(NT, a.KT, planes) +
                                   static_cast<uint64_t>(kt0) * tile;
            for (int i = 0; i < n_it; ++i) {
                if (fills >= stages) {
                    ok = mx_wait_warp(C, &C.empty[w_stage], w_phase ^ 1u, a);
                    if (!ok) break;
                }
                if (i >= early || item != item0) fill_weights(on, wat, i, tile, pol_w);
                if (!DIRECT)
                    bulk_g2s_if(on, ring0 + w_stage * stage_bytes + MXP_TPS * MATS * MX_TILE, image, tiles_of(i) * tile,
                                full0 + 8 * w_stage, pol_x);
                image += MXP_TPS * tile;
                ++fills;
                if (++w_stage == static_cast<uint32_t>(stages)) { w_stage = 0; w_phase ^= 1u; }
            }
        }
    } else if (warp == 1) {
        const uint32_t sf0 = tmem + static_cast<uint32_t>(acc * MATS * NT);   // scale columns, a slot per stage
        constexpr uint32_t SFB = NT > 128 ? 8 : 4;                              // columns of a plane's scales
        constexpr uint32_t sf_tile = 4u * MATS + SFB * planes, sf_slot = MXP_TPS * sf_tile;
        const uint32_t empty0 = smem_u32(C.empty), acc0 = smem_u32(C.acc_full);
        uint32_t s = 0, ph = 0, n = 0;
        bool ok = true;
        Item next = item_at(item0);
        for (int item = item0; item < n_items && ok; item += item_step, ++n) {
            const uint32_t ab = acc == 2 ? n & 1u : 0u, aph = acc == 2 ? (n >> 1) & 1u : n & 1u;
            const Item I = next;
            if (item + item_step < n_items) next = item_at(item + item_step);      // asked for one item ahead
            const int N = __shfl_sync(0xffffffffu, mx_round16(I.count), 0);
            if (n >= static_cast<uint32_t>(acc)) ok = mx_wait_warp(C, &C.acc_empty[ab], aph ^ 1u, a);
            const uint32_t id0 = mx_idesc(N, 0), id1 = mx_idesc(N, 1);
            const uint32_t d0 = tmem + ab * (MATS * NT);
            const uint32_t bp = mx_image_plane(N) >> 4, bh = 2u * N;   // next plane, next K = 64 (descriptor units)
            bool ready = false;
            for (int i = 0; i < n_it && ok; ++i) {
                if (!ready) ok = mx_wait_warp(C, &C.full[s], ph, a);
                if (DIRECT && ok) ok = mx_wait_warp(C, &C.rows[s], ph, a);
                if (!ok) break;
                tc_fence_after();
                const uint32_t A = ring0 + s * stage_bytes, B = A + MXP_TPS * MATS * MX_TILE, sf = sf0 + s * sf_slot;
                const uint32_t al = mx_desc_lo(A, 16 * MX_M), bl = mx_desc_lo(B, 16 * N);
                const uint32_t asf = mx_desc_lo(A + MX_CODES, 0u), bsf = mx_desc_lo(B + 64 * N, 0u);
                // in descriptor units: next tile, next matrix, next K = 64
                constexpr uint32_t AT = MX_TILE >> 4, AM = MXP_TPS * AT, AH = (2 * 16 * MX_M) >> 4;
                const int n = tiles_of(i);
                const uint32_t free_bar = empty0 + 8 * s;
                if (++s == static_cast<uint32_t>(stages)) { s = 0; ph ^= 1u; }
#pragma unroll
                for (int t = 0; t < MXP_TPS; ++t) {
                    // the next stage's barrier is looked at while this one's first MMAs run
                    if (t == MXP_TPS - 1) ready = i + 1 < n_it && __all_sync(0xffffffffu, mbar_test_wait(&C.full[s], ph));
                    if (t >= n) break;
                    const uint32_t sft = sf + t * sf_tile, bt = t * planes * bp;
#pragma unroll
                    for (int m = 0; m < MATS; ++m)
                        tmem_cp_scales(on, sft + 4 * m, asf + t * AT + m * AM);
#pragma unroll
                    for (int p = 0; p < planes; ++p) {
                        tmem_cp_scales(on, sft + 4 * MATS + SFB * p, bsf + bt + p * bp);
                        if (NT > 128 && N > 128) tmem_cp_scales(on, sft + 4 * MATS + SFB * p + 4, bsf + bt + p * bp + (MX_SF >> 4));
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int p = 0; p < planes; ++p)
#pragma unroll
                            for (int m = 0; m < MATS; ++m)
                                umma_mxf4(on, d0 + m * NT, al + t * AT + m * AM + h * AH, bl + bt + p * bp + h * bh,
                                          h ? id1 : id0, sft + 4 * m, sft + 4 * MATS + SFB * p,
                                          t + h + p > 0 || i > 0 ? 1u : 0u);
                }
                umma_commit_if(on, free_bar);
            }
            if (ok) umma_commit_if(on, acc0 + 8 * ab);
        }
    } else {
        // ---- epilogue -------------------------------------------------------
        // Thread = weight row. Group g takes columns 16 (g + EPI q), round q. All of them go to
        // registers first: the accumulators are free for the next item but one at once.
        const int grp = (warp - 2) >> 2;
        const int quarter = warp & 3;                 // TMEM lanes this warp may read
        const int r = 32 * quarter + lane;            // weight row of the tile
        MxRing at{0, 0, 0};                           // (direct form)
        constexpr int ROUNDS = (NT + 16 * MXP_EPI - 1) / (16 * MXP_EPI);
        uint32_t n = 0;
        Item next = item_at(item0);
        // the direct form enters one item early, with the first one's rows (one place in the code:
        // fetching a second copy took longer than what it does)
        for (int item = DIRECT ? item0 - item_step : item0; item < n_items; item += item_step) {
            const Item I = next;
            if (item + item_step < n_items) {
                next = item_at(item + item_step);
                if constexpr (DIRECT) {   // while this one multiplies (a wait that gives up: the epilogue's gives up with it)
                    mx_rows<NT, PLANES, MATS>(C, a, next.first, next.count, kt0, n_it, at, warp - 2, lane, ring);
                    if (item < item0) continue;
                }
            }
            const uint32_t ab = acc == 2 ? n & 1u : 0u, aph = acc == 2 ? (n >> 1) & 1u : n & 1u;
            ++n;
            const int row = I.rt * MX_M + r;
            const bool row_ok = row < a.rows;
            auto bias_of = [&](const float *b, int at) { return b[static_cast<int64_t>(I.expert) * a.rows + at]; };
            const float bu = a.bias && row_ok ? bias_of(a.bias, row) : 0.f;
            const float bg = GLU && a.gate_bias && row_ok ? bias_of(a.gate_bias, row) : 0.f;
            float *out = a.dst + row;
            // lane j: entry of column j of each round, asked for before the wait
            int ens[ROUNDS];
#pragma unroll
            for (int q = 0; q < ROUNDS; ++q) {
                const int c = 16 * (grp + MXP_EPI * q) + (lane & 15);
                ens[q] = c < I.count ? entry_of(I, c) : 0;
            }
            if (!mx_wait_warp(C, &C.acc_full[ab], aph, a)) break;
            tc_fence_after();
            const uint32_t cols = tmem + ab * (MATS * NT) + (static_cast<uint32_t>(32 * quarter) << 16);
            auto column0 = [&](int q) { return 16 * (grp + MXP_EPI * q); };
            auto load = [&](int q, uint32_t (&u)[16], uint32_t (&gt)[16]) {
                if (column0(q) < I.count) {
                    tmem_ld16(cols + column0(q), u);
                    if (GLU) tmem_ld16(cols + NT + column0(q), gt);
                }
            };
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&C.acc_empty[ab]);
            };
            // one round's results in place of its accumulators
            auto finish = [&](uint32_t (&u)[16], uint32_t (&gt)[16]) {
                auto apply = [&](auto op) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        u[j] = __float_as_uint(mx_glu<decltype(op)::value>(__uint_as_float(gt[j]) + bg, __uint_as_float(u[j]) + bu,
                                                                         a.glu_limit));
                };
                if (GLU) {
                    switch (a.glu_op) {
                        case 0: apply(std::integral_constant<int, 0>{}); break;
                        case 1: apply(std::integral_constant<int, 1>{}); break;
                        case 2: apply(std::integral_constant<int, 2>{}); break;
                        case 3: apply(std::integral_constant<int, 3>{}); break;
                        default: apply(std::integral_constant<int, 4>{}); break;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(__uint_as_float(u[j]) + bu);
                }
            };
            auto store = [&](int q, const uint32_t (&u)[16]) {
                // every address first: a shuffle between the stores would hold each store back
                float *at[16];
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    at[j] = out + static_cast<int64_t>(__shfl_sync(0xffffffffu, ens[q], j)) * a.rows;
                const int live = row_ok ? I.count - column0(q) : 0;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (j < live) __stcs(at[j], __uint_as_float(u[j]));   // the weights keep the L2
            };
            if (a.split > 1) {   // this rank's partial sums, for the cluster
                float *part = reinterpret_cast<float *>(ring);
                for (int q = 0; q < ROUNDS && column0(q) < I.count; ++q) {
                    uint32_t u[16], gt[16];
                    load(q, u, gt);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        part[(column0(q) + j) * MX_M + r] = __uint_as_float(u[j]);
                        if (GLU) part[(NT + column0(q) + j) * MX_M + r] = __uint_as_float(gt[j]);
                    }
                }
                release();
            } else {
                uint32_t us[ROUNDS][16], gs[MATS == 2 ? ROUNDS : 1][16];
#pragma unroll
                for (int q = 0; q < ROUNDS; ++q) load(q, us[q], gs[MATS == 2 ? q : 0]);
                tmem_wait_ld();
                release();
#pragma unroll
                for (int q = 0; q < ROUNDS; ++q)
                    if (column0(q) < I.count) {
                        finish(us[q], gs[MATS == 2 ? q : 0]);
                        store(q, us[q]);
                    }
            }
        }
    }
    __syncwarp();
    if (a.split > 1) {
        cluster_sync();
        if (warp >= 2 && *reinterpret_cast<volatile int32_t *>(&C.abort) == 0) {
            const Item I = item_at(item0);
            const int r = (tid - 64) & (MX_M - 1), row = I.rt * MX_M + r;
            if (row < a.rows) {
                const float bu = a.bias ? a.bias[static_cast<int64_t>(I.expert) * a.rows + row] : 0.f;
                const float bg = GLU && a.gate_bias ? a.gate_bias[static_cast<int64_t>(I.expert) * a.rows + row] : 0.f;
                for (int j = rank + a.split * ((tid - 64) / MX_M); j < I.count; j += a.split * MXP_EPI) {
                    float u = 0.f, gt = 0.f;
                    for (int q = 0; q < a.split; ++q) {
                        u += ld_cluster_f32(ring0 + 4 * (j * MX_M + r), q);
                        if (GLU) gt += ld_cluster_f32(ring0 + 4 * ((NT + j) * MX_M + r), q);
                    }
                    u += bu;
                    if (GLU) u = mx_glu_any(a.glu_op, gt + bg, u, a.glu_limit);
                    a.dst[static_cast<int64_t>(entry_of(I, j)) * a.rows + row] = u;
                }
            }
        }
        cluster_sync();   // the partial sums stay until every rank has read them
    }
    if (*reinterpret_cast<volatile int32_t *>(&C.abort) != 0 && warp == 0 && lane == 0) {
        // a wait ran out: let the copies in flight land before the shared memory goes
        const uint64_t lim = drain_limit_ns(a.timeout_ns);
        for (int i = fills > stages ? fills - stages : 0; i < fills; ++i)
            if (!mbar_wait_bounded(&C.full[i % stages], (i / stages) & 1, lim)) set_error(a.err, DERR_DRAIN);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*reinterpret_cast<volatile int32_t *>(&C.abort) != 0 && warp == 1) {
        // whichever warp gave up, the MMAs in flight end before the memory they use goes
        if (on) {
            umma_commit(&C.drain);
            if (!mbar_wait_bounded(&C.drain, 0, drain_limit_ns(a.timeout_ns))) set_error(a.err, DERR_DRAIN);
        }
        __syncwarp();
    }
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}

template <int XT>
void quantize_t(const void *x, int64_t stride, int64_t n_blocks, int nb, int planes, uint8_t *y, cudaStream_t st) {
    using T = typename MxElem<XT>::T;
    const unsigned grid = static_cast<unsigned>((n_blocks + MXQ_BLK - 1) / MXQ_BLK);
    if (mx_vec_ok<XT>(x, stride))
        mx_quantize_kernel<XT, true><<<grid, MXQ_THREADS, 0, st>>>(static_cast<const T *>(x), stride, n_blocks, nb, planes, y);
    else
        mx_quantize_kernel<XT, false><<<grid, MXQ_THREADS, 0, st>>>(static_cast<const T *>(x), stride, n_blocks, nb, planes, y);
}

template <int OT>
void dequantize_t(const uint8_t *y, int64_t n_blocks, int nb, int planes, void *out, int64_t stride, cudaStream_t st) {
    using T = typename MxElem<OT>::T;
    const unsigned grid = static_cast<unsigned>((n_blocks + MXQ_BLK - 1) / MXQ_BLK);
    if (mx_vec_ok<OT>(out, stride))
        mx_dequantize_kernel<OT, true><<<grid, MXQ_THREADS, 0, st>>>(y, n_blocks, nb, planes, stride, static_cast<T *>(out));
    else
        mx_dequantize_kernel<OT, false><<<grid, MXQ_THREADS, 0, st>>>(y, n_blocks, nb, planes, stride, static_cast<T *>(out));
}

template <int XT, bool VEC, int RUN>
cudaError_t images_run(const MxPrep &a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((a.n_rows * ((a.KT + RUN - 1) / RUN) * 16 + 255) / 256));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // overlaps the grouping
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, mx_images_kernel<XT, VEC, RUN>, a);
}

template <int XT, bool VEC>
cudaError_t images_t(const MxPrep &a, cudaStream_t st) {
    // a small call spreads over the SMs
    return a.n_rows * a.KT < 16384 ? images_run<XT, VEC, 1>(a, st) : images_run<XT, VEC, 2>(a, st);
}

template <int XT>
cudaError_t images_x(const MxPrep &a, cudaStream_t st) {
    return mx_vec_ok<XT>(a.x, a.stride) ? images_t<XT, true>(a, st) : images_t<XT, false>(a, st);
}

constexpr uint32_t kSmemMax = 227u * 1024u;

template <int NT, bool GLU, bool DIRECT, int PLANES>
cudaError_t product_p(MxArgs &a, int64_t units, cudaStream_t st) {
    constexpr int MATS = GLU ? 2 : 1, MXP_TPS = mxp_tps<NT>();
    auto kern = mx_product_kernel<NT, GLU, DIRECT, PLANES>;
    constexpr uint32_t fixed = (sizeof(MxCtl<DIRECT ? MX_DIRECT : 1>) + 127u) / 128u * 128u + 1024u;   // static part and the system's 1 KB
    const uint32_t sb = mx_stage_bytes<NT>(MATS, PLANES), sf = MXP_TPS * (4u * MATS + (NT > 128 ? 8u : 4u) * PLANES);
    const bool single = a.split > 1;                 // one item per CTA
    a.acc = single ? 1 : 2;
    const int tiles = (a.KT + a.split - 1) / a.split;
    const int most = single ? (tiles + MXP_TPS - 1) / MXP_TPS : MX_MAX_STAGES;   // stages that would be used
    const uint32_t part = a.split > 1 ? MATS * NT * MX_M * 4u : 0u;
    const uint32_t acc_cols = a.acc * MATS * NT;
    // two CTAs per SM where their accumulators fit in half the tensor memory each, else one
    const uint32_t least = std::min(most, 2);
    const int per_sm = acc_cols + least * sf <= 256u && least * sb <= kSmemMax / 2 - fixed ? 2 : 1;
    int stages = static_cast<int>((kSmemMax / per_sm - fixed) / sb);
    stages = std::min(stages, static_cast<int>((512u / per_sm - acc_cols) / sf));
    stages = std::min(std::min(stages, most), MX_MAX_STAGES);
    a.stages = stages;
    a.tmem_cols = 32;
    while (a.tmem_cols < acc_cols + stages * sf) a.tmem_cols *= 2;
    // shared memory in proportion to the tensor memory: CTAs that fit an SM together never wait for
    // columns, so ranks of a cluster cannot wait for one another through them
    uint32_t smem = std::max(stages * sb, part);
    const uint32_t fair = static_cast<uint32_t>((static_cast<uint64_t>(kSmemMax) * a.tmem_cols + 511) / 512);
    if (smem + fixed < fair) smem = (fair - fixed + 127u) / 128u * 128u;
    int dev = 0, n_sm = 148;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    static int configured[64] = {};   // SMs of a device that knows the kernel's limit
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(kSmemMax - fixed + 1024u));
        if (e != cudaSuccess) return e;
        cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev);
        configured[dev] = n_sm;
    }
    n_sm = configured[dev];
    int64_t grid = units * a.RT * a.split;
    if (!single) grid = std::min<int64_t>(grid, static_cast<int64_t>(n_sm) * per_sm);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(mxp_threads<NT>());
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = static_cast<unsigned>(a.split);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = DIRECT ? 1 : 2;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int NT, bool GLU, bool DIRECT>
cudaError_t product_t(MxArgs &a, int64_t units, cudaStream_t st) {
    return a.planes == 1 ? product_p<NT, GLU, DIRECT, 1>(a, units, st) : product_p<NT, GLU, DIRECT, 2>(a, units, st);
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

// The direct form, while its four quantising warps keep up with the weights. Kernel times of it and of the other
// form's three, added up, GLU, two planes: one token's 8 of 64 experts (K = 2048, 768 rows) 8.6 and 14.9 us, 64 tokens'
// one of 8 experts 14.5 and 15.2, 21 tokens' 3 of 8 (K = 4096, 1536 rows) 25.6 and 21.2, 16 tokens' 4 of 4 28.2 and
// 22.9. (In a replayed graph the three overlap: 8.5 and 12.3, 14.3 and 12.6, 25.2 and 18.3, 27.8 and 19.6; a call
// outside one pays the host for two launches more.)
bool mx_direct(int64_t n_tok, int64_t k, int64_t n_experts, int64_t K) {
    const int64_t n = n_tok * k, most = n < n_experts ? n : n_experts;
    return n <= MX_DIRECT && (n == 0 || std::min<int64_t>((n + most - 1) / most, 16) * K <= MX_DIRECT_VALUES);
}

// Entries per chunk: by the entries an expert has on average. Replayed calls with 16, 64 and the widest chunks, two planes,
// us: gate and up (64 experts, K = 2048, 768 rows) at 8 entries per expert 27.4, 26.0, 27.1, at 16 27.2, 26.9, 27.5, at 36 38.3,
// 30.0, 31.0, at 48 45.3, 31.3, 32.2, at 64 53.1, 35.4, 34.6, at 96 72.4, 46.2, 42.0; down (32 experts, K = 768, 2048 rows) at 8
// 11.3, 12.1, 14.2, at 12 11.9, 12.0, 14.2, at 16 13.6, 12.9, 14.8, at 48 20.0, 15.0, 16.8, at 64 23.5, 17.9, 18.6, at 96 29.2,
// 20.0, 19.6. Picks as a skewed router makes them, at 8: 22.0, 18.7, 19.7 and 11.5, 12.1, 14.4; at 48: 47.2, 33.1, 35.1 and
// 19.9, 15.8, 17.3.
int mx_chunk_tokens(int64_t n_tok, int64_t k, int64_t n_experts, int64_t K, bool glu) {
    const int64_t n = n_tok * k;
    if (mx_direct(n_tok, k, n_experts, K)) return 16;
    const int64_t per = n / (n < n_experts ? n : n_experts);
    return per <= 12 ? 16 : per <= 48 ? 64 : glu ? MXP_WIDE_GLU : MXP_WIDE;
}

int64_t mx_max_experts() { return MXG_MAX_EXPERTS; }

uint64_t mx_images_bytes(int64_t chunks, int NT, int64_t K, int planes) {
    return static_cast<uint64_t>(chunks) * mx_image_bytes(NT, static_cast<int>((K + MX_KT - 1) / MX_KT), planes);
}

cudaError_t launch_mx_prep(const void *x, int xt, int64_t stride, int64_t n_rows, int64_t K, const MxArgs &a, int NT,
                           cudaStream_t st) {
    MxPrep p{};
    p.x = x;
    p.stride = stride;
    p.n_rows = n_rows;
    p.nb = static_cast<int32_t>(K / 32);
    p.KT = a.KT;
    p.planes = a.planes;
    p.per_pick = a.per_pick;
    p.images = const_cast<uint8_t *>(a.images);
    p.ids = a.ids;
    p.ids_stride = a.ids_stride;
    p.n_entries = a.n_entries;
    p.k = a.k;
    p.n_experts = a.n_experts;
    p.NT = NT;
    p.err = a.err;
    p.entries = const_cast<int32_t *>(a.entries);
    p.n_chunks = const_cast<int32_t *>(a.n_chunks);
    p.chunks = const_cast<int4 *>(a.chunks);
    p.where = a.where;
    p.experts = a.experts;
    const size_t smem = (3 + static_cast<size_t>(mx_group_sets(a.n_experts))) * a.n_experts * sizeof(int);   // 64 KB at most
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(mx_group_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   4 * MXG_MAX_EXPERTS * static_cast<int>(sizeof(int)));
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    const int threads = a.n_entries <= 2048 * MXG_CTAS / 8 ? 256 : a.n_entries <= 1024 * MXG_CTAS ? 512 : MXG_THREADS;
    mx_group_kernel<<<MXG_CTAS, threads, smem, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    if (xt == MX_F32) return images_x<MX_F32>(p, st);
    if (xt == MX_F16) return images_x<MX_F16>(p, st);
    return images_x<MX_BF16>(p, st);
}

cudaError_t launch_mx_product(MxArgs &a, int NT, int64_t units, cudaStream_t st) {
    const bool glu = a.gate != nullptr, direct = a.chunks == nullptr;
    // few tiles: a cluster of 2, 4 or 8 CTAs shares a tile's K, until every SM has work (one token's gate
    // and up, K = 2048 and 48 tiles: 10.7 us without, 8.5, 8.6 and 11.9 by clusters of 2, 4 and 8)
    int split = 1;
    if (NT <= 64)
        while (split < 8 && units * a.RT * split < 148 && a.KT / (2 * split) >= 2) split *= 2;
    a.split = split;
    if (NT == 16) {
        if (glu) return direct ? product_t<16, true, true>(a, units, st) : product_t<16, true, false>(a, units, st);
        return direct ? product_t<16, false, true>(a, units, st) : product_t<16, false, false>(a, units, st);
    }
    if (NT == 64) {
        return glu ? product_t<64, true, false>(a, units, st) : product_t<64, false, false>(a, units, st);
    }
    return glu ? product_t<MXP_WIDE_GLU, true, false>(a, units, st) : product_t<MXP_WIDE, false, false>(a, units, st);
}

}  // namespace moe
