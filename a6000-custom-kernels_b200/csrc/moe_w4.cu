// moe_w4.cu -- products of a few tokens with 4-bit matrices that have group scales.
//
//   dst[i][r] = sum over groups of s[r][group] * sum over the group of (q[r][c] - z[r][group]) x[c]
//
// A batch of decode tokens reads every weight once, so the weights' bytes bound it, and the
// instructions between a byte and its product come right behind: at 6.5 TB/s an SM
// takes in a 512-byte tile every 22 cycles, and a scheduler has 88 issue slots for it. Hence
// * mma.sync m16n8k16 with the weights as A, straight from the registers they were unpacked
//   in. Its eight columns are the batch (or the planes of a 32-bit x), so up to eight tokens
//   cost what one does. (tcgen05 would take the weights through tensor memory, and the groups'
//   sums back out of it for their scales.)
// * codes become 16-bit floats by bits: 128 + q in bf16, 1024 + q in f16 are an OR; one
//   subtraction of 128 + z leaves q - z exactly. Products and the sums of a group's 64 values
//   are the tensor cores', in 32 bits; the scale is applied to those, in 32 bits.
// * a 32-bit x is split into three bf16 planes that add up to it exactly (8 + 8 + 8 bits), each
//   a column; 16-bit x are one plane of their own type. So x is never rounded.
// * each lane copies what it will read itself into a ring in shared memory (cp.async, 16 bytes of
//   codes and 4 of scales): no barrier between copy and use, and the ring, not the
//   registers, holds what is in flight.
// * the warps of a CTA share K (sums meet in shared memory in a fixed order), because
//   rows / 16 tiles are too few for the 2368 warps of the GPU.
#include "moe_aux.h"
#include "moe_mx.cuh"
#include "moe_w4.cuh"

#include <cuda_bf16.h>

namespace moe {

namespace {

constexpr int W4_WARPS = 8;
constexpr int W4_THREADS = 32 * W4_WARPS;
constexpr int W4_RED = 20;               // floats between two columns of a warp's sums: no bank conflicts
constexpr int W4_PAD = 64;               // bytes behind a column of x: two columns fill the banks
constexpr int W4_SMEM = 111 * 1024;      // of a CTA: two fit an SM
constexpr int W4_ACC = 16 * 1024;        // of it at most for sums kept over K passes

// ---- layout ----------------------------------------------------------------------
// one thread per word of codes, scales or zeros
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                                      const uint8_t *__restrict__ zeros, int64_t E, int rows, int K, int groups,
                                                      int RT, int KS, int G, uint32_t *out, int64_t n_codes, int64_t n_scales,
                                                      int64_t n_zeros, int *err) {
    const int64_t half_k = (K + 1) / 2;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n_codes + n_scales + n_zeros;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        uint32_t word = 0;
        if (i < n_codes) {
            const int w = static_cast<int>(i & 3), lane = static_cast<int>(i >> 2) & 31, g = lane >> 2, t = lane & 3;
            const int64_t tile = i >> 7;
            const int s = static_cast<int>(tile % KS);
            const int64_t et = tile / KS, e = et / RT;
            const int rt = static_cast<int>(et % RT);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = rt * W4_M + g + 8 * (j & 1), c = s * W4_KT + 32 * (w >> 1) + 8 * t + 4 * (w & 1) + 2 * (j >> 1);
                if (r < rows && c < K) {
                    const uint32_t b = codes[(e * rows + r) * half_k + (c >> 1)];
                    word |= ((b & 15u) << (4 * j)) | ((c + 1 < K ? b >> 4 : 0u) << (16 + 4 * j));
                }
            }
        } else if (i < n_codes + n_scales) {
            const int64_t o = i - n_codes, eg = o >> 3;
            const int g = static_cast<int>(o & 7), gi = static_cast<int>(eg % G);
            const int64_t et = eg / G, e = et / RT;
            const int rt = static_cast<int>(et % RT);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = rt * W4_M + g + 8 * h;
                if (r < rows && gi < groups) word |= static_cast<uint32_t>(scales[(e * rows + r) * groups + gi]) << (16 * h);
            }
        } else {
            const int64_t o = i - n_codes - n_scales, eg = o >> 2;
            const int g2 = static_cast<int>(o & 3), gi = static_cast<int>(eg % G);
            const int64_t et = eg / G, e = et / RT;
            const int rt = static_cast<int>(et % RT);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int r = rt * W4_M + 2 * g2 + (b >> 1) + 8 * (b & 1);
                if (r < rows && gi < groups) {
                    uint32_t z = zeros[(e * rows + r) * groups + gi];
                    if (z > W4_MAX_ZERO) {
                        set_error(err, DERR_BAD_ZERO);
                        z = W4_MAX_ZERO;
                    }
                    word |= z << (8 * b);
                }
            }
        }
        out[i] = word;
    }
}

// ---- product ---------------------------------------------------------------------

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds4(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

template <int T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (T == MX_F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t b, __half2 *) {
    const __half2 r = __hadd2(reinterpret_cast<const __half2 &>(a), reinterpret_cast<const __half2 &>(b));
    return reinterpret_cast<const uint32_t &>(r);
}
__device__ __forceinline__ uint32_t add2(uint32_t a, uint32_t b, __nv_bfloat162 *) {
    const __nv_bfloat162 r = __hadd2(reinterpret_cast<const __nv_bfloat162 &>(a), reinterpret_cast<const __nv_bfloat162 &>(b));
    return reinterpret_cast<const uint32_t &>(r);
}
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(reinterpret_cast<const __half2 &>(a), reinterpret_cast<const __half2 &>(b),
                              reinterpret_cast<const __half2 &>(c));
    return reinterpret_cast<const uint32_t &>(r);
}

// What a group subtracts, for rows g and g + 8: -(128 + z) twice in bf16; -(1024 + z) and -(64 + z) in f16.
template <int T>
struct Zeros {
    uint32_t a[2], b[2];
    // byte 2 (g & 1) + h of the word is row g + 8 h's zero
    __device__ __forceinline__ void set(uint32_t word, bool odd) {
        constexpr uint32_t top = T == MX_F16 ? 0xE4E4E4E4u : 0xC3C3C3C3u;
        a[0] = __byte_perm(word, top, odd ? 0x4242 : 0x4040);
        a[1] = __byte_perm(word, top, odd ? 0x4343 : 0x4141);
        if constexpr (T == MX_F16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) b[h] = add2(a[h], 0x63806380u, static_cast<__half2 *>(nullptr));   // + 960, exact
        }
    }
};

// A word's eight codes as the A fragment of one MMA, less the zeros.
template <int T>
__device__ __forceinline__ void unpack_codes(uint32_t w, const Zeros<T> &z, uint32_t (&a)[4]) {
    if constexpr (T == MX_F16) {
        // 1024 + q from bits 0..3, 1024 + 16 q from bits 4..7 (times 2^-4: 64 + q)
        const uint32_t hi = w >> 8;
        a[0] = add2((w & 0x000F000Fu) | 0x64006400u, z.a[0], static_cast<__half2 *>(nullptr));
        a[1] = fma2((w & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, z.b[1]);
        a[2] = add2((hi & 0x000F000Fu) | 0x64006400u, z.a[0], static_cast<__half2 *>(nullptr));
        a[3] = fma2((hi & 0x00F000F0u) | 0x64006400u, 0x2C002C00u, z.b[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            a[j] = add2(((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u, z.a[j & 1], static_cast<__nv_bfloat162 *>(nullptr));
    }
}

// A warp's way through the tiles of its CTA: chunks (an expert and up to nc entries) x row blocks, the row
// blocks of a run (of one chunk, at most seg of them where K takes several passes) once for each pass,
// the gate's matrix before the other's, then this warp's steps of the pass.
struct Cursor {
    int item, run_end;      // within [item of the run's first block, run_end)
    int run0, pass, mat, s, s_end;
    const uint8_t *codes, *scales, *zeros;
};

struct W4Ctl {              // the direct form's chunks
    int expert[W4_DIRECT], first[W4_DIRECT], count[W4_DIRECT], entry[W4_DIRECT];
    int n;
};

// Groups up to 64 ids, every CTA for itself: experts follow one another as they first appear.
__device__ void w4_group(const W4Args &a, W4Ctl &C, int *ids) {
    const int i = threadIdx.x, n = a.n_entries;
    if (i < n) {
        const int t = i / a.k;
        int id = a.ids[static_cast<int64_t>(t) * a.ids_stride + (i - t * a.k)];
        if (id < 0 || id >= a.n_experts) {
            if (id != -1 && blockIdx.x == 0) set_error(a.err, DERR_BAD_ID);
            id = -1;
        }
        ids[i] = id;
    }
    __syncthreads();
    if (i < n) {
        const int id = ids[i];
        int before = 0, all = 0, first = i;
        for (int j = 0; j < n; ++j) {
            const bool same = ids[j] == id;
            all += same;
            before += same && j < i;
            if (same && j < first) first = j;
        }
        // entries and chunks of the experts that appeared before this one did
        int e0 = 0, c0 = 0;
        for (int j = 0; j < first; ++j) {
            if (ids[j] < 0 || id < 0) continue;
            int seen = 0, cnt = 0;
            for (int q = 0; q < n; ++q) {
                const bool same = ids[q] == ids[j];
                seen += same && q < j;
                cnt += same;
            }
            if (seen == 0) {
                e0 += cnt;
                c0 += (cnt + a.nc - 1) / a.nc;
            }
        }
        if (id >= 0) {
            C.entry[e0 + before] = i;
            if (before % a.nc == 0) {
                const int c = c0 + before / a.nc;
                C.expert[c] = id;
                C.first[c] = e0 + before;
                C.count[c] = min(a.nc, all - before);
            }
            atomicMax(&C.n, c0 + (all + a.nc - 1) / a.nc);
        }
    }
    __syncthreads();
}

template <int T, int NT, bool ZERO, bool G32>
__global__ void __launch_bounds__(W4_THREADS, 2) w4_kernel(const __grid_constant__ W4Args a) {
    constexpr int D = NT == 1 ? 8 : NT == 2 ? 6 : 4;                     // tiles in flight per warp
    constexpr int GW = G32 ? 2 : 1;                                      // groups of a tile
    constexpr uint32_t STAGE = W4_TILE + 128 * GW * (ZERO ? 2 : 1);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ W4Ctl C;
    __shared__ int ids[W4_DIRECT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int WK = 1 << a.wk_shift, wk = warp & (WK - 1), wm = warp >> a.wk_shift, WM = W4_WARPS >> a.wk_shift;
    int n_chunks;
    if (a.chunks) {
        n_chunks = *a.n_chunks;
    } else if (!a.ids) {
        n_chunks = (a.n_entries + a.nc - 1) / a.nc;
    } else {
        if (tid == 0) C.n = 0;
        w4_group(a, C, ids);
        n_chunks = C.n;
    }
    const int items = n_chunks * a.tiles;
    const int i0 = static_cast<int>(static_cast<int64_t>(items) * blockIdx.x / gridDim.x);
    const int i1 = static_cast<int>(static_cast<int64_t>(items) * (blockIdx.x + 1) / gridDim.x);
    if (i0 == i1) return;

    auto expert_of = [&](int c) { return a.chunks ? a.chunks[c].x : a.ids ? C.expert[c] : 0; };
    auto first_of = [&](int c) { return a.chunks ? a.chunks[c].y : a.ids ? C.first[c] : c * a.nc; };
    auto count_of = [&](int c) {
        return a.chunks ? a.chunks[c].z : a.ids ? C.count[c] : min(a.nc, a.n_entries - c * a.nc);
    };
    auto run_of = [&](int item) {   // the run's end
        const int end = min(i1, (item / a.tiles + 1) * a.tiles);
        return a.passes > 1 ? min(end, item + a.seg) : end;
    };
    auto steps_of = [&](int pass) { return min(a.KS, (pass + 1) * a.sp); };   // the pass's end

    // prefetch
    const uint32_t ring = smem_u32(smem) + warp * D * STAGE;
    Cursor P{};
    auto seek = [&]() {   // the matrices' addresses at the cursor
        const int chunk = P.item / a.tiles, rt = min((P.item - chunk * a.tiles) * WM + wm, a.RT - 1);
        const int64_t row = static_cast<int64_t>(expert_of(chunk)) * a.RT + rt;
        const W4Matrix &m = a.w[P.mat];
        P.s = P.pass * a.sp + wk;
        P.s_end = steps_of(P.pass);
        P.codes = m.codes + (row * a.KS + P.s) * W4_TILE + 16 * lane;
        P.scales = m.scales + row * a.G * 32 + 4 * g;
        if (ZERO) P.zeros = m.zeros + row * a.G * 16 + 4 * (g >> 1);
    };
    auto next = [&]() {   // the next matrix, row block, pass or run; false behind the last
        if (++P.mat < a.mats) return true;
        P.mat = 0;
        if (++P.item < P.run_end) return true;
        if (++P.pass < a.passes) {
            P.item = P.run0;
            return true;
        }
        P.pass = 0;
        if (P.item >= i1) return false;
        P.run0 = P.item;
        P.run_end = run_of(P.item);
        return true;
    };
    bool more = true;
    P.item = P.run0 = i0;
    P.run_end = run_of(i0);
    P.pass = P.mat = 0;
    seek();
    auto fetch = [&](int slot) {
        while (more && P.s >= P.s_end) {
            more = next();
            if (more) seek();
        }
        if (more) {
            const uint32_t at = ring + slot * STAGE;
            cp16(at + 16 * lane, P.codes);
#pragma unroll
            for (int h = 0; h < GW; ++h) {
                const int gi = G32 ? 2 * P.s + h : P.s >> a.gshift;
                cp4(at + W4_TILE + 128 * h + 4 * lane, P.scales + 32 * static_cast<int64_t>(gi));
                if (ZERO) cp4(at + W4_TILE + 128 * (GW + h) + 4 * lane, P.zeros + 16 * static_cast<int64_t>(gi));
            }
            P.codes += static_cast<int64_t>(WK) * W4_TILE;
            P.s += WK;
        }
        cp_commit();
    };
#pragma unroll
    for (int d = 0; d < D; ++d) fetch(d);

    float *red = reinterpret_cast<float *>(smem + a.red_off);
    float *acc = reinterpret_cast<float *>(smem + a.acc_off);
    const int pitch = 2 * W4_KT * a.sp + W4_PAD;   // bytes of a staged column
    const uint32_t xs = smem_u32(smem) + a.x_off;
    constexpr uint32_t RED_BUF = W4_WARPS * NT * 8 * W4_RED;
    int slot = 0, buf = 0;

    for (int run0 = i0; run0 < i1;) {
        const int run_end = run_of(run0), chunk = run0 / a.tiles, count = count_of(chunk), first = first_of(chunk);
        const int expert = expert_of(chunk), cols = count * a.planes;
        for (int pass = 0; pass < a.passes; ++pass) {
            const int s0 = pass * a.sp, s1 = steps_of(pass);
            __syncthreads();   // everyone is done with the x of the pass before
            {
                const int per = (s1 - s0) * (W4_KT / 8), n = per * count;
                for (int v = tid; v < n; v += W4_THREADS) {
                    const int col = v / per, c8 = v - col * per, kk = s0 * W4_KT + 8 * c8;
                    int entry = first + col;
                    if (a.chunks) entry = a.entries[entry];
                    else if (a.ids) entry = C.entry[entry];
                    const int64_t row = a.per_pick ? entry : entry / a.k;
                    uint8_t *to = smem + a.x_off + static_cast<int64_t>(col) * a.planes * pitch + 16 * c8;
                    if (a.x_type == MX_F32) {
                        const float *src = static_cast<const float *>(a.x) + row * a.x_stride + kk;
                        float f[8];
                        if (a.x_vec && kk + 8 <= a.K) {
                            *reinterpret_cast<float4 *>(f) = *reinterpret_cast<const float4 *>(src);
                            *reinterpret_cast<float4 *>(f + 4) = *reinterpret_cast<const float4 *>(src + 4);
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) f[i] = kk + i < a.K ? src[i] : 0.f;
                        }
                        uint32_t p[3][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                // by truncation: 8 bits, the next 8, the last 8. A NaN keeps a quiet payload
                                const float v0 = f[2 * i + h];
                                const bool fin = fabsf(v0) < INFINITY;
                                uint32_t u0 = __float_as_uint(v0) & 0xFFFF0000u;
                                if (v0 != v0) u0 |= 0x00400000u;
                                const float r1 = fin ? v0 - __uint_as_float(u0) : 0.f;
                                const uint32_t u1 = __float_as_uint(r1) & 0xFFFF0000u;
                                const uint32_t u2 = __float_as_uint(r1 - __uint_as_float(u1));
                                p[0][i] = h ? p[0][i] | u0 : u0 >> 16;
                                p[1][i] = h ? p[1][i] | u1 : u1 >> 16;
                                p[2][i] = h ? p[2][i] | (u2 & 0xFFFF0000u) : u2 >> 16;
                            }
                        }
#pragma unroll
                        for (int q = 0; q < 3; ++q)
                            *reinterpret_cast<uint4 *>(to + q * pitch) = make_uint4(p[q][0], p[q][1], p[q][2], p[q][3]);
                    } else {
                        const uint16_t *src = static_cast<const uint16_t *>(a.x) + row * a.x_stride + kk;
                        uint4 q;
                        if (a.x_vec && kk + 8 <= a.K) {
                            q = *reinterpret_cast<const uint4 *>(src);
                        } else {
                            uint32_t h[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) h[i] = kk + i < a.K ? src[i] : 0u;
                            q = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
                        }
                        *reinterpret_cast<uint4 *>(to) = q;
                    }
                }
            }
            __syncthreads();
            for (int item = run0; item < run_end; ++item) {
                for (int mat = 0; mat < a.mats; ++mat) {
                    float sum[NT][4] = {};
                    for (int s = s0 + wk; s < s1; s += WK) {
                        cp_wait<D - 1>();
                        const uint32_t at = ring + slot * STAGE;
                        const uint4 w = lds16(at + 16 * lane);
                        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                        uint32_t A[4][4];
                        float sc[GW][2];
#pragma unroll
                        for (int h = 0; h < GW; ++h) {
                            const uint32_t sw = lds4(at + W4_TILE + 128 * h + 4 * lane);
                            if (a.scale_type == W4_BF16) {
                                sc[h][0] = __uint_as_float(sw << 16);
                                sc[h][1] = __uint_as_float(sw & 0xFFFF0000u);
                            } else {
                                const float2 f = __half22float2(reinterpret_cast<const __half2 &>(sw));
                                sc[h][0] = f.x;
                                sc[h][1] = f.y;
                            }
                            Zeros<T> z;
                            z.set(ZERO ? lds4(at + W4_TILE + 128 * (GW + h) + 4 * lane) : 0x08080808u, ZERO && (g & 1));
#pragma unroll
                            for (int i = 4 / GW * h; i < 4 / GW * (h + 1); ++i) unpack_codes<T>(words[i], z, A[i]);
                        }
                        const uint32_t xk = xs + (s - s0) * 2 * W4_KT + 16 * t;
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            if (NT > 1 && 8 * j >= cols) break;
                            // (columns past the last repeat the first one's: nothing reads their sums)
                            const uint32_t xc = xk + (8 * j + g < cols ? 8 * j + g : 0) * pitch;
                            const uint4 b0 = lds16(xc), b1 = lds16(xc + 64);
#pragma unroll
                            for (int h = 0; h < GW; ++h) {
                                float d[4] = {};
                                if (GW == 1 || h == 0) {
                                    mma<T>(d, A[0], b0.x, b0.y);
                                    mma<T>(d, A[1], b0.z, b0.w);
                                }
                                if (GW == 1 || h == 1) {
                                    mma<T>(d, A[2], b1.x, b1.y);
                                    mma<T>(d, A[3], b1.z, b1.w);
                                }
#pragma unroll
                                for (int i = 0; i < 4; ++i) sum[j][i] = fmaf(sc[h][i >> 1], d[i], sum[j][i]);
                            }
                        }
                        fetch(slot);
                        slot = slot + 1 == D ? 0 : slot + 1;
                    }
                    // the warps' sums meet
                    float *mine = red + buf * RED_BUF + warp * NT * 8 * W4_RED;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) mine[(8 * j + 2 * t + (i & 1)) * W4_RED + g + 8 * (i >> 1)] = sum[j][i];
                    __syncthreads();
                    const int outs = count * WM * W4_M;
                    const bool last = pass + 1 == a.passes;
                    const int tile = item - chunk * a.tiles;
                    float *keep = acc + ((a.passes > 1 ? item - run0 : 0) * a.mats + mat) * a.nc * WM * W4_M;
                    for (int o = tid; o < outs; o += W4_THREADS) {
                        const int r = o & (W4_M - 1), m = (o >> 4) & (WM - 1), col = o >> (4 + 3 - a.wk_shift);
                        const float *from = red + buf * RED_BUF + (m << a.wk_shift) * NT * 8 * W4_RED + r;
                        float v = 0.f;
                        for (int q = a.planes - 1; q >= 0; --q)   // the small planes first
                            for (int w = 0; w < WK; ++w) v += from[(w * NT * 8 + col * a.planes + q) * W4_RED];
                        if (pass > 0) v += keep[o];
                        if (!last || mat + 1 < a.mats) {
                            keep[o] = v;
                            continue;
                        }
                        const int row = (tile * WM + m) * W4_M + r;
                        if (row >= a.rows) continue;
                        int entry = first + col;
                        if (a.chunks) entry = a.entries[entry];
                        else if (a.ids) entry = C.entry[entry];
                        const int64_t b = static_cast<int64_t>(expert) * a.rows + row;
                        if (a.mats > 1) {
                            float gate = keep[o - a.nc * WM * W4_M];
                            if (a.bias[0]) gate += a.bias[0][b];
                            if (a.bias[1]) v += a.bias[1][b];
                            v = mx_glu_any(a.glu_op, gate, v, a.glu_limit);
                        } else if (a.bias[0]) {
                            v += a.bias[0][b];
                        }
                        a.dst[static_cast<int64_t>(entry) * a.rows + row] = v;
                    }
                    if (NT > 2) __syncthreads();   // one buffer
                    else buf ^= 1;
                }
            }
        }
        run0 = run_end;
    }
    cp_wait<0>();
}

template <int T, int NT, bool ZERO, bool G32>
cudaError_t w4_t(W4Args &a, int64_t max_chunks, cudaStream_t st) {
    constexpr int D = NT == 1 ? 8 : NT == 2 ? 6 : 4;
    constexpr uint32_t STAGE = W4_TILE + 128 * (G32 ? 2 : 1) * (ZERO ? 2 : 1);
    constexpr uint32_t ring = W4_WARPS * D * STAGE, red = (NT > 2 ? 1 : 2) * W4_WARPS * NT * 8 * W4_RED * 4;
    // warps that share K: at least three tiles each
    a.wk_shift = a.KS >= 24 ? 3 : a.KS >= 12 ? 2 : a.KS >= 6 ? 1 : 0;
    const int WM = W4_WARPS >> a.wk_shift, WK = 1 << a.wk_shift;
    a.tiles = (a.RT + WM - 1) / WM;
    const uint32_t one = static_cast<uint32_t>(a.nc * WM * W4_M * a.mats) * 4;     // a row block's sums
    const int cols = (a.n_entries < a.nc ? a.n_entries : a.nc) * a.planes;
    const uint32_t room = W4_SMEM - ring - red - (a.mats > 1 ? one : 0);
    const int fit = static_cast<int>((room / cols - W4_PAD) / (2 * W4_KT));
    a.passes = 1;
    a.seg = 1;
    a.sp = a.KS;
    uint32_t acc = a.mats > 1 ? one : 0;
    if (fit < a.KS) {
        acc = one > W4_ACC ? one : W4_ACC / one * one;
        a.seg = static_cast<int32_t>(acc / one);
        int sp = static_cast<int>(((W4_SMEM - ring - red - acc) / cols - W4_PAD) / (2 * W4_KT));
        sp = sp / WK * WK;
        if (sp < 1) return cudaErrorInvalidConfiguration;
        a.passes = (a.KS + sp - 1) / sp;
        a.sp = (a.KS + a.passes - 1) / a.passes;
        a.sp = (a.sp + WK - 1) / WK * WK;
        a.passes = (a.KS + a.sp - 1) / a.sp;
    }
    a.red_off = ring;
    a.acc_off = ring + red;
    a.x_off = (ring + red + acc + 15) / 16 * 16;
    const size_t smem = a.x_off + static_cast<size_t>(cols) * (2 * W4_KT * a.sp + W4_PAD);
    static bool configured[64] = {};
    int dev = 0, n_sm = 148;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev);
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(w4_kernel<T, NT, ZERO, G32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   W4_SMEM + 16);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    const int64_t items = max_chunks * a.tiles;
    const int64_t grid = items < 2 * n_sm ? items : 2 * n_sm;
    w4_kernel<T, NT, ZERO, G32><<<static_cast<unsigned>(grid), W4_THREADS, smem, st>>>(a);
    return cudaGetLastError();
}

template <int T, int NT>
cudaError_t w4_nt(W4Args &a, int64_t max_chunks, bool g32, cudaStream_t st) {
    const bool zero = a.w[0].zeros != nullptr;
    if (zero) return g32 ? w4_t<T, NT, true, true>(a, max_chunks, st) : w4_t<T, NT, true, false>(a, max_chunks, st);
    return g32 ? w4_t<T, NT, false, true>(a, max_chunks, st) : w4_t<T, NT, false, false>(a, max_chunks, st);
}

// MMA columns of 8: as few as hold a call's rows, for experts the average load and a half
int w4_tiles_n(int64_t n_tok, int64_t k, int64_t n_experts, bool one_matrix, int planes) {
    int64_t most = n_tok;
    if (!one_matrix) {
        const int64_t mean = (3 * n_tok * k + 2 * n_experts - 1) / (2 * n_experts);
        most = mean < n_tok ? mean : n_tok;
    }
    return most * planes <= 8 ? 1 : most * planes <= 16 ? 2 : 4;
}

}  // namespace

int w4_chunk_entries(int64_t n_tok, int64_t k, int64_t n_experts, bool one_matrix, int x_type) {
    const int planes = x_type == MX_F32 ? 3 : 1;
    return 8 * w4_tiles_n(n_tok, k, n_experts, one_matrix, planes) / planes;
}

cudaError_t launch_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int64_t E, int64_t rows, int64_t K,
                           int64_t groups, int64_t G, uint8_t *out, int *err, cudaStream_t st) {
    const int64_t RT = (rows + W4_M - 1) / W4_M, KS = (K + W4_KT - 1) / W4_KT;
    const int64_t nc = E * RT * KS * (W4_TILE / 4), ns = E * RT * G * 8, nz = zeros ? E * RT * G * 4 : 0;
    const int64_t blocks = (nc + ns + nz + 255) / 256;
    w4_pack_kernel<<<static_cast<unsigned>(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, st>>>(
        codes, static_cast<const uint16_t *>(scales), zeros, E, static_cast<int>(rows), static_cast<int>(K),
        static_cast<int>(groups), static_cast<int>(RT), static_cast<int>(KS), static_cast<int>(G),
        reinterpret_cast<uint32_t *>(out), nc, ns, nz, err);
    return cudaGetLastError();
}

cudaError_t launch_w4(W4Args &a, int64_t n_tok, int64_t max_chunks, bool g32, cudaStream_t st) {
    a.planes = a.x_type == MX_F32 ? 3 : 1;
    const int NT = w4_tiles_n(n_tok, a.k, a.n_experts, a.ids == nullptr, a.planes);
    a.nc = 8 * NT / a.planes;
    if (a.x_type == MX_F16) {
        if (NT == 1) return w4_nt<MX_F16, 1>(a, max_chunks, g32, st);
        return NT == 2 ? w4_nt<MX_F16, 2>(a, max_chunks, g32, st) : w4_nt<MX_F16, 4>(a, max_chunks, g32, st);
    }
    if (NT == 1) return w4_nt<MX_BF16, 1>(a, max_chunks, g32, st);
    return NT == 2 ? w4_nt<MX_BF16, 2>(a, max_chunks, g32, st) : w4_nt<MX_BF16, 4>(a, max_chunks, g32, st);
}

}  // namespace moe
