// moe_w4.cu -- products of a few tokens with 4-bit matrices that have group scales.
//
//   dst[i][r] = sum over groups of s[r][group] * sum over the group of (q[r][c] - z[r][group]) x[c]
//
// A batch of decode tokens reads every weight once, so the weights' bytes would bound it, but the
// instructions between a byte and its product come right behind: at 6.5 TB/s an SM takes in 512
// bytes (1024 codes) every 22 cycles, and a scheduler has 88 issue slots for them. Hence
// * mma.sync m16n8k16 in f16 with the weights as A, straight from the registers they were unpacked
//   in. Its eight columns are the batch, so up to eight tokens cost what one does. (tcgen05 would
//   take the weights through tensor memory, and the groups' sums back out of it for their scales.)
// * four bits in an f16's mantissa are a number as they are: the subnormal q 2^-22 at bits 2 to 5, q 2^-18 at bits 6
//   to 9 (the tile's other eight rows). So unpacking eight codes is four ANDs and a rotation; the powers of two
//   come off at the end. The tensor cores line products up by their exponents, so zeros ahead of a subnormal's
//   bits cost the sums as many of theirs: at bits 0 and 4 results were off by 1e-6, here by 3e-7.
// * zeros: sum (q - z) x = sum q x - z sum x. The sums of x per group are made once, when x is staged
//   (32 bits; errors are relative to sum |s| (q + z) |x|: about one bit more than with (q - z) x where x is of one size and
//   zeros are codes; a large x on a code that is its zero, or zeros up to 127, cost more).
// * x: f16 as it is. bf16 times a power of two per 256 values, so that their largest is just below
//   2^15: what f16 then cuts off is below 2^-39 of that largest. f32 likewise in two planes (two columns)
//   of 11 bits each, off by 2^-22 of the value at most. Everything behind the products is in 32 bits.
// * a warp copies what it will read itself into a ring in shared memory (cp.async): no barrier
//   between copy and use but the warp's, and the ring, not the registers, holds what is in
//   flight. A stage is 16 rows x 256 values with their scales and zeros, one piece of memory.
// * warps that share no K need no barrier; where rows are few, the warps of a CTA, and where rows are
//   very few or x is large the CTAs of a cluster, share K (the sums meet in shared memory, in a fixed
//   order), and a CTA then holds its share of x only.
// Measured (one B200, us per call among others, bytes of the weights a second): 32768 x 4096, groups of 64 with zeros, one
// bf16 token 18.0 (4.0 TB/s); 64 tokens' 8 of 64 experts, gate and up of 1024 x 2048 52.3 (2.0 TB/s of the 47 experts' that picks
// drawn with a skew touch); 4096 x 4096, groups of 32 with zeros, 24 f16 tokens 14.3; 768 x 2048, one f32 token 3.0 in a
// graph (weights in L2: latency).
// The first: 322 warp instructions per stage, 58 % of the active cycles' issue slots (46 % of all) with 3.7 warps per scheduler,
// the ALU 47 %, the tensor pipe 22 %, DRAM 42 %: warps wait for issue, for fixed latencies and for the math pipes. The
// second leaves a third of the SMs' time idle: a CTA's share is a number of blocks, which cost more the more rows a chunk has
// (cycles at work 38 k to 93 k of 100 k).
#include "moe_aux.h"
#include "moe_mx.cuh"
#include "moe_mmq.cuh"
#include "moe_w4.cuh"

#include <type_traits>
#include <cstring>

namespace moe {

namespace {

constexpr int W4_WARPS = 16;             // of a CTA, one to an SM: x lies there once
constexpr int W4_RED = 20;               // floats between two columns of a warp's sums: no bank conflicts
constexpr int W4_PAD = 64;               // bytes behind a column of x: two columns fill the banks
constexpr int W4_SMEM = 224 * 1024;
constexpr int W4_ACC = 8 * 1024;         // of it at most for sums kept to a run's end, where one block's fit
constexpr float W4_CODE = 0x1p-22f;      // a code's unit in rows g (times 16 in rows g + 8)
constexpr float W4_UP = 2048.f;          // which comes off in two factors: with x's power of two, and at the end
constexpr float W4_PLANE = 4096.f;       // the second plane of an f32 x holds what the first one leaves, times this

// What plans count with, in us: a stage of each of the warps that share an SM's issue slots, of one by itself, adding up a block
constexpr float W4_STAGE = 0.0596f, W4_STAGE_ALONE = 0.325f, W4_BLOCK_US = 0.8f;
__host__ __device__ __forceinline__ float w4_stage_us(int warps) { return W4_STAGE * warps * powf(16.f / warps, 0.3f); }

// stages in flight per warp
template <int NT>
__host__ __device__ constexpr int w4_stages() { return NT == 1 ? 3 : 2; }

// ---- layout ----------------------------------------------------------------------
// one thread per word
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t *__restrict__ codes, const uint16_t *__restrict__ scales,
                                                      const uint8_t *__restrict__ zeros, int rows, int K, int group, int groups,
                                                      int RT, int KS, int per_stage, uint32_t *out, int64_t n, int *err) {
    const int64_t half_k = (K + 1) / 2;
    const int words = w4_stage_bytes(per_stage, zeros != nullptr) / 4;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        uint32_t word = 0;
        const int64_t stage = i / words, et = stage / KS, e = et / RT;
        const int s = static_cast<int>(stage - et * KS), r0 = static_cast<int>(et - e * RT) * W4_M;
        int o = static_cast<int>(i - stage * words);
        if (o < W4_CODES / 4) {
            const int w = o & 3, lane = (o >> 2) & 31, g = lane >> 2, t = lane & 3;
            const int c0 = s * W4_KS + (o >> 7) * W4_KT + 32 * (w >> 1) + 8 * t + 4 * (w & 1);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r0 + g + 8 * (j & 1), c = c0 + 2 * (j >> 1);
                if (r < rows && c < K) {
                    const uint32_t b = codes[(e * rows + r) * half_k + (c >> 1)];
                    const uint32_t hi = c + 1 < K ? b >> 4 : 0u;
                    word |= ((b & 15u) << (2 + 4 * j)) | __funnelshift_l(hi, hi, 18 + 4 * j);
                }
            }
        } else {
            o -= W4_CODES / 4;
            const bool zero = o >= 8 * per_stage;
            if (zero) o -= 8 * per_stage;
            const int gi_stage = zero ? o >> 2 : o >> 3;
            const int64_t c = static_cast<int64_t>(s) * W4_KS + gi_stage * (W4_KS / per_stage);
            const int64_t gi = c / group;
            if (c < K && !zero) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = r0 + (o & 7) + 8 * h;
                    if (r < rows) word |= static_cast<uint32_t>(scales[(e * rows + r) * groups + gi]) << (16 * h);
                }
            } else if (c < K) {
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int r = r0 + 2 * (o & 3) + (b >> 1) + 8 * (b & 1);
                    if (r >= rows) continue;
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
// (those not committed to a group, too)
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ uint4 lds16(const uint8_t *p) { return *reinterpret_cast<const uint4 *>(p); }
__device__ __forceinline__ uint32_t lds4(const uint8_t *p) { return *reinterpret_cast<const uint32_t *>(p); }

// d = a b + c; the first of a chain starts from zeros
template <bool FIRST>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (FIRST)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A word's eight codes as the A fragment of one MMA: rows g as q 2^-22, rows g + 8 as q 2^-18
__device__ __forceinline__ void unpack_codes(uint32_t w, uint32_t (&a)[4]) {
    const uint32_t r = __funnelshift_r(w, w, 8);
    a[0] = w & 0x003C003Cu;
    a[1] = w & 0x03C003C0u;
    a[2] = r & 0x003C003Cu;
    a[3] = r & 0x03C003C0u;
}

// Behind w4_pack_kernel and any other kernel that writes packed bytes. A product may start when the blocks of the kernel before
// it have ended, and what those wrote is only sure to be seen behind dep_wait, but products read the matrices ahead of it. This
// launch is an ordinary one: it starts when what is before it is complete, and a product behind it later still. (Matrices
// read behind dep_wait, only brought to the L2 ahead of it, would need none: us in a graph 3.1 -> 3.7 for 768 x 2048 and one
// f32 token, 17.6 -> 18.4 for 32768 x 4096 and one bf16 token, 5.6 -> 6.1 for 4096 x 4096.)
__global__ void w4_settled_kernel() {}

// Programmatic dependent launch: calls follow one another without the gap between kernels. Behind dep_wait everything
// before this kernel in the stream is complete; ahead of it nothing is read but the matrices, which launch_w4_settle has
// settled, and by a product behind w4_stage_kernel the ids, which that one has waited for.
__device__ __forceinline__ void dep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ void w4_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster(uint32_t saddr, int rank) {
    uint32_t a;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

// Groups up to W4_DIRECT picks, every CTA for itself: entry[] by (expert, pick), chunk[] = {expert | count << 16,
// first entry}; returns the number of chunks. Every CTA has to find the same order, so counts belong to
// warps (count[W4_WARPS][E], scratch) and a warp's picks are ranked by its ballots.
// Only the warps that hold picks are counted up, in rolled loops (us in a graph, all 16 warps / these, both built and timed in
// turn: 4 tokens' 8 of 1000 experts 9.7 / 8.5, 3 tokens' 8 of 64 13.6 / 13.3, 8 tokens' 8 of 64 15.7 / 15.5, one token's 11.1 /
// 10.9; 64 tokens' 8 of 64 52.4 / 52.7). One warp that orders up to 64 picks by ballots instead was 0.4 to 0.7 faster for three
// calls, but the longer kernel took 3 % from the last.
__device__ int w4_group(const W4Args &a, int2 *chunk, uint16_t *entry, int *count) {
    __shared__ int warp_sum[W4_WARPS];
    constexpr int THREADS = 32 * W4_WARPS, PER = W4_DIRECT / THREADS, EPT = W4_MAX_EXPERTS / THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n_entries, E = a.n_experts;
    const int held = (n + 32 * PER - 1) / (32 * PER);   // warps that hold picks: few, mostly
    for (int e = tid; e < held * E; e += THREADS) count[e] = 0;
    __syncthreads();
    int id[PER], at[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const int i = (warp * PER + u) * 32 + lane;
        id[u] = -1;
        if (i < n) {
            const int t = i / a.k;
            id[u] = a.ids[static_cast<int64_t>(t) * a.ids_stride + (i - t * a.k)];
            if (id[u] < 0 || id[u] >= E) {
                if (id[u] != -1 && blockIdx.x == 0) set_error(a.err, DERR_BAD_ID);
                id[u] = -1;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        if ((warp * PER + u) * 32 >= n) break;
        const unsigned peers = __match_any_sync(0xffffffffu, id[u]);
        const int leader = __ffs(peers) - 1;
        int before = 0;
        if (id[u] >= 0 && lane == leader) {
            before = count[warp * E + id[u]];
            count[warp * E + id[u]] = before + __popc(peers);
        }
        at[u] = __shfl_sync(0xffffffffu, before, leader) + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
    }
    __syncthreads();
    // first entries and first chunks: scans over the experts, EPT consecutive ones per thread (halves of a word)
    int c[EPT], sum = 0;
#pragma unroll
    for (int u = 0; u < EPT; ++u) {
        const int e = EPT * tid + u;
        c[u] = 0;
        if (e < E)
#pragma unroll 1
            for (int w = 0; w < held; ++w) c[u] += count[w * E + e];
        sum += c[u] + ((c[u] + a.nc - 1) / a.nc << 16);
    }
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int at0 = incl - sum, total = 0;
#pragma unroll
    for (int w = 0; w < W4_WARPS; ++w) {
        at0 += w < warp ? warp_sum[w] : 0;
        total += warp_sum[w];
    }
#pragma unroll
    for (int u = 0; u < EPT; ++u) {
        const int e = EPT * tid + u;
        if (e >= E) break;
        int first = at0 & 0xFFFF, q = at0 >> 16, next = first;
        at0 += c[u] + ((c[u] + a.nc - 1) / a.nc << 16);
#pragma unroll 1
        for (int w = 0; w < held; ++w) {
            const int mine = count[w * E + e];
            count[w * E + e] = next;
            next += mine;
        }
        for (int left = c[u]; left > 0; left -= a.nc, first += a.nc)
            chunk[q++] = make_int2(e | min(left, a.nc) << 16, first);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < PER; ++u)
        if (id[u] >= 0) entry[count[warp * E + id[u]] + at[u]] = static_cast<uint16_t>((warp * PER + u) * 32 + lane);
    __syncthreads();
    return total >> 16;
}

// A warp brings 256 values of a row of x (from kk on, zeros behind K) to shared memory, eight per lane: the column (two,
// pitch bytes apart, for f32), the sums of its groups (negative, in units of the codes', gap floats apart) and
// the power of two that takes the column's products back. A NaN or an infinity makes the sums NaN, and so the row's outputs.
template <int GROUPS>
__device__ __forceinline__ void stage_x(const W4Args &a, int64_t row, int kk, int lane, uint8_t *to, int pitch, float *sums,
                                        float *back, int gap) {
    kk += 8 * lane;
    float v[8];
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (a.x_type == MX_F32) {
        const float *src = static_cast<const float *>(a.x) + row * a.x_stride + kk;
        if (a.x_vec && kk + 8 <= a.K) {
            *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(src);
            *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(src + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = kk + i < a.K ? src[i] : 0.f;
        }
    } else {
        const uint16_t *src = static_cast<const uint16_t *>(a.x) + row * a.x_stride + kk;
        if (a.x_vec && kk + 8 <= a.K) {
            raw = *reinterpret_cast<const uint4 *>(src);
        } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = kk + i < a.K ? src[i] : 0u;
            raw = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
        }
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (a.x_type == MX_BF16) {
                v[2 * i] = __uint_as_float(words[i] << 16);
                v[2 * i + 1] = __uint_as_float(words[i] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(reinterpret_cast<const __half2 &>(words[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
    uint32_t top = 0;
    bool odd = false;   // a NaN or an infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool fin = fabsf(v[i]) < INFINITY;
        odd |= !fin;
        v[i] = fin ? v[i] : 0.f;
        top = max(top, __float_as_uint(fabsf(v[i])));
    }
    odd = __any_sync(0xffffffffu, odd);
    int e = 0;
    if (a.x_type != MX_F16) {
        // the largest to [2^14, 2^15); above 2^-106 (values that small lose f16's subnormals at 2^-144)
        top = __reduce_max_sync(0xffffffffu, top);
        e = top ? min(141 - static_cast<int>(top >> 23), 120) : 0;
        const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        uint32_t h[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= up;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 p = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            h[i] = reinterpret_cast<const uint32_t &>(p);
        }
        raw = make_uint4(h[0], h[1], h[2], h[3]);
        if (a.x_type == MX_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(reinterpret_cast<const __half2 &>(h[i]));
                const __half2 p = __floats2half2_rn((v[2 * i] - f.x) * W4_PLANE, (v[2 * i + 1] - f.y) * W4_PLANE);
                h[i] = reinterpret_cast<const uint32_t &>(p);
                const float2 l = __half22float2(p);   // the sums are of what the planes hold
                v[2 * i] = fmaf(l.x, 1.f / W4_PLANE, f.x);
                v[2 * i + 1] = fmaf(l.y, 1.f / W4_PLANE, f.y);
            }
            *reinterpret_cast<uint4 *>(to + pitch + 16 * lane) = make_uint4(h[0], h[1], h[2], h[3]);
        }
    } else if (odd) {
        raw = make_uint4(0, 0, 0, 0);
    }
    *reinterpret_cast<uint4 *>(to + 16 * lane) = raw;
    float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
#pragma unroll
    for (int off = 1; off < 32 / GROUPS; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane % (32 / GROUPS) == 0) {
        sums[lane / (32 / GROUPS) * gap] = odd ? NAN : sum * -W4_CODE;
        if (a.x_type == MX_F32) sums[lane / (32 / GROUPS) * gap + 1] = 0.f;
    }
    if (lane == 0) {
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        back[0] = down * W4_UP;
        if (a.x_type == MX_F32) back[1] = down * (W4_UP / W4_PLANE);
    }
}

// The rows of x brought into that form once, for calls whose CTAs would all do it for the same rows: a unit per row and
// stage, planes x 512 bytes of columns, then [GROUPS + 1][planes] floats. One warp per unit.
template <int GROUPS>
__global__ void __launch_bounds__(256) w4_stage_kernel(const __grid_constant__ W4Args a, int64_t units, uint8_t *out) {
    dep_wait();
    dep_launch();   // (the product comes up meanwhile; what this call reads is complete then)
    const int64_t u = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (u >= units) return;
    const int64_t row = u / a.KS;
    uint8_t *to = out + u * a.unit;
    float *sums = reinterpret_cast<float *>(to + a.planes * 2 * W4_KS);
    stage_x<GROUPS>(a, row, static_cast<int>(u - row * a.KS) * W4_KS, threadIdx.x & 31, to, 2 * W4_KS, sums, sums + GROUPS * a.planes,
                    a.planes);
}

// A warp's way through its stages, ahead of their use: chunks (an expert and up to nc entries) x row blocks, the
// row blocks of a run (of one chunk, at most seg of them) once for each pass over K, the gate's matrix before the
// other's, then this warp's stages of the pass. Nothing here divides: it runs for every row block.
struct Cursor {
    int left, chunk, tile0, len, i, pass, mat;   // blocks left; the run [tile0, tile0 + len) and the block in it
    int begin, mine;                             // this warp's stages of the pass: first, number
    int todo;                                    // of them left at src
    const uint8_t *src;
    int64_t expert;                              // offset of the expert's matrix
};

template <int NT, bool ZERO, int GROUPS, bool SCALE_BF16>
__global__ void __launch_bounds__(32 * W4_WARPS, 1) w4_kernel(const __grid_constant__ W4Args a) {
    constexpr int D = w4_stages<NT>(), GW = GROUPS == 8 ? 2 : 1;   // groups of a stage, of a tile
    constexpr int COLS = 8 * NT, XGAP = (GROUPS + 1) * COLS;       // floats of a stage's sums of x, and its powers of two
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    // WK warps from wm * WK on share K of the block's row tile wm
    const int WK = 1 << a.wk_shift, wk = warp & (WK - 1), wm = warp >> a.wk_shift;
    const int S = 1 << a.split_shift, rank = static_cast<int>(blockIdx.x) & (S - 1);
    float *red = reinterpret_cast<float *>(smem + a.red_off);
    int2 *chunk_tab = reinterpret_cast<int2 *>(smem + a.tab_off);
    uint16_t *entry_tab = reinterpret_cast<uint16_t *>(chunk_tab + a.n_entries);
    dep_launch();
    bool waited = a.ids && !(a.staged && !a.chunks);
    if (waited) dep_wait();
    int n_chunks;
    if (a.chunks) n_chunks = *a.n_chunks;
    else if (!a.ids) n_chunks = (a.n_entries + a.nc - 1) / a.nc;
    else n_chunks = w4_group(a, chunk_tab, entry_tab, reinterpret_cast<int *>(smem));   // (the ring is not in use yet)
    const int cluster = static_cast<int>(blockIdx.x) >> a.split_shift, clusters = static_cast<int>(gridDim.x) >> a.split_shift;
    // row tiles of a block: as planned, or for experts, whose chunks only the GPU knows, by the plan's count of a round's time
    int WM = a.wm;
    if (a.ids) {
        const int w = lane + 1, rounds = (n_chunks * ((a.RT + w - 1) / w) + clusters - 1) / clusters;
        const float us = a.deep * fmaxf(W4_STAGE_ALONE, w4_stage_us(w << a.wk_shift)) + a.per_block;
        const uint32_t cost = w <= a.wm ? __float_as_uint(rounds * us) : 0xFFFFFFFFu;
        WM = __ffs(__ballot_sync(0xffffffffu, cost == __reduce_min_sync(0xffffffffu, cost)));
    }
    const int tiles = (a.RT + WM - 1) / WM, items = n_chunks * tiles;   // blocks of a chunk, of all
    const int i0 = static_cast<int>(static_cast<int64_t>(items) * cluster / clusters);
    int left = static_cast<int>(static_cast<int64_t>(items) * (cluster + 1) / clusters) - i0;
    if (left == 0) {   // the whole cluster's
        dep_wait();
        return;
    }
    int chunk = i0 / tiles, tile0 = i0 - chunk * tiles;

    auto expert_of = [&](int c) { return a.chunks ? a.chunks[c].x : a.ids ? chunk_tab[c].x & 0xFFFF : 0; };
    auto entry_of = [&](int i) { return a.chunks ? a.entries[i] : a.ids ? static_cast<int>(entry_tab[i]) : i; };
    auto run_of = [&](int left, int tile0) { return min(min(left, tiles - tile0), a.seg); };
    // the first of rank r's stages of a pass
    auto share = [&](int pass, int r) {
        const int s0 = pass * a.sp, n = min(a.KS, s0 + a.sp) - s0;
        return s0 + (n * r >> a.split_shift);
    };

    constexpr uint32_t stage_bytes = w4_stage_bytes(GROUPS, ZERO);
    const uint32_t ring = warp * D * stage_bytes, ring_end = ring + D * stage_bytes;   // (offsets)
    Cursor P{};
    auto seek_chunk = [&]() {
        P.expert = static_cast<int64_t>(expert_of(P.chunk)) * a.RT * a.KS * stage_bytes + 16 * lane;
    };
    auto seek_pass = [&]() {
        P.begin = share(P.pass, rank) + wk;
        P.mine = max(0, (share(P.pass, rank + 1) - P.begin + WK - 1) >> a.wk_shift);
    };
    auto seek = [&]() {   // the first of the warp's stages of a matrix and pass
        const int rt = (P.tile0 + P.i) * WM + wm;
        P.src = (P.mat ? a.w[1] : a.w[0]) + P.expert + (static_cast<int64_t>(rt) * a.KS + P.begin) * stage_bytes;
        P.todo = rt < a.RT ? P.mine : 0;
    };
    auto next = [&]() {   // the next matrix, row block, pass or run; nothing behind the last (left 0)
        if (++P.mat == a.mats) {
            P.mat = 0;
            if (++P.i == P.len) {
                P.i = 0;
                if (++P.pass == a.passes) {
                    P.pass = 0;
                    P.left -= P.len;
                    if (P.left == 0) return;
                    P.tile0 += P.len;
                    if (P.tile0 == tiles) {
                        P.tile0 = 0;
                        ++P.chunk;
                        seek_chunk();
                    }
                    P.len = run_of(P.left, P.tile0);
                }
                if (a.passes > 1) seek_pass();
            }
        }
        seek();
    };
    if (wm < WM) {
        P.left = left;
        P.chunk = chunk;
        P.tile0 = tile0;
        P.len = run_of(left, tile0);
        seek_chunk();
        seek_pass();
        seek();
    }
    const uint32_t step = stage_bytes << a.wk_shift, lane_at = smem_u32(smem) + 16 * lane;
    auto fetch = [&](uint32_t stage) {   // (its offset)
        if (P.todo == 0)
            while (P.left && P.todo == 0) next();
        if (P.todo) {
#pragma unroll
            for (int i = 0; i < 4; ++i) cp16(lane_at + stage + 512 * i, P.src + 512 * i);
            if (16 * lane < stage_bytes - W4_CODES) cp16(lane_at + stage + W4_CODES, P.src + W4_CODES);
            P.src += step;
            --P.todo;
        }
        cp_commit();
    };
#pragma unroll 1
    for (int d = 0; d < D; ++d) fetch(ring + d * stage_bytes);

    float *acc = reinterpret_cast<float *>(smem + a.acc_off);
    const int outs1 = a.nc * W4_M;        // sums of a row tile
    const bool hold = S > 1 || a.passes > 1;
    constexpr int RED_BUF = W4_WARPS * COLS * W4_RED;
    uint32_t at = ring;
    int buf = 0, x_chunk = -1;            // whose x is staged

    while (left) {
        const int len = run_of(left, tile0);
        int count, first, expert;
        if (a.chunks) {
            const int4 c = a.chunks[chunk];
            expert = c.x, first = c.y, count = c.z;
        } else if (a.ids) {
            const int2 c = chunk_tab[chunk];
            expert = c.x & 0xFFFF, first = c.y, count = c.x >> 16;
        } else {
            expert = 0, first = chunk * a.nc, count = min(a.nc, a.n_entries - first);
        }
        const int cols = count * a.planes, outs = count * (W4_M / 4);   // a thread takes four rows of an entry
        const int64_t row_base = static_cast<int64_t>(expert) * a.rows;
        auto emit = [&](int row, int col, float4 v, float4 gate) {   // the biases, the GLU, the result
            const int n = min(4, a.rows - row);
            if (n <= 0) return;
            float u[4] = {v.x, v.y, v.z, v.w};
            const float gt[4] = {gate.x, gate.y, gate.z, gate.w};
            float *to = a.dst + static_cast<int64_t>(entry_of(first + col)) * a.rows + row;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i >= n) break;
                if (a.mats > 1) {
                    const float gi = a.bias[0] ? gt[i] + a.bias[0][row_base + row + i] : gt[i];
                    if (a.bias[1]) u[i] += a.bias[1][row_base + row + i];
                    u[i] = mx_glu_any(a.glu_op, gi, u[i], a.glu_limit);
                } else if (a.bias[0]) {
                    u[i] += a.bias[0][row_base + row + i];
                }
            }
            if (a.dst_vec) {   // (rows a multiple of 4)
                *reinterpret_cast<float4 *>(to) = make_float4(u[0], u[1], u[2], u[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < n) to[i] = u[i];
            }
        };
        auto add4 = [](float4 p, float4 q) { return make_float4(p.x + q.x, p.y + q.y, p.z + q.z, p.w + q.w); };
        for (int pass = 0; pass < a.passes; ++pass) {
            const int s0 = share(pass, rank), n_st = share(pass, rank + 1) - s0;
            const int pitch = n_st * 2 * W4_KS + W4_PAD;   // bytes of a column of x
            float *xsum = reinterpret_cast<float *>(smem + a.x_off + cols * pitch);   // [stage][GROUPS + 1][COLS]
            if (chunk != x_chunk || a.passes > 1) {
                __syncthreads();   // everyone is done with the x of before
                if (!waited) {
                    dep_wait();
                    waited = true;
                }
                // 1 << x_shift warps to an entry, a stage each at a time
                const int st0 = warp & ((1 << a.x_shift) - 1), dst_step = 1 << a.x_shift;
                for (int col = warp >> a.x_shift; col < count; col += W4_WARPS >> a.x_shift) {
                    const int entry = entry_of(first + col);
                    const int64_t row = a.per_pick || a.k == 1 ? entry : entry / a.k;
                    uint8_t *to = smem + a.x_off + col * a.planes * pitch + st0 * 2 * W4_KS;
                    float *sums = xsum + st0 * XGAP + col * a.planes;
                    if (a.staged) {   // (cp.async)
                        const uint8_t *from = a.staged + (row * a.KS + s0 + st0) * a.unit;
                        const int gi = a.planes > 1 ? lane >> 1 : lane, q = a.planes > 1 ? lane & 1 : 0;
                        uint32_t to32 = smem_u32(to + 16 * lane), sums32 = smem_u32(sums + gi * COLS + q);
                        for (int st = st0; st < n_st; st += dst_step) {
                            cp16(to32, from + 16 * lane);
                            if (a.planes > 1) cp16(to32 + pitch, from + 2 * W4_KS + 16 * lane);
                            if (lane < (GROUPS + 1) * a.planes) cp4(sums32, from + a.planes * 2 * W4_KS + 4 * lane);
                            from += a.unit << a.x_shift;
                            to32 += 2 * W4_KS << a.x_shift;
                            sums32 += 4 * XGAP << a.x_shift;
                        }
                    } else {
                        for (int st = st0; st < n_st; st += dst_step) {
                            stage_x<GROUPS>(a, row, (s0 + st) * W4_KS, lane, to, pitch, sums, sums + GROUPS * COLS, COLS);
                            to += 2 * W4_KS << a.x_shift;
                            sums += XGAP << a.x_shift;
                        }
                    }
                }
                if (a.staged) cp_wait_all();   // (and the stages in flight)
                __syncthreads();
                x_chunk = chunk;
            }
            const uint8_t *xcol[NT];   // (columns past the last repeat the first one's: nothing reads their sums)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                xcol[j] = smem + a.x_off + (8 * j + g < cols ? 8 * j + g : 0) * pitch + 16 * t + wk * 2 * W4_KS;
            const int mine = wm < WM ? max(0, (n_st - wk + WK - 1) >> a.wk_shift) : 0;
            for (int it = 0; it < len; ++it) {
                const int rt = (tile0 + it) * WM + wm;
                if (wm >= WM || rt >= a.RT) break;
                for (int mat = 0; mat < a.mats; ++mat) {
                    float sum[NT][4] = {};
                    // this warp's stages, for J tiles of columns
                    auto run = [&](auto columns) {
                        constexpr int J = decltype(columns)::value;
                        uint32_t xk = 0;
                        const float *xs = xsum + wk * XGAP + 2 * t;
                        for (int s = 0; s < mine; ++s) {
                            cp_wait<D - 1>();
                            __syncwarp();
                            float part[J][4], dots[J][GW][4], sc[GW][2], sz[GW][2];
#pragma unroll
                            for (int i = 0; i < W4_KS / W4_KT; ++i) {
                                const uint4 w = lds16(smem + at + 16 * lane + W4_TILE * i);
                                uint32_t A[4][4];
                                unpack_codes(w.x, A[0]);
                                unpack_codes(w.y, A[1]);
                                unpack_codes(w.z, A[2]);
                                unpack_codes(w.w, A[3]);
#pragma unroll
                                for (int h = 0; h < GW; ++h) {
                                    if (GW == 1 && i * GROUPS % 4) continue;   // the group goes on
                                    const int gi = GW == 2 ? 2 * i + h : i * GROUPS / 4;
                                    const uint32_t sw = lds4(smem + at + W4_CODES + 32 * gi + 4 * g);
                                    if constexpr (SCALE_BF16) {
                                        sc[h][0] = __uint_as_float(sw << 16);
                                        sc[h][1] = __uint_as_float(sw & 0xFFFF0000u);
                                    } else {
                                        const float2 f = __half22float2(reinterpret_cast<const __half2 &>(sw));
                                        sc[h][0] = f.x;
                                        sc[h][1] = f.y;
                                    }
                                    // scale * zero; rows g + 8 in their codes' units
                                    if constexpr (ZERO) {
                                        const uint32_t zw = lds4(smem + at + W4_CODES + 32 * GROUPS + 16 * gi + 4 * (g >> 1));
                                        // 2^23 + zero, by bits
                                        const float z0 = __uint_as_float(__byte_perm(zw, 0x4B000000u, g & 1 ? 0x7552 : 0x7550));
                                        const float z1 = __uint_as_float(__byte_perm(zw, 0x4B000000u, g & 1 ? 0x7553 : 0x7551));
                                        sz[h][0] = sc[h][0] * (z0 - 8388608.f);
                                        sz[h][1] = sc[h][1] * fmaf(z1, 16.f, -16.f * 8388608.f);
                                    } else {
                                        sz[h][0] = sc[h][0] * 8.f;
                                        sz[h][1] = sc[h][1] * 128.f;
                                    }
                                }
#pragma unroll
                                for (int j = 0; j < J; ++j) {
                                    const uint8_t *xb = xcol[j] + xk + 2 * W4_KT * i;
                                    const uint4 b0 = lds16(xb), b1 = lds16(xb + 64);
                                    // (groups of 128 and more: two tiles' products meet in the tensor cores)
                                    constexpr bool PAIRS = GROUPS <= 2;
                                    float (&d)[GW][4] = dots[j];
                                    if (PAIRS && i % 2) mma<false>(d[0], A[0], b0.x, b0.y);
                                    else mma<true>(d[0], A[0], b0.x, b0.y);
                                    mma<false>(d[0], A[1], b0.z, b0.w);
                                    mma<GW == 2>(d[GW - 1], A[2], b1.x, b1.y);
                                    mma<false>(d[GW - 1], A[3], b1.z, b1.w);
                                    if (PAIRS && i % 2 == 0) continue;
#pragma unroll
                                    for (int h = 0; h < GW; ++h) {
#pragma unroll
                                        for (int q = 0; q < 4; ++q)
                                            part[j][q] = i / (PAIRS ? 2 : 1) + h == 0 ? sc[h][q >> 1] * d[h][q]
                                                                                      : fmaf(sc[h][q >> 1], d[h][q], part[j][q]);
                                        if (GW == 1 && (i + 1) * GROUPS % 4) continue;   // the group's last tile
                                        const int gi = GW == 2 ? 2 * i + h : i * GROUPS / 4;
                                        const float2 x = *reinterpret_cast<const float2 *>(xs + gi * COLS + 8 * j);
#pragma unroll
                                        for (int q = 0; q < 4; ++q) part[j][q] = fmaf(sz[h][q >> 1], q & 1 ? x.y : x.x, part[j][q]);
                                    }
                                }
                            }
#pragma unroll
                            for (int j = 0; j < J; ++j) {
                                const float2 x = *reinterpret_cast<const float2 *>(xs + GROUPS * COLS + 8 * j);
#pragma unroll
                                for (int q = 0; q < 4; ++q) sum[j][q] = fmaf(q & 1 ? x.y : x.x, part[j][q], sum[j][q]);
                            }
                            xk += 2 * W4_KS << a.wk_shift;
                            xs += XGAP << a.wk_shift;
                            __syncwarp();   // all lanes have read the stage
                            fetch(at);
                            at = at + stage_bytes == ring_end ? ring : at + stage_bytes;
                        }
                    };
                    if constexpr (NT == 1) {
                        run(std::integral_constant<int, 1>{});
                    } else {
                        if (cols <= 8) run(std::integral_constant<int, 1>{});
                        else run(std::integral_constant<int, 2>{});
                    }
                    // the sums of the warps that share K meet; codes' units come off
                    float *mine_at = red + buf * RED_BUF + warp * COLS * W4_RED + 2 * t * W4_RED + g;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            mine_at[(8 * j + (q & 1)) * W4_RED + 8 * (q >> 1)] = sum[j][q] * (q < 2 ? W4_UP : W4_UP / 16.f);
                    auto group_sync = [&]() {
                        if (WK == 1) __syncwarp();
                        else asm volatile("bar.sync %0, %1;" ::"r"(1 + wm), "r"(32 << a.wk_shift) : "memory");
                    };
                    group_sync();
                    const float *from = red + buf * RED_BUF + (wm << a.wk_shift) * COLS * W4_RED;
                    float *keep = acc + (((hold ? it : 0) * a.mats + mat) * WM + wm) * outs1;
                    for (int o = 32 * wk + lane; o < outs; o += 32 << a.wk_shift) {
                        const int r = 4 * (o & 3), col = o >> 2;
                        const float *p = from + col * a.planes * W4_RED + r;
                        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (a.planes > 1)   // the small plane first
                            for (int w = 0; w < WK; ++w) v = add4(v, *reinterpret_cast<const float4 *>(p + (w * COLS + 1) * W4_RED));
                        for (int w = 0; w < WK; ++w) v = add4(v, *reinterpret_cast<const float4 *>(p + w * COLS * W4_RED));
                        float4 *kept = reinterpret_cast<float4 *>(keep) + o;
                        if (pass > 0) v = add4(v, *kept);
                        if (S > 1 || pass + 1 < a.passes || mat + 1 < a.mats) *kept = v;
                        else emit(rt * W4_M + r, col, v, a.mats > 1 ? kept[-(WM * outs1 / 4)] : v);
                    }
                    buf ^= 1;
                }
            }
        }
        if (S > 1) {   // the run's outputs, from the sums of every CTA of the cluster
            w4_cluster_sync();
            for (int it = 0, turn = 0; it < len; ++it)
                for (int m = 0; m < WM; ++m, ++turn) {
                    const int rt = (tile0 + it) * WM + m;
                    if (rt >= a.RT) break;
                    // the warps of the cluster in turn
                    int o = ((rank * W4_WARPS + warp + (turn << 3) - turn) & ((W4_WARPS << a.split_shift) - 1)) * 32 + lane;
                    for (; o < outs; o += 32 * W4_WARPS << a.split_shift) {
                        auto total = [&](int mat) {
                            const uint32_t at4 = smem_u32(reinterpret_cast<float4 *>(acc + ((it * a.mats + mat) * WM + m) * outs1) + o);
                            float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (S == 2) {
                                const float4 p = ld_cluster(at4, 0), q = ld_cluster(at4, 1);
                                return add4(p, q);
                            }
                            for (int q = 0; q < S; q += 4) {   // (loads of four CTAs in flight)
                                const float4 p0 = ld_cluster(at4, q), p1 = ld_cluster(at4, q + 1), p2 = ld_cluster(at4, q + 2),
                                             p3 = ld_cluster(at4, q + 3);
                                u = add4(u, add4(add4(p0, p1), add4(p2, p3)));
                            }
                            return u;
                        };
                        const float4 v = total(0);
                        emit(rt * W4_M + 4 * (o & 3), o >> 2, a.mats > 1 ? total(1) : v, v);
                    }
                }
            w4_cluster_sync();   // the sums stay until every CTA has read them
        }
        left -= len;
        tile0 += len;
        if (tile0 == tiles) {
            tile0 = 0;
            ++chunk;
        }
    }
    cp_wait_all();
}

// How the columns, the rows and K are shared out. A CTA has up to 16 warps at work: wm row tiles, K of each shared by
// 1 << wk_shift warps and `split` CTAs; chunks have up to 8 nt MMA columns. Of all such plans the one with the least
// time by the count below is taken; its constants were fitted to 22 calls (one matrix of 768 x 2048 to 32768 x 4096 with 1 to
// 64 rows of x, experts with 1 to 64 tokens) timed in every plan: its choice is 5 % slower than the best of them on average,
// 27 % at most (1024 x 8192, one row: 6.5 us, 5.1 without a cluster). For experts, whose chunks depend on the picks, the GPU
// takes wm when it has counted them (64 of them, 4 tokens' 6: 20.5 us, 27.3 with the wm that a guess gave).
// (Plans with 32 columns or with clusters of eight were never better by more than 1 %.)
struct W4Plan {
    int nt, split, wk_shift, wm, passes, sp, seg, deep;
    uint32_t acc, tab;
    double us;
};

// what a plan depends on
struct W4Key {
    int64_t n_tok, RT, KS;
    int32_t k, n_experts, one_matrix, planes, mats, groups, zeros;
    int32_t slots[3];   // CTAs, clusters of 2 and clusters of 4 that run at once
};

int w4_ring(int nt) { return nt == 1 ? w4_stages<1>() : w4_stages<2>(); }
uint32_t w4_red_bytes(int nt) { return 2 * W4_WARPS * nt * 8 * W4_RED * 4; }

void w4_plan(const W4Key &c, int nt, W4Plan &best) {
    const int nc = 8 * nt / c.planes;
    const int64_t n = c.n_tok * c.k;
    const int cols = static_cast<int>(n < nc ? n : nc) * c.planes;
    const uint32_t tab = !c.one_matrix && n <= W4_DIRECT ? (static_cast<uint32_t>(n) * 10 + 15) / 16 * 16 : 0;
    const int64_t fixed = static_cast<int64_t>(W4_WARPS) * w4_ring(nt) * w4_stage_bytes(c.groups, c.zeros != 0) + w4_red_bytes(nt) + tab;
    const int x_stage = (c.groups + 1) * 8 * nt * 4;   // bytes of a stage's sums of x
    // chunks to expect: those of the experts that even picks would touch, and some of the crowded ones'
    int64_t chunks = (n + nc - 1) / nc;
    if (!c.one_matrix) {
        const int64_t touched = n < c.n_experts ? n : c.n_experts;
        chunks = touched + n / (2 * nc) < n ? touched + n / (2 * nc) : n;
    }
    const double mean = c.one_matrix ? cols / c.planes : static_cast<double>(n) / static_cast<double>(chunks);
    const double entries = mean < 1.0 ? 1.0 : mean < nc ? mean : nc;   // of a chunk
    const bool wide = entries * c.planes > 8, staged = w4_staged(c.n_tok, c.KS);
    for (int split = 1; split <= 4 && (split == 1 || split <= c.KS); split *= 2) {
        if (c.slots[split / 2] < 1) continue;
        for (int wk = 0; wk <= 4; ++wk)
            for (int wm = 1; wm << wk <= W4_WARPS; ++wm) {
                const int WK = 1 << wk, KS = static_cast<int>(c.KS), spr = (KS + split - 1) / split;
                if ((WK > 1 && WK / 2 >= spr) || (wm > 1 && wm > c.RT)) continue;
                const int most = c.one_matrix ? wm : W4_WARPS >> wk;              // row tiles that a block may have
                const uint32_t one = static_cast<uint32_t>(nc * most * W4_M * c.mats) * 4;   // its sums
                W4Plan p{nt, split, wk, most, 1, KS, 1 << 24, 0, 0, tab, 0.0};
                bool hold = split > 1;
                auto room_for_x = [&]() {   // stages of x that fit
                    p.acc = hold ? (one > W4_ACC ? one : W4_ACC / one * one) : c.mats > 1 ? one : 0;
                    const int64_t left = W4_SMEM - fixed - p.acc - cols * W4_PAD;
                    return left < 0 ? 0 : static_cast<int>(left / (cols * 2 * W4_KS + x_stage));
                };
                int fit = room_for_x();
                if (fit < spr) {
                    hold = true;
                    fit = room_for_x();
                    if (fit < 1) continue;
                    p.passes = (spr + fit - 1) / fit;
                    p.sp = (KS + p.passes - 1) / p.passes;
                    if ((p.sp + split - 1) / split > fit) p.sp = fit * split;
                    p.passes = (KS + p.sp - 1) / p.sp;
                }
                if (hold) p.seg = static_cast<int>(p.acc / one);
                const int mine = (p.sp + split - 1) / split;                    // stages of a CTA in a pass
                const int sums = c.mats * p.passes, deep = sums * ((mine + WK - 1) / WK);   // of a warp, for a row block
                p.deep = deep;
                const int64_t blocks = (c.RT + wm - 1) / wm, items = chunks * blocks, slots = c.slots[split / 2];
                const double rounds = static_cast<double>((items + slots - 1) / slots);
                // the SM's issue slots, and the way through one CTA's row blocks
                const double full = rounds * (deep * (w4_stage_us(wm * WK) + (wide ? 0.0086 * wm * WK : 0.0)) +
                                             sums * 0.0588 * wm * WK * (0.5 + entries / 8));
                const double one_by_one = rounds * (deep * (wide ? 0.63 : W4_STAGE_ALONE) + sums * W4_BLOCK_US);
                // bringing x, once for every chunk that a CTA meets, or for every pass of every run
                const double runs = p.passes > 1 || split > 1 ? static_cast<double>((static_cast<int64_t>(rounds) + p.seg - 1) / p.seg) : 1.0;
                const double met = 1.0 + rounds / static_cast<double>(blocks);
                const double bring = 1.15 + entries * mine * c.planes * (staged ? 0.001 : 0.026);
                p.us = (full > one_by_one ? full : one_by_one) + (p.passes > 1 ? runs * p.passes : rounds < met ? rounds : met) * bring +
                       (split > 1 ? runs * (1.55 + 0.0107 * wm * entries) : 0.0);
                if (p.us < best.us) best = p;
            }
    }
}

// the plan of a call, remembered by its sizes (working it out takes some microseconds; the caller holds the library's lock)
const W4Plan &w4_plan_of(const W4Key &c) {
    static struct { W4Key key; W4Plan plan; } seen[256];
    uint64_t h = 0;
    for (size_t i = 0; i < sizeof(W4Key) / 4; ++i) {
        uint32_t v;
        memcpy(&v, reinterpret_cast<const char *>(&c) + 4 * i, 4);
        h = (h ^ v) * 0x9E3779B97F4A7C15ull;
    }
    auto &slot = seen[h >> 56];
    if (slot.plan.nt == 0 || memcmp(&slot.key, &c, sizeof(c))) {
        W4Plan best{};
        best.us = 1e30;
        w4_plan(c, 1, best);
        w4_plan(c, 2, best);
        slot.key = c;
        slot.plan = best;
    }
    return slot.plan;
}

template <int NT, bool ZERO, int GROUPS, bool SCALE_BF16>
cudaError_t w4_t(W4Args &a, const W4Plan &p, int64_t max_chunks, int slots, cudaStream_t st) {
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(w4_kernel<NT, ZERO, GROUPS, SCALE_BF16>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, W4_SMEM);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    static_assert(W4_WARPS * w4_stages<NT>() * W4_CODES >= W4_WARPS * W4_MAX_EXPERTS * 4, "the grouping counts in the ring");
    const int most = a.n_entries < a.nc ? a.n_entries : a.nc, mine = (p.sp + p.split - 1) / p.split;
    a.split_shift = p.split == 1 ? 0 : p.split == 2 ? 1 : 2;
    a.wk_shift = p.wk_shift;
    a.wm = p.wm;
    a.deep = static_cast<float>(p.deep);
    a.per_block = static_cast<float>(a.mats * p.passes) * W4_BLOCK_US;
    a.x_shift = most >= 16 ? 0 : most >= 8 ? 1 : most >= 4 ? 2 : most >= 2 ? 3 : 4;
    a.dst_vec = a.rows % 4 == 0 && reinterpret_cast<uintptr_t>(a.dst) % 16 == 0;
    a.passes = p.passes;
    a.sp = p.sp;
    a.seg = p.seg;
    a.red_off = W4_WARPS * w4_stages<NT>() * w4_stage_bytes(GROUPS, ZERO);
    a.tab_off = a.red_off + w4_red_bytes(NT);
    a.acc_off = a.tab_off + p.tab;
    a.x_off = a.acc_off + p.acc;
    const size_t smem = a.x_off + static_cast<size_t>(most * a.planes) * (mine * 2 * W4_KS + W4_PAD) +
                        static_cast<size_t>(mine) * (GROUPS + 1) * 8 * NT * 4;
    if (smem > W4_SMEM) return cudaErrorInvalidConfiguration;
    const int64_t blocks = a.ids ? a.RT : (a.RT + p.wm - 1) / p.wm, items = max_chunks * blocks;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>((items < slots ? items : slots) * p.split));
    cfg.blockDim = dim3(32 * W4_WARPS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = static_cast<unsigned>(p.split);
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.split > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, w4_kernel<NT, ZERO, GROUPS, SCALE_BF16>, a);
}

template <int NT, bool ZERO, bool SCALE_BF16>
cudaError_t w4_groups(W4Args &a, const W4Plan &p, int64_t max_chunks, int slots, cudaStream_t st) {
    switch (a.groups) {
        case 8: return w4_t<NT, ZERO, 8, SCALE_BF16>(a, p, max_chunks, slots, st);
        case 4: return w4_t<NT, ZERO, 4, SCALE_BF16>(a, p, max_chunks, slots, st);
        case 2: return w4_t<NT, ZERO, 2, SCALE_BF16>(a, p, max_chunks, slots, st);
        default: return w4_t<NT, ZERO, 1, SCALE_BF16>(a, p, max_chunks, slots, st);
    }
}

template <int NT>
cudaError_t w4_nt(W4Args &a, const W4Plan &p, int64_t max_chunks, int slots, cudaStream_t st) {
    if (a.scale_type == MX_BF16)
        return a.zeros ? w4_groups<NT, true, true>(a, p, max_chunks, slots, st) : w4_groups<NT, false, true>(a, p, max_chunks, slots, st);
    return a.zeros ? w4_groups<NT, true, false>(a, p, max_chunks, slots, st) : w4_groups<NT, false, false>(a, p, max_chunks, slots, st);
}

}  // namespace

// Whether a call brings x into the products' form first, once, rather than in every CTA (us in a graph, every CTA / once):
// n_tok KS up to 32 the launch costs 0.7 to 1.3 (one bf16 token 2048 x 2048 4.7 / 5.9); 40 to 64 it costs up to 0.7 (12 tokens
// 2048 x 1024 5.5 / 6.2) or saves up to 6 (4 f32 tokens 4096 x 4096 14.1 / 8.2, 6 tokens' 4 of 16 experts 20.0 / 16.4); from
// 128 on it saves (8 bf16 tokens 4096 x 4096 14.7 / 8.7) but for 32 tokens 2048 x 2048 (7.9 / 8.1).
bool w4_staged(int64_t n_tok, int64_t KS) { return n_tok * KS > 32; }

// bytes of a row of x in that form
int64_t w4_row_bytes(int64_t KS, int groups, int x_type) {
    const int planes = x_type == MX_F32 ? 2 : 1;
    return KS * ((planes * (2 * W4_KS + 4 * (groups + 1)) + 15) / 16 * 16);
}

// entries of a chunk at least
int w4_min_chunk(int x_type) { return x_type == MX_F32 ? 4 : 8; }

cudaError_t launch_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int64_t E, int64_t rows, int64_t K,
                           int64_t group, int per_stage, uint8_t *out, int *err, cudaStream_t st) {
    const int64_t RT = (rows + W4_M - 1) / W4_M, KS = (K + W4_KS - 1) / W4_KS, g = group < K ? group : K;
    const int64_t n = E * RT * KS * (w4_stage_bytes(per_stage, zeros != nullptr) / 4), blocks = (n + 255) / 256;
    w4_pack_kernel<<<static_cast<unsigned>(blocks < 148 * 64 ? blocks : 148 * 64), 256, 0, st>>>(
        codes, static_cast<const uint16_t *>(scales), zeros, static_cast<int>(rows), static_cast<int>(K), static_cast<int>(g),
        static_cast<int>((K + g - 1) / g), static_cast<int>(RT), static_cast<int>(KS), per_stage, reinterpret_cast<uint32_t *>(out),
        n, err);
    const cudaError_t e = cudaGetLastError();
    return e != cudaSuccess ? e : launch_w4_settle(st);
}

cudaError_t launch_w4_settle(cudaStream_t st) {
    w4_settled_kernel<<<1, 1, 0, st>>>();
    return cudaGetLastError();
}

// How many CTAs, clusters of 2 and clusters of 4 run at once, one CTA to an SM: clusters do not span GPCs (one B200: 148, 74
// and 33; 37 clusters of 4 ran in two rounds: us for 8 bf16 tokens 4096 x 14336 23.6 -> 13.6, 16 f16 tokens 3718 x 6968
// 19.7 -> 11.9 in a graph).
cudaError_t w4_slots(int32_t (&out)[3]) {
    static int32_t known[64][3] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    int32_t (&n)[3] = known[dev];
    if (!n[0]) {
        auto *kern = w4_kernel<1, true, 8, false>;
        int sms = 0, clusters[2] = {};
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_SMEM);
        if (e != cudaSuccess) return e;
        for (int i = 0; i < 2; ++i) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(148 * 4);
            cfg.blockDim = dim3(32 * W4_WARPS);
            cfg.dynamicSmemBytes = W4_SMEM;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 2u << i;
            at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
            cfg.attrs = at;
            cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&clusters[i], kern, &cfg) != cudaSuccess) {
                cudaGetLastError();
                clusters[i] = 0;   // plans do without
            }
        }
        e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        n[1] = clusters[0], n[2] = clusters[1], n[0] = sms;
    }
    for (int i = 0; i < 3; ++i) out[i] = n[i];
    return cudaSuccess;
}

static W4Key w4_key(const W4Args &a, int64_t n_tok, const int32_t (&slots)[3]) {
    W4Key c;
    memset(&c, 0, sizeof(c));   // (compared byte by byte)
    c.n_tok = n_tok, c.RT = a.RT, c.KS = a.KS;
    c.k = a.k, c.n_experts = a.n_experts, c.one_matrix = a.ids == nullptr, c.planes = a.x_type == MX_F32 ? 2 : 1, c.mats = a.mats;
    c.groups = a.groups, c.zeros = a.zeros;
    memcpy(c.slots, slots, sizeof(slots));
    return c;
}

bool w4_plan_for(const W4Args &a, int64_t n_tok, const int32_t (&slots)[3], int32_t (&out)[6]) {
    const W4Plan p = w4_plan_of(w4_key(a, n_tok, slots));
    if (p.nt == 0) return false;
    out[0] = p.nt, out[1] = p.split, out[2] = 1 << p.wk_shift, out[3] = p.wm, out[4] = p.passes, out[5] = w4_staged(n_tok, a.KS);
    return true;
}

cudaError_t launch_w4(W4Args &a, int64_t n_tok, uint8_t *staged, cudaStream_t st) {
    int32_t slots[3];
    const cudaError_t known = w4_slots(slots);
    if (known != cudaSuccess) return known;
    a.planes = a.x_type == MX_F32 ? 2 : 1;
    const W4Plan p = w4_plan_of(w4_key(a, n_tok, slots));
    if (p.nt == 0) return cudaErrorInvalidConfiguration;
    a.nc = 8 * p.nt / a.planes;
    int64_t max_chunks = (a.n_entries + a.nc - 1) / a.nc;
    if (a.ids) {
        max_chunks = mmq_max_chunks(a.n_entries, a.n_experts, a.nc);
        if (max_chunks > a.n_entries) max_chunks = a.n_entries;
    }
    if (a.chunks) {
        const cudaError_t e = launch_mmq_group(a.ids, a.ids_stride, static_cast<int>(n_tok), a.k, a.n_experts, a.nc,
                                               const_cast<int32_t *>(a.entries), const_cast<int4 *>(a.chunks),
                                               const_cast<int32_t *>(a.n_chunks), a.err, st, true);
        if (e != cudaSuccess) return e;
    }
    if (staged) {
        a.unit = static_cast<int32_t>(w4_row_bytes(1, a.groups, a.x_type));
        const int64_t units = (a.per_pick ? static_cast<int64_t>(a.n_entries) : n_tok) * a.KS;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>((units + 7) / 8));
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        const cudaError_t e = a.groups == 8   ? cudaLaunchKernelEx(&cfg, w4_stage_kernel<8>, a, units, staged)
                              : a.groups == 4 ? cudaLaunchKernelEx(&cfg, w4_stage_kernel<4>, a, units, staged)
                              : a.groups == 2 ? cudaLaunchKernelEx(&cfg, w4_stage_kernel<2>, a, units, staged)
                                              : cudaLaunchKernelEx(&cfg, w4_stage_kernel<1>, a, units, staged);
        if (e != cudaSuccess) return e;
        a.staged = staged;
    }
    const int n = slots[p.split / 2];
    return p.nt == 1 ? w4_nt<1>(a, p, max_chunks, n, st) : w4_nt<2>(a, p, max_chunks, n, st);
}

}  // namespace moe
