// moe_router.cu -- routing with the scores of current MoE routers: softmax or
// sigmoid scores (or a softmax over the picks), a bias that only the choice
// sees, groups of experts, top-k, renormalised and scaled gating weights.
//
// One warp per token; lane l holds experts l + 32 j in registers. What ranks
// the experts is a key that orders like the score: the logit itself where no
// bias and no group sum enters (all three scores grow with it), else the score
// in 64 bits -- sigmoid(l) + bias brings experts closer together than the last
// places of 32-bit arithmetic can tell apart, and the pick would then depend on
// how an exp rounds. Weights are 32-bit throughout.
#include "moe_aux.h"
#include "moe_common.cuh"
#include "moe_mx.cuh"
#include "moe_route.cuh"

#include <cfloat>
#include <cuda_bf16.h>

namespace moe {

namespace {

constexpr int RT_WARPS = 4;   // tokens per CTA

// The logit as the router takes it: a NaN counts as -inf, +inf as the largest number.
__device__ __forceinline__ float clean_logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

template <int LT>
__device__ __forceinline__ float logit_at(const void *p, int64_t i) {
    if constexpr (LT == MX_F32) return static_cast<const float *>(p)[i];
    else if constexpr (LT == MX_F16) return __half2float(static_cast<const __half *>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

// order-preserving 64-bit key; 0 is below every key
__device__ __forceinline__ uint64_t key64(double d) {
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(d + 0.0));
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

// the largest key of the warp and the lowest id that has it
__device__ __forceinline__ void warp_best(uint32_t k, int id, uint32_t &bk, int &bi) {
    bk = __reduce_max_sync(0xffffffffu, k);
    bi = static_cast<int>(__reduce_min_sync(0xffffffffu, k == bk ? static_cast<uint32_t>(id) : 0xFFFFFFFFu));
}
__device__ __forceinline__ void warp_best(uint64_t k, int id, uint64_t &bk, int &bi) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
    bk = (static_cast<uint64_t>(hi) << 32) | lo;
    bi = static_cast<int>(__reduce_min_sync(0xffffffffu, k == bk ? static_cast<uint32_t>(id) : 0xFFFFFFFFu));
}

// the k largest keys, ties to the lower id: lane q keeps pick q and its key
template <int NV, typename KEY>
__device__ __forceinline__ void pick_k(KEY (&key)[NV], int k, int lane, int &pick, KEY &pick_key) {
    pick = 0;
    pick_key = 0;
    for (int q = 0; q < k; ++q) {
        KEY m = key[0];
        int mj = 0;
#pragma unroll
        for (int j = 1; j < NV; ++j)
            if (key[j] > m) { m = key[j]; mj = j; }
        KEY bk;
        int bi;
        warp_best(m, lane + 32 * mj, bk, bi);
        if ((bi & 31) == lane) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (bi == lane + 32 * j) key[j] = 0;
        }
        if (lane == q) { pick = bi; pick_key = bk; }
    }
}

template <int LT, int NV, bool RANK64>
__global__ void __launch_bounds__(32 * RT_WARPS) route_kernel(const RouteArgs a) {
    extern __shared__ double smem[];   // RANK64 with groups: the warp's scores [E]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * RT_WARPS + warp;
    if (t >= a.n_tok) return;
    const int E = a.n_experts, k = a.k;
    float l[NV];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = lane + 32 * j;
        l[j] = e < E ? clean_logit(logit_at<LT>(a.logits, t * a.row_stride + e)) : -INFINITY;
        top = max(top, logit_key(l[j]));
    }
    const float mx = key_logit(__reduce_max_sync(0xffffffffu, top));   // -inf: the row has no expert to offer

    int pick;
    bool live;      // the pick's selection score is above -inf
    if constexpr (!RANK64) {
        uint32_t key[NV], pk;
#pragma unroll
        for (int j = 0; j < NV; ++j) key[j] = lane + 32 * j < E ? logit_key(l[j]) : 0u;
        pick_k<NV>(key, k, lane, pick, pk);
        live = pk > logit_key(-INFINITY);
    } else {
        double c[NV];
        if (a.score == ROUTE_SOFTMAX) {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                c[j] = l[j] > -INFINITY ? exp(static_cast<double>(l[j]) - static_cast<double>(mx)) : 0.0;
                sum += c[j];
            }
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll
            for (int j = 0; j < NV; ++j) c[j] /= sum;
        } else if (a.score == ROUTE_SIGMOID) {
#pragma unroll
            for (int j = 0; j < NV; ++j) c[j] = 1.0 / (1.0 + exp(-static_cast<double>(l[j])));
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) c[j] = static_cast<double>(l[j]);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = lane + 32 * j;
            if (a.bias && e < E) c[j] += static_cast<double>(a.bias[e]);
            if (!(l[j] > -INFINITY) || c[j] != c[j]) c[j] = -INFINITY;
        }
        uint32_t kept = 0xffffffffu;   // bit g: group g stays
        const int gsz = E / a.n_group;
        if (a.n_group > 1) {
            double *s = smem + static_cast<size_t>(warp) * E;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane + 32 * j < E) s[lane + 32 * j] = c[j];
            __syncwarp();
            int per = 1;                                        // lanes per group
            while (per * 2 * a.n_group <= 32) per *= 2;
            const int grp = lane / per, sub = lane % per;
            double m1 = -INFINITY, m2 = -INFINITY;              // the group's two largest
            if (grp < a.n_group)
                for (int i = sub; i < gsz; i += per) {
                    const double v = s[grp * gsz + i];
                    if (v > m1) { m2 = m1; m1 = v; }
                    else if (v > m2) m2 = v;
                }
            for (int off = 1; off < per; off <<= 1) {
                const double o1 = __shfl_xor_sync(0xffffffffu, m1, off), o2 = __shfl_xor_sync(0xffffffffu, m2, off);
                m2 = fmax(fmin(m1, o1), fmax(m2, o2));
                m1 = fmax(m1, o1);
            }
            const double gs = a.group_score == ROUTE_GROUP_MAX || gsz == 1 ? m1 : m1 + m2;
            // a group stays when fewer than topk_group others are ahead of it
            uint64_t gk[1] = {grp < a.n_group && sub == 0 ? key64(gs) : 0ull};
            int ahead = 0;
            for (int h = 0; h < a.n_group; ++h) {
                const uint64_t o = __shfl_sync(0xffffffffu, gk[0], h * per);
                ahead += (o > gk[0] || (o == gk[0] && h < grp)) ? 1 : 0;
            }
            const uint32_t in = __ballot_sync(0xffffffffu, grp < a.n_group && sub == 0 && ahead < a.topk_group);
            kept = 0;
            for (int h = 0; h < a.n_group; ++h) kept |= ((in >> (h * per)) & 1u) << h;
        }
        uint64_t key[NV], pk;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = lane + 32 * j;
            const bool in = a.n_group == 1 || ((kept >> (e / gsz)) & 1u);
            key[j] = e < E ? key64(in ? c[j] : -INFINITY) : 0ull;
        }
        pick_k<NV>(key, k, lane, pick, pk);
        live = pk > key64(-INFINITY);
    }

    // gating weights of the picks, from the scores without the bias
    live = live && lane < k;
    const float lp = lane < k ? clean_logit(logit_at<LT>(a.logits, t * a.row_stride + pick)) : -INFINITY;
    float w = 0.f;
    if (a.score == ROUTE_SIGMOID) {
        w = live ? 1.0f / (1.0f + expf(-lp)) : 0.f;
    } else if (a.score == ROUTE_SOFTMAX) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) sum += l[j] > -INFINITY ? expf(l[j] - mx) : 0.f;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        w = live ? expf(lp - mx) / sum : 0.f;
    } else {
        const float pm = key_logit(__reduce_max_sync(0xffffffffu, live ? logit_key(lp) : 0u));
        const float x = live ? expf(lp - pm) : 0.f;
        float sum = x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        w = live ? x / sum : 0.f;
    }
    if (a.norm_w) {
        float sum = w;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        w /= fmaxf(sum, ROUTE_MIN_SUM);
    }
    if (lane < k) {
        a.ids[t * k + lane] = pick;
        a.weights[t * k + lane] = w * a.scale;
    }
}

template <int LT, int NV>
cudaError_t route_nv(const RouteArgs &a, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>((a.n_tok + RT_WARPS - 1) / RT_WARPS);
    if (!a.bias && a.n_group == 1) {
        route_kernel<LT, NV, false><<<grid, 32 * RT_WARPS, 0, st>>>(a);
    } else {
        const size_t smem = a.n_group > 1 ? static_cast<size_t>(RT_WARPS) * a.n_experts * sizeof(double) : 0;
        route_kernel<LT, NV, true><<<grid, 32 * RT_WARPS, smem, st>>>(a);
    }
    return cudaGetLastError();
}

template <int LT>
cudaError_t route_t(const RouteArgs &a, cudaStream_t st) {
    if (a.n_experts <= 256) return route_nv<LT, 8>(a, st);
    if (a.n_experts <= 512) return route_nv<LT, 16>(a, st);
    return route_nv<LT, 32>(a, st);
}

}  // namespace

cudaError_t launch_route(const RouteArgs &a, int logits_type, cudaStream_t st) {
    if (a.n_tok == 0) return cudaSuccess;
    if (logits_type == MX_F32) return route_t<MX_F32>(a, st);
    if (logits_type == MX_F16) return route_t<MX_F16>(a, st);
    return route_t<MX_BF16>(a, st);
}

}  // namespace moe
