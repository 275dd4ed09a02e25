// moe_router.cu -- routing with the scores of current MoE routers: softmax or
// sigmoid scores (or a softmax over the picks), a bias that only the choice
// sees, groups of experts, top-k, renormalised and scaled gating weights.
//
// One warp per token; lane l holds experts l + 32 j in registers. Where no bias
// and no group sum enters, the logit itself ranks (all three scores grow with
// it). Otherwise the ranking is the one that 64-bit scores give: sigmoid(l) +
// bias brings experts closer together than the last places of 32-bit arithmetic
// can tell apart, and a pick would then depend on how an exp rounds. 64-bit exp
// for every expert made the kernel twice as slow, so scores are 32-bit first,
// with a bound on their error: where all gaps that decide (between consecutive
// picks, behind the last one, behind the last kept group) exceed it, the order
// is the 64-bit one; a token with a closer pair is ranked again in 64 bits.
// Weights are 32-bit throughout. 8192 tokens, 256 experts in 8 groups with a bias, top-8: 21.3 to
// 23.5 us, bound by issue; one token 8.2 us, the latency of its serial steps (a call 12.8).
#include "moe_aux.h"
#include "moe_common.cuh"
#include "moe_mx.cuh"
#include "moe_route.cuh"

#include <cfloat>
#include <cuda_bf16.h>

namespace moe {

namespace {

constexpr int RT_WARPS = 4;   // tokens per CTA; 12 CTAs' registers fit an SM (up to 256 experts)

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

// the largest of the warp's keys leaves them (ties: the lowest id)
template <int NV, typename KEY>
__device__ __forceinline__ void pick_one(KEY (&key)[NV], int lane, int &id, KEY &id_key) {
    KEY m = key[0];
    int mj = 0;
#pragma unroll
    for (int j = 1; j < NV; ++j)
        if (key[j] > m) { m = key[j]; mj = j; }
    warp_best(m, lane + 32 * mj, id_key, id);
    if ((id & 31) == lane) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (id == lane + 32 * j) key[j] = 0;
    }
}
// k of them: lane q keeps pick q and its key
template <int NV, typename KEY>
__device__ __forceinline__ void pick_k(KEY (&key)[NV], int k, int lane, int &pick, KEY &pick_key) {
    pick = 0;
    pick_key = 0;
    for (int q = 0; q < k; ++q) {
        KEY bk;
        int bi;
        pick_one<NV>(key, lane, bi, bk);
        if (lane == q) { pick = bi; pick_key = bk; }
    }
}

// e / (E / n_group) for e < 1024: magic = ceil(2^20 / size) is off by less than one part in the size
__device__ __forceinline__ int group_of(int e, uint32_t magic) { return static_cast<int>((static_cast<uint32_t>(e) * magic) >> 20); }

// The two largest of each group's scores s[E], by 32 / n_group lanes (a power of
// two) per group; the group's score where sub == 0. Lanes of different groups
// start at different elements, which keeps them on different banks.
template <typename T>
__device__ __forceinline__ T group_score_of(const T *s, int gsz, int n_group, int group_score, int per, int grp, int sub) {
    T m1 = -INFINITY, m2 = -INFINITY;
    const int cnt = (gsz + per - 1) / per;
    if (grp < n_group) {
        int i = grp % cnt;
        for (int c = 0; c < cnt; ++c) {
            const int at = sub + per * i;
            const T v = at < gsz ? s[grp * gsz + at] : static_cast<T>(-INFINITY);
            m2 = v > m1 ? m1 : (v > m2 ? v : m2);
            m1 = v > m1 ? v : m1;
            i = i + 1 == cnt ? 0 : i + 1;
        }
    }
    for (int off = 1; off < per; off <<= 1) {
        const T o1 = __shfl_xor_sync(0xffffffffu, m1, off), o2 = __shfl_xor_sync(0xffffffffu, m2, off);
        const T lo = m1 < o1 ? m1 : o1, hi = m2 > o2 ? m2 : o2;
        m2 = lo > hi ? lo : hi;
        m1 = m1 > o1 ? m1 : o1;
    }
    // (one expert left in the group counts alone)
    return group_score == ROUTE_GROUP_MAX || !(m2 > -INFINITY) ? m1 : m1 + m2;
}
__device__ __forceinline__ int lanes_per_group(int n_group) {
    int per = 1;
    while (per * 2 * n_group <= 32) per *= 2;
    return per;
}
// bit h: group h stays, being behind fewer than topk_group others (ties to the lower group)
template <typename KEY>
__device__ __forceinline__ uint32_t kept_groups(KEY k, int n_group, int topk_group, int per, int grp, int sub) {
    int ahead = 0;
    for (int h = 0; h < n_group; ++h) {
        const KEY o = __shfl_sync(0xffffffffu, k, h * per);
        ahead += (o > k || (o == k && h < grp)) ? 1 : 0;
    }
    const uint32_t in = __ballot_sync(0xffffffffu, grp < n_group && sub == 0 && ahead < topk_group);
    uint32_t kept = 0;
    for (int h = 0; h < n_group; ++h) kept |= ((in >> (h * per)) & 1u) << h;
    return kept;
}

// Picks of token t by 64-bit scores, in E doubles of shared memory. Written as
// loops: the code runs once in a while and its time is that of fetching it
// (unrolled over the experts it took 10 us).
template <int LT>
__device__ __noinline__ void rank_exact(const RouteArgs &a, int64_t t, int lane, float mx, double *s, int &pick, bool &live) {
    const int E = a.n_experts;
    double sum = 0.0;
#pragma unroll 1
    for (int e = lane; e < E; e += 32) {
        const float l = clean_logit(logit_at<LT>(a.logits, t * a.row_stride + e));
        const bool has = l > -INFINITY;
        double c = static_cast<double>(l);
        if (a.score != ROUTE_SOFTMAX_TOPK) {
            const double x = exp(a.score == ROUTE_SOFTMAX ? c - static_cast<double>(mx) : -c);
            c = a.score == ROUTE_SOFTMAX ? x : 1.0 / (1.0 + x);
        }
        c = has ? c : 0.0;
        sum += c;
        s[e] = c;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
#pragma unroll 1
    for (int e = lane; e < E; e += 32) {
        double c = s[e];
        if (a.score == ROUTE_SOFTMAX) c /= sum;
        if (a.bias) c += static_cast<double>(a.bias[e]);
        const float l = clean_logit(logit_at<LT>(a.logits, t * a.row_stride + e));
        s[e] = l > -INFINITY && c == c ? c : -INFINITY;
    }
    __syncwarp();
    if (a.n_group > 1) {
        const int gsz = E / a.n_group, per = lanes_per_group(a.n_group);
        const int grp = lane >> (31 - __clz(per)), sub = lane & (per - 1);
        const double gs = group_score_of(s, gsz, a.n_group, a.group_score, per, grp, sub);
        const uint32_t kept = kept_groups(key64(gs), a.n_group, a.topk_group, per, grp, sub);
        __syncwarp();
#pragma unroll 1
        for (int e = lane; e < E; e += 32)
            if (!((kept >> group_of(e, a.group_magic)) & 1u)) s[e] = -INFINITY;
    }
    // a pick leaves the row as a NaN, which no key exceeds
    uint64_t pk = 0;
#pragma unroll 1
    for (int q = 0; q < a.k; ++q) {
        uint64_t m = 0;
        int id = 0x7fffffff;
        for (int e = lane; e < E; e += 32) {
            const double c = s[e];
            const uint64_t key = c == c ? key64(c) : 0ull;
            if (key > m) { m = key; id = e; }
        }
        uint64_t bk;
        int bi;
        warp_best(m, id, bk, bi);
        if ((bi & 31) == lane) s[bi] = __longlong_as_double(0x7ff8000000000000ll);
        if (lane == q) { pick = bi; pk = bk; }
    }
    live = pk > key64(-INFINITY);
}

// Lanes 0..k hold candidates (the k picks and the next one): their order by
// 64-bit scores, one per lane. Sigmoid or plain logits.
template <int LT>
__device__ __noinline__ int reorder_exact(const RouteArgs &a, int64_t t, int lane, int cand) {
    double c = -INFINITY;
    if (lane <= a.k) {
        const float l = clean_logit(logit_at<LT>(a.logits, t * a.row_stride + cand));
        c = static_cast<double>(l);
        if (a.score == ROUTE_SIGMOID) c = 1.0 / (1.0 + exp(-c));
        if (a.bias) c += static_cast<double>(a.bias[cand]);
        if (!(l > -INFINITY) || c != c) c = -INFINITY;
    }
    int ahead = 0;
#pragma unroll 1
    for (int j = 0; j <= a.k; ++j) {
        const double o = __shfl_sync(0xffffffffu, c, j);
        const int oid = __shfl_sync(0xffffffffu, cand, j);
        ahead += (o > c || (o == c && oid < cand)) ? 1 : 0;
    }
    int pick = 0;
#pragma unroll 1
    for (int j = 0; j <= a.k; ++j) {
        const int at = __shfl_sync(0xffffffffu, ahead, j), id = __shfl_sync(0xffffffffu, cand, j);
        if (at == lane) pick = id;
    }
    return pick;
}

template <int LT, int NV, bool SCORED>
__global__ void __launch_bounds__(32 * RT_WARPS, NV == 8 ? 12 : 1) route_kernel(const __grid_constant__ RouteArgs a) {
    extern __shared__ double smem[];   // SCORED: each warp's scores [E]
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
    float sum = 0.f;                                                    // softmax's denominator
    if (a.score == ROUTE_SOFTMAX) {
#pragma unroll
        for (int j = 0; j < NV; ++j) sum += l[j] > -INFINITY ? expf(l[j] - mx) : 0.f;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }

    int pick;
    bool live;      // the pick's selection score is above -inf
    if constexpr (!SCORED) {
        uint32_t key[NV], pk;
#pragma unroll
        for (int j = 0; j < NV; ++j) key[j] = lane + 32 * j < E ? logit_key(l[j]) : 0u;
        pick_k<NV>(key, k, lane, pick, pk);
        live = pk > logit_key(-INFINITY);
    } else {
        // Scores in 32 bits, and how far they may be off: exp and the quotient to 2 ulp, a
        // rounding of 1 + e -- below 8e-7 of the largest score for sigmoid, and 2^-126 where the quotient
        // of a denominator above 2^126 is 0; for softmax also l - mx (|l - mx|
        // e^(l - mx) <= 0.37) and up to 37 additions, below 4e-6; half an ulp of the sum with the bias.
        // Nothing where the logit is the score.
        float c[NV], big = 0.f, bigs = 0.f;
        const float rs = 1.0f / sum;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = lane + 32 * j;
            const bool has = l[j] > -INFINITY;
            c[j] = a.score == ROUTE_SOFTMAX ? (has ? expf(l[j] - mx) * rs : 0.f)
                 : a.score == ROUTE_SIGMOID ? __fdividef(1.0f, 1.0f + expf(-l[j])) : l[j];
            if (has) bigs = fmaxf(bigs, fabsf(c[j]));
            if (a.bias && e < E) c[j] += a.bias[e];
            if (!has || c[j] != c[j]) c[j] = -INFINITY;
            if (fabsf(c[j]) < INFINITY) big = fmaxf(big, fabsf(c[j]));
        }
        big = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big)));
        bigs = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(bigs)));
        const float err = (a.score == ROUTE_SOFTMAX ? 4e-6f * bigs : a.score == ROUTE_SIGMOID ? 8e-7f * bigs + 1.2e-38f : 0.f) +
                          (a.bias ? 1.2e-7f * big : 0.f);
        // (sums of a bias with a score, and of two scores, that 32 bits do not hold: by 64 bits)
        bool close_group = fmaxf(big, bigs) > 1.7e38f;
        uint32_t kept = 0xffffffffu;
        const int gsz = E / a.n_group;
        if (a.n_group > 1) {
            float *s = reinterpret_cast<float *>(smem + static_cast<size_t>(warp) * E);
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (lane + 32 * j < E) s[lane + 32 * j] = c[j];
            __syncwarp();
            const int per = lanes_per_group(a.n_group), grp = lane >> (31 - __clz(per)), sub = lane & (per - 1);
            const float gs = group_score_of(s, gsz, a.n_group, a.group_score, per, grp, sub);
            kept = kept_groups(logit_key(gs), a.n_group, a.topk_group, per, grp, sub);
            __syncwarp();
            // the least kept group against the best of the others
            const bool mine = grp < a.n_group && sub == 0, in = mine && ((kept >> grp) & 1u);
            const float worst = key_logit(__reduce_min_sync(0xffffffffu, in ? logit_key(gs) : 0xFFFFFFFFu));
            const uint32_t rest = __reduce_max_sync(0xffffffffu, mine && !in ? logit_key(gs) : 0u);
            // (a sum of two scores has twice the error and a rounding of its own)
            if (rest > logit_key(-INFINITY)) close_group |= !(worst - key_logit(rest) > 2.f * (2.f * err + 1.2e-7f * 2.f * big));
        }
        uint32_t key[NV], pk;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = lane + 32 * j;
            const bool in = a.n_group == 1 || (e < E && ((kept >> group_of(e, a.group_magic)) & 1u));
            key[j] = e < E ? logit_key(in ? c[j] : -INFINITY) : 0u;
        }
        pick_k<NV>(key, k, lane, pick, pk);
        live = pk > logit_key(-INFINITY);
        // pick q against pick q + 1, the last one against the best of the rest
        const uint32_t none = logit_key(-INFINITY);
        uint32_t next_key;
        int next_id;
        pick_one<NV>(key, lane, next_id, next_key);
        uint32_t behind = __shfl_down_sync(0xffffffffu, pk, 1);
        if (lane == k - 1) behind = next_key;
        const bool close = lane < k && behind > none && !(key_logit(pk) - key_logit(behind) > 2.f * err);
        if (__any_sync(0xffffffffu, close || close_group)) {
            // mostly the picks and the next one hold all that could be meant: the one behind them is
            // clearly less than the last pick
            uint32_t third_key;
            int third_id;
            pick_one<NV>(key, lane, third_id, third_key);
            const float last = key_logit(__shfl_sync(0xffffffffu, pk, k - 1));
            if (!__any_sync(0xffffffffu, close_group) && a.score != ROUTE_SOFTMAX && k < 32 && next_key > none &&
                last - key_logit(max(third_key, none)) > 2.f * err)
                pick = reorder_exact<LT>(a, t, lane, lane < k ? pick : lane == k ? next_id : 0x7fffffff);
            else
                rank_exact<LT>(a, t, lane, mx, smem + static_cast<size_t>(warp) * E, pick, live);
        }
    }

    // gating weights of the picks, from the scores without the bias
    live = live && lane < k;
    const float lp = lane < k ? clean_logit(logit_at<LT>(a.logits, t * a.row_stride + pick)) : -INFINITY;
    float w = 0.f;
    if (a.score == ROUTE_SIGMOID) {
        w = live ? 1.0f / (1.0f + expf(-lp)) : 0.f;
    } else if (a.score == ROUTE_SOFTMAX) {
        w = live ? expf(lp - mx) / sum : 0.f;
    } else {
        const float pm = key_logit(__reduce_max_sync(0xffffffffu, live ? logit_key(lp) : 0u));
        const float x = live ? expf(lp - pm) : 0.f;
        float total = x;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        w = live ? x / total : 0.f;
    }
    if (a.norm_w) {
        float total = w;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
        w /= fmaxf(total, ROUTE_MIN_SUM);
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
        const size_t smem = static_cast<size_t>(RT_WARPS) * a.n_experts * sizeof(double);   // 32 KB at most
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

cudaError_t launch_route(RouteArgs a, int logits_type, cudaStream_t st) {
    if (a.n_tok == 0) return cudaSuccess;
    const uint32_t size = static_cast<uint32_t>(a.n_experts / a.n_group);
    a.group_magic = ((1u << 20) + size - 1) / size;
    if (logits_type == MX_F32) return route_t<MX_F32>(a, st);
    if (logits_type == MX_F16) return route_t<MX_F16>(a, st);
    return route_t<MX_BF16>(a, st);
}

}  // namespace moe
