// moe_sort.cu -- tokens sorted by expert and back: the stable order of the
// (token, pick) entries by expert, the tokens' rows in that order, the weighted
// sum of the sorted rows back into the tokens, and the gradients of both.
//
//   entry i = t k + j, expert ids[i]; the M entries with 0 <= id < E, ordered by (id, i)
//   gather    out[p] = x[rows[p] / k]                      d_x[t] = sum_j d_out[pos[t][j]]
//   combine   out[t] = sum_j w[t][j] y[pos[t][j]] + shared[t]
//             d_y[pos[t][j]] = w[t][j] d_out[t]            d_w[t][j] = <d_out[t], y[pos[t][j]]>
//
// All of it moves bytes: nothing is computed that HBM does not hide. 16384 tokens of 2048 bf16 values, 8 of 256
// experts each (one B200): sort 13.8 us, gather 107 (waiting for the order included; 5.6 TB/s), weighted sum 110 (5.5),
// gradient of the gather 97 (6.2), of the sum 173 (6.6; up to 126 MB of what a kernel writes may reach HBM after
// its end); the pass 497. One f32 token with 8 picks: 4.2 us and 3.3, the latency of the steps.
#include "moe_aux.h"
#include "moe_common.cuh"
#include "moe_mx.cuh"

#include <cuda_bf16.h>

namespace moe {

namespace {

// ---- the order -----------------------------------------------------------------
// A counting sort whose counts belong to warps: warp w of CTA c owns a stretch of
// consecutive entries and a column of counts of its own, so that an entry's
// place is (entries of lower experts) + (of its expert in earlier CTAs) + (in
// earlier warps) + (earlier in its warp), the same whatever ran first. Few entries
// take one CTA, many one cluster, whose totals meet in distributed shared memory: of 8 CTAs,
// or of 16 (where the GPU runs such clusters) from 32768 entries on. Its time is the instructions of so few SMs: 65536 entries
// 12.6 us by 8 and 9.9 by 16, 131072 20.9 and 13.9.
constexpr int SORT_THREADS = 1024;
constexpr int SORT_AHEAD = 8;   // loads in flight per lane

__device__ __forceinline__ void sort_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_cluster_s32(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// The places of a warp's entries among its earlier ones of their expert, whose counts go up; -1 for id -1. Lanes of one
// expert are found by a ballot per bit of the ids (bits of them), which costs less than __match_any_sync on many
// different ones.
__device__ __forceinline__ int warp_rank(int *count, int id, int lane, int bits) {
    unsigned peers = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool one = (id >> b) & 1;
        const unsigned m = __ballot_sync(0xffffffffu, one);
        peers &= one ? m : ~m;
    }
    const unsigned with = __ballot_sync(0xffffffffu, id >= 0);
    peers &= id >= 0 ? with : ~with;
    const int leader = __ffs(peers) - 1;
    int before = 0;
    if (id >= 0 && lane == leader) {
        before = count[id];
        count[id] = before + __popc(peers);
    }
    before = __shfl_sync(0xffffffffu, before, leader);
    __syncwarp();
    return id >= 0 ? before + __popc(peers & ((1u << lane) - 1u)) : -1;
}

template <int CTAS>
__global__ void __launch_bounds__(SORT_THREADS) sort_kernel(const SortArgs a) {
    extern __shared__ int sort_smem[];   // counts [warps][E], totals of this CTA [E], first places [E]
    __shared__ int warp_sum[32];
    if (CTAS > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (they wait for the order)
    const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nth >> 5;
    const int rank = CTAS > 1 ? static_cast<int>(blockIdx.x) : 0;
    const int E = a.n_experts, N = a.n_entries, k = a.k;
    const int bits = 32 - __clz(E - 1);
    int *count = sort_smem + warp * E, *total = sort_smem + warps * E, *first = total + E;
    for (int i = tid; i < warps * E; i += nth) sort_smem[i] = 0;
    __syncthreads();
    // a warp's stretch: whole groups of 32 entries
    const int groups = (N + 31) >> 5, per = (groups + CTAS * warps - 1) / (CTAS * warps);
    const int64_t lo = (static_cast<int64_t>(rank) * warps + warp) * per * 32;
    const int64_t hi = lo + static_cast<int64_t>(per) * 32 < N ? lo + static_cast<int64_t>(per) * 32 : N;
    auto id_of = [&](int i) {
        if (a.ids_stride == k) return a.ids[i];
        const int t = i / k;
        return a.ids[static_cast<int64_t>(t) * a.ids_stride + (i - t * k)];
    };
    for (int64_t i0 = lo; i0 < hi; i0 += 32 * SORT_AHEAD) {
        int id[SORT_AHEAD];
#pragma unroll
        for (int u = 0; u < SORT_AHEAD; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            id[u] = i < hi ? id_of(static_cast<int>(i)) : -1;
        }
#pragma unroll
        for (int u = 0; u < SORT_AHEAD; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            if (i0 + 32 * u >= hi) break;
            const bool ok = id[u] >= 0 && id[u] < E;
            if (!ok && id[u] != -1) set_error(a.err, DERR_BAD_ID);
            const int local = warp_rank(count, ok ? id[u] : -1, lane, bits);
            // (the place in the warp's stretch, until the counts of the others are known)
            if (i < hi) a.positions[i] = local;
        }
    }
    __syncthreads();
    for (int e = tid; e < E; e += nth) {
        int sum = 0;
        for (int w = 0; w < warps; ++w) {
            const int c = sort_smem[w * E + e];
            sort_smem[w * E + e] = sum;
            sum += c;
        }
        total[e] = sum;
    }
    if (CTAS > 1) sort_cluster_sync();
    // first[e]: entries of lower experts, plus those of e in earlier CTAs
    int carry = 0;
    for (int base = 0; base < E; base += nth) {
        const int e = base + tid;
        int all = 0, earlier = 0;
        if (e < E) {
            if (CTAS > 1) {
#pragma unroll
                for (int c = 0; c < CTAS; ++c) {
                    const int v = ld_cluster_s32(smem_u32(&total[e]), c);
                    all += v;
                    earlier += c < rank ? v : 0;
                }
            } else {
                all = total[e];
            }
        }
        int incl = all;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int ahead = carry, sum = 0;
        for (int w = 0; w < warps; ++w) {
            const int s = warp_sum[w];
            ahead += w < warp ? s : 0;
            sum += s;
        }
        if (e < E) {
            first[e] = ahead + incl - all + earlier;
            if (rank == 0) a.offsets[e] = ahead + incl - all;
        }
        carry += sum;
        __syncthreads();
    }
    if (rank == 0 && tid == 0) a.offsets[E] = carry;
    __syncthreads();
    for (int64_t i0 = lo; i0 < hi; i0 += 32 * SORT_AHEAD) {
        int id[SORT_AHEAD], local[SORT_AHEAD];
#pragma unroll
        for (int u = 0; u < SORT_AHEAD; ++u) {
            const int64_t i = i0 + 32 * u + lane;
            local[u] = i < hi ? a.positions[i] : -1;
            id[u] = i < hi ? id_of(static_cast<int>(i)) : -1;
        }
#pragma unroll
        for (int u = 0; u < SORT_AHEAD; ++u) {
            if (local[u] < 0) continue;
            const int i = static_cast<int>(i0) + 32 * u + lane, p = first[id[u]] + count[id[u]] + local[u];
            a.positions[i] = p;
            if (CTAS == 1) {
                a.rows[p] = i;
                a.experts[p] = id[u];
            }
        }
    }
    if constexpr (CTAS > 1) {
        sort_cluster_sync();   // the totals stay until every CTA has read them
    } else {
        for (int p = carry + tid; p < N; p += nth) a.rows[p] = a.experts[p] = -1;
    }
}

// What the cluster leaves to the whole GPU: rows and experts. These writes are scattered, and an SM sends off one sector
// per cycle (8 of them took 31 us for 131072 entries, 21 without these writes). The row kernel does it where one follows.
__device__ __forceinline__ void place_entry(const SortArgs &s, int64_t i, int64_t t, int j) {
    const int p = s.positions[i];
    if (p < 0) return;
    s.rows[p] = static_cast<int>(i);
    s.experts[p] = s.ids[t * s.ids_stride + j];
}
__global__ void __launch_bounds__(256) place_kernel(const SortArgs s) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // (the order)
    const int i = blockIdx.x * 256 + threadIdx.x, live = s.offsets[s.n_experts];
    if (i >= s.n_entries) return;
    place_entry(s, i, i / s.k, i % s.k);
    if (i >= live) s.rows[i] = s.experts[i] = -1;
}

// ---- rows -----------------------------------------------------------------------
// 1 << tpt threads work on a token, V bytes each at a time (the widest that the row, its
// stride and the addresses allow), so that short rows leave no thread of a CTA idle. 8192 tokens, 8 of 64 experts, bf16,
// gather and weighted sum (us, one B200): rows of 2048 values by 16 bytes 51 and 61, of 2052 by 4 72 and 72, of 2047 by 2
// 98 and 131.
constexpr int ROW_THREADS = 256;

template <int V> struct vec;
template <> struct vec<16> { using t = uint4; };
template <> struct vec<4> { using t = uint32_t; };
template <> struct vec<2> { using t = uint16_t; };

template <int V>
__device__ __forceinline__ typename vec<V>::t zero_vec() {
    typename vec<V>::t z{};
    return z;
}

// V bytes as floats and back, rounded to the nearest
template <int T, int V>
__device__ __forceinline__ void unpack(const typename vec<V>::t &v, float *f) {
    if constexpr (T == MX_F32) {
        memcpy(f, &v, V);
    } else {
        uint16_t h[V / 2];
        memcpy(h, &v, V);
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            f[i] = T == MX_F16 ? __half2float(__ushort_as_half(h[i])) : __uint_as_float(static_cast<uint32_t>(h[i]) << 16);
    }
}
template <int T, int V>
__device__ __forceinline__ typename vec<V>::t pack(const float *f) {
    typename vec<V>::t v;
    if constexpr (T == MX_F32) {
        memcpy(&v, f, V);
    } else {
        uint16_t h[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            h[i] = T == MX_F16 ? __half_as_ushort(__float2half_rn(f[i])) : __bfloat16_as_ushort(__float2bfloat16_rn(f[i]));
        memcpy(&v, h, V);
    }
    return v;
}

// out[p] = 0 for the rows behind the last sorted one
template <int V>
__device__ __forceinline__ void zero_tail(char *out, int64_t row_bytes, int live, int N) {
    for (int64_t p = static_cast<int64_t>(live) + blockIdx.x; p < N; p += gridDim.x)
        for (int64_t c = threadIdx.x; c < row_bytes / V; c += blockDim.x)
            reinterpret_cast<typename vec<V>::t *>(out + p * row_bytes)[c] = zero_vec<V>();
}

// A token's row is read once and written to its picks' places. PLACES: right behind sort_kernel's cluster, whose rows and
// experts it writes; a token's first vectors arrive meanwhile.
template <int V, bool PLACES>
__global__ void __launch_bounds__(ROW_THREADS) gather_kernel(const RowArgs a, const SortArgs s) {
    using vt = typename vec<V>::t;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) << a.per_cta) + (threadIdx.x >> a.tpt);
    const int nv = static_cast<int>(a.row_bytes / V), step = static_cast<int>(gridDim.y) << a.tpt;
    const int col = threadIdx.x & ((1 << a.tpt) - 1);
    int c = (static_cast<int>(blockIdx.y) << a.tpt) + col;
    if (t < a.n_tok) {
        const vt *src = reinterpret_cast<const vt *>(a.src + t * a.src_stride);
        const int32_t *pos = a.positions + t * a.k;
        vt v = c < nv ? src[c] : zero_vec<V>();
        if (PLACES) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            if (blockIdx.y == 0)
                for (int j = col; j < a.k; j += 1 << a.tpt) place_entry(s, t * a.k + j, t, j);
        }
        for (; c < nv;) {
#pragma unroll 4
            for (int j = 0; j < a.k; ++j) {
                const int p = pos[j];
                if (p >= 0) reinterpret_cast<vt *>(a.out + p * a.row_bytes)[c] = v;
            }
            c += step;
            if (c < nv) v = src[c];
        }
    } else if (PLACES) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    if (blockIdx.y == 0) {
        const int live = *a.live;
        zero_tail<V>(a.out, a.row_bytes, live, a.n_entries);
        if (PLACES)
            for (int64_t p = static_cast<int64_t>(live) + static_cast<int64_t>(blockIdx.x) * ROW_THREADS + threadIdx.x; p < a.n_entries;
                 p += static_cast<int64_t>(gridDim.x) * ROW_THREADS)
                s.rows[p] = s.experts[p] = -1;
    }
}

// Both in one launch for few entries: every CTA finds the whole order by itself (as sort_kernel's CTAs do; two
// microseconds, against those of a second launch) and copies its tokens' rows; the first one writes the order down.
constexpr int DISPATCH_PER = 8;   // entries of a thread at most
constexpr int DISPATCH_CTAS = 592;   // more would sort in several waves (2048 tokens' one expert each)

template <int V>
__global__ void __launch_bounds__(ROW_THREADS) dispatch_kernel(const SortArgs s, const RowArgs a) {
    using vt = typename vec<V>::t;
    constexpr int WARPS = ROW_THREADS / 32;
    extern __shared__ int sort_smem[];   // counts [WARPS][E], then the positions [N]
    __shared__ int warp_sum[WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, E = s.n_experts, N = s.n_entries, k = s.k;
    const bool writes = blockIdx.x == 0 && blockIdx.y == 0;
    const int bits = 32 - __clz(E - 1);
    int *count = sort_smem + warp * E, *positions = sort_smem + WARPS * E;
    for (int i = tid; i < WARPS * E; i += ROW_THREADS) sort_smem[i] = 0;
    __syncthreads();
    const int per = (N + 32 * WARPS - 1) / (32 * WARPS);   // groups of 32 entries of a warp
    int id[DISPATCH_PER], local[DISPATCH_PER];
#pragma unroll
    for (int u = 0; u < DISPATCH_PER; ++u) {
        const int i = (warp * per + u) * 32 + lane;
        id[u] = -1;
        if (u < per && i < N) {
            const int t = i / k;
            id[u] = s.ids[static_cast<int64_t>(t) * s.ids_stride + (i - t * k)];
            if (id[u] < 0 || id[u] >= E) {
                if (id[u] != -1 && writes) set_error(s.err, DERR_BAD_ID);
                id[u] = -1;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < DISPATCH_PER; ++u)
        if (u < per) local[u] = warp_rank(count, id[u], lane, bits);
    __syncthreads();
    int carry = 0;
    for (int base = 0; base < E; base += ROW_THREADS) {
        const int e = base + tid;
        int all = 0;
        if (e < E)
            for (int w = 0; w < WARPS; ++w) all += sort_smem[w * E + e];
        int incl = all;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += o;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int first = carry + incl - all;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            first += w < warp ? warp_sum[w] : 0;
            carry += warp_sum[w];
        }
        if (e < E) {
            if (writes) s.offsets[e] = first;
            for (int w = 0; w < WARPS; ++w) {
                const int c = sort_smem[w * E + e];
                sort_smem[w * E + e] = first;
                first += c;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < DISPATCH_PER; ++u) {
        const int i = (warp * per + u) * 32 + lane;
        if (u >= per || i >= N) continue;
        const int p = id[u] >= 0 ? count[id[u]] + local[u] : -1;
        positions[i] = p;
        if (writes) {
            s.positions[i] = p;
            if (p >= 0) {
                s.rows[p] = i;
                s.experts[p] = id[u];
            }
        }
    }
    if (writes) {
        if (tid == 0) s.offsets[E] = carry;
        for (int p = carry + tid; p < N; p += ROW_THREADS) s.rows[p] = s.experts[p] = -1;
    }
    __syncthreads();
    const int64_t t = (static_cast<int64_t>(blockIdx.x) << a.per_cta) + (tid >> a.tpt);
    const int nv = static_cast<int>(a.row_bytes / V), step = static_cast<int>(gridDim.y) << a.tpt;
    if (t < a.n_tok) {
        const vt *src = reinterpret_cast<const vt *>(a.src + t * a.src_stride);
        const int *pos = positions + t * k;
        for (int c = (static_cast<int>(blockIdx.y) << a.tpt) + (tid & ((1 << a.tpt) - 1)); c < nv; c += step) {
            const vt v = src[c];
            for (int j = 0; j < k; ++j)
                if (pos[j] >= 0) reinterpret_cast<vt *>(a.out + pos[j] * a.row_bytes)[c] = v;
        }
    }
    if (blockIdx.y == 0) zero_tail<V>(a.out, a.row_bytes, carry, N);
}

// The sum of a token's rows in pick order, in 32 bits, rounded once; WEIGHTED: times the
// gating weights. A pick without a row adds nothing, whatever its weight holds.
constexpr int COMBINE_AHEAD = 8;   // rows in flight per thread

template <int T, int V, bool WEIGHTED>
__global__ void __launch_bounds__(ROW_THREADS) combine_sorted_kernel(const RowArgs a) {
    using vt = typename vec<V>::t;
    constexpr int n = T == MX_F32 ? V / 4 : V / 2;
    const int64_t t = (static_cast<int64_t>(blockIdx.x) << a.per_cta) + (threadIdx.x >> a.tpt);
    if (t >= a.n_tok) return;
    const int nv = static_cast<int>(a.row_bytes / V), step = static_cast<int>(gridDim.y) << a.tpt;
    const int32_t *pos = a.positions + t * a.k;
    const float *w = WEIGHTED ? a.weights + t * a.k : nullptr;
    for (int c = (static_cast<int>(blockIdx.y) << a.tpt) + (threadIdx.x & ((1 << a.tpt) - 1)); c < nv; c += step) {
        float acc[n] = {};
        for (int j0 = 0; j0 < a.k; j0 += COMBINE_AHEAD) {
            vt v[COMBINE_AHEAD];
            float wj[COMBINE_AHEAD];
            bool on[COMBINE_AHEAD];
#pragma unroll
            for (int u = 0; u < COMBINE_AHEAD; ++u) {
                const int p = j0 + u < a.k ? pos[j0 + u] : -1;
                on[u] = p >= 0;
                v[u] = zero_vec<V>();
                wj[u] = 1.f;
                if (on[u]) {
                    v[u] = reinterpret_cast<const vt *>(a.src + p * a.src_stride)[c];
                    if (WEIGHTED) wj[u] = w[j0 + u];
                }
            }
#pragma unroll
            for (int u = 0; u < COMBINE_AHEAD; ++u)
                if (on[u]) {
                    float f[n];
                    unpack<T, V>(v[u], f);
#pragma unroll
                    for (int i = 0; i < n; ++i) acc[i] = WEIGHTED ? fmaf(wj[u], f[i], acc[i]) : acc[i] + f[i];
                }
        }
        if (a.shared) {
            float f[n];
            unpack<T, V>(reinterpret_cast<const vt *>(a.shared + t * a.shared_stride)[c], f);
#pragma unroll
            for (int i = 0; i < n; ++i) acc[i] += f[i];
        }
        reinterpret_cast<vt *>(a.out + t * a.row_bytes)[c] = pack<T, V>(acc);
    }
}

// One warp per entry: d_out's row against y's (the lanes' sums meet in a fixed order) and
// scaled into d_y's. The k warps of a token run side by side, so that its row comes from L1.
template <int T, int V, bool DY, bool DW>
__global__ void __launch_bounds__(ROW_THREADS) combine_grad_kernel(const RowArgs a) {
    using vt = typename vec<V>::t;
    constexpr int n = T == MX_F32 ? V / 4 : V / 2;
    constexpr int U = V == 16 ? 4 : 8;   // loads in flight of either row
    const int lane = threadIdx.x & 31;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * (ROW_THREADS / 32) + (threadIdx.x >> 5);
    if (i < a.n_entries) {
        const int p = a.positions[i];
        const int64_t t = i / a.k;
        const int nv = static_cast<int>(a.row_bytes / V);
        float dot = 0.f;
        if (p >= 0) {
            const float w = a.weights ? a.weights[i] : 1.f;
            const vt *d = reinterpret_cast<const vt *>(a.src + t * a.src_stride);
            const vt *y = DW ? reinterpret_cast<const vt *>(a.y + p * a.y_stride) : nullptr;
            vt *dy = DY ? reinterpret_cast<vt *>(a.out + p * a.row_bytes) : nullptr;
            for (int c0 = lane; c0 < nv; c0 += 32 * U) {
                vt dv[U], yv[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    dv[u] = yv[u] = zero_vec<V>();
                    if (c0 + 32 * u < nv) {
                        dv[u] = d[c0 + 32 * u];
                        if (DW) yv[u] = y[c0 + 32 * u];
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (c0 + 32 * u >= nv) continue;
                    float f[n], g[n];
                    unpack<T, V>(dv[u], f);
                    if (DW) {
                        unpack<T, V>(yv[u], g);
#pragma unroll
                        for (int e = 0; e < n; ++e) dot = fmaf(f[e], g[e], dot);
                    }
                    if (DY) {
#pragma unroll
                        for (int e = 0; e < n; ++e) f[e] *= w;
                        dy[c0 + 32 * u] = pack<T, V>(f);
                    }
                }
            }
        }
        if (DW) {
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
            if (lane == 0) a.d_weights[i] = dot;
        }
    }
    if (DY) zero_tail<V>(a.out, a.row_bytes, *a.live, a.n_entries);
}

// threads of a token and the launch of a kernel whose CTAs hold ROW_THREADS >> tpt tokens; few tokens spread
// their rows over more CTAs
dim3 row_grid(RowArgs &a, int V) {
    const int64_t nv = a.row_bytes / V;
    a.tpt = 2;
    while ((1 << a.tpt) < nv && (1 << a.tpt) < ROW_THREADS) ++a.tpt;
    a.per_cta = 8 - a.tpt;
    const int64_t x = (a.n_tok + (1 << a.per_cta) - 1) >> a.per_cta;
    int64_t y = 1;
    if (a.tpt == 8 && x < 296) {
        y = (nv + ROW_THREADS - 1) / ROW_THREADS;
        y = y < 296 / x + 1 ? y : 296 / x + 1;
    }
    return dim3(static_cast<unsigned>(x), static_cast<unsigned>(y));
}

int vec_bytes(const RowArgs &a, int elem) {
    uint64_t bits = reinterpret_cast<uintptr_t>(a.src) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.y) |
                    reinterpret_cast<uintptr_t>(a.shared) | static_cast<uint64_t>(a.row_bytes) |
                    static_cast<uint64_t>(a.src_stride);
    if (a.y) bits |= static_cast<uint64_t>(a.y_stride);
    if (a.shared) bits |= static_cast<uint64_t>(a.shared_stride);
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : elem;
}

template <int T, int V>
cudaError_t combine_tv(RowArgs &a, cudaStream_t st) {
    const dim3 grid = row_grid(a, V);
    if (a.weights) combine_sorted_kernel<T, V, true><<<grid, ROW_THREADS, 0, st>>>(a);
    else combine_sorted_kernel<T, V, false><<<grid, ROW_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}
template <int T, int V>
cudaError_t grad_tv(const RowArgs &a, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(a.n_entries) + ROW_THREADS / 32 - 1) / (ROW_THREADS / 32));
    if (a.out && a.d_weights) combine_grad_kernel<T, V, true, true><<<grid, ROW_THREADS, 0, st>>>(a);
    else if (a.out) combine_grad_kernel<T, V, true, false><<<grid, ROW_THREADS, 0, st>>>(a);
    else combine_grad_kernel<T, V, false, true><<<grid, ROW_THREADS, 0, st>>>(a);
    return cudaGetLastError();
}
template <int T>
cudaError_t combine_t(RowArgs &a, cudaStream_t st) {
    const int v = vec_bytes(a, T == MX_F32 ? 4 : 2);
    if (v == 16) return combine_tv<T, 16>(a, st);
    if (T == MX_F32 || v == 4) return combine_tv<T, 4>(a, st);
    if constexpr (T != MX_F32) return combine_tv<T, 2>(a, st);
    return cudaErrorInvalidValue;
}
template <int T>
cudaError_t grad_t(const RowArgs &a, cudaStream_t st) {
    const int v = vec_bytes(a, T == MX_F32 ? 4 : 2);
    if (v == 16) return grad_tv<T, 16>(a, st);
    if (T == MX_F32 || v == 4) return grad_tv<T, 4>(a, st);
    if constexpr (T != MX_F32) return grad_tv<T, 2>(a, st);
    return cudaErrorInvalidValue;
}

size_t sort_smem_bytes(int warps, int E) { return sizeof(int) * static_cast<size_t>(warps + 2) * E; }

// the launch of one CTA or cluster; cudaErrorNotSupported where the GPU runs no such cluster
template <int CTAS>
cudaError_t sort_launch(const SortArgs &a, int threads, cudaStream_t st) {
    static int state[64] = {};   // by device: 1 fit to run, -1 not
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(CTAS);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = sort_smem_bytes(SORT_THREADS / 32, SORT_MAX_EXPERTS);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CTAS;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CTAS > 1 ? 1 : 0;
    if (!state[dev]) {
        cudaError_t e = cudaFuncSetAttribute(sort_kernel<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(cfg.dynamicSmemBytes));
        if (e != cudaSuccess) return e;
        state[dev] = 1;
        if (CTAS > 8) {
            int clusters = 0;
            e = cudaFuncSetAttribute(sort_kernel<CTAS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&clusters, sort_kernel<CTAS>, &cfg);
            if (e != cudaSuccess || clusters < 1) {
                cudaGetLastError();
                state[dev] = -1;
            }
        }
    }
    if (state[dev] < 0) return cudaErrorNotSupported;
    cfg.dynamicSmemBytes = sort_smem_bytes(threads / 32, a.n_experts);
    return cudaLaunchKernelEx(&cfg, sort_kernel<CTAS>, a);
}

}  // namespace

namespace {

// the launch of a kernel that waits for sort_kernel's cluster by itself
template <typename... P, typename... A>
cudaError_t behind_sort(void (*kernel)(P...), dim3 grid, cudaStream_t st, const A &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(ROW_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

bool sort_by_cluster(const SortArgs &a) { return a.n_entries > 4096; }

cudaError_t sort_order(const SortArgs &a, cudaStream_t st) {
    if (a.n_entries >= 32768) {
        const cudaError_t e = sort_launch<16>(a, SORT_THREADS, st);
        if (e != cudaErrorNotSupported) return e;
    }
    if (sort_by_cluster(a)) return sort_launch<8>(a, SORT_THREADS, st);
    int threads = 32;
    while (threads < a.n_entries && threads < SORT_THREADS) threads <<= 1;
    return sort_launch<1>(a, threads, st);
}

}  // namespace

cudaError_t launch_sort(const SortArgs &a, cudaStream_t st) {
    const cudaError_t e = sort_order(a, st);
    if (e != cudaSuccess || !sort_by_cluster(a)) return e;
    static_assert(ROW_THREADS == 256, "place_kernel's CTAs");
    return behind_sort(place_kernel, dim3(static_cast<unsigned>((static_cast<int64_t>(a.n_entries) + 255) / 256)), st, a);
}

cudaError_t launch_gather_sorted(RowArgs a, int type, cudaStream_t st) {
    if (a.n_tok == 0) return cudaSuccess;
    const int v = vec_bytes(a, type == MX_F32 ? 4 : 2);
    const dim3 grid = row_grid(a, v);
    const SortArgs none{};
    if (v == 16) gather_kernel<16, false><<<grid, ROW_THREADS, 0, st>>>(a, none);
    else if (v == 4) gather_kernel<4, false><<<grid, ROW_THREADS, 0, st>>>(a, none);
    else gather_kernel<2, false><<<grid, ROW_THREADS, 0, st>>>(a, none);
    return cudaGetLastError();
}

template <int V>
cudaError_t dispatch_v(const SortArgs &s, const RowArgs &a, dim3 grid, cudaStream_t st) {
    static bool configured[64] = {};
    constexpr size_t most = sizeof(int) * (ROW_THREADS / 32 * static_cast<size_t>(SORT_MAX_EXPERTS) + DISPATCH_PER * ROW_THREADS);
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(dispatch_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    dispatch_kernel<V><<<grid, ROW_THREADS, sizeof(int) * (ROW_THREADS / 32 * static_cast<size_t>(s.n_experts) + s.n_entries), st>>>(s, a);
    return cudaGetLastError();
}

cudaError_t launch_dispatch_sorted(const SortArgs &s, RowArgs a, int type, cudaStream_t st) {
    if (a.n_tok == 0) return launch_sort(s, st);
    const int v = vec_bytes(a, type == MX_F32 ? 4 : 2);
    const dim3 grid = row_grid(a, v);
    if (s.n_entries > DISPATCH_PER * ROW_THREADS || grid.x * grid.y > DISPATCH_CTAS) {
        const cudaError_t e = sort_order(s, st);
        if (e != cudaSuccess) return e;
        if (!sort_by_cluster(s)) return launch_gather_sorted(a, type, st);
        return v == 16 ? behind_sort(gather_kernel<16, true>, grid, st, a, s)
             : v == 4 ? behind_sort(gather_kernel<4, true>, grid, st, a, s) : behind_sort(gather_kernel<2, true>, grid, st, a, s);
    }
    return v == 16 ? dispatch_v<16>(s, a, grid, st) : v == 4 ? dispatch_v<4>(s, a, grid, st) : dispatch_v<2>(s, a, grid, st);
}

cudaError_t launch_combine_sorted(RowArgs a, int type, cudaStream_t st) {
    if (a.n_tok == 0) return cudaSuccess;
    return type == MX_F32 ? combine_t<MX_F32>(a, st) : type == MX_F16 ? combine_t<MX_F16>(a, st) : combine_t<MX_BF16>(a, st);
}

cudaError_t launch_combine_sorted_grad(const RowArgs &a, int type, cudaStream_t st) {
    if (a.n_tok == 0 || (!a.out && !a.d_weights)) return cudaSuccess;
    return type == MX_F32 ? grad_t<MX_F32>(a, st) : type == MX_F16 ? grad_t<MX_F16>(a, st) : grad_t<MX_BF16>(a, st);
}

}  // namespace moe
