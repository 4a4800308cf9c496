// The router over many tokens and its balance loss, forward and backward.
//
// Routing (decode_step.route_tokens; NemotronHMoE.route_tokens_to_experts, tf:697-720): score = sigmoid(logit) (or the
// softmax of the row), choice = score + bias, optionally only the best expert groups, the top_k choices in decreasing
// order (ties to the lower id, a NaN as if it were -inf), weight = score (/ (their sum + 1e-20)) * scaling, and how
// many tokens chose each expert. The choice of a softmax row is its logit, which has the scores' order; the sum of a
// group's two best logits has that of the product of its two best scores (not of their sum). A group that is left out
// counts as 0 with sigmoids, so that its experts come before negative choices, as the model's router has it; of a
// softmax none of them is ever chosen.
//   backward, dw -> dlogits: ds_i = scaling dw_i, or with the sum S over the chosen scaling (dw_i - sum_j dw_j s_j / S) / S;
//   sigmoid: dl_i = ds_i s_i (1 - s_i) at the chosen; softmax: dl_j = p_j (ds_j - sum_i ds_i p_i) everywhere.
// Balance loss: p_te = score_te / sum_e score_te, P_e = mean of p_te over the T' unmasked tokens, f_e = E count_e / (k T'),
//   loss = coef sum_e f_e P_e;  with c_e = coef f_e / T': dl_tj = p_tj (c_j - sum_e c_e p_te) (times 1 - s_tj for sigmoid).
//
// All four kernels give a token to a warp, which holds its logits in registers, one per lane and 32 experts: the row is
// read once and every sum over experts is a warp's. The loss's gradient runs near the logits' bytes (32768 x 512 fp32 with
// a fifth masked: 121 MB in 21 us). Its sums (54 MB in 20 us) and the routing (16384 x 512: 34 MB in 25 us) take twice the
// time of their instructions at the full issue rate (9 and 13 us): a token's load and its chains of shuffles, with eight
// warps per scheduler and nothing of the next token in flight, are the rest.
#include <cmath>

#include "common.cuh"
#include "host.h"

namespace qmoe {
namespace rt {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int MAX_E = 1024, MAX_K = 32;

__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float wide(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Clusters: a barrier of all threads that makes shared memory visible, and a word of CTA `rank`'s shared memory.
constexpr int CLUSTER = 8;
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t word_of(const void *p, int rank) {
    uint32_t v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.b32 %0, [r];\n\t}"
                 : "=r"(v) : "r"(smem_u32(p)), "r"(rank) : "memory");
    return v;
}
// A launch as clusters of n CTAs; pdl: it may begin before the kernel in front of it has ended (and waits in it).
template <typename K, typename A>
static int launch_cluster(K kern, unsigned grid, int threads, size_t smem, int n, bool pdl, cudaStream_t st, const A &a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)n;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) {
        cudaGetLastError();
        return QMOE_ERR_LAUNCH;
    }
    return launch_status();
}

// torch's fp32 sigmoid, bit for bit (expf, IEEE division).
__device__ __forceinline__ float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// Which expert lane `lane`'s register i holds. Up to 128 experts one per lane and 32, so that every lane has some; more:
// four consecutive ones per lane and 128, which one wide load brings.
template <int EPL> __device__ __forceinline__ int expert(int i, int lane) {
    return EPL == 4 ? i * 32 + lane : (i >> 2) * 128 + lane * 4 + (i & 3);
}

// A lane's logits; -inf past ne. vec: rows allow four elements per load.
template <typename T, int EPL> __device__ __forceinline__ void load_row(const T *row, int ne, int lane, bool vec, float (&x)[EPL]) {
#pragma unroll
    for (int i = 0; i < EPL; i += 4) {
        if (EPL > 4 && vec) {
            const int e = expert<EPL>(i, lane);   // ne is a multiple of 4: all four or none
            if constexpr (sizeof(T) == 4) {
                float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                if (e < ne) v = *reinterpret_cast<const float4 *>(row + e);
                x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
            } else {
                uint2 v = make_uint2(0u, 0u);
                if (e < ne) v = *reinterpret_cast<const uint2 *>(row + e);
                const T *h = reinterpret_cast<const T *>(&v);
#pragma unroll
                for (int j = 0; j < 4; j++) x[i + j] = e < ne ? wide(h[j]) : -INFINITY;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int e = expert<EPL>(i + j, lane);
                x[i + j] = e < ne ? wide(row[e]) : -INFINITY;
            }
        }
    }
}

// The same places of a row, stored.
template <typename T, int EPL> __device__ __forceinline__ void store_row(T *row, int ne, int lane, bool vec, const float (&x)[EPL]) {
#pragma unroll
    for (int i = 0; i < EPL; i += 4) {
        if (EPL > 4 && vec) {
            const int e = expert<EPL>(i, lane);
            if (e >= ne) continue;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(row + e) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
            } else {
                uint2 v;
                T *h = reinterpret_cast<T *>(&v);
#pragma unroll
                for (int j = 0; j < 4; j++) h[j] = narrow<T>(x[i + j]);
                *reinterpret_cast<uint2 *>(row + e) = v;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int e = expert<EPL>(i + j, lane);
                if (e < ne) row[e] = narrow<T>(x[i + j]);
            }
        }
    }
}

// Softmax of a row, in place.
template <int EPL> __device__ __forceinline__ void softmax_row(float (&x)[EPL], int ne, int lane) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) m = fmaxf(m, x[i]);
    m = warp_max(m);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        x[i] = expert<EPL>(i, lane) < ne ? expf(x[i] - m) : 0.f;
        s += x[i];
    }
    s = 1.f / warp_sum(s);
#pragma unroll
    for (int i = 0; i < EPL; i++) x[i] *= s;
}

struct Route {
    const void *logits;
    int64_t ld;
    const float *bias;   // may be null
    int64_t T;
    int ne, k, n_group, topk_group, norm, softmax, vec;
    int cluster;         // the CTAs are one cluster
    float scaling;
    int64_t *ids;        // [T, k]
    float *w;            // [T, k]
    int *counts;         // [ne]
    const float *dw;     // backward
    void *dl;
};

// Order of choices (no NaN, no -0) as unsigned keys: larger choice, larger key; 0 is below every choice.
__device__ __forceinline__ uint32_t key_of(float c) {
    const uint32_t b = __float_as_uint(c);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}

// Keeps the choices of the topk_group groups with the largest sums of their two best choices (ties to the lower group),
// the others become `fill`. buf: ne floats of this warp. Returns which of the lane's choices became so.
template <int EPL>
__device__ __forceinline__ uint32_t keep_groups(float (&c)[EPL], const Route &a, float fill, float *buf, int lane) {
    const int size = a.ne / a.n_group;
#pragma unroll
    for (int i = 0; i < EPL; i++)
        if (expert<EPL>(i, lane) < a.ne) buf[expert<EPL>(i, lane)] = c[i];
    __syncwarp();
    float mine = -INFINITY;   // lane g: group g's sum
    for (int g = 0; g < a.n_group; g++) {
        float b1 = -INFINITY, b2 = -INFINITY;
        for (int j = lane; j < size; j += 32) {
            const float v = buf[g * size + j];
            b2 = fmaxf(b2, fminf(b1, v));
            b1 = fmaxf(b1, v);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const float o1 = __shfl_xor_sync(0xffffffffu, b1, o), o2 = __shfl_xor_sync(0xffffffffu, b2, o);
            b2 = fmaxf(fmaxf(b2, o2), fminf(b1, o1));
            b1 = fmaxf(b1, o1);
        }
        if (lane == g) mine = fmaxf(b1 + b2, -INFINITY);   // of opposite infinities: last
    }
    int rank = 0;
    for (int g = 0; g < a.n_group; g++) {
        const float v = __shfl_sync(0xffffffffu, mine, g);
        rank += v > mine || (v == mine && g < lane);
    }
    const uint32_t kept = __ballot_sync(0xffffffffu, lane < a.n_group && rank < a.topk_group);
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < EPL; i++)
        if (expert<EPL>(i, lane) < a.ne && !(kept >> (expert<EPL>(i, lane) / size) & 1u)) {
            c[i] = fill;
            out |= 1u << i;
        }
    __syncwarp();
    return out;
}

// The lane's value of a descending bitonic sort of the warp's 32 values.
__device__ __forceinline__ float sort_desc(float v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, j);
            v = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}

constexpr int MAX_CAND = 64;
struct Candidates {   // of one warp: choice (as a key) and expert, the lower expert larger; score
    unsigned long long key[MAX_CAND];
    float s[MAX_CAND];
};

// k rounds of the warp's largest key, of equal ones the lowest expert: lane r gets the r-th. For rows with many equal
// choices; on random logits of 16384 x 512 these rounds alone took 94 us. FAST: v holds logits, else scores, c choices.
// Choices in `out` take no part, also where others are -inf (there are k of those).
template <int EPL, bool FAST>
__device__ __noinline__ void choose_by_rounds(const Route &a, int lane, const float (&c)[EPL], const float (&v)[EPL], uint32_t out, const float *bias, int &id, float &sc) {
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const int e = expert<EPL>(i, lane);
        key[i] = e < a.ne && !(out >> i & 1u) ? key_of(FAST ? fmaxf(sigmoid(v[i]) + bias[e], -INFINITY) : c[i]) : 0u;
    }
    for (int r = 0; r < a.k; r++) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < EPL; i++) m = max(m, key[i]);
        m = __reduce_max_sync(0xffffffffu, m);
        uint32_t e = 0xFFFFFFFFu;
#pragma unroll
        for (int i = EPL - 1; i >= 0; i--)
            if (key[i] == m) e = expert<EPL>(i, lane);
        e = __reduce_min_sync(0xffffffffu, e);
        float x = 0.f;
        bool here = false;
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (e == (uint32_t)expert<EPL>(i, lane)) {
                key[i] = 0u;
                x = v[i];
                here = true;
            }
        x = __shfl_sync(0xffffffffu, x, __ffs(__ballot_sync(0xffffffffu, here)) - 1);
        if (lane == r) id = (int)e, sc = FAST ? sigmoid(x) : x;
    }
}

// One token. The k-th largest of the 32 lanes' largest choices bounds the k-th largest choice from below, so only those
// from there on can be chosen: about 34 of 512 experts for k = 22. They are gathered in shared memory, and the rank of
// each among them is its place, since (choice, lower expert first) is unique: a lane counts the rank of one, and what is
// beyond 32 the warp counts by votes. More than MAX_CAND, or a bound of -inf: by rounds.
//
// FAST (sigmoid scores, no groups): c holds choices of approximate scores and v the logits. An approximate score is off by
// under 2^-21 (its exponent's rounding, |x| 2^-24, shrinks by s (1 - s); two approximate instructions), so with twice
// that and two places of the sum as a margin no choice at or above the bound is missed; torch's bits are computed for
// the gathered ones alone. With exact scores for all it was 1,580 instructions a token, now 940 (512 experts, ncu):
// 16384 x 512 in 43, now 25 us.
template <int EPL, bool FAST>
__device__ __forceinline__ void choose(const Route &a, int64_t t, int lane, const float (&c)[EPL], const float (&v)[EPL], uint32_t out, const float *bias, Candidates &cand, int *hist) {
    float top = c[0];
#pragma unroll
    for (int i = 1; i < EPL; i++) top = fmaxf(top, c[i]);
    float bound = __shfl_sync(0xffffffffu, sort_desc(top, lane), a.k - 1);
    if (FAST) bound -= 4e-6f + fabsf(bound) * 0x1p-21f;
    uint32_t in = 0;
#pragma unroll
    for (int i = 0; i < EPL; i++) in |= (uint32_t)(c[i] >= bound) << i;
    const int cnt = __popc(in);
    int off = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, off, o);
        if (lane >= o) off += u;
    }
    const int n = __shfl_sync(0xffffffffu, off, 31);
    off -= cnt;
    int id = 0, rank = MAX_K, id2 = 0, rank2 = MAX_K;
    float sc = 0.f, sc2 = 0.f;
    if (n <= MAX_CAND && bound > -INFINITY) {
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (in >> i & 1u) {
                const uint32_t e = expert<EPL>(i, lane);
                cand.key[off] = (FAST ? 0ull : (unsigned long long)key_of(c[i]) << 32) | (0xFFFFFFFFu - e);
                cand.s[off++] = v[i];
            }
        __syncwarp();
        unsigned long long mine = ~0ull, mine2 = 0;
        auto take = [&](int j, unsigned long long &key, int &e, float &score) {
            key = cand.key[j];
            e = (int)~(uint32_t)key;
            score = cand.s[j];
            if (FAST) {
                score = sigmoid(score);
                key |= (unsigned long long)key_of(fmaxf(score + bias[e], -INFINITY)) << 32;
                cand.key[j] = key;
            }
        };
        if (lane < n) {
            take(lane, mine, id, sc);
            rank = 0;
        }
        if (lane + 32 < n) take(lane + 32, mine2, id2, sc2);
        if (lane == 0 && (n & 1)) cand.key[n] = 0;   // the loop takes two at a time; n odd is below MAX_CAND
        __syncwarp();
#pragma unroll 4
        for (int j = 0; j < n; j += 2) {
            const ulonglong2 u = *reinterpret_cast<const ulonglong2 *>(&cand.key[j]);
            rank += u.x > mine;
            rank += u.y > mine;
        }
        for (int j = 32; j < n; j++) {
            const unsigned long long u = cand.key[j];
            const int r = __popc(__ballot_sync(0xffffffffu, lane < n && mine > u)) + __popc(__ballot_sync(0xffffffffu, mine2 > u));
            if (lane + 32 == j) rank2 = r;
        }
        __syncwarp();
    } else {
        choose_by_rounds<EPL, FAST>(a, lane, c, v, out, bias, id, sc);
        if (lane < a.k) rank = lane;
    }
    float total = 1.f;
    if (a.norm) total = warp_sum((rank < a.k ? sc : 0.f) + (rank2 < a.k ? sc2 : 0.f)) + 1e-20f;
    if (rank < a.k) {
        a.ids[t * a.k + rank] = id;
        a.w[t * a.k + rank] = (a.norm ? sc / total : sc) * a.scaling;
        atomicAdd(&hist[id], 1);
    }
    if (rank2 < a.k) {
        a.ids[t * a.k + rank2] = id2;
        a.w[t * a.k + rank2] = (a.norm ? sc2 / total : sc2) * a.scaling;
        atomicAdd(&hist[id2], 1);
    }
}

// blockDim.x / 32 tokens at a time, up to ROUTE_WARPS. Every CTA adds its counts to the global ones at its end, so many
// tokens take one large CTA per SM, up to 20 tokens per SM small CTAs of WARPS, up to four per SM (T x 512, small against
// large: 1184 tokens 8.3 and 10.4 us, 2960 12.2 and 12.4, 4736 14.4 and 11.8, 37888 47 and 42). What CLUSTER small
// CTAs hold at a token per warp is one cluster, whose CTAs add up each other's counts: no clearing before the launch (64 x
// 512: 6.3 and 4.7 us; with CLUSTER large CTAs 256 tokens took 7.5 instead of 6.3).
template <int EPL> constexpr int ROUTE_WARPS = EPL > 16 ? 16 : 32;
template <typename T, int EPL, bool FAST> __global__ void __launch_bounds__(ROUTE_WARPS<EPL> * 32) route_kernel(const Route a) {
    constexpr int SLOTS = EPL * 32;
    extern __shared__ __align__(16) uint8_t raw[];
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Candidates &cand = reinterpret_cast<Candidates *>(raw)[warp];
    float *bias = reinterpret_cast<float *>(raw + warps * sizeof(Candidates));   // [SLOTS], 0 without one
    int *hist = reinterpret_cast<int *>(bias + SLOTS);                           // [ne]
    float *buf = reinterpret_cast<float *>(hist + a.ne) + warp * a.ne;           // [warps][ne], only with groups
    for (int e = threadIdx.x; e < SLOTS; e += blockDim.x) {
        bias[e] = a.bias && e < a.ne ? a.bias[e] : 0.f;
        if (e < a.ne) hist[e] = 0;
    }
    __syncthreads();
    for (int64_t t = blockIdx.x * (int64_t)warps + warp; t < a.T; t += (int64_t)gridDim.x * warps) {
        float v[EPL], c[EPL];   // logits (FAST) or scores; choices
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, a.vec, v);
        if constexpr (FAST) {
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                float e, s;
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v[i] * -1.44269504f));
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
                c[i] = fmaxf(s + bias[expert<EPL>(i, lane)], -INFINITY);         // a NaN last
            }
        } else if (a.softmax) {
#pragma unroll
            for (int i = 0; i < EPL; i++) c[i] = fmaxf(v[i], -INFINITY) + 0.f;   // the two zeros are equal
            softmax_row<EPL>(v, a.ne, lane);
        } else {
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                v[i] = sigmoid(v[i]);
                c[i] = fmaxf(v[i] + bias[expert<EPL>(i, lane)], -INFINITY);      // no score is -0, so no choice is
            }
        }
        uint32_t out = 0;   // choices that are none
        if constexpr (!FAST)
            if (a.n_group > 1) {
                const uint32_t u = keep_groups<EPL>(c, a, a.softmax ? -INFINITY : 0.f, buf, lane);
                if (a.softmax) out = u;
            }
        if (a.ne < SLOTS)
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (expert<EPL>(i, lane) >= a.ne) c[i] = -INFINITY;
        choose<EPL, FAST>(a, t, lane, c, v, out, bias, cand, hist);
    }
    if (a.cluster) {
        cluster_sync();
        for (int e = blockIdx.x * blockDim.x + threadIdx.x; e < a.ne; e += gridDim.x * blockDim.x) {
            int n = 0;
            for (int r = 0; r < (int)gridDim.x; r++) n += (int)word_of(&hist[e], r);
            a.counts[e] = n;
        }
        cluster_sync();   // no CTA leaves while another reads its counts
        return;
    }
    __syncthreads();
    const int turn = (int)(blockIdx.x * 96u % a.ne);   // CTAs that end together start at different experts
    for (int i = threadIdx.x; i < a.ne; i += blockDim.x) {   // integers: the order of the additions does not matter
        const int e = i + turn < a.ne ? i + turn : i + turn - a.ne;
        if (gridDim.x == 1) a.counts[e] = hist[e];
        else if (hist[e]) atomicAdd(&a.counts[e], hist[e]);
    }
}

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS) route_backward_kernel(const Route a) {
    extern __shared__ float sm[];
    float *row = sm + (threadIdx.x >> 5) * a.ne;
    const int lane = threadIdx.x & 31;
    for (int e = lane; e < a.ne; e += 32) row[e] = 0.f;
    __syncwarp();
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * WARPS) {
        const T *x = static_cast<const T *>(a.logits) + t * a.ld;
        const int64_t id64 = lane < a.k ? a.ids[t * a.k + lane] : -1;
        const bool on = id64 >= 0 && id64 < a.ne;   // an id that route cannot have given takes no part
        const int id = on ? (int)id64 : 0;
        float ds = on ? a.dw[t * a.k + lane] * a.scaling : 0.f;
        float p[EPL];
        float s = 0.f;
        if (a.softmax) {
            load_row<T, EPL>(x, a.ne, lane, a.vec, p);
            softmax_row<EPL>(p, a.ne, lane);
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (expert<EPL>(i, lane) < a.ne) row[expert<EPL>(i, lane)] = p[i];
            __syncwarp();
            if (on) s = row[id];
            __syncwarp();
            for (int e = lane; e < a.ne; e += 32) row[e] = 0.f;
            __syncwarp();
        } else if (on) {
            s = sigmoid(wide(x[id]));
        }
        if (a.norm) {
            const float total = warp_sum(s) + 1e-20f;
            ds = (ds - warp_sum(ds * s) / total) / total;
        }
        const float dot = a.softmax ? warp_sum(on ? ds * s : 0.f) : 0.f;
        if (on) row[id] = a.softmax ? ds : ds * s * (1.f - s);
        __syncwarp();
        float d[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = expert<EPL>(i, lane);
            d[i] = e < a.ne ? row[e] : 0.f;
            if (a.softmax) d[i] = p[i] * (d[i] - dot);
        }
        store_row<T, EPL>(static_cast<T *>(a.dl) + t * a.ne, a.ne, lane, a.vec, d);
        __syncwarp();
        if (on) row[id] = 0.f;
        __syncwarp();
    }
}

struct Balance {
    const void *logits;
    int64_t ld;
    const void *ids;          // [T, k] int64 or int32; outside [0, ne): not counted
    int ids64;
    const uint8_t *mask;      // [T] or null: tokens with 0 take no part
    int64_t T;
    int ne, k, softmax, parts, vec;
    float coef;
    float *part_p;            // [parts, ne] sums of p
    int *part_n;              // [parts, ne + 1] counts, then unmasked tokens
    float *loss;
    int *counts;
    float *c;                 // [ne] coef * f_e / T'
    const float *grad;        // backward: d loss
    void *dl;
};

constexpr int MAX_PARTS = 160;
// A CTA per SM: 32 warps of 64 registers, 16 where a lane holds 32 experts.
template <int EPL> constexpr int BAL_WARPS = EPL > 16 ? 16 : 32;

// sigmoid and 1 - sigmoid as products of one reciprocal (1 ulp), where nothing is decided by their last bit, as it is in
// the routing: neither loses digits near 1. e^-x is 2^y for y = fl(-x log2 e), corrected by what that rounding left.
// x is kept to [-87, 126] (a NaN stays one), where no step overflows; what lies outside counts as the border. From 87.3 on
// e^-x lies below the normal numbers and is 0, and 1 - sigmoid with it.
__device__ __forceinline__ void sigmoid_pair(float x, float &s, float &r) {
    asm("max.NaN.f32 %0, %0, 0fC2AE0000;\n\tmin.NaN.f32 %0, %0, 0f42FC0000;" : "+f"(x));
    constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;
    const float y = -x * LOG2E;
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(y));
    e = fmaf(e, fmaf(-x, LOG2E, -y) * LN2, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
    r = e * s;
}

// A row whose scores sum to less is under -20 everywhere: sigmoid(x) is e^x to fp32's last place there, and p the softmax.
// Its sigmoids may all underflow, their ratios need not.
constexpr float LOW = 2e-9f;

// Up to so many tokens per warp of CLUSTER CTAs are one kernel instead of two (256 x 512: 8.5 and 9.7 us, 512 x 512 10.0 and
// 9.7, 1024 x 512 13.3 and 9.8; and a launch less for the host).
constexpr int ONE_TOKENS = 2;

// An expert's count and coefficient stored; its term of the loss.
__device__ __forceinline__ float expert_term(const Balance &a, int e, float p, int n, int rows) {
    const float f = rows ? (float)n * ((float)a.ne / ((float)a.k * (float)rows)) : 0.f;
    a.counts[e] = n;
    a.c[e] = rows ? a.coef * f / (float)rows : 0.f;
    return rows ? f * (p / (float)rows) : 0.f;
}

// The sum of the CTAs' terms in their order, by the first one.
__device__ __forceinline__ void store_loss(const Balance &a, const float *mine, int ctas) {
    cluster_sync();
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        float sum = 0.f;
        for (int i = 0; i < ctas; i++) sum += __uint_as_float(word_of(mine, i));
        *a.loss = a.coef * sum;
    }
    cluster_sync();   // no CTA leaves before its term is read
}

// ONE: few tokens, all CTAs in one cluster, which adds their sums as well: no second kernel.
template <typename T, int EPL, bool ONE> __global__ void __launch_bounds__(BAL_WARPS<EPL> * 32) balance_kernel(const Balance a) {
    constexpr int W = BAL_WARPS<EPL>;
    extern __shared__ float sm[];
    float *sums = sm;                                     // [W][ne]
    int *hist = reinterpret_cast<int *>(sm + W * a.ne);   // [ne + 1]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e <= a.ne; e += W * 32) hist[e] = 0;
    __syncthreads();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) acc[i] = 0.f;
    int rows = 0;
    const int64_t step = (int64_t)gridDim.x * W;
    uint32_t live = 0;   // masks of the warp's next 32 tokens, fetched together
    int left = 0;
    for (int64_t t = blockIdx.x * (int64_t)W + warp; t < a.T; t += step, live >>= 1, left--) {
        if (a.mask && left == 0) {
            live = __ballot_sync(0xffffffffu, t + lane * step < a.T && a.mask[t + lane * step]);
            left = 32;
        }
        if (a.mask && !(live & 1u)) continue;
        rows++;
        const T *row = static_cast<const T *>(a.logits) + t * a.ld;
        float s[EPL];
        load_row<T, EPL>(row, a.ne, lane, a.vec, s);
        for (int j = lane; j < a.k; j += 32) {
            const int64_t e = a.ids64 ? static_cast<const int64_t *>(a.ids)[t * a.k + j] : static_cast<const int *>(a.ids)[t * a.k + j];
            if (e >= 0 && e < a.ne) atomicAdd(&hist[e], 1);
        }
        float inv = 1.f;
        if (!a.softmax) {   // past ne x is -inf: 1e-38 each, nothing beside LOW
            float total = 0.f, r;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                sigmoid_pair(s[i], s[i], r);
                total += s[i];
            }
            total = warp_sum(total);
            inv = 1.f / total;
            if (total < LOW) load_row<T, EPL>(row, a.ne, lane, a.vec, s);
            if (total < LOW) inv = 0.f;
        }
        if (a.softmax || inv == 0.f) {
            softmax_row<EPL>(s, a.ne, lane);
            inv = 1.f;
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) acc[i] = fmaf(s[i], inv, acc[i]);
    }
    if (lane == 0 && rows) atomicAdd(&hist[a.ne], rows);
#pragma unroll
    for (int i = 0; i < EPL; i++)
        if (expert<EPL>(i, lane) < a.ne) sums[warp * a.ne + expert<EPL>(i, lane)] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < a.ne; e += W * 32) {   // the warps in order: the same sums every time
        float p = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) p += sums[w * a.ne + e];
        if (ONE) sums[e] = p;   // column e is this thread's alone
        else a.part_p[(int64_t)blockIdx.x * a.ne + e] = p;
    }
    if constexpr (ONE) {
        __shared__ float red[W], mine;
        cluster_sync();
        rows = 0;
        for (int r = 0; r < a.parts; r++) rows += (int)word_of(&hist[a.ne], r);
        float term = 0.f;
        for (int e = blockIdx.x * W * 32 + threadIdx.x; e < a.ne; e += a.parts * W * 32) {
            float p = 0.f;
            int n = 0;
            for (int r = 0; r < a.parts; r++) {
                p += __uint_as_float(word_of(&sums[e], r));
                n += (int)word_of(&hist[e], r);
            }
            term += expert_term(a, e, p, n, rows);
        }
        term = warp_sum(term);
        if (lane == 0) red[warp] = term;
        __syncthreads();
        if (warp == 0) {
            term = warp_sum(lane < W ? red[lane] : 0.f);
            if (lane == 0) mine = term;
        }
        store_loss(a, &mine, a.parts);
    } else {
        for (int e = threadIdx.x; e <= a.ne; e += W * 32) a.part_n[(int64_t)blockIdx.x * (a.ne + 1) + e] = hist[e];
    }
}

// The parts' sums: a cluster of FIN CTAs, each every FIN-th run of 32 experts, 32 rows of parts at a time (one CTA with a
// thread per expert took 250 us for 592 parts). Every sum runs in a fixed order.
constexpr int FIN = CLUSTER;
__global__ void __launch_bounds__(1024) balance_final_kernel(const Balance a) {
    __shared__ float sp[32][33];
    __shared__ int sn[32][33];
    __shared__ int rows_of[32];
    __shared__ float mine;
    const int lane = threadIdx.x & 31, y = threadIdx.x >> 5, rank = blockIdx.x;
    pdl_wait();
    int r = 0;
    for (int i = threadIdx.x; i < a.parts; i += 1024) r += a.part_n[(int64_t)i * (a.ne + 1) + a.ne];
    r = __reduce_add_sync(0xffffffffu, r);
    if (lane == 0) rows_of[y] = r;
    __syncthreads();
    const int rows = __reduce_add_sync(0xffffffffu, rows_of[lane]);
    float term = 0.f;
    for (int e0 = rank * 32; e0 < a.ne; e0 += FIN * 32) {
        const int e = e0 + lane;
        float p = 0.f;
        int n = 0;
        if (e < a.ne)
#pragma unroll 4
            for (int i = y; i < a.parts; i += 32) {
                p += a.part_p[(int64_t)i * a.ne + e];
                n += a.part_n[(int64_t)i * (a.ne + 1) + e];
            }
        sp[y][lane] = p;
        sn[y][lane] = n;
        __syncthreads();
        // warp y sums expert e0 + y over the 32 rows
        p = warp_sum(sp[lane][y]);
        n = __reduce_add_sync(0xffffffffu, sn[lane][y]);
        if (lane == 0 && e0 + y < a.ne) term += expert_term(a, e0 + y, p, n, rows);
        __syncthreads();
    }
    if (lane == 0) sp[0][y] = term;
    __syncthreads();
    if (y == 0) {
        term = warp_sum(sp[0][lane]);
        if (lane == 0) mine = term;
    }
    store_loss(a, &mine, FIN);
}

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS, EPL > 16 ? 2 : 4) balance_backward_kernel(const Balance a) {
    const int lane = threadIdx.x & 31;
    const float g = *a.grad;
    float c[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) c[i] = expert<EPL>(i, lane) < a.ne ? a.c[expert<EPL>(i, lane)] : 0.f;
    const int64_t step = (int64_t)gridDim.x * WARPS;
    uint32_t live = 0;   // as in balance_kernel
    int left = 0;
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += step, live >>= 1, left--) {
        if (a.mask && left == 0) {
            live = __ballot_sync(0xffffffffu, t + lane * step < a.T && a.mask[t + lane * step]);
            left = 32;
        }
        T *out = static_cast<T *>(a.dl) + t * a.ne;
        const T *row = static_cast<const T *>(a.logits) + t * a.ld;
        float u[EPL];   // p before its division, times 1 - s
        if (a.mask && !(live & 1u)) {
#pragma unroll
            for (int i = 0; i < EPL; i++) u[i] = 0.f;
            store_row<T, EPL>(out, a.ne, lane, a.vec, u);
            continue;
        }
        load_row<T, EPL>(row, a.ne, lane, a.vec, u);
        float total = 1.f, dot = 0.f;
        if (!a.softmax) {
            total = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                float s, r;
                sigmoid_pair(u[i], s, r);
                total += s;
                dot = fmaf(c[i], s, dot);
                u[i] = s * r;
            }
            total = warp_sum(total);
            if (total < LOW) load_row<T, EPL>(row, a.ne, lane, a.vec, u);
        }
        if (a.softmax || total < LOW) {
            softmax_row<EPL>(u, a.ne, lane);
            total = 1.f;
            dot = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; i++) dot = fmaf(c[i], u[i], dot);
        }
        const float inv = 1.f / total;
        dot = warp_sum(dot) * inv;
        const float f = g * inv;
#pragma unroll
        for (int i = 0; i < EPL; i++) u[i] = f * u[i] * (c[i] - dot);
        store_row<T, EPL>(out, a.ne, lane, a.vec, u);
    }
}

// f(T{}, EPL constant) for the logits' type and the number of experts.
template <typename T, typename F> static int by_width(int ne, F f) {
    if (ne <= 128) return f(T{}, std::integral_constant<int, 4>{});
    if (ne <= 256) return f(T{}, std::integral_constant<int, 8>{});
    if (ne <= 512) return f(T{}, std::integral_constant<int, 16>{});
    return f(T{}, std::integral_constant<int, 32>{});
}
template <typename F> static int by_type(int dt, int ne, F f) {
    if (dt == QMOE_DT_BF16) return by_width<__nv_bfloat16>(ne, f);
    if (dt == QMOE_DT_F16) return by_width<__half>(ne, f);
    return by_width<float>(ne, f);
}

// Rows of `rows` elements apart, read or written four at a time: their start and length allow it.
static bool four(const void *p, int dt, int64_t stride, int ne) {
    const int size = dt == QMOE_DT_F32 ? 4 : 2;
    return ne % 4 == 0 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & (4 * size - 1)) == 0;
}

static unsigned grid_of(int64_t T, const DeviceInfo &di, int per_sm) {
    const int64_t g = (T + WARPS - 1) / WARPS, most = (int64_t)di.sms * per_sm;
    return (unsigned)(g < most ? g : most);
}

static bool aligned(const void *p, int dt) { return reinterpret_cast<uintptr_t>(p) % (dt == QMOE_DT_F32 ? 4 : 2) == 0; }

static int check_logits(const void *logits, int dt, int64_t ld, int64_t T, int ne, int k, int score) {
    if (!logits) return QMOE_ERR_NULL;
    if (T < 1 || T > 0x7FFFFFFF || ne < 1 || ne > MAX_E || k < 1 || ld < ne || score < 0 || score > 1) return QMOE_ERR_SHAPE;
    if (!valid_dtype(dt)) return QMOE_ERR_DTYPE;
    return aligned(logits, dt) ? QMOE_OK : QMOE_ERR_ALIGN;
}

} // namespace rt
} // namespace qmoe

using namespace qmoe;

extern "C" {

int qmoe_route(const void *logits, int x_dtype, int64_t ld, const float *bias, int64_t T, int n_experts, int top_k,
               int n_group, int topk_group, int norm, int score, float scaling, int64_t *ids, float *weights,
               int32_t *counts, void *stream) {
    if (!ids || !weights || !counts) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, top_k, score)) return e;
    if (top_k > rt::MAX_K || top_k > n_experts || n_group < 1 || n_group > 32 || n_experts % n_group || topk_group < 1 ||
        topk_group > n_group || (n_group > 1 && n_experts / n_group < 2) || (bias && score == 1) ||
        (score == 1 && top_k > n_experts / n_group * topk_group))
        return QMOE_ERR_SHAPE;
    if (!aligned4(bias) || !aligned8(ids) || !aligned4(weights) || !aligned4(counts)) return QMOE_ERR_ALIGN;
    DeviceInfo *di;
    int dev;
    if (int e = current_device(&dev, &di)) return e;
    rt::Route a{};
    a.logits = logits;
    a.ld = ld;
    a.bias = bias;
    a.T = T;
    a.ne = n_experts;
    a.k = top_k;
    a.n_group = n_group;
    a.topk_group = topk_group;
    a.norm = norm != 0;
    a.softmax = score == 1;
    a.scaling = scaling;
    a.ids = ids;
    a.w = weights;
    a.counts = counts;
    a.vec = rt::four(logits, x_dtype, ld, n_experts);
    cudaStream_t st = as_stream(stream);
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) -> int {
        constexpr int EPL = decltype(w)::value;
        using X = decltype(t);
        const int warps = T <= (int64_t)di->sms * 20 ? rt::WARPS : rt::ROUTE_WARPS<EPL>;
        const int64_t ctas = (T + warps - 1) / warps;
        a.cluster = ctas > 1 && ctas <= rt::CLUSTER;
        const unsigned grid = (unsigned)(ctas < di->sms * (warps == rt::WARPS ? 4 : 1) ? ctas : di->sms * (warps == rt::WARPS ? 4 : 1));
        const size_t smem = warps * sizeof(rt::Candidates) + sizeof(float) * (EPL * 32 + n_experts * (n_group > 1 ? 1 + warps : 1));
        auto launch = [&](auto kern, std::atomic<uint64_t> &done) -> int {
            if (!(done.load(std::memory_order_acquire) >> (dev & 63) & 1) && !ensure_smem(kern, smem, dev, done)) return QMOE_ERR_LAUNCH;
            if (a.cluster) return rt::launch_cluster(kern, grid, warps * 32, smem, (int)grid, false, st, a);
            if (grid > 1 && cudaMemsetAsync(counts, 0, sizeof(int) * n_experts, st) != cudaSuccess) return QMOE_ERR_LAUNCH;
            kern<<<grid, warps * 32, smem, st>>>(a);
            return launch_status();
        };
        static std::atomic<uint64_t> done_fast{0}, done_full{0};
        return a.softmax || a.n_group > 1 ? launch(rt::route_kernel<X, EPL, false>, done_full) : launch(rt::route_kernel<X, EPL, true>, done_fast);
    });
}

int qmoe_route_backward(const void *logits, int x_dtype, int64_t ld, int64_t T, int n_experts, int top_k, int norm, int score,
                        float scaling, const int64_t *ids, const float *dweights, void *dlogits, void *stream) {
    if (!ids || !dweights || !dlogits) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, top_k, score)) return e;
    if (top_k > rt::MAX_K || top_k > n_experts) return QMOE_ERR_SHAPE;
    if (!aligned8(ids) || !aligned4(dweights) || !rt::aligned(dlogits, x_dtype)) return QMOE_ERR_ALIGN;
    DeviceInfo *di;
    if (int e = current_device(nullptr, &di)) return e;
    rt::Route a{};
    a.logits = logits;
    a.ld = ld;
    a.T = T;
    a.ne = n_experts;
    a.k = top_k;
    a.norm = norm != 0;
    a.softmax = score == 1;
    a.scaling = scaling;
    a.ids = const_cast<int64_t *>(ids);
    a.dw = dweights;
    a.dl = dlogits;
    a.vec = rt::four(logits, x_dtype, ld, n_experts) && rt::four(dlogits, x_dtype, n_experts, n_experts);
    const unsigned grid = rt::grid_of(T, *di, 8);
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::route_backward_kernel<decltype(t), decltype(w)::value>
            <<<grid, rt::THREADS, sizeof(float) * n_experts * rt::WARPS, as_stream(stream)>>>(a);
        return launch_status();
    });
}

size_t qmoe_balance_workspace_bytes(int64_t T, int n_experts) {
    if (T < 1 || n_experts < 1 || n_experts > rt::MAX_E) return 0;
    const int64_t parts = (T + 15) / 16;   // at least
    return (size_t)(parts < rt::MAX_PARTS ? parts : rt::MAX_PARTS) * (2 * n_experts + 1) * 4;
}

int qmoe_balance(const void *logits, int x_dtype, int64_t ld, const void *ids, int ids_64, const uint8_t *mask, int64_t T,
                 int n_experts, int top_k, int score, float coef, float *loss, int32_t *counts, float *c, void *workspace,
                 size_t workspace_bytes, void *stream) {
    if (!ids || !loss || !counts || !c || !workspace) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, top_k, score)) return e;
    if (T * top_k > INT32_MAX) return QMOE_ERR_SHAPE;   // counts are 32 bits
    if (!aligned4(workspace) || !(ids_64 ? aligned8(ids) : aligned4(ids)) || !aligned4(loss) || !aligned4(counts) || !aligned4(c)) return QMOE_ERR_ALIGN;
    if (workspace_bytes < qmoe_balance_workspace_bytes(T, n_experts)) return QMOE_ERR_WORKSPACE;
    DeviceInfo *di;
    int dev;
    if (int e = current_device(&dev, &di)) return e;
    rt::Balance a{};
    a.logits = logits;
    a.ld = ld;
    a.ids = ids;
    a.ids64 = ids_64 != 0;
    a.mask = mask;
    a.T = T;
    a.ne = n_experts;
    a.k = top_k;
    a.softmax = score == 1;
    a.coef = coef;
    a.loss = loss;
    a.counts = counts;
    a.c = c;
    a.vec = rt::four(logits, x_dtype, ld, n_experts);
    const int warps = n_experts > 512 ? rt::BAL_WARPS<32> : rt::BAL_WARPS<16>;
    const int64_t parts = (T + warps - 1) / warps;
    const int most = di->sms < rt::MAX_PARTS ? di->sms : rt::MAX_PARTS;
    a.parts = (int)(parts < most ? parts : most);
    a.part_p = static_cast<float *>(workspace);
    a.part_n = static_cast<int *>(workspace) + (int64_t)a.parts * n_experts;
    cudaStream_t st = as_stream(stream);
    const bool one = T <= rt::ONE_TOKENS * rt::CLUSTER * warps;
    if (one && a.parts > rt::CLUSTER) a.parts = rt::CLUSTER;
    const int rc = rt::by_type(x_dtype, n_experts, [&](auto t, auto w) -> int {
        static std::atomic<uint64_t> done_one{0}, done_parts{0};
        using X = decltype(t);
        constexpr int EPL = decltype(w)::value, W = rt::BAL_WARPS<EPL>;
        const size_t smem = sizeof(float) * ((W + 1) * n_experts + 1);   // at most 68 KB
        auto launch = [&](auto kern, std::atomic<uint64_t> &done) -> int {
            if (!(done.load(std::memory_order_acquire) >> (dev & 63) & 1) && !ensure_smem(kern, smem, dev, done)) return QMOE_ERR_LAUNCH;
            return rt::launch_cluster(kern, (unsigned)a.parts, W * 32, smem, one ? a.parts : 1, false, st, a);
        };
        return one ? launch(rt::balance_kernel<X, EPL, true>, done_one) : launch(rt::balance_kernel<X, EPL, false>, done_parts);
    });
    if (rc || one) return rc;
    return rt::launch_cluster(rt::balance_final_kernel, rt::FIN, 1024, 0, rt::FIN, true, st, a);
}

int qmoe_balance_backward(const void *logits, int x_dtype, int64_t ld, const uint8_t *mask, int64_t T, int n_experts,
                          int score, const float *c, const float *dloss, void *dlogits, void *stream) {
    if (!c || !dloss || !dlogits) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, 1, score)) return e;
    if (!aligned4(c) || !aligned4(dloss) || !rt::aligned(dlogits, x_dtype)) return QMOE_ERR_ALIGN;
    DeviceInfo *di;
    if (int e = current_device(nullptr, &di)) return e;
    rt::Balance a{};
    a.logits = logits;
    a.ld = ld;
    a.mask = mask;
    a.T = T;
    a.ne = n_experts;
    a.softmax = score == 1;
    a.c = const_cast<float *>(c);
    a.grad = dloss;
    a.dl = dlogits;
    a.vec = rt::four(logits, x_dtype, ld, n_experts) && rt::four(dlogits, x_dtype, n_experts, n_experts);
    const unsigned grid = rt::grid_of(T, *di, 4);
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::balance_backward_kernel<decltype(t), decltype(w)::value><<<grid, rt::THREADS, 0, as_stream(stream)>>>(a);
        return launch_status();
    });
}

} // extern "C"
