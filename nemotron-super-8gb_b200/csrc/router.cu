// The router over many tokens and its balance loss, forward and backward.
//
// Routing (decode_step.route_tokens; NemotronHMoE.route_tokens_to_experts, tf:697-720): score = sigmoid(logit) (or the
// softmax of the row), choice = score + bias, optionally only the best expert groups, the top_k choices in decreasing
// order (ties to the lower id, a NaN never before a number), weight = score (/ (their sum + 1e-20)) * scaling, and how
// many tokens chose each expert. Softmax rows are chosen by their logits, which have the same order.
//   backward, dw -> dlogits: ds_i = scaling dw_i, or with the sum S over the chosen scaling (dw_i - sum_j dw_j s_j / S) / S;
//   sigmoid: dl_i = ds_i s_i (1 - s_i) at the chosen; softmax: dl_j = p_j (ds_j - sum_i ds_i p_i) everywhere.
// Balance loss: p_te = score_te / sum_e score_te, P_e = mean of p_te over the T' unmasked tokens, f_e = E count_e / (k T'),
//   loss = coef sum_e f_e P_e;  with c_e = coef f_e / T': dl_tj = p_tj (c_j - sum_e c_e p_te) (times 1 - s_tj for sigmoid).
//
// All four kernels give a token to a warp, which holds its logits in registers, one per lane and 32 experts: the row is
// read once and every sum over experts is a warp's. They are bound by the logits' bytes, and by issue (the exact
// sigmoid, the selection) next to them.
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
    float scaling;
    int64_t *ids;        // [T, k]
    float *w;            // [T, k]
    int *counts;         // [ne]
    const float *dw;     // backward
    void *dl;
};

// Order of choices as unsigned keys: larger choice, larger key; 0 is below every choice.
__device__ __forceinline__ uint32_t key_of(float c) {
    c = c != c ? -INFINITY : c + 0.f;   // + 0: the two zeros are equal
    const uint32_t b = __float_as_uint(c);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Keeps the choices of the topk_group groups with the largest sums of their two best choices (ties to the lower group),
// the others become `fill`. buf: ne floats of this warp.
template <int EPL>
__device__ __forceinline__ void keep_groups(float (&c)[EPL], const Route &a, float fill, float *buf, int lane) {
    const int size = a.ne / a.n_group;
#pragma unroll
    for (int i = 0; i < EPL; i++)
        if (expert<EPL>(i, lane) < a.ne) buf[expert<EPL>(i, lane)] = c[i] != c[i] ? -INFINITY : c[i];
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
        if (lane == g) mine = b1 + b2;
    }
    int rank = 0;
    for (int g = 0; g < a.n_group; g++) {
        const float v = __shfl_sync(0xffffffffu, mine, g);
        rank += v > mine || (v == mine && g < lane);
    }
    const uint32_t kept = __ballot_sync(0xffffffffu, lane < a.n_group && rank < a.topk_group);
#pragma unroll
    for (int i = 0; i < EPL; i++)
        if (expert<EPL>(i, lane) < a.ne && !(kept >> (expert<EPL>(i, lane) / size) & 1u)) c[i] = fill;
    __syncwarp();
}

// The lane's value of a descending bitonic sort of the warp's 32 keys.
__device__ __forceinline__ uint32_t sort_desc(uint32_t v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) {
            const uint32_t o = __shfl_xor_sync(0xffffffffu, v, j);
            v = ((lane & j) == 0) == ((lane & k) == 0) ? max(v, o) : min(v, o);
        }
    return v;
}

constexpr int MAX_CAND = 64;

// One token. The k-th largest of the 32 lanes' largest keys bounds the k-th largest key from below, so only the keys
// from there on can be chosen: about 34 for 512 experts and k = 22. They are gathered in shared memory, and the rank of
// each among them, counted by a lane, is its place: (key, lower expert first) is unique. Rows with many equal keys, or
// too few lanes with experts, can have more than MAX_CAND; those take k rounds of the warp's maximum. On random logits
// of 16384 x 512 the rounds alone took 94 us.
template <int EPL>
__device__ __forceinline__ void choose(const Route &a, int64_t t, int lane, uint32_t (&key)[EPL], const float (&s)[EPL], uint4 *cand, int *hist) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < EPL; i++) top = max(top, key[i]);
    const uint32_t bound = max(__shfl_sync(0xffffffffu, sort_desc(top, lane), a.k - 1), 1u);
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < EPL; i++) cnt += key[i] >= bound;
    int off = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, off, o);
        if (lane >= o) off += v;
    }
    const int n = __shfl_sync(0xffffffffu, off, 31);
    off -= cnt;
    int id[2] = {0, 0}, rank[2] = {MAX_K, MAX_K};
    float sc[2] = {0.f, 0.f};
    if (n <= MAX_CAND) {
#pragma unroll
        for (int i = 0; i < EPL; i++)
            if (key[i] >= bound) cand[off++] = make_uint4(~(uint32_t)expert<EPL>(i, lane), key[i], __float_as_uint(s[i]), 0u);
        __syncwarp();
        unsigned long long mine[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int c = lane + 32 * u;
            mine[u] = ~0ull;   // none: ranks behind nothing, and is not stored
            if (c < n) {
                const uint4 v = cand[c];
                mine[u] = (unsigned long long)v.y << 32 | v.x;
                id[u] = (int)~v.x;
                sc[u] = __uint_as_float(v.z);
                rank[u] = 0;
            }
        }
        for (int j = 0; j < n; j++) {
            const unsigned long long v = *reinterpret_cast<const unsigned long long *>(&cand[j]);
            rank[0] += v > mine[0];
            if (n > 32) rank[1] += v > mine[1];
        }
        __syncwarp();
    } else {
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
            float v = 0.f;
            bool here = false;
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (e == (uint32_t)expert<EPL>(i, lane)) {
                    key[i] = 0u;
                    v = s[i];
                    here = true;
                }
            v = __shfl_sync(0xffffffffu, v, __ffs(__ballot_sync(0xffffffffu, here)) - 1);
            if (lane == r) id[0] = (int)e, sc[0] = v, rank[0] = r;
        }
    }
    float total = 1.f;
    if (a.norm) total = warp_sum((rank[0] < a.k ? sc[0] : 0.f) + (rank[1] < a.k ? sc[1] : 0.f)) + 1e-20f;
#pragma unroll
    for (int u = 0; u < 2; u++)
        if (rank[u] < a.k) {
            a.ids[t * a.k + rank[u]] = id[u];
            a.w[t * a.k + rank[u]] = (a.norm ? sc[u] / total : sc[u]) * a.scaling;
            atomicAdd(&hist[id[u]], 1);
        }
}

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS, EPL > 16 ? 2 : 4) route_kernel(const Route a) {
    extern __shared__ float sm[];
    __shared__ uint4 cands[WARPS][MAX_CAND];
    int *hist = reinterpret_cast<int *>(sm);
    float *buf = sm + a.ne + (threadIdx.x >> 5) * a.ne;   // only with groups
    const int lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < a.ne; e += THREADS) hist[e] = 0;
    __syncthreads();
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * WARPS) {
        float s[EPL], c[EPL];
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, a.vec, s);
        if (a.softmax) {
#pragma unroll
            for (int i = 0; i < EPL; i++) c[i] = s[i];
            softmax_row<EPL>(s, a.ne, lane);
        } else {
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                const int e = expert<EPL>(i, lane);
                s[i] = sigmoid(s[i]);
                c[i] = a.bias && e < a.ne ? s[i] + a.bias[e] : s[i];
            }
        }
        if (a.n_group > 1) keep_groups<EPL>(c, a, a.softmax ? -INFINITY : 0.f, buf, lane);
        uint32_t key[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) key[i] = expert<EPL>(i, lane) < a.ne ? key_of(c[i]) : 0u;
        choose<EPL>(a, t, lane, key, s, cands[threadIdx.x >> 5], hist);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < a.ne; e += THREADS) {   // integers: the order of the additions does not matter
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
        const int id = lane < a.k ? (int)a.ids[t * a.k + lane] : 0;
        float ds = lane < a.k ? a.dw[t * a.k + lane] * a.scaling : 0.f;
        float p[EPL];
        float s = 0.f;
        if (a.softmax) {
            load_row<T, EPL>(x, a.ne, lane, a.vec, p);
            softmax_row<EPL>(p, a.ne, lane);
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (expert<EPL>(i, lane) < a.ne) row[expert<EPL>(i, lane)] = p[i];
            __syncwarp();
            if (lane < a.k) s = row[id];
            __syncwarp();
            for (int e = lane; e < a.ne; e += 32) row[e] = 0.f;
            __syncwarp();
        } else if (lane < a.k) {
            s = sigmoid(wide(x[id]));
        }
        if (a.norm) {
            const float total = warp_sum(s) + 1e-20f;
            ds = (ds - warp_sum(ds * s) / total) / total;
        }
        const float dot = a.softmax ? warp_sum(lane < a.k ? ds * s : 0.f) : 0.f;
        if (lane < a.k) row[id] = a.softmax ? ds : ds * s * (1.f - s);
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
        if (lane < a.k) row[id] = 0.f;
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

constexpr int BAL_WARPS = 16, BAL_THREADS = BAL_WARPS * 32, MAX_PARTS = 320;

// sigmoid and 1 - sigmoid as products of one reciprocal (1 ulp): neither loses digits near 1, and nothing is decided
// by their last bit, as it is in the routing.
__device__ __forceinline__ void sigmoid_pair(float x, float &s, float &r) {
    const float e = fminf(expf(-x), 8e37f);   // its reciprocal is still a normal number
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + e));
    r = e * s;
}

// Whether a row's p are its softmax: asked for, or scores so low (all under 2e-9) that sigmoid(x) is e^x to fp32's last
// place. Their sigmoids may all underflow, their ratios need not.
template <int EPL> __device__ __forceinline__ bool as_softmax(const float (&x)[EPL], bool softmax) {
    if (softmax) return true;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) m = fmaxf(m, x[i]);
    return warp_max(m) < -20.f;
}

template <typename T, int EPL> __global__ void __launch_bounds__(BAL_THREADS) balance_kernel(const Balance a) {
    extern __shared__ float sm[];
    int *hist = reinterpret_cast<int *>(sm);              // [ne + 1]
    float *sums = sm + a.ne + 1;                          // [ne]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < 2 * a.ne + 1; e += BAL_THREADS) sm[e] = 0.f;   // zero bits for both
    __syncthreads();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) acc[i] = 0.f;
    int rows = 0;
    for (int64_t t = blockIdx.x * (int64_t)BAL_WARPS + warp; t < a.T; t += (int64_t)gridDim.x * BAL_WARPS) {
        if (a.mask && !a.mask[t]) continue;
        rows++;
        float s[EPL];
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, a.vec, s);
        for (int j = lane; j < a.k; j += 32) {
            const int64_t e = a.ids64 ? static_cast<const int64_t *>(a.ids)[t * a.k + j] : static_cast<const int *>(a.ids)[t * a.k + j];
            if (e >= 0 && e < a.ne) atomicAdd(&hist[e], 1);
        }
        float inv = 1.f;
        if (as_softmax<EPL>(s, a.softmax)) {
            softmax_row<EPL>(s, a.ne, lane);
        } else {
            float total = 0.f, r;
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                sigmoid_pair(s[i], s[i], r);
                s[i] = expert<EPL>(i, lane) < a.ne ? s[i] : 0.f;
                total += s[i];
            }
            inv = 1.f / warp_sum(total);
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) acc[i] = fmaf(s[i], inv, acc[i]);
    }
    if (lane == 0 && rows) atomicAdd(&hist[a.ne], rows);
    for (int w = 0; w < BAL_WARPS; w++) {   // the warps in order: the same sums every time
        if (warp == w) {
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (expert<EPL>(i, lane) < a.ne) sums[expert<EPL>(i, lane)] += acc[i];
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.ne; e += BAL_THREADS) a.part_p[(int64_t)blockIdx.x * a.ne + e] = sums[e];
    for (int e = threadIdx.x; e <= a.ne; e += BAL_THREADS) a.part_n[(int64_t)blockIdx.x * (a.ne + 1) + e] = hist[e];
}

// The parts' sums: a cluster of FIN CTAs, each every FIN-th run of 32 experts, 32 rows of parts at a time (one CTA with a
// thread per expert took 250 us for 592 parts). Every sum runs in a fixed order.
constexpr int FIN = 8;
__global__ void __launch_bounds__(1024) __cluster_dims__(FIN, 1, 1) balance_final_kernel(const Balance a) {
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
        if (lane == 0 && e0 + y < a.ne) {
            const float f = rows ? (float)n * ((float)a.ne / ((float)a.k * (float)rows)) : 0.f;
            a.counts[e0 + y] = n;
            a.c[e0 + y] = rows ? a.coef * f / (float)rows : 0.f;
            term += rows ? f * (p / (float)rows) : 0.f;
        }
        __syncthreads();
    }
    if (lane == 0) sp[0][y] = term;
    __syncthreads();
    if (y == 0) {
        term = warp_sum(sp[0][lane]);
        if (lane == 0) mine = term;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
        float sum = 0.f;
        for (int i = 0; i < FIN; i++) {
            float v;
            asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}"
                         : "=f"(v) : "r"(smem_u32(&mine)), "r"(i) : "memory");
            sum += v;
        }
        *a.loss = a.coef * sum;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS, EPL > 16 ? 2 : 4) balance_backward_kernel(const Balance a) {
    const int lane = threadIdx.x & 31;
    const float g = *a.grad;
    float c[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) c[i] = expert<EPL>(i, lane) < a.ne ? a.c[expert<EPL>(i, lane)] : 0.f;
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * WARPS) {
        T *out = static_cast<T *>(a.dl) + t * a.ne;
        float s[EPL];
        if (a.mask && !a.mask[t]) {
#pragma unroll
            for (int i = 0; i < EPL; i++) s[i] = 0.f;
            store_row<T, EPL>(out, a.ne, lane, a.vec, s);
            continue;
        }
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, a.vec, s);
        float r[EPL], total = 0.f, dot = 0.f;
        const bool soft = as_softmax<EPL>(s, a.softmax);
        if (soft) softmax_row<EPL>(s, a.ne, lane);
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            r[i] = 1.f;
            if (!soft) {
                sigmoid_pair(s[i], s[i], r[i]);
                s[i] = expert<EPL>(i, lane) < a.ne ? s[i] : 0.f;
            }
            total += s[i];
            dot = fmaf(c[i], s[i], dot);
        }
        const float inv = soft ? 1.f : 1.f / warp_sum(total);
        dot = warp_sum(dot) * inv;
#pragma unroll
        for (int i = 0; i < EPL; i++) s[i] = g * (s[i] * inv) * (c[i] - dot) * r[i];
        store_row<T, EPL>(out, a.ne, lane, a.vec, s);
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

static int check_logits(const void *logits, int dt, int64_t ld, int64_t T, int ne, int k, int score) {
    if (!logits) return QMOE_ERR_NULL;
    if (T < 1 || T > 0x7FFFFFFF || ne < 1 || ne > MAX_E || k < 1 || ld < ne || score < 0 || score > 1) return QMOE_ERR_SHAPE;
    if (!valid_dtype(dt)) return QMOE_ERR_DTYPE;
    return reinterpret_cast<uintptr_t>(logits) % (dt == QMOE_DT_F32 ? 4 : 2) ? QMOE_ERR_ALIGN : QMOE_OK;
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
        topk_group > n_group || (n_group > 1 && n_experts / n_group < 2) || (bias && score == 1))
        return QMOE_ERR_SHAPE;
    DeviceInfo *di;
    if (int e = current_device(nullptr, &di)) return e;
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
    const unsigned grid = rt::grid_of(T, *di, 4);
    if (grid > 1 && cudaMemsetAsync(counts, 0, sizeof(int) * n_experts, st) != cudaSuccess) return QMOE_ERR_LAUNCH;
    const size_t smem = sizeof(float) * n_experts * (n_group > 1 ? 1 + rt::WARPS : 1);   // at most 36 KB
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::route_kernel<decltype(t), decltype(w)::value><<<grid, rt::THREADS, smem, st>>>(a);
        return launch_status();
    });
}

int qmoe_route_backward(const void *logits, int x_dtype, int64_t ld, int64_t T, int n_experts, int top_k, int norm, int score,
                        float scaling, const int64_t *ids, const float *dweights, void *dlogits, void *stream) {
    if (!ids || !dweights || !dlogits) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, top_k, score)) return e;
    if (top_k > rt::MAX_K || top_k > n_experts) return QMOE_ERR_SHAPE;
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
    const int64_t parts = (T + rt::BAL_WARPS - 1) / rt::BAL_WARPS;
    return (size_t)(parts < rt::MAX_PARTS ? parts : rt::MAX_PARTS) * (2 * n_experts + 1) * 4;
}

int qmoe_balance(const void *logits, int x_dtype, int64_t ld, const void *ids, int ids_64, const uint8_t *mask, int64_t T,
                 int n_experts, int top_k, int score, float coef, float *loss, int32_t *counts, float *c, void *workspace,
                 size_t workspace_bytes, void *stream) {
    if (!ids || !loss || !counts || !c || !workspace) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, top_k, score)) return e;
    if (!aligned4(workspace) || (reinterpret_cast<uintptr_t>(ids) & (ids_64 ? 7u : 3u))) return QMOE_ERR_ALIGN;
    if (workspace_bytes < qmoe_balance_workspace_bytes(T, n_experts)) return QMOE_ERR_WORKSPACE;
    DeviceInfo *di;
    if (int e = current_device(nullptr, &di)) return e;
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
    int64_t parts = (T + rt::BAL_WARPS - 1) / rt::BAL_WARPS;
    const int most = 2 * di->sms < rt::MAX_PARTS ? 2 * di->sms : rt::MAX_PARTS;
    a.parts = (int)(parts < most ? parts : most);
    a.part_p = static_cast<float *>(workspace);
    a.part_n = static_cast<int *>(workspace) + (int64_t)a.parts * n_experts;
    cudaStream_t st = as_stream(stream);
    const int rc = rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::balance_kernel<decltype(t), decltype(w)::value>
            <<<a.parts, rt::BAL_THREADS, sizeof(float) * (2 * n_experts + 1), st>>>(a);
        return launch_status();
    });
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rt::FIN);
    cfg.blockDim = dim3(1024);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, rt::balance_final_kernel, a) != cudaSuccess) {
        cudaGetLastError();
        return QMOE_ERR_LAUNCH;
    }
    return launch_status();
}

int qmoe_balance_backward(const void *logits, int x_dtype, int64_t ld, const uint8_t *mask, int64_t T, int n_experts,
                          int score, const float *c, const float *dloss, void *dlogits, void *stream) {
    if (!c || !dloss || !dlogits) return QMOE_ERR_NULL;
    if (int e = rt::check_logits(logits, x_dtype, ld, T, n_experts, 1, score)) return e;
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
    const unsigned grid = rt::grid_of(T, *di, 8);
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::balance_backward_kernel<decltype(t), decltype(w)::value><<<grid, rt::THREADS, 0, as_stream(stream)>>>(a);
        return launch_status();
    });
}

} // extern "C"
