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

// A lane's logits: expert i * 32 + lane; -inf past ne.
template <typename T, int EPL> __device__ __forceinline__ void load_row(const T *row, int ne, int lane, float (&x)[EPL]) {
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        const int e = i * 32 + lane;
        x[i] = e < ne ? wide(row[e]) : -INFINITY;
    }
}

// x -> scores; for softmax the probabilities.
template <int EPL> __device__ __forceinline__ void scores(float (&x)[EPL], int ne, int lane, bool softmax) {
    if (!softmax) {
#pragma unroll
        for (int i = 0; i < EPL; i++) x[i] = i * 32 + lane < ne ? sigmoid(x[i]) : 0.f;
        return;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPL; i++) m = fmaxf(m, x[i]);
    m = warp_max(m);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; i++) {
        x[i] = i * 32 + lane < ne ? expf(x[i] - m) : 0.f;
        s += x[i];
    }
    s = warp_sum(s);
#pragma unroll
    for (int i = 0; i < EPL; i++) x[i] /= s;
}

struct Route {
    const void *logits;
    int64_t ld;
    const float *bias;   // may be null
    int64_t T;
    int ne, k, n_group, topk_group, norm, softmax;
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
        if (i * 32 + lane < a.ne) buf[i * 32 + lane] = c[i] != c[i] ? -INFINITY : c[i];
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
        if (i * 32 + lane < a.ne && !(kept >> ((i * 32 + lane) / size) & 1u)) c[i] = fill;
    __syncwarp();
}

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS) route_kernel(const Route a) {
    extern __shared__ float sm[];
    int *hist = reinterpret_cast<int *>(sm);
    float *buf = sm + a.ne + (threadIdx.x >> 5) * a.ne;   // only with groups
    const int lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < a.ne; e += THREADS) hist[e] = 0;
    __syncthreads();
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * WARPS) {
        float s[EPL], c[EPL];
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, s);
#pragma unroll
        for (int i = 0; i < EPL; i++) c[i] = s[i];
        scores<EPL>(s, a.ne, lane, a.softmax);
        if (!a.softmax) {
#pragma unroll
            for (int i = 0; i < EPL; i++) c[i] = i * 32 + lane < a.ne ? s[i] + (a.bias ? a.bias[i * 32 + lane] : 0.f) : 0.f;
        }
        if (a.n_group > 1) keep_groups<EPL>(c, a, a.softmax ? -INFINITY : 0.f, buf, lane);
        uint32_t key[EPL];
#pragma unroll
        for (int i = 0; i < EPL; i++) key[i] = i * 32 + lane < a.ne ? key_of(c[i]) : 0u;
        // k rounds: the largest key of the warp, of equal ones the lowest expert
        int id = 0;
        float sc = 0.f;
        for (int r = 0; r < a.k; r++) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < EPL; i++) m = max(m, key[i]);
            m = __reduce_max_sync(0xffffffffu, m);
            uint32_t e = 0xFFFFFFFFu;
#pragma unroll
            for (int i = EPL - 1; i >= 0; i--)
                if (key[i] == m) e = i * 32 + lane;
            e = __reduce_min_sync(0xffffffffu, e);
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (e == (uint32_t)(i * 32 + lane)) {
                    key[i] = 0u;
                    v = s[i];
                }
            v = __shfl_sync(0xffffffffu, v, e & 31);
            if (lane == r) id = (int)e, sc = v;
        }
        float w = sc;
        if (a.norm) w = sc / (warp_sum(lane < a.k ? sc : 0.f) + 1e-20f);
        if (lane < a.k) {
            a.ids[t * a.k + lane] = id;
            a.w[t * a.k + lane] = w * a.scaling;
            atomicAdd(&hist[id], 1);
        }
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
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * WARPS) {
        const T *x = static_cast<const T *>(a.logits) + t * a.ld;
        T *out = static_cast<T *>(a.dl) + t * a.ne;
        const int id = lane < a.k ? (int)a.ids[t * a.k + lane] : 0;
        float ds = lane < a.k ? a.dw[t * a.k + lane] * a.scaling : 0.f;
        float p[EPL];
        float s = 0.f;
        if (a.softmax) {
            load_row<T, EPL>(x, a.ne, lane, p);
            scores<EPL>(p, a.ne, lane, true);
#pragma unroll
            for (int i = 0; i < EPL; i++) {
                if (i * 32 >= a.ne) break;
                const float v = __shfl_sync(0xffffffffu, p[i], id & 31);
                if (id >> 5 == i) s = v;
            }
            if (lane >= a.k) s = 0.f;
        } else if (lane < a.k) {
            s = sigmoid(wide(x[id]));
        }
        if (a.norm) {
            const float total = warp_sum(s) + 1e-20f;
            ds = (ds - warp_sum(ds * s) / total) / total;
        }
        const float dot = a.softmax ? warp_sum(lane < a.k ? ds * s : 0.f) : 0.f;
        for (int e = lane; e < a.ne; e += 32) row[e] = 0.f;
        __syncwarp();
        if (lane < a.k) row[id] = a.softmax ? ds : ds * s * (1.f - s);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = i * 32 + lane;
            if (e < a.ne) out[e] = narrow<T>(a.softmax ? p[i] * (row[e] - dot) : row[e]);
        }
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
    int ne, k, softmax, parts;
    float coef;
    float *part_p;            // [parts, ne] sums of p
    int *part_n;              // [parts, ne + 1] counts, then unmasked tokens
    float *loss;
    int *counts;
    float *c;                 // [ne] coef * f_e / T'
    const float *grad;        // backward: d loss
    void *dl;
};

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS) balance_kernel(const Balance a) {
    extern __shared__ float sm[];
    int *hist = reinterpret_cast<int *>(sm);              // [ne + 1]
    float *sums = sm + a.ne + 1;                          // [ne]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < 2 * a.ne + 1; e += THREADS) sm[e] = 0.f;   // zero bits for both
    __syncthreads();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) acc[i] = 0.f;
    int rows = 0;
    for (int64_t t = blockIdx.x * (int64_t)WARPS + warp; t < a.T; t += (int64_t)gridDim.x * WARPS) {
        if (a.mask && !a.mask[t]) continue;
        rows++;
        float s[EPL];
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, s);
        for (int j = lane; j < a.k; j += 32) {
            const int64_t e = a.ids64 ? static_cast<const int64_t *>(a.ids)[t * a.k + j] : static_cast<const int *>(a.ids)[t * a.k + j];
            if (e >= 0 && e < a.ne) atomicAdd(&hist[e], 1);
        }
        scores<EPL>(s, a.ne, lane, a.softmax);
        float inv = 1.f;
        if (!a.softmax) {
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < EPL; i++) total += s[i];
            inv = 1.f / warp_sum(total);
        }
#pragma unroll
        for (int i = 0; i < EPL; i++) acc[i] += s[i] * inv;
    }
    if (lane == 0 && rows) atomicAdd(&hist[a.ne], rows);
    for (int w = 0; w < WARPS; w++) {   // the warps in order: the same sums every time
        if (warp == w) {
#pragma unroll
            for (int i = 0; i < EPL; i++)
                if (i * 32 + lane < a.ne) sums[i * 32 + lane] += acc[i];
        }
        __syncthreads();
    }
    for (int e = threadIdx.x; e < a.ne; e += THREADS) a.part_p[(int64_t)blockIdx.x * a.ne + e] = sums[e];
    for (int e = threadIdx.x; e <= a.ne; e += THREADS) a.part_n[(int64_t)blockIdx.x * (a.ne + 1) + e] = hist[e];
}

// One CTA: the parts' sums in order, one expert per thread.
__global__ void __launch_bounds__(MAX_E) balance_final_kernel(const Balance a) {
    __shared__ int rows;
    __shared__ float red[MAX_E / 32];
    const int e = threadIdx.x;
    if (e == 0) rows = 0;
    __syncthreads();
    for (int i = e; i < a.parts; i += blockDim.x) {
        const int v = a.part_n[(int64_t)i * (a.ne + 1) + a.ne];
        if (v) atomicAdd(&rows, v);
    }
    float p = 0.f;
    int n = 0;
    if (e < a.ne)
        for (int i = 0; i < a.parts; i++) {
            p += a.part_p[(int64_t)i * a.ne + e];
            n += a.part_n[(int64_t)i * (a.ne + 1) + e];
        }
    __syncthreads();
    float term = 0.f;
    if (e < a.ne) {
        const float f = rows ? (float)n * ((float)a.ne / ((float)a.k * (float)rows)) : 0.f;
        term = rows ? f * (p / (float)rows) : 0.f;
        a.counts[e] = n;
        a.c[e] = rows ? a.coef * f / (float)rows : 0.f;
    }
    term = warp_sum(term);
    if (!(e & 31)) red[e >> 5] = term;
    __syncthreads();
    if (e < 32) {
        term = warp_sum(e < (int)(blockDim.x >> 5) ? red[e] : 0.f);
        if (e == 0) *a.loss = a.coef * term;
    }
}

template <typename T, int EPL> __global__ void __launch_bounds__(THREADS) balance_backward_kernel(const Balance a) {
    const int lane = threadIdx.x & 31;
    const float g = *a.grad;
    float c[EPL];
#pragma unroll
    for (int i = 0; i < EPL; i++) c[i] = i * 32 + lane < a.ne ? a.c[i * 32 + lane] : 0.f;
    for (int64_t t = blockIdx.x * (int64_t)WARPS + (threadIdx.x >> 5); t < a.T; t += (int64_t)gridDim.x * WARPS) {
        T *out = static_cast<T *>(a.dl) + t * a.ne;
        if (a.mask && !a.mask[t]) {
            for (int e = lane; e < a.ne; e += 32) out[e] = narrow<T>(0.f);
            continue;
        }
        float s[EPL];
        load_row<T, EPL>(static_cast<const T *>(a.logits) + t * a.ld, a.ne, lane, s);
        scores<EPL>(s, a.ne, lane, a.softmax);
        float total = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            total += s[i];
            dot += c[i] * s[i];
        }
        const float inv = a.softmax ? 1.f : 1.f / warp_sum(total);
        dot = warp_sum(dot) * inv;
#pragma unroll
        for (int i = 0; i < EPL; i++) {
            const int e = i * 32 + lane;
            const float d = g * (s[i] * inv) * (c[i] - dot);
            if (e < a.ne) out[e] = narrow<T>(a.softmax ? d : d * (1.f - s[i]));
        }
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
    const unsigned grid = rt::grid_of(T, *di, 8);
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::route_backward_kernel<decltype(t), decltype(w)::value>
            <<<grid, rt::THREADS, sizeof(float) * n_experts * rt::WARPS, as_stream(stream)>>>(a);
        return launch_status();
    });
}

size_t qmoe_balance_workspace_bytes(int64_t T, int n_experts) {
    if (T < 1 || n_experts < 1 || n_experts > rt::MAX_E) return 0;
    const int64_t parts = (T + rt::WARPS - 1) / rt::WARPS;
    return (size_t)(parts < 4 * 160 ? parts : 4 * 160) * (2 * n_experts + 1) * 4;
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
    int64_t parts = (T + rt::WARPS - 1) / rt::WARPS;
    const int most = 4 * (di->sms < 160 ? di->sms : 160);
    a.parts = (int)(parts < most ? parts : most);
    a.part_p = static_cast<float *>(workspace);
    a.part_n = static_cast<int *>(workspace) + (int64_t)a.parts * n_experts;
    cudaStream_t st = as_stream(stream);
    const int rc = rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::balance_kernel<decltype(t), decltype(w)::value>
            <<<a.parts, rt::THREADS, sizeof(float) * (2 * n_experts + 1), st>>>(a);
        return launch_status();
    });
    if (rc) return rc;
    rt::balance_final_kernel<<<1, (n_experts + 31) / 32 * 32, 0, st>>>(a);
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
    const unsigned grid = rt::grid_of(T, *di, 8);
    return rt::by_type(x_dtype, n_experts, [&](auto t, auto w) {
        rt::balance_backward_kernel<decltype(t), decltype(w)::value><<<grid, rt::THREADS, 0, as_stream(stream)>>>(a);
        return launch_status();
    });
}

} // extern "C"
