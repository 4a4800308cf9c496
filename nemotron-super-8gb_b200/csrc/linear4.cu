// The linear on four-bit activations and weights (dq_linear_a4): the rows of x quantised as dq_quantize_nvfp4 does, then
// multiplied as dq_gemm_nvfp4 does. Up to TOKENS rows are one kernel: the weights' bytes bound it, so tensor cores have
// nothing to give, and a second launch and a cluster's hand-offs cost more than the product (one token on
// 2688 x 4096, caches cold: quantiser 3.5 and tensor-core kernel 9.4 us, this one 6.5). More rows are the two kernels.
//
// Each CTA quantises the rows itself, into shared memory as f16: a code times its block scale has 6 significant bits
// between 2^-10 and 2688, so that is exact. A warp streams two weight rows at a time with 16-byte loads and sums
// code x value products in fp32 (mixed-precision FMA: products exact), scaled per 16-element group by the weight's scale,
// as the GEMVs of gemv.cuh do.
#include "common.cuh"
#include "epilogue4.cuh"
#include "host.h"
#include "quant.cuh"

namespace qmoe {
namespace g4 {

constexpr int TOKENS = 4, TOK_THREADS = 256, TOK_WARPS = TOK_THREADS / 32;

struct TokenArgs {
    const uint8_t *w, *sc;
    const float *sw;
    int sw_step;
    const void *x;
    int64_t ldx;
    int N, K, vec, rows;   // rows: weight rows per CTA
    int epilogue;
    const void *res;
    void *y;
};

// Two e2m1 codes' f16x2 times a block scale's f16x2 (both halves the same): exact.
__device__ __forceinline__ uint32_t mul_h2(uint32_t a, uint32_t b) { return h2_as_u(__hmul2(as_h2(a), as_h2(b))); }

template <typename T, int M, int CPL> __global__ void __launch_bounds__(TOK_THREADS) token_kernel(const TokenArgs a) {
    extern __shared__ uint4 xs[];   // [m][q][chunk]: eight f16 of chunk's 32 elements, so that lanes read side by side
    __shared__ uint32_t red[TOK_WARPS][M];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nch = a.K / 32, nb = a.K / 16;
    pdl_wait();

    // ---- rows of x: largest magnitudes, then codes
    uint32_t top[M];
#pragma unroll
    for (int m = 0; m < M; m++) {
        top[m] = 0;
        for (int b = tid; b < nb; b += TOK_THREADS) {
            qz::Raw<T> v;
            qz::load16(static_cast<const T *>(a.x) + m * a.ldx + b * 16, a.vec, v);
            top[m] = max(top[m], qz::block_max(v) & ~qz::NONFINITE);
        }
        top[m] = __reduce_max_sync(0xffffffffu, top[m]);
        if (lane == 0) red[warp][m] = top[m];
    }
    __syncthreads();
    float sx[M];
#pragma unroll
    for (int m = 0; m < M; m++) {
#pragma unroll
        for (int i = 0; i < TOK_WARPS; i++) top[m] = max(top[m], red[i][m]);
        const int e = qz::scale_exp(top[m]);
        sx[m] = pow2f(e);
        for (int b = tid; b < nb; b += TOK_THREADS) {
            qz::Raw<T> v;
            qz::load16(static_cast<const T *>(a.x) + m * a.ldx + b * 16, a.vec, v);
            uint2 c;
            const uint32_t s1 = qz::block16<T>(v, qz::block_max(v), e, c), s2 = e4m3x2_f16x2((uint16_t)(s1 | (s1 << 8)));
            uint32_t o[8];
            e2m1x8_f16x2(c.x, reinterpret_cast<uint32_t(&)[4]>(o[0]));
            e2m1x8_f16x2(c.y, reinterpret_cast<uint32_t(&)[4]>(o[4]));
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = mul_h2(o[i], s2);
            uint4 *dst = xs + ((size_t)m * 4 + (b & 1) * 2) * nch + (b >> 1);
            dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
            dst[nch] = make_uint4(o[4], o[5], o[6], o[7]);
        }
    }
    __syncthreads();

    // ---- weight rows, two per warp and round
    const int row0 = blockIdx.x * a.rows, end = min(row0 + a.rows, a.N);
    for (int r = row0 + warp * 2; r < end; r += TOK_WARPS * 2) {
        float acc[2][M];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int m = 0; m < M; m++) acc[i][m] = 0.f;
        for (int cb = 0; cb < nch; cb += 32 * CPL) {
            uint4 wv[2][CPL];
            uint16_t sv[2][CPL];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int64_t row = min(r + i, end - 1);
#pragma unroll
                for (int k = 0; k < CPL; k++) {
                    const int c = cb + lane + 32 * k;
                    if (c < nch) {
                        wv[i][k] = ldg_stream(a.w + row * (a.K / 2) + 16 * c);
                        sv[i][k] = __ldg(reinterpret_cast<const uint16_t *>(a.sc + row * nb) + c);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < CPL; k++) {
                const int c = cb + lane + 32 * k;
                if (c >= nch) continue;
#pragma unroll
                for (int m = 0; m < M; m++) {
                    uint4 xq[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) xq[q] = xs[((size_t)m * 4 + q) * nch + c];
                    const uint32_t *xw = reinterpret_cast<const uint32_t *>(xq);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t *ww = reinterpret_cast<const uint32_t *>(&wv[i][k]);
                        float g[2][2] = {{0.f, 0.f}, {0.f, 0.f}};   // the chunk's two groups
#pragma unroll
                        for (int wd = 0; wd < 4; wd++) {
                            uint32_t o[4];
                            e2m1x8_f16x2(ww[wd], o);
#pragma unroll
                            for (int j = 0; j < 4; j++) fma2_f16_f32(o[j], xw[4 * wd + j], g[wd >> 1][0], g[wd >> 1][1]);
                        }
                        const float2 sf = __half22float2(as_h2(e4m3x2_f16x2(sv[i][k])));
                        acc[i][m] = fmaf(g[0][0] + g[0][1], sf.x, acc[i][m]);
                        acc[i][m] = fmaf(g[1][0] + g[1][1], sf.y, acc[i][m]);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int o = 16; o; o >>= 1) acc[i][m] += __shfl_xor_sync(0xffffffffu, acc[i][m], o);
        const int n = r + lane;
        if (lane < 2 && n < end) {
            const float sw = a.sw[(int64_t)n * a.sw_step];
#pragma unroll
            for (int m = 0; m < M; m++) {
                const float v = lane ? acc[1][m] : acc[0][m];
                const int64_t at = (int64_t)m * a.N + n;
                if (a.epilogue == 0) store_one<T, 0>(a.y, a.res, at, v, sx[m], sw);
                else if (a.epilogue == 1) store_one<T, 1>(a.y, a.res, at, v, sx[m], sw);
                else store_one<T, 2>(a.y, a.res, at, v, sx[m], sw);
            }
        }
    }
}

template <typename T, int M, int CPL> static int launch_tokens(const TokenArgs &a, cudaStream_t st, int dev) {
    static std::atomic<uint64_t> done{0};
    auto kern = token_kernel<T, M, CPL>;
    const size_t smem = (size_t)M * a.K * 2;
    if (!(done.load(std::memory_order_acquire) >> (dev & 63) & 1) && !ensure_smem(kern, smem, dev, done)) return QMOE_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.N + a.rows - 1) / a.rows));
    cfg.blockDim = dim3(TOK_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, a) != cudaSuccess) {
        cudaGetLastError();
        return QMOE_ERR_LAUNCH;
    }
    return launch_status();
}

template <typename T, int M> static int launch_tokens(const TokenArgs &a, cudaStream_t st, int dev) {
    return a.K <= 2048 ? launch_tokens<T, M, 2>(a, st, dev) : launch_tokens<T, M, 4>(a, st, dev);
}

template <typename T> static int launch_tokens(const TokenArgs &a, int M, cudaStream_t st, int dev) {
    switch (M) {
    case 1: return launch_tokens<T, 1>(a, st, dev);
    case 2: return launch_tokens<T, 2>(a, st, dev);
    case 3: return launch_tokens<T, 3>(a, st, dev);
    default: return launch_tokens<T, 4>(a, st, dev);
    }
}

} // namespace g4
} // namespace qmoe

using namespace qmoe;

extern "C" {

size_t dq_linear_a4_workspace_bytes(int64_t M, int64_t K) {
    if (M < 1 || M > (1 << 24) || K < 32 || (K % 32) || K > (1 << 24)) return 0;
    return (size_t)(M * (K / 2) + (M + 127) / 128 * ((K + 63) / 64) * 512 + (M + 3) / 4 * 16 + M * (K / 16));
}

int dq_linear_a4(const uint8_t *w, const uint8_t *w_sc, const uint8_t *w_atoms, const float *sw, int sw_per_row, const void *x,
                 int x_dtype, int64_t ldx, int M, int N, int K, int epilogue, const void *residual, void *y, void *workspace,
                 size_t workspace_bytes, void *stream) {
    const bool few = M <= g4::TOKENS && K <= 16384;   // up to 128 KB of quantised rows in shared memory
    if (!w || !w_sc || !sw || !x || !y || (!few && (!w_atoms || !workspace)) || (epilogue == 2 && !residual)) return QMOE_ERR_NULL;
    const size_t need = dq_linear_a4_workspace_bytes(M, K);
    if (!need || N < 1 || N > (1 << 24) || epilogue < 0 || epilogue > 2 || ldx < K) return QMOE_ERR_SHAPE;
    if (!valid_dtype(x_dtype)) return QMOE_ERR_DTYPE;
    const int size = x_dtype == QMOE_DT_F32 ? 4 : 2;
    if ((!few && !aligned16(workspace)) || !aligned16(w) || (reinterpret_cast<uintptr_t>(w_sc) & 1u) || !aligned4(sw) ||
        reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(y) % size || reinterpret_cast<uintptr_t>(residual) % size)
        return QMOE_ERR_ALIGN;
    if (!few && workspace_bytes < need) return QMOE_ERR_WORKSPACE;
    int dev;
    DeviceInfo *di;
    if (int e = current_device(&dev, &di)) return e;
    if (few) {
        g4::TokenArgs a{};
        a.w = w;
        a.sc = w_sc;
        a.sw = sw;
        a.sw_step = sw_per_row != 0;
        a.x = x;
        a.ldx = ldx;
        a.N = N;
        a.K = K;
        a.vec = qz::row_vec(x, ldx * size);
        const int unit = 2 * g4::TOK_WARPS, target = 2 * di->sms;   // about two CTAs per SM, whole rounds of rows
        a.rows = ((N + target - 1) / target + unit - 1) / unit * unit;
        a.epilogue = epilogue;
        a.res = residual;
        a.y = y;
        cudaStream_t st = as_stream(stream);
        if (x_dtype == QMOE_DT_BF16) return g4::launch_tokens<__nv_bfloat16>(a, M, st, dev);
        if (x_dtype == QMOE_DT_F16) return g4::launch_tokens<__half>(a, M, st, dev);
        return g4::launch_tokens<float>(a, M, st, dev);
    }
    uint8_t *codes = static_cast<uint8_t *>(workspace), *atoms = codes + (int64_t)M * (K / 2);
    uint8_t *s = atoms + (int64_t)((M + 127) / 128) * ((K + 63) / 64) * 512, *sc = s + (int64_t)(M + 3) / 4 * 16;
    if (int e = dq_quantize_nvfp4(x, x_dtype, ldx, M, K, 1, codes, sc, reinterpret_cast<float *>(s), atoms, stream)) return e;
    return dq_gemm_nvfp4(w, w_atoms, sw, sw_per_row, codes, atoms, reinterpret_cast<float *>(s), 1, M, N, K, epilogue, residual, y, x_dtype, stream);
}

} // extern "C"
