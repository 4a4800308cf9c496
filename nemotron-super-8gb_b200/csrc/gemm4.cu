// Four-bit product (dq_gemm_nvfp4): y[m, n] = sx[m] * sw[n] * sum_k (q_x sc_x)[m, k] * (q_w sc_w)[n, k] for NVFP4
// activations and NVFP4 weights, on block-scaled tcgen05.mma with fp32 accumulators in tensor memory.
//
// A CTA computes tiles of 128 weight rows (the MMA's M) x TN tokens (its N): the weights are on the M side whatever
// the number of tokens, so a few tokens cost a narrow MMA instead of a padded one. Per 256-element stage, TMA brings
// 128 x 128 B of weight codes and TN x 128 B of activation codes (128-byte swizzle), and bulk copies bring both
// operands' scales, which lie in global memory as the tensor core's 512-byte atoms (128 rows x 4 scales per 64-wide
// k-step). One thread copies the stage's atoms to tensor memory (tcgen05.cp) and issues its MMAs; the tensor pipe runs
// both in the order issued, so the scale slots, two of them, need no barrier.
#include "common.cuh"
#include "host.h"
#include "tc.cuh"

namespace qmoe {
namespace g4 {

constexpr int BM = 128;              // weight rows of a tile
constexpr int BK = 256;              // elements of k per stage: four MMA k-steps
constexpr int ROWB = BK / 2;         // bytes of codes per row and stage
constexpr int ATOM = 512;
constexpr int A_BYTES = BM * ROWB;
constexpr int SFA_BYTES = 4 * ATOM;
constexpr int THREADS = 192;         // warps 0..3 epilogue, 4 loads, 5 MMA
constexpr int MAX_SPLIT = 8;

__device__ int g_status;             // first error of this device's calls since it was last cleared

template <int TN> struct Plan {
    static constexpr int NA = (TN + 127) / 128;        // scale atoms of the tokens per k-step
    static constexpr int B_BYTES = TN * ROWB;
    static constexpr int SFB_BYTES = NA * 4 * ATOM;
    static constexpr int OFF_B = A_BYTES, OFF_SFA = OFF_B + B_BYTES, OFF_SFB = OFF_SFA + SFA_BYTES;
    static constexpr int STAGE = (OFF_SFB + SFB_BYTES + 1023) / 1024 * 1024;
    static constexpr int STAGES = 221184 / STAGE < 8 ? 221184 / STAGE : 8;
    static constexpr int OFF_BAR = STAGES * STAGE;
    static constexpr int NBAR = 2 * STAGES + 5;
    static constexpr int OFF_MISC = OFF_BAR + (NBAR * 8 + 15) / 16 * 16;
    static constexpr int SMEM = OFF_MISC + 16 + 1024;
    static_assert(SMEM <= 232448, "fits the 227 KB opt-in");
    // Tensor memory: two accumulators of TN columns and two scale slots. At TN = 256 the accumulators overlap in 96
    // columns (0..255 and 160..415), which the epilogue drains first, so that the next tile starts before it is done.
    static constexpr int ACC1 = TN == 256 ? 160 : TN;
    static constexpr int SF_COL = ACC1 + TN;
    static constexpr int SF_SLOT = 4 * 4 * (1 + NA);
    static constexpr int NEED = SF_COL + 2 * SF_SLOT;
    static constexpr int COLS = NEED <= 128 ? 128 : NEED <= 256 ? 256 : 512;
    static_assert(NEED <= 512, "tensor memory");
    static constexpr int LAG = TN == 256 ? 1 : 2;      // tile t's MMAs wait for the release of tile t - LAG
};

struct Params {
    const uint8_t *sfa, *sfb;   // scale atoms of the weights and of the tokens
    const float *sw, *sx;
    int sw_step, sx_step;       // 0: one scale, 1: one per row
    int M, N, nks, nst;         // tokens, weight rows, 64-wide k-steps, 256-wide stages
    int nbn, ntiles, split;
    int epilogue, dtype;
    const void *res;
    void *y;
    long long wait;
};

__device__ __forceinline__ void cp_sf(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float ld_cluster(uint32_t addr, int rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
                 : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// The product is rounded before a residual is added to it: no fused multiply-add.
__device__ __forceinline__ float scaled(float v, float sx, float sw) { return __fmul_rn(__fmul_rn(v, sx), sw); }

// One result: the linear's value rounded to the output type, then (in fp32, rounded again) its squared ReLU or the
// sum with the residual, as the unfused operators round.
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float wide(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ void store(const Params &p, int64_t at, float v) {
    T o = narrow<T>(v);
    if (p.epilogue == 1) {
        float b = wide(o);
        b = b > 0.f ? b : (b != b ? b : 0.f);
        o = narrow<T>(b * b);
    } else if (p.epilogue == 2) {
        o = narrow<T>(wide(o) + wide(static_cast<const T *>(p.res)[at]));
    }
    static_cast<T *>(p.y)[at] = o;
}

template <int TN, typename T>
__global__ void __launch_bounds__(THREADS, 1)
    gemm_kernel(const Params p, const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b) {
    using P = Plan<TN>;
    constexpr int S = P::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const uint32_t sbase = smem_u32(sm);
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + P::OFF_BAR);
    uint64_t *empty = full + S;
    uint64_t *acc_full = empty + S;      // [2]
    uint64_t *acc_free = acc_full + 2;   // [2] tile t (at t & 1): the columns that tile t + LAG needs are drained
    uint64_t *drain = acc_free + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + P::OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sm + P::OFF_MISC + 8);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // A cluster of `split` CTAs shares one tile, each a part of the stages; without it a CTA walks tiles.
    const int split = p.split, part = split > 1 ? (int)(blockIdx.x % split) : 0;
    const int first = split > 1 ? (int)(blockIdx.x / split) : (int)blockIdx.x;
    const int step = split > 1 ? p.ntiles : (int)gridDim.x;
    const int k0 = (int)((int64_t)p.nst * part / split), k1 = (int)((int64_t)p.nst * (part + 1) / split);

    if (tid == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&acc_full[0], 1);
        mbar_init(&acc_full[1], 1);
        mbar_init(&acc_free[0], 4);
        mbar_init(&acc_free[1], 4);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(P::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    uint32_t q = 0;   // stages loaded (warp 4) or consumed (warp 5)

    if (warp == 4) {
        // ------------------------------------------------------------ loads
        if (lane == 0) {
            bool ok = true;
            for (int i = first; i < p.ntiles && ok; i += step) {
                const int n0 = i % p.nbn * BM, m0 = i / p.nbn * TN;
                const uint8_t *fa = p.sfa + (int64_t)(n0 >> 7) * p.nks * ATOM, *fb = p.sfb + (int64_t)(m0 >> 7) * p.nks * ATOM;
                const int na = P::NA > 1 && m0 + 128 >= p.M ? 1 : P::NA;   // no tokens, and no atoms, past M
                for (int kt = k0; kt < k1; kt++, q++) {
                    const int s = q % S;
                    if (!lane_wait(&empty[s], ((q / S) & 1) ^ 1, abort_flag, &g_status, p.wait)) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = sm + s * P::STAGE;
                    const uint32_t sf = (uint32_t)min(4, p.nks - 4 * kt) * ATOM;
                    mbar_expect_tx(&full[s], A_BYTES + P::B_BYTES + sf * (1 + na));
                    tma_load_2d(st, &tm_a, kt * ROWB, n0, &full[s]);
                    tma_load_2d(st + P::OFF_B, &tm_b, kt * ROWB, m0, &full[s]);
                    bulk_g2s_nohint(st + P::OFF_SFA, fa + (int64_t)kt * SFA_BYTES, sf, &full[s]);
                    for (int a = 0; a < na; a++)
                        bulk_g2s_nohint(st + P::OFF_SFB + a * SFA_BYTES, fb + ((int64_t)a * p.nks + 4 * kt) * ATOM, sf, &full[s]);
                }
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        // ------------------------------------------------------------ scales to tensor memory, MMAs
        if (lane == 0) {
            const uint64_t dbase = smem_desc(0, 16, 1024, 2);   // K-major, 128-byte swizzle
            const uint64_t fbase = smem_desc(0, 16, 128, 0);    // an atom: 32 rows of 16 bytes
            int t = 0;
            bool ok = true;
            for (int i = first; i < p.ntiles && ok; i += step, t++) {
                const int m0 = i / p.nbn * TN;
                const uint32_t idesc = instr_desc_nvfp4((min(TN, p.M - m0) + 15) & ~15);
                const int f = t - P::LAG;
                if (f >= 0 && !lane_wait(&acc_free[f & 1], (f >> 1) & 1, abort_flag, &g_status, p.wait)) break;
                tc_fence_after();
                const uint32_t d = tmem + (t & 1) * P::ACC1;
                for (int kt = k0; kt < k1; kt++, q++) {
                    const int s = q % S;
                    if (!lane_wait(&full[s], (q / S) & 1, abort_flag, &g_status, p.wait)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t st = sbase + s * P::STAGE;
                    const uint32_t slot = tmem + P::SF_COL + (q & 1) * P::SF_SLOT;
                    const int nk = min(4, p.nks - 4 * kt);
                    for (int kk = 0; kk < nk; kk++) {
                        const uint32_t c = slot + kk * 4 * (1 + P::NA);
                        cp_sf(c, fbase + ((st + P::OFF_SFA + kk * ATOM) >> 4));
#pragma unroll
                        for (int a = 0; a < P::NA; a++)
                            cp_sf(c + 4 + 4 * a, fbase + ((st + P::OFF_SFB + a * SFA_BYTES + kk * ATOM) >> 4));
                    }
                    for (int kk = 0; kk < nk; kk++) {
                        const uint32_t c = slot + kk * 4 * (1 + P::NA);
                        mma_nvfp4(d, dbase + (st >> 4) + 2 * kk, dbase + ((st + P::OFF_B) >> 4) + 2 * kk, idesc, (kt > k0) | (kk > 0), c, c + 4);
                    }
                    mma_commit(&empty[s]);
                }
                mma_commit(&acc_full[t & 1]);
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue: lane = weight row, column = token
        int t = 0;
        for (int i = first; i < p.ntiles; i += step, t++) {
            if (!warp_wait_bo(&acc_full[t & 1], (t >> 1) & 1, lane, abort_flag, &g_status, p.wait)) break;
            tc_fence_after();
            const int n = i % p.nbn * BM + tid, m0 = i / p.nbn * TN, cols = min(TN, p.M - m0);
            const uint32_t d = tmem + (t & 1) * P::ACC1 + ((uint32_t)(warp * 32) << 16);
            if (split > 1) {
                float *dump = reinterpret_cast<float *>(sm);   // every stage has been read
                for (int c0 = 0; c0 < cols; c0 += 32) {
                    float v[32];
                    tmem_ld32(d + c0, v);
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (c0 + j < cols) dump[(c0 + j) * BM + tid] = v[j];
                }
                break;
            }
            const float sw = n < p.N ? p.sw[(int64_t)n * p.sw_step] : 0.f;
            // TN = 256: the 96 shared columns first (accumulator 0: its last, accumulator 1: its first)
            for (int u = 0; u < TN; u += 32) {
                const int c0 = TN == 256 && !(t & 1) ? (u < 96 ? 160 + u : u - 96) : u;
                float v[32];
                if (c0 < cols) tmem_ld32(d + c0, v);
                if (u == (TN == 256 ? 64 : (TN - 1) / 32 * 32)) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_free[t & 1]);
                }
                if (n < p.N)
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (c0 + j < cols)
                            store<T>(p, (int64_t)(m0 + c0 + j) * p.N + n, scaled(v[j], p.sx[(int64_t)(m0 + c0 + j) * p.sx_step], sw));
            }
        }
    }
    if (split > 1) {
        // The parts' sums are added in rank order, each CTA a slice of the tile, through distributed shared memory.
        tc_fence_before();
        __syncthreads();
        cluster_sync();
        const int n0 = first % p.nbn * BM, m0 = first / p.nbn * TN, total = min(TN, p.M - m0) * BM;
        for (int e = part * THREADS + tid; e < total; e += split * THREADS) {
            float v = 0.f;
            for (int r = 0; r < split; r++) v += ld_cluster(sbase + e * 4, r);
            const int n = n0 + e % BM, m = m0 + e / BM;
            if (n < p.N) store<T>(p, (int64_t)m * p.N + n, scaled(v, p.sx[(int64_t)m * p.sx_step], p.sw[(int64_t)n * p.sw_step]));
        }
        cluster_sync();   // no CTA leaves while another reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && lane == 0) {
        // A wait ran out: what is still in flight ends before the CTA does (bounded waits). Copies: of every stage
        // its last use, since an earlier one was consumed before the stage was loaded again. MMAs: one more commit.
        if (warp == 4)
            for (uint32_t u = q > (uint32_t)S ? q - S : 0; u < q; u++) mbar_wait(&full[u % S], (u / S) & 1);
        if (warp == 5) {
            mma_commit(drain);
            mbar_wait(drain, 0);
        }
    }
    __syncwarp();
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::COLS) : "memory");
    }
}

// Codes [rows][K / 2] as a 2-D u8 tensor, boxes of 128 B x `box` rows with the 128-byte swizzle; out of range reads zero.
static bool code_map(CUtensorMap *m, const void *base, int64_t rows, int64_t bytes, int box) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)bytes};
    const cuuint32_t b[2] = {ROWB, (cuuint32_t)box}, one[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN, typename T>
static int launch(Params p, const CUtensorMap &a, const uint8_t *x, int64_t bytes, cudaStream_t st, int dev, const DeviceInfo &di) {
    using P = Plan<TN>;
    static std::atomic<uint64_t> done{0};
    auto kern = gemm_kernel<TN, T>;
    CUtensorMap b;
    if (!code_map(&b, x, p.M, bytes, TN)) return QMOE_ERR_LAUNCH;
    if (!ensure_smem(kern, P::SMEM, dev, done)) return QMOE_ERR_LAUNCH;
    p.ntiles = p.nbn * ((p.M + TN - 1) / TN);
    p.split = 1;
    if constexpr (TN <= 128) {   // too few tiles for the SMs: a cluster per tile, each CTA an even part of the stages
        int s = di.sms / p.ntiles;
        s = s < 1 ? 1 : s > MAX_SPLIT ? MAX_SPLIT : s;
        if (s > p.nst) s = p.nst;
        const int each = (p.nst + s - 1) / s;
        p.split = (p.nst + each - 1) / each;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.split > 1 ? p.ntiles * p.split : p.ntiles < di.sms ? p.ntiles : di.sms));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, p, a, b) != cudaSuccess) {
        cudaGetLastError();
        return QMOE_ERR_LAUNCH;
    }
    return launch_status();
}

template <typename T>
static int pick(const Params &p, const CUtensorMap &a, const uint8_t *x, int64_t bytes, cudaStream_t st, int dev, const DeviceInfo &di) {
    if (p.M <= 16) return launch<16, T>(p, a, x, bytes, st, dev, di);
    if (p.M <= 32) return launch<32, T>(p, a, x, bytes, st, dev, di);
    if (p.M <= 64) return launch<64, T>(p, a, x, bytes, st, dev, di);
    if (p.M <= 128 || (int64_t)p.nbn * ((p.M + 127) / 128) <= di.sms) return launch<128, T>(p, a, x, bytes, st, dev, di);
    return launch<256, T>(p, a, x, bytes, st, dev, di);
}

} // namespace g4
} // namespace qmoe

using namespace qmoe;

extern "C" {

int dq_gemm_nvfp4(const uint8_t *w, const uint8_t *w_atoms, const float *sw, int sw_per_row, const uint8_t *x,
                  const uint8_t *x_atoms, const float *sx, int sx_per_row, int M, int N, int K, int epilogue,
                  const void *residual, void *y, int y_dtype, void *stream) {
    if (!w || !w_atoms || !sw || !x || !x_atoms || !sx || !y || (epilogue == 2 && !residual)) return QMOE_ERR_NULL;
    if (epilogue < 0 || epilogue > 2 || M < 1 || N < 1 || K < 32 || (K % 32) || K > (1 << 24)) return QMOE_ERR_SHAPE;
    if (M > (1 << 24) || N > (1 << 24)) return QMOE_ERR_SHAPE;
    if (!valid_dtype(y_dtype)) return QMOE_ERR_DTYPE;
    const int size = y_dtype == QMOE_DT_F32 ? 4 : 2;
    if (!aligned16(w) || !aligned16(x) || !aligned16(w_atoms) || !aligned16(x_atoms) || !aligned4(sw) || !aligned4(sx) ||
        reinterpret_cast<uintptr_t>(y) % size || (residual && reinterpret_cast<uintptr_t>(residual) % size))
        return QMOE_ERR_ALIGN;
    int dev;
    DeviceInfo *di;
    if (int e = current_device(&dev, &di)) return e;
    g4::Params p{};
    p.sfa = w_atoms;
    p.sfb = x_atoms;
    p.sw = sw;
    p.sx = sx;
    p.sw_step = sw_per_row != 0;
    p.sx_step = sx_per_row != 0;
    p.M = M;
    p.N = N;
    p.nks = (K + 63) / 64;
    p.nst = (K + g4::BK - 1) / g4::BK;
    p.nbn = (N + g4::BM - 1) / g4::BM;
    p.epilogue = epilogue;
    p.dtype = y_dtype;
    p.res = residual;
    p.y = y;
    p.wait = wait_cycles(dev);
    CUtensorMap a;
    if (!g4::code_map(&a, w, N, K / 2, g4::BM)) return QMOE_ERR_LAUNCH;
    cudaStream_t st = as_stream(stream);
    if (y_dtype == QMOE_DT_BF16) return g4::pick<__nv_bfloat16>(p, a, x, K / 2, st, dev, *di);
    if (y_dtype == QMOE_DT_F16) return g4::pick<__half>(p, a, x, K / 2, st, dev, *di);
    return g4::pick<float>(p, a, x, K / 2, st, dev, *di);
}

int dq_gemm_nvfp4_status(int clear, void *stream) {
    if (int e = current_device(nullptr, nullptr)) return e;
    int v = 0;
    const int zero = 0;
    cudaStream_t st = as_stream(stream);
    if (cudaMemcpyFromSymbolAsync(&v, g4::g_status, sizeof(int), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess) return QMOE_ERR_LAUNCH;
    if (cudaStreamSynchronize(st) != cudaSuccess) return QMOE_ERR_LAUNCH;
    if (clear && v != 0) {
        if (cudaMemcpyToSymbolAsync(g4::g_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st) != cudaSuccess) return QMOE_ERR_LAUNCH;
        if (cudaStreamSynchronize(st) != cudaSuccess) return QMOE_ERR_LAUNCH;
    }
    return v;
}

} // extern "C"
