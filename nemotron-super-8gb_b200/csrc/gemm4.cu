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
#include "epilogue4.cuh"
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

constexpr int MOST = 64;             // most tokens of a tile of gemm_kernel

template <int TN> struct Plan {   // TN <= 128: a stage holds one atom of token scales per k-step
    static constexpr int B_BYTES = TN * ROWB;
    static constexpr int OFF_B = A_BYTES, OFF_SFA = OFF_B + B_BYTES, OFF_SFB = OFF_SFA + SFA_BYTES;
    static constexpr int STAGE = (OFF_SFB + SFA_BYTES + 1023) / 1024 * 1024;
    static constexpr int STAGES = 221184 / STAGE < 8 ? 221184 / STAGE : 8;
    static constexpr int OFF_BAR = STAGES * STAGE;
    static constexpr int NBAR = 2 * STAGES + 5;
    static constexpr int OFF_MISC = OFF_BAR + (NBAR * 8 + 15) / 16 * 16;
    static constexpr int OFF_COL = OFF_MISC + 16;      // [4][MOST] each epilogue warp's copy of the token scales
    static constexpr int SMEM = OFF_COL + 4 * MOST * 4 + 1024;
    static_assert(SMEM <= 232448, "fits the 227 KB opt-in");
    // Tensor memory: two accumulators of TN columns and two scale slots.
    static constexpr int SF_COL = 2 * TN;
    static constexpr int SF_SLOT = 4 * 4 * 2;
    static constexpr int NEED = SF_COL + 2 * SF_SLOT;
    static constexpr int COLS = NEED <= 128 ? 128 : NEED <= 256 ? 256 : 512;
};

struct Params {
    const uint8_t *sfa, *sfb;   // scale atoms of the weights and of the tokens
    const float *sw, *sx;
    int sw_step, sx_step;       // 0: one scale, 1: one per row
    int M, N, nks, nst;         // tokens, weight rows, 64-wide k-steps, 256-wide stages
    int nbn, ntiles, split;
    int epilogue;
    const void *res;
    void *y;
    long long wait;
};

// The load and MMA warps run their loops with all lanes, so that addresses and descriptors stay in uniform registers;
// only the instruction itself is one lane's. (From a loop that one lane runs alone, every such instruction cost 100 to
// 150 cycles to issue: 8192 x 12288 x 4096 took 413 us.)
__device__ __forceinline__ bool elect_one() {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(v));
    return v != 0;
}

// Bounded wait of a whole warp. The result comes from a vote, so that the compiler sees that it is the same in every lane.
__device__ __forceinline__ bool all_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, long long limit) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = lane_wait(bar, parity, abort_flag, &g_status, limit);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) mbar_try_wait(bar, parity);   // a completed phase: the acquire of the other lanes
    return ok;
}

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

__device__ __forceinline__ float4 ld_cluster(uint32_t addr, int rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// 32 tokens' columns of one weight row (a lane): element j at y[at + j * N], for the first `left` of them, their scales in
// cs[0 .. 31]. The residuals and the scales are loaded before the first store: for all the compiler knows y is the same
// memory, and between stores each load waits by itself (2048 x 4097 x 2688: 26 us instead of 15; with a residual 100
// instead of 45). FULL: no column is missing; 32 tests between the stores cost as much again.
template <typename T, int EPI, bool FULL>
__device__ __forceinline__ void store_tokens(T *y, const T *res, int64_t N, int left, const float (&v)[32], float sw, const float *cs) {
    T r[32];
    float s[32];
    if (EPI == 2) {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (FULL || j < left) r[j] = res[j * N];
    }
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(cs + j);
        s[j] = f.x, s[j + 1] = f.y, s[j + 2] = f.z, s[j + 3] = f.w;
    }
#pragma unroll
    for (int j = 0; j < 32; j++)
        if (FULL || j < left) y[j * N] = narrow<T>(finish<T, EPI>(v[j], s[j], sw, EPI == 2 ? wide(r[j]) : 0.f));
}

template <typename T, int EPI>
__device__ __forceinline__ void store_tokens(void *y, const void *res, int64_t at, int64_t N, bool in, int left, const float (&v)[32], float sw, const float *cs) {
    if (!in) return;
    T *dst = static_cast<T *>(y) + at;
    const T *src = static_cast<const T *>(res) + at;
    if (left >= 32) store_tokens<T, EPI, true>(dst, src, N, left, v, sw, cs);
    else store_tokens<T, EPI, false>(dst, src, N, left, v, sw, cs);
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
    uint64_t *acc_free = acc_full + 2;   // [2] the accumulator is drained
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
    pdl_wait();   // what comes before may write an operand: nothing of it is read earlier
    uint32_t q = 0;   // stages loaded (warp 4) or consumed (warp 5)

    if (warp == 4) {
        // ------------------------------------------------------------ loads
        {
            bool ok = true;
            for (int i = first; i < p.ntiles && ok; i += step) {
                const int n0 = i % p.nbn * BM, m0 = i / p.nbn * TN;
                const uint8_t *fa = p.sfa + (int64_t)(n0 >> 7) * p.nks * ATOM, *fb = p.sfb + (int64_t)(m0 >> 7) * p.nks * ATOM;
                for (int kt = k0; kt < k1; kt++, q++) {
                    const int s = q % S;
                    if (!all_wait(&empty[s], ((q / S) & 1) ^ 1, abort_flag, p.wait)) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = sm + s * P::STAGE;
                    const uint32_t sf = (uint32_t)min(4, p.nks - 4 * kt) * ATOM;
                    if (elect_one()) {
                        mbar_expect_tx(&full[s], A_BYTES + P::B_BYTES + 2 * sf);
                        tma_load_2d(st, &tm_a, kt * ROWB, n0, &full[s]);
                        tma_load_2d(st + P::OFF_B, &tm_b, kt * ROWB, m0, &full[s]);
                        bulk_g2s_nohint(st + P::OFF_SFA, fa + (int64_t)kt * SFA_BYTES, sf, &full[s]);
                        bulk_g2s_nohint(st + P::OFF_SFB, fb + (int64_t)kt * SFA_BYTES, sf, &full[s]);
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        // ------------------------------------------------------------ scales to tensor memory, MMAs
        {
            const uint64_t dbase = smem_desc(0, 16, 1024, 2);   // K-major, 128-byte swizzle
            const uint64_t fbase = smem_desc(0, 16, 128, 0);    // an atom: 32 rows of 16 bytes
            int t = 0;
            bool ok = true;
            for (int i = first; i < p.ntiles && ok; i += step, t++) {
                const int m0 = i / p.nbn * TN;
                const uint32_t idesc = instr_desc_nvfp4((min(TN, p.M - m0) + 15) & ~15);
                const int f = t - 2;   // the tile that had this accumulator before
                if (f >= 0 && !all_wait(&acc_free[f & 1], (f >> 1) & 1, abort_flag, p.wait)) break;
                tc_fence_after();
                const uint32_t d = tmem + (t & 1) * TN;
                for (int kt = k0; kt < k1; kt++, q++) {
                    const int s = q % S;
                    if (!all_wait(&full[s], (q / S) & 1, abort_flag, p.wait)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t st = sbase + s * P::STAGE;
                    const uint32_t slot = tmem + P::SF_COL + (q & 1) * P::SF_SLOT;
                    const int nk = min(4, p.nks - 4 * kt);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            if (kk >= nk) break;
                            cp_sf(slot + 8 * kk, fbase + ((st + P::OFF_SFA + kk * ATOM) >> 4));
                            cp_sf(slot + 8 * kk + 4, fbase + ((st + P::OFF_SFB + kk * ATOM) >> 4));
                        }
#pragma unroll
                        for (int kk = 0; kk < 4; kk++) {
                            if (kk >= nk) break;
                            const uint32_t c = slot + 8 * kk;
                            mma_nvfp4(d, dbase + (st >> 4) + 2 * kk, dbase + ((st + P::OFF_B) >> 4) + 2 * kk, idesc, (kt > k0) | (kk > 0), c, c + 4);
                        }
                        mma_commit(&empty[s]);
                        if (kt == k1 - 1) mma_commit(&acc_full[t & 1]);
                    }
                    __syncwarp();
                }
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
            const uint32_t d = tmem + (t & 1) * TN + ((uint32_t)(warp * 32) << 16);
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
            float *cs = reinterpret_cast<float *>(sm + P::OFF_COL) + warp * MOST;   // a copy per warp: no barrier between warps
            __syncwarp();
            for (int c = lane; c < cols; c += 32) cs[c] = p.sx[(int64_t)(m0 + c) * p.sx_step];
            __syncwarp();
#pragma unroll 1
            for (int c0 = 0; c0 < TN; c0 += 32) {
                float v[32];
                const int left = cols - c0;
                if (left > 0) tmem_ld32(d + c0, v);
                if (c0 + 32 >= TN) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_free[t & 1]);
                }
                if (left <= 0) continue;
                const int64_t at = (int64_t)(m0 + c0) * p.N + n;
                if (p.epilogue == 0) store_tokens<T, 0>(p.y, p.res, at, p.N, n < p.N, left, v, sw, cs + c0);
                else if (p.epilogue == 1) store_tokens<T, 1>(p.y, p.res, at, p.N, n < p.N, left, v, sw, cs + c0);
                else store_tokens<T, 2>(p.y, p.res, at, p.N, n < p.N, left, v, sw, cs + c0);
            }
        }
    }
    if (split > 1) {
        // The parts' sums are added in rank order, each CTA a slice of the tile, through distributed shared memory.
        tc_fence_before();
        __syncthreads();
        cluster_sync();
        const int n0 = first % p.nbn * BM, m0 = first / p.nbn * TN, total = min(TN, p.M - m0) * BM;
        for (int e = (part * THREADS + tid) * 4; e < total; e += split * THREADS * 4) {   // four weight rows of a token
            float4 v[MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; r++)
                if (r < split) v[r] = ld_cluster(sbase + e * 4, r);   // all in flight together
            float4 o = v[0];
#pragma unroll
            for (int r = 1; r < MAX_SPLIT; r++)
                if (r < split) o.x += v[r].x, o.y += v[r].y, o.z += v[r].z, o.w += v[r].w;
            const int n = n0 + e % BM, m = m0 + e / BM;
            const float sx = p.sx[(int64_t)m * p.sx_step];
            const int64_t at = (int64_t)m * p.N + n;
            const float u[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (n + j >= p.N) break;
                const float sw = p.sw[(int64_t)(n + j) * p.sw_step];
                if (p.epilogue == 0) store_one<T, 0>(p.y, p.res, at + j, u[j], sx, sw);
                else if (p.epilogue == 1) store_one<T, 1>(p.y, p.res, at + j, u[j], sx, sw);
                else store_one<T, 2>(p.y, p.res, at + j, u[j], sx, sw);
            }
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
    }
    if (warp == 5 && *abort_flag) {   // the lane that issued the MMAs: elect picks the same one every time
        if (elect_one()) {
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

// ------------------------------------------------------------------------------------------ pairs of CTAs
// The same product for many tokens: a cluster of two CTAs computes 256 x TN with cta_group::2 MMAs. Each CTA holds 128
// rows of the one operand and half of the other's TN, so that a stage costs each SM 70 KB of shared-memory traffic
// for 512 cycles of tensor work at TN = 256; one CTA alone on 128 x 256 needs 102 KB, which is what bounded it.
// Which operand has the 256 rows (the lanes of tensor memory) is the caller's choice: with the tokens there, a thread
// holds consecutive columns of one row of y and stores 32 bytes at a time; with the weights there, a warp's lanes are
// consecutive in a row of y, which suits rows of y that are not 32-byte aligned.
// One warp issues everything for both tensor cores, a stage in one elected block: the scale copies of k-step k + 1, then
// the MMA of k-step k, so that a copy runs while the MMA before it does. The pipe runs them in the order issued, which
// makes two k-steps' worth of scale columns enough. (Two stages' worth, with a warp of its own for the copies, needed two
// more hand-offs per stage.) What bounds it is the tensor pipe at the clock the power limit leaves: 8192 x 12288 x
// 4096 runs at 5.3 PFLOP/s, 0.78 of four times the bf16 rate of the library's product, and a version without any loads
// took 0.96 of the time of the same version with them.
// TN = 320 is for products of at most one tile per pair: one accumulator, two MMAs (192 and 128 columns) per k-step.
template <int TN> struct PairPlan {
    static constexpr int NA = (TN + 127) / 128;
    static constexpr int N0 = TN > 256 ? 192 : TN, N1 = TN - N0;   // columns of an MMA, of a second one
    static constexpr int BOX = N1 ? 32 : TN / 2;                   // token or weight rows of a copy
    static constexpr int B_BYTES = TN / 2 * ROWB;
    static constexpr int OFF_B = A_BYTES, OFF_SFA = OFF_B + B_BYTES, OFF_SFB = OFF_SFA + SFA_BYTES;
    static constexpr int BYTES = OFF_SFB + NA * SFA_BYTES;
    static constexpr int STAGE = (BYTES + 1023) / 1024 * 1024;
    static constexpr int STAGES = 221184 / STAGE < 8 ? 221184 / STAGE : 8;
    static constexpr int OFF_BAR = STAGES * STAGE;
    static constexpr int NBAR = 2 * STAGES + 5;
    static constexpr int OFF_MISC = OFF_BAR + (NBAR * 8 + 15) / 16 * 16;
    static constexpr int OFF_COL = OFF_MISC + 16;   // [4][TN] each epilogue warp's copy of the columns' scales of its tile
    static constexpr int SMEM = OFF_COL + 4 * TN * 4 + 1024;
    static_assert(SMEM <= 232448, "fits the 227 KB opt-in");
    // Tensor memory: two accumulators and two k-steps of scales. At TN = 256 the accumulators share 32 columns, which the
    // epilogue reads first, so that the next tile's MMAs wait for those alone; else for the tile before the last.
    static constexpr int ACC1 = N1 ? 0 : TN == 256 ? 224 : TN;
    static constexpr int SF_COL = ACC1 + TN;
    static constexpr int SF_SLOT = 4 * (1 + NA);
    static constexpr int LAG = TN == 256 ? 1 : 2;
    static_assert(SF_COL + 2 * SF_SLOT <= 512, "tensor memory");
};

struct PairParams {
    const float *sa, *sb;   // scales of the lanes' and of the columns' operand
    int sa_step, sb_step;
    int A, B;               // rows of the two operands
    int nks, nst, nba, ntiles;
    int tokens_on_lanes;
    int N;                  // row length of y
    const void *res;
    void *y;
    long long wait;
};

__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// Descriptors in halves: the upper is constant, the lower (address / 16 and the leading offset) takes one addition.
constexpr uint32_t LO = 1u << 16, HI_SF = (128u >> 4) | (1u << 14), HI_TILE = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void cp_sf_pair(uint32_t taddr, uint32_t lo) {
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(taddr), "r"(lo), "r"(HI_SF)
                 : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc, uint32_t sfa, uint32_t sfb) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], a, b, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb), "r"(HI_TILE)
        : "memory");
}
// Arrives on both CTAs' barrier at this offset once the MMAs issued so far have completed.
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ uint32_t in_leader(const void *p) {   // the same place in the pair's first CTA
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}

// A word of the other CTA's shared memory, at this one's place.
__device__ __forceinline__ void tell(const volatile uint32_t *p, int rank, uint32_t v) {
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\tst.shared::cluster.b32 [r], %2;\n\t}" ::"r"(
                     smem_u32(const_cast<const uint32_t *>(p))),
                 "r"(rank), "r"(v)
                 : "memory");
}
// Counts `bytes` as copied on a barrier of this CTA.
__device__ __forceinline__ void mbar_complete_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// tmem_ld32 in two halves, so that several loads are in flight; the wait takes the registers, so that none is used before.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) asm volatile("" : "+f"(v[i]));
}

// Only tensor-memory reads come before it, and those are waited for. (With .release.cluster it waits for the thread's
// global stores too: 1300 cycles.)
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<float>(float, float) { return 0; }
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u)); }
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) { return __half22float2(as_h2(v)); }
__device__ __forceinline__ float2 unpack2(uint32_t, float) { return make_float2(0.f, 0.f); }

__device__ __forceinline__ void st32(void *p, const uint32_t (&v)[8]) {   // 32 bytes, 32-byte aligned
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void ld32(const void *p, uint32_t (&v)[8]) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(p));
}

// 32 weight rows' columns of one token (a lane): y[at ..], for the first `left` of them, 32 bytes at a time (left, like the
// row length, is a multiple of those). EACH: cs holds the columns' scales, else sw is all of theirs.
template <typename T, int EPI, bool EACH>
__device__ __forceinline__ void store_run(void *y, const void *res, int64_t at, bool in, int left, const float (&v)[32], float sx, float sw, const float *cs) {
    constexpr int EPV = 32 / sizeof(T);   // elements per store
    uint32_t rs[32 / EPV][8] = {};
    if (EPI == 2) {   // all loads before the first store, as in store_tokens
#pragma unroll
        for (int u = 0; u < 32 / EPV; u++)
            if (in && u * EPV < left) ld32(static_cast<const T *>(res) + at + u * EPV, rs[u]);
    }
#pragma unroll
    for (int u = 0; u < 32 / EPV; u++) {
        const bool live = in && u * EPV < left;
        const uint32_t(&r)[8] = rs[u];
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (sizeof(T) == 4) {
                const int c = u * EPV + j;
                o[j] = __float_as_uint(finish<T, EPI>(v[c], sx, EACH ? cs[c] : sw, __uint_as_float(r[j])));
            } else {
                const int c = u * EPV + 2 * j;
                const float2 q = unpack2(r[j], T{});
                const float lo = finish<T, EPI>(v[c], sx, EACH ? cs[c] : sw, q.x);
                const float hi = finish<T, EPI>(v[c + 1], sx, EACH ? cs[c + 1] : sw, q.y);
                o[j] = pack2<T>(lo, hi);
            }
        }
        if (live) st32(static_cast<T *>(y) + at + u * EPV, o);
    }
}

template <int TN, typename T, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
    pair_kernel(const PairParams p, const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                const __grid_constant__ CUtensorMap tm_sa, const __grid_constant__ CUtensorMap tm_sb) {
    using P = PairPlan<TN>;
    constexpr int S = P::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t *sm = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const uint32_t sbase = smem_u32(sm);
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + P::OFF_BAR);   // the first CTA's count both CTAs' copies
    uint64_t *empty = full + S;
    uint64_t *acc_full = empty + S;      // [2]
    uint64_t *acc_free = acc_full + 2;   // [2], the first CTA's
    uint64_t *drain = acc_free + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + P::OFF_MISC);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sm + P::OFF_MISC + 8);
    volatile uint32_t *other_loaded = tmem_slot + 1, *other_abort = tmem_slot + 3;   // written by the other CTA
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x & 1, first = blockIdx.x >> 1, step = gridDim.x >> 1;

    if (tid == 0) {
        for (int s = 0; s < S; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&acc_full[0], 1);
        mbar_init(&acc_full[1], 1);
        mbar_init(&acc_free[0], 8);
        mbar_init(&acc_free[1], 8);
        mbar_init(drain, 1);
        *abort_flag = 0;
        *other_loaded = *other_abort = 0;
        fence_mbar_init();
    }
    if (warp == 5) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();   // both CTAs' barriers exist before either is signalled
    tc_fence_after();   // all 512 columns are this CTA's, so they start at column 0
    pdl_wait();         // what comes before may write an operand: nothing of it is read earlier
    uint32_t q = 0;     // stages loaded

    if (warp == 4) {
        // ------------------------------------------------------------ loads: each CTA its own half of the stage
        {
            bool ok = true;
            for (int i = first; i < p.ntiles && ok; i += step) {
                const int a0 = i % p.nba * 256 + rank * 128, b0 = i / p.nba * TN;
                const int fa = (a0 >> 7) * p.nks, fb = (b0 >> 7) * p.nks;
                for (int kt = 0; kt < p.nst; kt++, q++) {
                    const int s = q % S;
                    if (!all_wait(&empty[s], ((q / S) & 1) ^ 1, abort_flag, p.wait)) {
                        ok = false;
                        break;
                    }
                    uint8_t *st = sm + s * P::STAGE;
                    const uint32_t bar = in_leader(&full[s]);
                    if (elect_one()) {
                        if (rank == 0) mbar_expect_tx(&full[s], 2 * P::BYTES);
                        tma_load_2d_pair(st, &tm_a, kt * ROWB, a0, bar);
#pragma unroll
                        for (int r = 0; r < P::N0 / 2; r += P::BOX) tma_load_2d_pair(st + P::OFF_B + r * ROWB, &tm_b, kt * ROWB, b0 + rank * (P::N0 / 2) + r, bar);
#pragma unroll
                        for (int r = 0; r < P::N1 / 2; r += P::BOX)
                            tma_load_2d_pair(st + P::OFF_B + (P::N0 / 2 + r) * ROWB, &tm_b, kt * ROWB, b0 + P::N0 + rank * (P::N1 / 2) + r, bar);
                        tma_load_2d_pair(st + P::OFF_SFA, &tm_sa, 0, fa + 4 * kt, bar);
#pragma unroll
                        for (int a = 0; a < P::NA; a++)
                            tma_load_2d_pair(st + P::OFF_SFB + a * SFA_BYTES, &tm_sb, 0, fb + a * p.nks + 4 * kt, bar);
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
        if (lane == 0) tell(other_loaded, rank ^ 1, q);
        __syncwarp();
    } else if (warp == 5) {
        // ------------------------------------------------------------ the first CTA's warp drives both tensor cores
        if (rank == 0) {
            constexpr uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(P::N0 >> 3) << 17) | (16u << 24);    // M = 256
            constexpr uint32_t idesc1 = (1u << 7) | (1u << 10) | ((uint32_t)(P::N1 >> 3) << 17) | (16u << 24);
            const bool lead = elect_one();
            const int tail = p.nks - 4 * (p.nst - 1);   // k-steps of a tile's last stage
            uint32_t ph = 0;                            // parity of stage s's current use
            int s = 0, sp = 0, t = 0;                   // sp: the stage before
            bool ok = true;
            for (int i = first; i < p.ntiles && ok; i += step, t++) {
                const uint32_t d = (t & 1) * P::ACC1;
                const uint32_t off = (uint32_t)(i / p.nba * TN & 127) >> 5;   // TN = 192, 320: a tile may start at row 64 of an atom
                for (int kt = 0; kt < p.nst; kt++) {
                    if (!all_wait(&full[s], ph, abort_flag, p.wait)) {
                        ok = false;
                        break;
                    }
                    if (kt == 0 && t >= P::LAG) {
                        const int f = t - P::LAG;
                        if (!all_wait(&acc_free[f & 1], (f >> 1) & 1, abort_flag, p.wait)) {
                            ok = false;
                            break;
                        }
                    }
                    tc_fence_after();
                    const uint32_t f = ((sbase + s * P::STAGE + P::OFF_SFA) >> 4) + LO;
                    const uint32_t a = ((sbase + s * P::STAGE) >> 4) + LO, ap = ((sbase + sp * P::STAGE) >> 4) + LO;
                    const int nk = kt == p.nst - 1 ? tail : 4;
                    auto copies = [&](int k) {
                        const uint32_t c = P::SF_COL + (k & 1) * P::SF_SLOT;
                        cp_sf_pair(c, f + k * (ATOM >> 4));
#pragma unroll
                        for (int j = 0; j < P::NA; j++) cp_sf_pair(c + 4 + 4 * j, f + ((SFA_BYTES + j * SFA_BYTES + k * ATOM) >> 4));
                    };
                    auto mma = [&](uint32_t at, int k, uint32_t acc) {
                        const uint32_t c = P::SF_COL + (k & 1) * P::SF_SLOT;
                        mma_pair(d, at + 2 * k, at + (P::OFF_B >> 4) + 2 * k, idesc, acc, c, c + 4 + off);
                        if constexpr (P::N1 > 0)
                            mma_pair(d + P::N0, at + 2 * k, at + ((P::OFF_B + P::N0 / 2 * ROWB) >> 4) + 2 * k, idesc1, acc, c, c + 4 + off + P::N0 / 32);
                    };
                    if (lead) {
                        copies(0);
                        if (kt > 0) {   // the stage before had four
                            mma(ap, 3, 1);
                            commit_pair(&empty[sp]);
                        }
#pragma unroll
                        for (int k = 1; k < 4; k++)
                            if (k < nk) {
                                copies(k);
                                mma(a, k - 1, kt + k - 1);
                            }
                        if (kt == p.nst - 1) {
                            mma(a, nk - 1, kt + nk - 1);
                            commit_pair(&empty[s]);
                            commit_pair(&acc_full[t & 1]);
                        }
                    }
                    __syncwarp();
                    sp = s;
                    if (++s == S) s = 0, ph ^= 1;
                }
            }
        }
        __syncwarp();
    } else {
        // ------------------------------------------------------------ epilogue: each CTA its 128 lanes
        const bool each = p.sb_step != 0;
        const float sb_all = p.sb[0];
        float *cs = reinterpret_cast<float *>(sm + P::OFF_COL) + warp * TN;   // a copy per warp: no barrier between warps
        int t = 0;
        for (int i = first; i < p.ntiles; i += step, t++) {
            const int a = i % p.nba * 256 + rank * 128 + tid, b0 = i / p.nba * TN;
            const uint32_t d = (t & 1) * P::ACC1 + ((uint32_t)(warp * 32) << 16);
            const bool in = a < p.A;
            const float sa = in ? p.sa[(int64_t)a * p.sa_step] : 0.f;
            __syncwarp();
            if (each || !p.tokens_on_lanes)
#pragma unroll
                for (int c = lane; c < TN; c += 32) cs[c] = b0 + c < p.B ? p.sb[(int64_t)(b0 + c) * p.sb_step] : 0.f;
            __syncwarp();
            const uint32_t free_bar = in_leader(&acc_free[t & 1]);
            if (!all_wait(&acc_full[t & 1], (t >> 1) & 1, abort_flag, p.wait)) break;
            tc_fence_after();
            auto put = [&](int c0, const float(&v)[32]) {
                const int left = p.B - b0 - c0;   // columns from here that exist
                if (left <= 0) return;
                if (!p.tokens_on_lanes) {
                    store_tokens<T, EPI>(p.y, p.res, (int64_t)(b0 + c0) * p.N + a, p.N, in, left, v, sa, cs + c0);
                } else {
                    const int64_t at = (int64_t)a * p.N + b0 + c0;
                    if (each) store_run<T, EPI, true>(p.y, p.res, at, in, left, v, sa, 0.f, cs + c0);
                    else store_run<T, EPI, false>(p.y, p.res, at, in, left, v, sa, sb_all, cs);
                }
            };
            // the 32 columns shared with the other accumulator first (accumulator 0's last, 1's first); a run is loaded while
            // the one before it is stored
            const int start = TN == 256 && !(t & 1) ? 224 : 0;
            auto at = [&](int k) { const int c = start + 32 * k; return c >= TN ? c - TN : c; };
            float v0[32], v1[32];
            tmem_ld32_issue(d + at(0), v0);
            tmem_ld_wait(v0);
            auto release = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_remote(free_bar);
            };
            if (TN == 256) release();
#pragma unroll 1
            for (int k = 0; k < TN / 32; k += 2) {
                tmem_ld32_issue(d + at(k + 1), v1);
                put(at(k), v0);
                tmem_ld_wait(v1);
                if (k + 2 < TN / 32) tmem_ld32_issue(d + at(k + 2), v0);
                else if (TN < 256) release();
                put(at(k + 1), v1);
                if (k + 2 < TN / 32) tmem_ld_wait(v0);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort_flag) tell(other_abort, rank ^ 1, 1u);
    __syncwarp();
    cluster_sync();   // neither CTA leaves while the other may still signal it or run on its memory
    if (*abort_flag || *other_abort) {   // the same in both CTAs
        // A wait ran out: as in gemm_kernel, what is in flight ends before the pair does. The two CTAs may have given up at
        // different stages. The first one's barriers count both halves: a stage that only the other loaded is expected
        // here, the missing half of one that only this CTA loaded counts as copied.
        if (rank == 0 && warp == 4 && lane == 0) {
            const uint32_t other = *other_loaded, most = max(q, other);
            for (uint32_t u = most > (uint32_t)S ? most - S : 0; u < most; u++) {
                if (u >= q) mbar_expect_tx(&full[u % S], P::BYTES);
                else if (u >= other) mbar_complete_tx(&full[u % S], P::BYTES);
                mbar_wait(&full[u % S], (u / S) & 1);
            }
        }
        if (warp == 5) {
            if (elect_one()) {
                if (rank == 0) commit_pair(drain);   // the lane that issued: elect picks the same one
                mbar_wait(drain, 0);
            }
        }
        __syncwarp();
        cluster_sync();
    }
    if (warp == 5) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(*tmem_slot) : "memory");
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
    if (!(done.load(std::memory_order_acquire) >> (dev & 63) & 1) && !ensure_smem(kern, P::SMEM, dev, done)) return QMOE_ERR_LAUNCH;
    p.ntiles = p.nbn * ((p.M + TN - 1) / TN);
    p.split = 1;
    {   // too few tiles for the SMs: a cluster per tile, each CTA an even part of the stages
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
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, kern, p, a, b) != cudaSuccess) {
        cudaGetLastError();
        return QMOE_ERR_LAUNCH;
    }
    return launch_status();
}

// Scale atoms as a 2-D u32 tensor [atoms][128], boxes of four (a stage's).
static bool atom_map(CUtensorMap *m, const void *base, int64_t rows, int nks) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {ATOM / 4, (cuuint64_t)((rows + 127) / 128 * nks)};
    const cuuint64_t strides[1] = {ATOM};
    const cuuint32_t b[2] = {ATOM / 4, 4}, one[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void *>(base), dims, strides, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tokens on the lanes wherever y's rows allow 32-byte stores.
template <typename T> static bool tokens_on_lanes(const Params &g) {
    return (int64_t)g.N * sizeof(T) % 32 == 0 && !((reinterpret_cast<uintptr_t>(g.y) | reinterpret_cast<uintptr_t>(g.res)) & 31u);
}

template <int TN, typename T, int EPI>
static int launch_pair(const Params &g, const uint8_t *w, const uint8_t *x, int64_t bytes, cudaStream_t st, int dev, const DeviceInfo &di) {
    static std::atomic<uint64_t> done{0};
    auto kern = pair_kernel<TN, T, EPI>;
    PairParams p{};
    p.tokens_on_lanes = tokens_on_lanes<T>(g);
    const bool t = p.tokens_on_lanes;
    p.sa = t ? g.sx : g.sw;
    p.sb = t ? g.sw : g.sx;
    p.sa_step = t ? g.sx_step : g.sw_step;
    p.sb_step = t ? g.sw_step : g.sx_step;
    p.A = t ? g.M : g.N;
    p.B = t ? g.N : g.M;
    p.nks = g.nks;
    p.nst = g.nst;
    p.nba = (p.A + 255) / 256;
    p.ntiles = p.nba * ((p.B + TN - 1) / TN);
    p.N = g.N;
    p.res = g.res;
    p.y = g.y;
    p.wait = g.wait;
    CUtensorMap a, b, sa, sb;
    if (!code_map(&a, t ? x : w, p.A, bytes, 128) || !code_map(&b, t ? w : x, p.B, bytes, PairPlan<TN>::BOX) ||
        !atom_map(&sa, t ? g.sfb : g.sfa, p.A, p.nks) || !atom_map(&sb, t ? g.sfa : g.sfb, p.B, p.nks))
        return QMOE_ERR_LAUNCH;
    if (!(done.load(std::memory_order_acquire) >> (dev & 63) & 1) && !ensure_smem(kern, PairPlan<TN>::SMEM, dev, done)) return QMOE_ERR_LAUNCH;
    cudaLaunchConfig_t cfg = {};
    const int pairs = di.sms / 2;
    cfg.gridDim = dim3((unsigned)(2 * (p.ntiles < pairs ? p.ntiles : pairs)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = PairPlan<TN>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, kern, p, a, b, sa, sb) != cudaSuccess) {
        cudaGetLastError();
        return QMOE_ERR_LAUNCH;
    }
    return launch_status();
}

template <int TN, typename T>
static int launch_pair(const Params &p, const uint8_t *w, const uint8_t *x, int64_t bytes, cudaStream_t st, int dev, const DeviceInfo &di) {
    if (p.epilogue == 0) return launch_pair<TN, T, 0>(p, w, x, bytes, st, dev, di);
    if (p.epilogue == 1) return launch_pair<TN, T, 1>(p, w, x, bytes, st, dev, di);
    return launch_pair<TN, T, 2>(p, w, x, bytes, st, dev, di);
}

// Up to 64 tokens: one tile of weight rows x all tokens per CTA, the stages split over a cluster where tiles are few. More:
// pairs, with the columns that take the least time: waves of tiles times a tile's time, 1, 0.86 and 0.72 for 256, 192
// and 128 columns (8192 x 12288 x 4096 in 155, 178 and 223 us); 128 x 4096 x 4096: 12.1, 11.5, 10.9, 128 taken (a cluster
// per tile of 128 x 128: 11.7). 320 columns (1.25) where they make one wave and the others two: 2048 x 2688 x 4096 in
// 12.7 us instead of 16.0 with 192, 512 x 10000 x 4096 in 12.0 instead of 15.3.
template <typename T>
static int pick(const Params &p, const CUtensorMap &a, const uint8_t *w, const uint8_t *x, int64_t bytes, cudaStream_t st, int dev, const DeviceInfo &di) {
    if (p.M <= 16) return launch<16, T>(p, a, x, bytes, st, dev, di);
    if (p.M <= 32) return launch<32, T>(p, a, x, bytes, st, dev, di);
    if (p.M <= 64) return launch<64, T>(p, a, x, bytes, st, dev, di);
    const int64_t A = tokens_on_lanes<T>(p) ? p.M : p.N, B = tokens_on_lanes<T>(p) ? p.N : p.M, pairs = di.sms / 2;
    auto cost = [&](int tn, int each) { return ((A + 255) / 256 * ((B + tn - 1) / tn) + pairs - 1) / pairs * each; };
    const int64_t c128 = cost(128, 72), c192 = cost(192, 86), c256 = cost(256, 100), c320 = cost(320, 125);
    if (c320 == 125 && c320 < c128 && c320 < c192 && c320 < c256) return launch_pair<320, T>(p, w, x, bytes, st, dev, di);
    if (c128 <= c192 && c128 <= c256) return launch_pair<128, T>(p, w, x, bytes, st, dev, di);
    if (c192 <= c256) return launch_pair<192, T>(p, w, x, bytes, st, dev, di);
    return launch_pair<256, T>(p, w, x, bytes, st, dev, di);
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
    p.res = residual;
    p.y = y;
    p.wait = wait_cycles(dev);
    CUtensorMap a;
    if (!g4::code_map(&a, w, N, K / 2, g4::BM)) return QMOE_ERR_LAUNCH;
    cudaStream_t st = as_stream(stream);
    if (y_dtype == QMOE_DT_BF16) return g4::pick<__nv_bfloat16>(p, a, w, x, K / 2, st, dev, *di);
    if (y_dtype == QMOE_DT_F16) return g4::pick<__half>(p, a, w, x, K / 2, st, dev, *di);
    return g4::pick<float>(p, a, w, x, K / 2, st, dev, *di);
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
