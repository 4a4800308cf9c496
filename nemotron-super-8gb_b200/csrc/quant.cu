// NVFP4 quantisation (dq_quantize_nvfp4), its inverse, and the tensor-core layout of block scales; the definition, and
// how its decisions are exact, in quant.cuh.
//
// Bounds: bytes, 2.56 an element for bf16 (131072 x 4096: 220 us, 6.25 TB/s), and next to them issue, 12 instructions an
// element (ncu). With IEEE divisions and a comparison per midpoint 16384 x 4096 bf16 took 61 us, now 33 (26 at the copy
// rate); the inverse takes 26 to 31 us for the same elements.
#include "common.cuh"
#include "host.h"
#include "quant.cuh"

namespace qmoe {
namespace qz {

constexpr int THREADS = 256;
constexpr int KEEP = 4;   // 16-element blocks a thread keeps in registers between the row maximum and the codes

struct Args {
    const void *x;
    int64_t ldx;   // row stride of x, in elements
    int64_t M;
    int nb;        // blocks per row, K / 16
    int vec;       // row_vec
    int words;     // whole k-steps per row: four scales are one aligned word
    uint8_t *w, *sc, *atoms;
    float *s;      // per row: written; per tensor: read
};

// Byte offset of the four scales of row r, k-step ks in a tensor-core scale layout: atoms of 512 bytes, 128 rows x 4
// scales, [row / 128][k-step], inside an atom row r at (r % 32) * 16 + (r % 128 / 32) * 4.
__device__ __forceinline__ int64_t atom_at(int64_t r, int ks, int nks) {
    return ((r >> 7) * nks + ks) * 512 + (r & 31) * 16 + ((r & 127) >> 5) * 4;
}

// Stores a block's codes and scale, and the k-step's four scales as one word of the atoms (b runs over whole k-steps;
// blocks at or past nb are padding with scale zero).
__device__ __forceinline__ void put(const Args &a, int64_t row, int b, bool live, uint2 codes, uint32_t sb) {
    if (live) *reinterpret_cast<uint2 *>(a.w + (row * a.nb + b) * 8) = codes;
    uint32_t v = live ? sb : 0u;
    v |= __shfl_down_sync(0xffffffffu, v, 1) << 8;
    v |= __shfl_down_sync(0xffffffffu, v, 2) << 16;
    const int nks = (a.nb + 3) >> 2;
    const bool first = !(b & 3) && (b >> 2) < nks;
    if (a.words) {
        if (first) *reinterpret_cast<uint32_t *>(a.sc + row * a.nb + b) = v;
    } else if (live) {
        a.sc[row * a.nb + b] = (uint8_t)sb;
    }
    if (a.atoms && first) *reinterpret_cast<uint32_t *>(a.atoms + atom_at(row, b >> 2, nks)) = v;
}

// One row per G threads, 256 / G rows a CTA: few enough threads that each has several blocks' loads in flight, more for
// few rows. Blocks past the KEEP a thread keeps are read again (from L2).
template <typename T, int G>
__global__ void __launch_bounds__(THREADS) rows_kernel(const Args a) {
    __shared__ uint32_t red[THREADS / 32];
    pdl_launch_dependents();   // a product that follows may set itself up meanwhile
    const int t = threadIdx.x % G;
    const int64_t row = blockIdx.x * (int64_t)(THREADS / G) + threadIdx.x / G;
    const bool in = row < a.M;   // a warp is all in or all out
    const T *x = static_cast<const T *>(a.x) + (in ? row : 0) * a.ldx;
    Raw<T> keep[KEEP];
    uint32_t top[KEEP];
    uint32_t m = 0;
    if (in) {
#pragma unroll
        for (int i = 0; i < KEEP; i++)
            if (t + i * G < a.nb) load16(x + (t + i * G) * 16, a.vec, keep[i]);
#pragma unroll
        for (int i = 0; i < KEEP; i++) {
            top[i] = t + i * G < a.nb ? block_max(keep[i]) : 0u;
            m = max(m, top[i] & ~NONFINITE);
        }
        for (int b = t + KEEP * G; b < a.nb; b += G) {
            Raw<T> v;
            load16(x + (int64_t)b * 16, a.vec, v);
            m = max(m, block_max(v) & ~NONFINITE);
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if constexpr (G > 32) {
        if (!(threadIdx.x & 31)) red[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < G / 32; i++) m = max(m, red[threadIdx.x / G * (G / 32) + i]);
    }
    if (!in) return;
    const int e = scale_exp(m);
    if (t == 0) a.s[row] = pow2f(e);
    const int lim = (a.nb + 31) & ~31;   // whole warps, for the shuffles of put()
#pragma unroll
    for (int i = 0; i < KEEP; i++) {
        const int b = t + i * G;
        if (b < lim) {
            uint2 c = make_uint2(0u, 0u);
            uint32_t sb = 0;
            if (b < a.nb) sb = block16<T>(keep[i], top[i], e, c);
            put(a, row, b, b < a.nb, c, sb);
        }
    }
    for (int b = t + KEEP * G; b < lim; b += G) {
        uint2 c = make_uint2(0u, 0u);
        uint32_t sb = 0;
        if (b < a.nb) {
            Raw<T> v;
            load16(x + (int64_t)b * 16, a.vec, v);
            sb = block16<T>(v, block_max(v), e, c);
        }
        put(a, row, b, b < a.nb, c, sb);
    }
}

// Tensor scale, first pass: s is monotone in the largest magnitude, so the largest of the CTAs' own s is the tensor's
// (an integer maximum of float bits: the order of the atomics does not matter). *s starts at zero.
template <typename T>
__global__ void __launch_bounds__(THREADS) tensor_scale_kernel(const Args a) {
    __shared__ uint32_t red[THREADS / 32];
    uint32_t m = 0;
    for (int64_t row = blockIdx.y; row < a.M; row += gridDim.y) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        for (int b = blockIdx.x * THREADS + threadIdx.x; b < a.nb; b += gridDim.x * THREADS) {
            Raw<T> v;
            load16(x + (int64_t)b * 16, a.vec, v);
            m = max(m, block_max(v) & ~NONFINITE);
        }
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (!(threadIdx.x & 31)) red[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < THREADS / 32; i++) m = max(m, red[i]);
        atomicMax(reinterpret_cast<uint32_t *>(a.s), __float_as_uint(pow2f(scale_exp(m))));
    }
}

// Tensor scale, second pass.
template <typename T>
__global__ void __launch_bounds__(THREADS) tensor_kernel(const Args a) {
    const int e = (int)(__float_as_uint(*a.s) >> 23) - 127;
    const int lim = (a.nb + 31) & ~31;
    for (int64_t i = blockIdx.y; i < a.M; i += gridDim.y) {
        const int64_t row = a.M - 1 - i;   // the first pass ended with the last rows: L2 still holds those
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        for (int b = blockIdx.x * THREADS + threadIdx.x; b < lim; b += gridDim.x * THREADS) {
            uint2 c = make_uint2(0u, 0u);
            uint32_t sb = 0;
            if (b < a.nb) {
                Raw<T> v;
                load16(x + (int64_t)b * 16, a.vec, v);
                sb = block16<T>(v, block_max(v), e, c);
            }
            put(a, row, b, b < a.nb, c, sb);
        }
    }
}

template <typename T>
static int launch(const Args &a, bool per_row, cudaStream_t st, const DeviceInfo &di) {
    if (per_row) {
        // the fewest threads whose registers hold a row, or more while the rows leave room on the SMs (bf16 x 4096, caches
        // cold, 32, 64, 128 and 256 threads: 8192 rows 26.0, 20.3, 22.5, 28.8 us; 512 rows 8.5, 4.3, 3.8, 3.6)
        int g = 32;
        while (g < THREADS && (a.nb > g * KEEP || (a.nb > g && a.M * g * 2 <= (int64_t)di.sms * 1024))) g *= 2;
        const unsigned grid = (unsigned)((a.M + THREADS / g - 1) / (THREADS / g));
        if (g == 32) rows_kernel<T, 32><<<grid, THREADS, 0, st>>>(a);
        else if (g == 64) rows_kernel<T, 64><<<grid, THREADS, 0, st>>>(a);
        else if (g == 128) rows_kernel<T, 128><<<grid, THREADS, 0, st>>>(a);
        else rows_kernel<T, 256><<<grid, THREADS, 0, st>>>(a);
        return launch_status();
    }
    if (cudaMemsetAsync(a.s, 0, sizeof(float), st) != cudaSuccess) return QMOE_ERR_LAUNCH;
    const unsigned gx = (unsigned)((a.nb + THREADS - 1) / THREADS);
    const dim3 grid(gx, (unsigned)(a.M < 32768 ? a.M : 32768));
    const unsigned scan = di.sms * 8 / gx > 0 ? di.sms * 8 / gx : 1;
    tensor_scale_kernel<T><<<dim3(gx, a.M < scan ? (unsigned)a.M : scan), THREADS, 0, st>>>(a);
    tensor_kernel<T><<<grid, THREADS, 0, st>>>(a);
    return launch_status();
}

// sc [N, nb] -> atoms; one thread per row and k-step (padding bytes of a last half k-step are zero).
__global__ void __launch_bounds__(256) scale_atoms_kernel(const uint8_t *__restrict__ sc, int64_t N, int nb, uint8_t *__restrict__ atoms) {
    const int nks = (nb + 3) >> 2;
    const int64_t total = N * nks;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t r = i / nks;
        const int ks = (int)(i - r * nks);
        uint32_t v = 0;
        for (int j = 0; j < 4; j++)
            if (4 * ks + j < nb) v |= (uint32_t)sc[r * nb + 4 * ks + j] << (8 * j);
        *reinterpret_cast<uint32_t *>(atoms + atom_at(r, ks, nks)) = v;
    }
}

// dense_q.py:179-188 for NVFP4: e2m1 * (e4m3 * s) in fp32, rounded to OUT. One thread per 16-element block.
template <typename OUT> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(a)) | ((uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(b)) << 16);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    return (uint32_t)__half_as_ushort(__float2half_rn(a)) | ((uint32_t)__half_as_ushort(__float2half_rn(b)) << 16);
}

template <typename OUT>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t *__restrict__ w, const uint8_t *__restrict__ sc,
                                                      const float *__restrict__ s, int per_row, int nb, int64_t r0,
                                                      int64_t total, int vec, OUT *__restrict__ out) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t row = r0 + i / nb, at = r0 * nb + i;   // block index in the weight
        const uint2 c = *reinterpret_cast<const uint2 *>(w + at * 8);
        const float f = __fmul_rn(e4m3_f32(sc[at]), s[per_row ? row : 0]);
        float v[16];
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            e2m1x8_f16x2(k ? c.y : c.x, o);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 q = __half22float2(as_h2(o[j]));
                v[8 * k + 2 * j] = __fmul_rn(q.x, f), v[8 * k + 2 * j + 1] = __fmul_rn(q.y, f);
            }
        }
        OUT *dst = out + i * 16;
        if constexpr (sizeof(OUT) == 4) {
            if (vec) {
#pragma unroll
                for (int j = 0; j < 4; j++) reinterpret_cast<float4 *>(dst)[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            } else {
                for (int j = 0; j < 16; j++) dst[j] = v[j];
            }
        } else {
            uint32_t p[8];
#pragma unroll
            for (int j = 0; j < 8; j++) p[j] = pack2<OUT>(v[2 * j], v[2 * j + 1]);
            if (vec) {
                reinterpret_cast<uint4 *>(dst)[0] = make_uint4(p[0], p[1], p[2], p[3]);
                reinterpret_cast<uint4 *>(dst)[1] = make_uint4(p[4], p[5], p[6], p[7]);
            } else {
                uint16_t *h = reinterpret_cast<uint16_t *>(dst);
                for (int j = 0; j < 8; j++) h[2 * j] = (uint16_t)p[j], h[2 * j + 1] = (uint16_t)(p[j] >> 16);
            }
        }
    }
}

} // namespace qz
} // namespace qmoe

using namespace qmoe;

extern "C" {

int dq_quantize_nvfp4(const void *x, int x_dtype, int64_t ldx, int64_t M, int64_t K, int per_row, uint8_t *w, uint8_t *sc,
                      float *s, uint8_t *atoms, void *stream) {
    if (!x || !w || !sc || !s) return QMOE_ERR_NULL;
    if (M < 1 || M > 0x7FFFFFFF || K < 16 || (K % 16) || K > (1 << 24) || ldx < K) return QMOE_ERR_SHAPE;
    if (!valid_dtype(x_dtype)) return QMOE_ERR_DTYPE;
    const int size = x_dtype == QMOE_DT_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(x) % size) || (reinterpret_cast<uintptr_t>(w) & 7u) || !aligned4(s) || !aligned4(atoms))
        return QMOE_ERR_ALIGN;
    DeviceInfo *di;
    if (int e = current_device(nullptr, &di)) return e;
    qz::Args a{};
    a.x = x;
    a.ldx = ldx;
    a.M = M;
    a.nb = (int)(K / 16);
    a.vec = qz::row_vec(x, ldx * size);
    a.words = a.nb % 4 == 0 && aligned4(sc);
    a.w = w;
    a.sc = sc;
    a.s = s;
    a.atoms = atoms;
    cudaStream_t st = as_stream(stream);
    if (x_dtype == QMOE_DT_BF16) return qz::launch<__nv_bfloat16>(a, per_row != 0, st, *di);
    if (x_dtype == QMOE_DT_F16) return qz::launch<__half>(a, per_row != 0, st, *di);
    return qz::launch<float>(a, per_row != 0, st, *di);
}

int dq_scale_atoms(const uint8_t *sc, int64_t N, int64_t K, uint8_t *atoms, void *stream) {
    if (!sc || !atoms) return QMOE_ERR_NULL;
    if (N < 1 || N > 0x7FFFFFFF || K < 16 || (K % 16) || K > (1 << 24)) return QMOE_ERR_SHAPE;
    if (!aligned4(atoms)) return QMOE_ERR_ALIGN;
    if (int e = current_device(nullptr, nullptr)) return e;
    const int nb = (int)(K / 16);
    int64_t blocks = (N * ((nb + 3) / 4) + 255) / 256;
    if (blocks > 148 * 16) blocks = 148 * 16;
    qz::scale_atoms_kernel<<<(unsigned)blocks, 256, 0, as_stream(stream)>>>(sc, N, nb, atoms);
    return launch_status();
}

int dq_dequant_nvfp4(const uint8_t *w, const uint8_t *sc, const float *s, int s_per_row, int64_t N, int64_t K, int64_t r0,
                     int64_t r1, void *out, int out_dtype, void *stream) {
    if (!w || !sc || !s || !out) return QMOE_ERR_NULL;
    if (K < 16 || (K % 16) || K > (1 << 24) || r0 < 0 || r1 < r0 || r1 > N) return QMOE_ERR_SHAPE;
    if (!valid_dtype(out_dtype)) return QMOE_ERR_DTYPE;
    if ((reinterpret_cast<uintptr_t>(w) & 7u) || !aligned4(s) || reinterpret_cast<uintptr_t>(out) % (out_dtype == QMOE_DT_F32 ? 4 : 2)) return QMOE_ERR_ALIGN;
    if (int e = current_device(nullptr, nullptr)) return e;
    if (r1 == r0) return QMOE_OK;
    const int nb = (int)(K / 16), vec = aligned16(out);
    const int64_t total = (r1 - r0) * nb;
    int64_t blocks = (total + 255) / 256;
    if (blocks > 148 * 64) blocks = 148 * 64;
    cudaStream_t st = as_stream(stream);
    if (out_dtype == QMOE_DT_BF16)
        qz::dequant_kernel<<<(unsigned)blocks, 256, 0, st>>>(w, sc, s, s_per_row, nb, r0, total, vec, static_cast<__nv_bfloat16 *>(out));
    else if (out_dtype == QMOE_DT_F16)
        qz::dequant_kernel<<<(unsigned)blocks, 256, 0, st>>>(w, sc, s, s_per_row, nb, r0, total, vec, static_cast<__half *>(out));
    else
        qz::dequant_kernel<<<(unsigned)blocks, 256, 0, st>>>(w, sc, s, s_per_row, nb, r0, total, vec, static_cast<float *>(out));
    return launch_status();
}

} // extern "C"
