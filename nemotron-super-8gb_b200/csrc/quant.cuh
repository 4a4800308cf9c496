// NVFP4 quantisation of a 16-element block, shared by the quantiser and the four-bit linear of few tokens.
//
// x [M, K] -> e2m1 codes, one e4m3 scale per 16 elements, and one fp32 scale s per row or per tensor:
//   s  = 2^e, the smallest power of two >= 2^-126 with amax <= 6 * 448 * s,
//   sc = e4m3(amax16 / (6 s)), nearest, ties to even,
//   q  = e2m1(x / (s sc)), nearest, ties to even; value = q * sc * s.
// Against s = amax / 2688 a power of two costs up to one binade at the lower end of the block scales' range, and nothing
// above it: the block scale is itself a floating-point number. x / s is exact. A block that holds an infinity or a NaN
// gets the scale NaN (0x7F) and zero codes; s ignores those elements.
//
// Every decision is the exact one, without a division. What is compared is x / s with midpoint * sc, or amax16 / s with
// 6 * midpoint: numbers of at most 7 significant bits. An fp32 x is first cut to 13 bits with the rest ORed into the last
// ("round to odd"), which keeps its order among such numbers; bf16 and f16 have fewer anyway. So a quotient that is no
// tie is at least 2^-12 of its size away from one. x * (1 / (s sc)) + 192 in one FMA rounds the quotient (below 10, its
// reciprocal off by 2^-23) to a multiple of 2^-16: a tie comes back as the tie, and nothing else reaches one, the smallest
// distance being 0.25 * 2^-12. amax16 / 6 is rounded to 18 bits to the same end.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace qmoe {
namespace qz {

// 16 consecutive elements as loaded.
template <typename T> struct Raw { uint32_t r[sizeof(T) * 4]; };

// How wide a block may be loaded: vec 2: rows are 32-byte aligned, 1: 16-byte, 0: neither. A lane's 32-byte load is whole
// sectors; in halves each sector passes L1 twice (12288 x 4096 fp32 with one scale: 86 us against 82).
template <typename T> __device__ __forceinline__ void load16(const T *p, int vec, Raw<T> &v) {
    if (vec == 2) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            uint32_t *r = v.r + 8 * i;
            asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                         : "l"(reinterpret_cast<const uint8_t *>(p) + 32 * i));
        }
    } else if (vec == 1) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T); i++) {
            const uint4 u = ldg_stream(reinterpret_cast<const uint8_t *>(p) + 16 * i);
            v.r[4 * i] = u.x, v.r[4 * i + 1] = u.y, v.r[4 * i + 2] = u.z, v.r[4 * i + 3] = u.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; i++) v.r[i] = __float_as_uint(p[i]);
    } else {
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) v.r[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
    }
}

template <typename T> __device__ __forceinline__ void widen(const Raw<T> &v, float (&f)[16]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if constexpr (sizeof(T) == 4) {
            f[2 * i] = __uint_as_float(v.r[2 * i]), f[2 * i + 1] = __uint_as_float(v.r[2 * i + 1]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 h = __half22float2(as_h2(v.r[i]));
            f[2 * i] = h.x, f[2 * i + 1] = h.y;
        } else {
            f[2 * i] = __uint_as_float(v.r[i] << 16), f[2 * i + 1] = __uint_as_float(v.r[i] & 0xFFFF0000u);
        }
    }
}

// fp32 bits of the largest finite magnitude of a block; with NONFINITE set where the block holds anything else.
constexpr uint32_t NONFINITE = 0x80000000u;
// The larger magnitudes of two pairs, NaN where either is; the signs are of no use.
template <typename T> __device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t block_max(const Raw<T> &v) {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; i++) m = max(m, v.r[i] & 0x7FFFFFFFu);
        if (m < 0x7F800000u) return m;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) m = larger2<T>(m, v.r[i]);
        m &= 0x7FFF7FFFu;
        m = max(m & 0xFFFFu, m >> 16);
        if (std::is_same<T, __half>::value && m < 0x7C00u) return __float_as_uint(__half2float(__ushort_as_half((uint16_t)m)));
        if (!std::is_same<T, __half>::value && m < 0x7F80u) return m << 16;
    }
    float f[16];
    widen(v, f);
    m = 0;
    for (int i = 0; i < 16; i++) {
        const uint32_t b = __float_as_uint(f[i]) & 0x7FFFFFFFu;
        m = max(m, b >= 0x7F800000u ? 0u : b);
    }
    return m | NONFINITE;
}

// Exponent e of s = 2^e for a largest magnitude with these bits: 2688 = 1.3125 * 2^11.
__device__ __forceinline__ int scale_exp(uint32_t bits) {
    const int e = (int)(bits >> 23) - 127 - ((bits & 0x7FFFFFu) <= 0x280000u ? 11 : 10);
    return max(e, -126);
}

// Round to odd at 13 significant bits (of a normal number's bits).
__device__ __forceinline__ uint32_t odd13(uint32_t b) { return (b | ((b & 0x7FFu) + 0x7FFu)) & ~0x7FFu; }

// a = a f + 192 - 192, each step rounded once, and b likewise: two elements per instruction.
__device__ __forceinline__ void snap2(float &a, float &b, float f) {
    asm("{\n\t.reg .b64 v, g, c, d;\n\t"
        "mov.b64 v, {%0, %1};\n\tmov.b64 g, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\tmov.b64 d, {%4, %4};\n\t"
        "fma.rn.f32x2 v, v, g, c;\n\tadd.rn.f32x2 v, v, d;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(a), "+f"(b) : "f"(f), "f"(192.f), "f"(-192.f));
}

// One block whose block_max is `top`: codes (element 2i in the low nibble of byte i) and scale byte, s = 2^e.
template <typename T> __device__ __forceinline__ uint32_t block16(const Raw<T> &v, uint32_t top, int e, uint2 &codes) {
    codes = make_uint2(0u, 0u);
    if (top & NONFINITE) return 0x7Fu;
    const float inv_s = pow2f(-e);
    uint32_t m = __float_as_uint(__uint_as_float(top) * inv_s);
    if constexpr (sizeof(T) == 4) m = odd13(m);
    m = (__float_as_uint(__uint_as_float(m) * (1.f / 6.f)) + 0x20u) & ~0x3Fu;
    uint32_t sb;
    asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %1, %2;\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(sb) : "f"(0.f), "f"(__uint_as_float(m)));
    sb &= 0xFFu;
    if (sb == 0u) return 0u;
    float f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(e4m3_f32((uint8_t)sb)));
    float q[16];
    widen(v, q);
    if (e >= -116) {   // one factor for x / (s sc), off by the reciprocal's error alone
        f *= inv_s;
    } else {           // rows of almost nothing: it would overflow
#pragma unroll
        for (int i = 0; i < 16; i++) q[i] *= inv_s;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 16; i++) q[i] = __uint_as_float(odd13(__float_as_uint(q[i])));
    }
#pragma unroll
    for (int i = 0; i < 16; i += 2) snap2(q[i], q[i + 1], f);
#pragma unroll
    for (int k = 0; k < 2; k++) {
        uint32_t &c = k ? codes.y : codes.x;
        const float *u = q + 8 * k;
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
            "mov.b32 %0, {a, b, c, d};\n\t}"
            : "=r"(c) : "f"(u[0]), "f"(u[1]), "f"(u[2]), "f"(u[3]), "f"(u[4]), "f"(u[5]), "f"(u[6]), "f"(u[7]));
    }
    return sb;
}

// vec of rows `stride` bytes apart from p on.
inline int row_vec(const void *p, int64_t stride) {
    const uint64_t a = reinterpret_cast<uintptr_t>(p) | (uint64_t)stride;
    return (a & 31u) == 0 ? 2 : (a & 15u) == 0 ? 1 : 0;
}

} // namespace qz
} // namespace qmoe
