// Block-scaled quantisation of values in registers: what the producers of E4M3 and E2M1 operands share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "ptx.cuh"

namespace dg {

// The group of the psum layout that row `row` lies in: the end of its valid rows, and of its padding (both `row` where no group
// reaches that far). The lanes of a warp look at 32 experts at a time, so the look-up is one round trip and not a binary
// search's five.
struct GroupEnd { uint32_t valid, whole; };
__device__ __forceinline__ GroupEnd group_end_of(const int32_t* psum, uint32_t num_experts, uint32_t alignment, uint32_t row, uint32_t lane) {
    for (uint32_t e0 = 0; e0 < num_experts; e0 += 32) {
        const uint32_t p = e0 + lane < num_experts ? (uint32_t)max((int32_t)ld_stream_u32(psum + e0 + lane), 0) : 0u;
        const uint32_t whole = (p + alignment - 1) / alignment * alignment;
        const uint32_t hit = __ballot_sync(0xffffffffu, whole > row);
        if (hit != 0) {
            const int first = __ffs(hit) - 1;
            return {__shfl_sync(0xffffffffu, p, first), __shfl_sync(0xffffffffu, whole, first)};
        }
    }
    return {row, row};
}

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// 2^x and 1 / x within 2 ulp, subnormal results as zeros.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two FP32 numbers in one instruction.
struct Pair {
    uint64_t v;
    Pair() = default;
    __device__ __forceinline__ Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Pair(float a) : Pair(a, a) {}
    __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Pair operator*(const Pair& a, const Pair& b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) {
    Pair d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair fma2(const Pair& a, const Pair& b, const Pair& c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
// The largest of m and both magnitudes (a NaN does not count).
__device__ __forceinline__ float larger_magnitude(float m, const Pair& p) {
    float a, b, d;
    p.get(a, b);
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}
constexpr float kLog2E = 1.4426950408889634f;

// ---- E4M3: scale = max(amax, floor) * (1/448) rounded up to a power of two, 2^-126 or more; exponent byte from the bit pattern (255 = NaN
// for an infinity)
__device__ __forceinline__ uint32_t e4m3_scale_byte(float amax, float floor = 1e-4f) {
    const uint32_t bits = __float_as_uint(fmaxf(amax, floor) * (1.0f / 448.0f));
    return max((bits + 0x7fffffu) >> 23, 1u);
}
// Eight values times the inverse of a scale of exponent byte `e`, rounded to E4M3.
__device__ __forceinline__ uint2 e4m3_pack8(const float (&v)[8], uint32_t e) {
    const float inv = __uint_as_float((254u - e) << 23);
    uint32_t q[2];
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const __nv_fp8x2_storage_t p0 = __nv_cvt_float2_to_fp8x2(make_float2(v[h * 4] * inv, v[h * 4 + 1] * inv), __NV_SATFINITE, __NV_E4M3);
        const __nv_fp8x2_storage_t p1 = __nv_cvt_float2_to_fp8x2(make_float2(v[h * 4 + 2] * inv, v[h * 4 + 3] * inv), __NV_SATFINITE, __NV_E4M3);
        q[h] = (uint32_t)p0 | ((uint32_t)p1 << 16);
    }
    return make_uint2(q[0], q[1]);
}

__device__ __forceinline__ uint2 e4m3_pack8(const Pair (&v)[4], uint32_t e) {
    const Pair inv(__uint_as_float((254u - e) << 23));
    uint32_t q[4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        float2 f;
        (v[j] * inv).get(f.x, f.y);
        q[j] = (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
    }
    return make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
}
// Four E4M3 codes as FP32, exactly.
__device__ __forceinline__ void e4m3_unpack4(uint32_t q, float (&v)[4]) {
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(q >> (16 * h)), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        v[2 * h] = f.x;
        v[2 * h + 1] = f.y;
    }
}
// A power of two from its exponent byte (0: 2^-127, a subnormal number; 255: NaN).
__device__ __forceinline__ float ue8m0_float(uint32_t e) { return __uint_as_float(max(e << 23, 0x00400000u) | (((e + 1u) << 14) & 0x00400000u)); }

// ---- E2M1: scale = the smallest power of two s with amax <= 6 s, from the bits of amax without a product that could round:
// 6 s = 1.5 x 2^(e + 2), so the exponent goes up by one where the mantissa is above 1.5. There is no floor under amax (small
// gradients keep their bits); the byte stays within 1 .. 253 for finite values (a subnormal scale would need a subnormal
// inverse), and 255 = NaN where the block holds an infinity or a NaN, which E2M1 cannot hold: the product then shows it.
__device__ __forceinline__ uint32_t e2m1_scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return 255u;
    const int32_t e = (int32_t)((amax_bits + 0x3fffffu) >> 23) - 2;
    return (uint32_t)max(e, 1);
}
// Exponent field of the factor that brings a block of scale byte `e` into E2M1's range (0 where the scale is NaN: the codes do not
// matter then).
__device__ __forceinline__ uint32_t e2m1_inverse(uint32_t e) { return e == 255u ? 0u : 254u - e; }
// Eight values, rounded to the nearest E2M1 (halves to the even code), the first in the lowest bits.
__device__ __forceinline__ uint32_t e2m1_pack8(const float (&v)[8]) {
    uint32_t q;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(q) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return q;
}
// Eight codes as BF16 pairs, exactly: the two bytes of a magnitude are looked up by its three bits in tables of eight bytes (a byte permute
// takes four of them at a time), the sign bits by a permute that repeats the top bit of its source where a code's fourth bit is set.
__device__ __forceinline__ void e2m1_to_bf16(uint32_t q, uint32_t (&w)[4]) {
    #pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t four = q >> (16 * h), magnitude = four & 0x7777u;
        const uint32_t low = __byte_perm(0xc0800000u, 0xc0804000u, magnitude);        // 0, .5, 1, 1.5 and 2, 3, 4, 6
        uint32_t high = __byte_perm(0x3f3f3f00u, 0x40404040u, magnitude);
        uint32_t sign;                                                                // 0x80 where positive, 0xff where negative
        asm("prmt.b32 %0, %1, %1, %2;" : "=r"(sign) : "r"(0x80808080u), "r"(four));
        high |= (sign << 7) & 0x80808080u;
        w[2 * h] = __byte_perm(low, high, 0x5140);
        w[2 * h + 1] = __byte_perm(low, high, 0x7362);
    }
}
// A power of two from its exponent byte, as BF16 bits: 2^-127 is a subnormal number, 255 is NaN.
__device__ __forceinline__ uint32_t ue8m0_bf16(uint32_t e) { return e == 0u ? 0x0040u : e == 255u ? 0x7fffu : e << 7; }
// Two products of BF16 values. (One factor is a power of two here: exact but where the result is subnormal.)
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 p = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&p);
}

}  // namespace dg
