// Device arithmetic of the 4-bit formats.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rfx_fp4.h"

namespace rfx {

namespace {

// Two floats -> two e4m3 bytes (nearest, ties to even, saturating at 448), lo in the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t d;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
    return d;
}

// e4m3 byte -> float, exactly (0x7F: NaN).
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)byte));
    return __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFF)));
}

// The two e4m3 bytes in the low half of w -> two floats, exactly.
__device__ __forceinline__ float2 e4m3_pair(uint32_t w) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)w));
    return make_float2(__half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu))),
                       __half2float(__ushort_as_half((unsigned short)(h2 >> 16))));
}

// e8m0 byte -> 2^(byte - 127) (0: the denormal 2^-127; 255: NaN).
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    if (byte == 255u) return __int_as_float(0x7fc00000);
    return __int_as_float(byte ? (int)(byte << 23) : 0x00400000);
}

__device__ __forceinline__ float f4_scale_value(int nv, uint32_t byte) {
    return nv ? e4m3_value(byte) : e8m0_value(byte);
}

// Eight floats -> eight e2m1 codes in a word, v[0] in the lowest nibble (nearest, ties to the
// even code, saturating at 6).
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float* v) {
    uint32_t d;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}\n"
        : "=r"(d)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}

// The same for four floats, in the lower half of a word.
__device__ __forceinline__ uint32_t cvt_e2m1x4(const float* v) {
    uint32_t d;
    asm("{\n\t.reg .b8 b0, b1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "mov.b32 %0, {b0, b1, b0, b1};\n\t}\n"
        : "=r"(d)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return d & 0xFFFFu;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;  // (__byte_perm drops the selectors' top bits)
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}

// Twice the magnitudes (0, 1, 2, 3, 4, 6, 8, 12) of those of the four codes in the low half of w
// that have no sign, as bytes; 0 for the others: a selector with its top bit set replicates the
// sign of the byte it selects, and no byte here has one.  With w ^ 0x8888: of those that have one.
__device__ __forceinline__ uint32_t e2m1_pos4(uint32_t w) { return prmt(0x03020100u, 0x0C080604u, w); }
// Of all four.
__device__ __forceinline__ uint32_t e2m1_mag4(uint32_t w) { return e2m1_pos4(w & 0x7777u); }

// 0x7F in the bytes whose code (low half of w) has its sign bit set, else 0.
__device__ __forceinline__ uint32_t e2m1_neg4(uint32_t w) {
    // a selector of 8 replicates the sign of byte 0 (0xFF), 0 copies it (0x80)
    return prmt(0x80u, 0u, w & 0x8888u) & 0x7F7F7F7Fu;
}

// The values of kN (4 or 8) codes in a word, through the upper bytes of their fp16 forms.
template <int kN>
__device__ __forceinline__ void e2m1_values(uint32_t w, float* v) {
#pragma unroll
    for (int q = 0; q < kN / 4; ++q) {
        const uint32_t x = w >> (16 * q);
        const uint32_t hi = __byte_perm(0x3E3C3800u, 0x46444240u, x & 0x7777u) | ((e2m1_neg4(x) & 0x01010101u) << 7);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t pair = __byte_perm(hi, 0u, e ? 0x3424u : 0x1404u);
            v[4 * q + 2 * e] = __half2float(__ushort_as_half((unsigned short)(pair & 0xFFFFu)));
            v[4 * q + 2 * e + 1] = __half2float(__ushort_as_half((unsigned short)(pair >> 16)));
        }
    }
}

// Value of one e2m1 code.
__device__ __forceinline__ float e2m1_value(uint32_t code) {
    const float m = 0.5f * (float)(e2m1_mag4(code & 7u) & 0xFFu);
    return (code & 8u) ? -m : m;
}

// acc + four times the dot product of sixteen codes (decoded as signed bytes of twice their values)
// with the sixteen codes of w0 and w1, exactly.
__device__ __forceinline__ int e2m1_dot16(int4 q, uint32_t w0, uint32_t w1, int acc) {
    const uint32_t x0 = w0 ^ 0x88888888u, x1 = w1 ^ 0x88888888u;
    int neg = __dp4a(q.x, (int)e2m1_pos4(x0), 0);
    acc = __dp4a(q.x, (int)e2m1_pos4(w0), acc);
    neg = __dp4a(q.y, (int)e2m1_pos4(x0 >> 16), neg);
    acc = __dp4a(q.y, (int)e2m1_pos4(w0 >> 16), acc);
    neg = __dp4a(q.z, (int)e2m1_pos4(x1), neg);
    acc = __dp4a(q.z, (int)e2m1_pos4(w1), acc);
    neg = __dp4a(q.w, (int)e2m1_pos4(x1 >> 16), neg);
    acc = __dp4a(q.w, (int)e2m1_pos4(w1 >> 16), acc);
    return acc - neg;
}

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

}  // namespace

}  // namespace rfx
