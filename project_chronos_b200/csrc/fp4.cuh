// fp4.cuh — pages of 4-bit values (include/chronos_paged4.h): where a slot's codes and
// scales lie, and the conversions.
#pragma once

#include "common.cuh"

namespace chronos {

// Columns of a stored slot: the head dimension rounded up to what the kernels are built for.
__host__ __device__ __forceinline__ int fp4_columns(int head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
// Bytes of a record of 16 slots, the codes first.
__host__ __device__ constexpr int fp4_record(int columns) { return 9 * columns; }

// 8 codes (column 0 in the lowest bits) as four pairs of halves, exact.
__device__ __forceinline__ void fp4_halves(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
}
// 8 values as codes: to the nearest, ties to even, beyond 6 to 6.
__device__ __forceinline__ uint32_t fp4_codes(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// Two scales (the first in the low byte) as halves, exact.
__device__ __forceinline__ uint32_t fp8_halves(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
    return r;
}
__device__ __forceinline__ float fp8_value(uint32_t scale) {
    const uint32_t h = fp8_halves(scale & 0xffu);
    return __low2float(*reinterpret_cast<const __half2*>(&h));
}
// lo and hi as scales, hi in the upper byte: to the nearest, ties to even, beyond 448 to 448.
__device__ __forceinline__ uint32_t fp8_scales(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t mul_halves(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// Halves of one operand twice (an operand of the multiplication itself, no instruction of its
// own): a * (s.low, s.low), a * (s.high, s.high).
__device__ __forceinline__ uint32_t mul_low(uint32_t a, uint32_t s) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t.reg .b32 t;\n\tmov.b32 {l, h}, %2;\n\tmov.b32 t, {l, l};\n\tmul.rn.f16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(a), "r"(s));
    return r;
}
__device__ __forceinline__ uint32_t mul_high(uint32_t a, uint32_t s) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\t.reg .b32 t;\n\tmov.b32 {l, h}, %2;\n\tmov.b32 t, {h, h};\n\tmul.rn.f16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(a), "r"(s));
    return r;
}
// (a.low * s.low, b.low * t.high) and (a.high * s.low, b.high * t.high) for s = (s, 0), t = (0, t).
__device__ __forceinline__ void pair_scaled(uint32_t a, uint32_t b, uint32_t s, uint32_t t, uint32_t& low, uint32_t& high) {
    asm("{\n\t.reg .b16 al, ah, bl, bh;\n\t.reg .b32 x, y, z;\n\t"
        "mov.b32 {al, ah}, %2;\n\tmov.b32 {bl, bh}, %3;\n\t"
        "mov.b32 x, {al, al};\n\tmov.b32 y, {bl, bl};\n\t"
        "mul.rn.f16x2 z, x, %4;\n\tfma.rn.f16x2 %0, y, %5, z;\n\t"
        "mov.b32 x, {ah, ah};\n\tmov.b32 y, {bh, bh};\n\t"
        "mul.rn.f16x2 z, x, %4;\n\tfma.rn.f16x2 %1, y, %5, z;\n\t}"
        : "=&r"(low), "=&r"(high)
        : "r"(a), "r"(b), "r"(s), "r"(t));
}
constexpr uint32_t kFp8Nan = 0x7fu;
// max(a, |b|), NaN where one of the two is.
__device__ __forceinline__ float max_magnitude(float a, float b) {
    float r;
    asm("{\n\t.reg .f32 m;\n\tabs.f32 m, %2;\n\tmax.NaN.f32 %0, %1, m;\n\t}" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 1 / x to 2^-22.
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

}  // namespace chronos
