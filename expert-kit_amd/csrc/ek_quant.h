// The codes of a row's values: q = rint(127 p / m), m = max |p| of the row.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ek {

// rint(127 p / m) for |p| <= m, as inv = 127 / m times p.  The fp32 product t is within 2^-22 relative of the real
// value, so it decides unless it lies within 2^-15 of a half-integer; there 254 |p| is compared with the
// odd multiple of m that the half-integer stands for, both exact in fp64 (24 + 8 bits).
//
// Adding 1.5 * 2^23 rounds t to the nearest integer, ties to even, and leaves it in the low byte of the sum as the
// two's complement code.
constexpr float kToInt = 12582912.f;
__device__ __forceinline__ uint32_t quant_exact(float p, float m, float inv)
{
    const float a = __builtin_fabsf(p);
    const float f = __builtin_floorf(a * inv);
    const double lhs = 254.0 * (double)a, rhs = (2.0 * (double)f + 1.0) * (double)m;
    const bool odd = ((int)f & 1) != 0;
    const int k = (int)f + (lhs > rhs || (lhs == rhs && odd) ? 1 : 0);
    return (uint32_t)(p < 0.f ? -k : k);
}
// 8 codes as bytes
__device__ __forceinline__ uint2 quant8(const float *p, float m, float inv)
{
    uint32_t u[8];
    float worst = 0.f;               // distance to the nearest integer: 1/2 on a border
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float t = p[j] * inv, s = t + kToInt;
        worst = __builtin_fmaxf(worst, __builtin_fabsf(t - (s - kToInt)));
        u[j] = __builtin_bit_cast(uint32_t, s);
    }
    if (worst > 0.5f - 0x1p-15f) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = p[j] * inv;
            if (__builtin_fabsf(t - ((t + kToInt) - kToInt)) > 0.5f - 0x1p-15f) u[j] = quant_exact(p[j], m, inv);
        }
    }
    uint2 o;
    o.x = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
    o.y = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[7], u[6], 0x0c0c0400u), __builtin_amdgcn_perm(u[5], u[4], 0x0c0c0400u), 0x05040100u);
    return o;
}

// A row by its maximum (an infinity or NaN: a row that is not finite, whose codes are 0 and whose scale is NaN).
struct QuantRow {
    float m, inv;
    bool finite, tiny;
    __device__ __forceinline__ explicit QuantRow(float max_abs)
    {
        // a row of tiny values is brought into the range of normal numbers (a power of two: exact) before 127 / m
        finite = max_abs < __builtin_huge_valf();
        tiny = max_abs < 0x1p-100f;
        m = tiny ? max_abs * 0x1p64f : max_abs;
        inv = m > 0.f && finite ? 127.f / m : 0.f;
    }
    // m / 127, and v / 127 for the row's maximum v in the units of what the codes stand for: rounded once
    __device__ __forceinline__ float scale() const { return finite ? (tiny ? m * 0x1p-64f : m) / 127.f : __builtin_nanf(""); }
    __device__ __forceinline__ float scale_of(double v) const { return finite ? (float)(v * (1.0 / 127.0)) : __builtin_nanf(""); }
    __device__ __forceinline__ uint2 codes(float *p) const
    {
        if (tiny) {
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] *= 0x1p64f;
        }
        uint2 o = quant8(p, m, inv);
        if (!finite) o = uint2{0, 0};
        return o;
    }
};

}  // namespace ek
