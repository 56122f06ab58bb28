// Quantisation of a row to INT8 with a scale of its own, shared by the kernels that produce such rows.
//
//   scale = amax / 127 (FP32), q = 127 x / amax rounded to the nearest whole number, halves to the even one.
// The rounding is that of the exact quotient, so a row has one right result and every path here gives it: t = x * inv, inv = 127 * r, r the
// reciprocal of amax after a Newton step (within 2^-23: 2^-45 of the step, its rounding and that of its residual), is off by less than 2^-22 relative,
// that is by less than 127 * 2^-22 < 2^-15 for |t| <= 127; a t that lies so near a half between two steps is decided by comparing 254 |x| with
// (2 k + 1) amax, both exact in 64 bits. About one value in 2^14 takes that path; an approximate t alone would put one value in 10^5 on
// the neighbouring step.
// A row of zeros has scale 0. A row with a NaN or an infinity has no scale: NaN, and its q are 0, so that what is multiplied with it is NaN.
#pragma once

#include "common.cuh"

namespace b200
{

struct RowScale
{
    float amax; // of the row, times `up`
    float inv;  // about 127 / amax; 0 for a row of zeros or without a scale
    float up;   // 1, or 2^64 / 2^-64 for rows so small / so large that the reciprocal would not be a normal number
};

constexpr float kNearHalf = 0.5f - 0x1p-15f;

__device__ __forceinline__ RowScale makeRowScale(float amax)
{
    RowScale s;
    s.up = amax < 0x1p-64f ? 0x1p64f : amax > 0x1p64f ? 0x1p-64f : 1.f;
    s.amax = amax * s.up;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s.amax));
    r = fmaf(r, fmaf(-s.amax, r, 1.f), r);
    s.inv = amax > 0.f && amax < __int_as_float(0x7f800000) ? 127.f * r : 0.f;
    return s;
}

// What is stored beside the row.
__device__ __forceinline__ float rowScaleValue(float amax)
{
    return amax < __int_as_float(0x7f800000) ? amax / 127.f : __int_as_float(0x7fffffff);
}

// q of one value whose quotient lies next to a half between two steps.
static __device__ __noinline__ int32_t quantNearHalf(float x, float amax, float t)
{
    int32_t const k = __float2int_rn(fabsf(t) - 0.5f);
    double const a = 254. * static_cast<double>(fabsf(x)), b = static_cast<double>(2 * k + 1) * static_cast<double>(amax);
    int32_t const q = k + (a > b || (a == b && (k & 1) != 0) ? 1 : 0);
    return x < 0.f ? -q : q;
}

// N values (a multiple of four) to N / 4 words; x is working space. kSmall: the values may be so small that they have to be scaled up first.
template <int N, bool kSmall>
__device__ __forceinline__ void quantRowChunk(float (&x)[N], RowScale const& s, uint32_t (&w)[N / 4])
{
    if (kSmall && s.up != 1.f) // the same for the whole row
    {
#pragma unroll
        for (int j = 0; j < N; ++j)
            x[j] *= s.up;
    }
    constexpr float kMagic = 12582912.f; // 1.5 * 2^23: adding it rounds to nearest even and leaves q in the low byte
    uint64_t const inv = pack2(s.inv, s.inv), magic = pack2(kMagic, kMagic), minusMagic = pack2(-kMagic, -kMagic);
    uint64_t const minusOne = pack2(-1.f, -1.f);
    uint64_t t[N / 2], r[N / 2];
    float far = 0.f;
#pragma unroll
    for (int j = 0; j < N / 2; ++j)
    {
        t[j] = mul2(pack2(x[2 * j], x[2 * j + 1]), inv);
        r[j] = add2(t[j], magic);
        float a, b;
        unpack2(fma2(add2(r[j], minusMagic), minusOne, t[j]), a, b); // how far t is from the whole number
        far = fmaxf(fmaxf(far, fabsf(a)), fabsf(b));
    }
    uint32_t u[N];
#pragma unroll
    for (int j = 0; j < N / 2; ++j)
    {
        float a, b;
        unpack2(r[j], a, b);
        u[2 * j] = __float_as_uint(a);
        u[2 * j + 1] = __float_as_uint(b);
    }
    if (far > kNearHalf)
    {
#pragma unroll
        for (int j = 0; j < N; ++j)
        {
            float a, b;
            unpack2(t[j / 2], a, b);
            float const v = j % 2 == 0 ? a : b;
            if (fabsf(v - (__uint_as_float(u[j]) - kMagic)) > kNearHalf)
                u[j] = static_cast<uint32_t>(quantNearHalf(x[j], s.amax, v));
        }
    }
#pragma unroll
    for (int j = 0; j < N / 4; ++j)
        w[j] = s.inv == 0.f ? 0u : __byte_perm(__byte_perm(u[4 * j], u[4 * j + 1], 0x0040), __byte_perm(u[4 * j + 2], u[4 * j + 3], 0x0040), 0x5410);
}

template <bool kSmall>
__device__ __forceinline__ int8_t quantRowValue(float x, RowScale const& s)
{
    constexpr float kMagic = 12582912.f;
    if (s.inv == 0.f)
        return 0;
    if (kSmall)
        x *= s.up;
    float const t = x * s.inv;
    float const r = t + kMagic;
    if (fabsf(t - (r - kMagic)) > kNearHalf)
        return static_cast<int8_t>(quantNearHalf(x, s.amax, t));
    return static_cast<int8_t>(__float_as_uint(r) & 0xffu);
}

} // namespace b200
