// Quantisation of a row to INT8 with a scale of its own, shared by the kernels that produce such rows.
//
//   scale = amax / 127 (FP32), q = 127 x / amax rounded to the nearest whole number, halves to the even one.
// The rounding is that of the exact quotient, so a row has one right result and every path here gives it: t = x * (127 / amax) is off by
// at most 2^-23 relative, that is by less than 2^-15 for |t| <= 127; a t that lies so near a half between two steps is decided by
// comparing 254 |x| with (2 k + 1) amax, both exact in 64 bits. About one value in 2^14 takes that path; an approximate t alone would
// put one value in 10^5 on the neighbouring step.
// A row of zeros has scale 0. A row with a NaN or an infinity has no scale: NaN, and its q are 0, so that what is multiplied with it is NaN.
#pragma once

#include "common.cuh"

namespace b200
{

struct RowScale
{
    float amax;  // of the row, times `up`
    float inv;   // 127 / amax
    float up;    // 1, or 2^64 for rows so small that 127 / amax would overflow
    float scale; // what is stored
};

__device__ __forceinline__ RowScale makeRowScale(float amax)
{
    RowScale s;
    bool const valid = amax < __int_as_float(0x7f800000); // neither infinite nor NaN
    s.scale = valid ? amax / 127.f : __int_as_float(0x7fffffff);
    s.up = amax < 0x1p-64f ? 0x1p64f : 1.f;
    s.amax = amax * s.up;
    s.inv = valid && amax > 0.f ? 127.f / s.amax : 0.f;
    return s;
}

// q of one value whose quotient lies next to a half between two steps.
static __device__ __noinline__ int32_t quantNearHalf(float x, float amax, float t)
{
    int32_t const k = __float2int_rn(fabsf(t) - 0.5f);
    double const a = 254. * static_cast<double>(fabsf(x)), b = static_cast<double>(2 * k + 1) * static_cast<double>(amax);
    int32_t const q = k + (a > b || (a == b && (k & 1) != 0) ? 1 : 0);
    return x < 0.f ? -q : q;
}

// N values (a multiple of four) to N / 4 words. kSmall: the values may be so small that they have to be scaled up first.
template <int N, bool kSmall>
__device__ __forceinline__ void quantRowChunk(float const (&x)[N], RowScale const& s, uint32_t (&w)[N / 4])
{
    constexpr float kMagic = 12582912.f; // 1.5 * 2^23: adding it rounds to nearest even and leaves q in the low byte
    float t[N], far = 0.f;
    uint32_t u[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
    {
        t[j] = (kSmall ? x[j] * s.up : x[j]) * s.inv;
        float const r = t[j] + kMagic;
        u[j] = __float_as_uint(r);
        far = fmaxf(far, fabsf(t[j] - (r - kMagic)));
    }
    if (far > 0.5f - 0x1p-15f)
    {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (fabsf(t[j] - (__uint_as_float(u[j]) - kMagic)) > 0.5f - 0x1p-15f)
                u[j] = static_cast<uint32_t>(quantNearHalf(kSmall ? x[j] * s.up : x[j], s.amax, t[j]));
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
    if (fabsf(t - (r - kMagic)) > 0.5f - 0x1p-15f)
        return static_cast<int8_t>(quantNearHalf(x, s.amax, t));
    return static_cast<int8_t>(__float_as_uint(r) & 0xffu);
}

} // namespace b200
