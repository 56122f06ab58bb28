// Rows of FP16 / FP32 activations to INT8, each with a scale of its own (see row_quant.cuh for the arithmetic): what the row-wise INT8
// layers multiply. No counterpart in the reference, whose INT8 plugins take one calibrated step per tensor.
#include "row_quant.cuh"

namespace b200
{
namespace
{

constexpr int kThreads = 256;

// The row's maximum over WPR warps; `slots`: this row's scratch, two lines used alternately (one barrier per call is enough, see rowSum
// in skip_ln.cu).
template <int WPR>
__device__ __forceinline__ float rowMax(float v, float (*slots)[WPR], int rowInCta, int wInRow, int lane, int& turn)
{
    v = warpMaxNan(v);
    if (WPR == 1)
        return v;
    float* const slot = slots[turn];
    turn ^= 1;
    if (lane == 0)
        slot[wInRow] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + rowInCta), "n"(WPR * 32) : "memory");
    float t = slot[0];
#pragma unroll
    for (int w = 1; w < WPR; ++w)
        t = maxNan(t, slot[w]);
    return t;
}

template <typename T>
struct Chunk;
template <>
struct Chunk<__half>
{
    static constexpr int kElems = 8;
    static __device__ __forceinline__ float absMax(uint4 const& v)
    {
        __half2 const* h = reinterpret_cast<__half2 const*>(&v);
        __half2 const m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
        return maxNan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ void unpack(uint4 const& v, float (&f)[8])
    {
        unpackHalf8(v, f);
    }
    // values `at` to at + 7 of the row, zeros where it has none
    static __device__ __forceinline__ uint4 loadPart(__half const* row, int at, int width)
    {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (at + j >= 0 && at + j < width)
                w[j / 2] |= static_cast<uint32_t>(ldGlobal(reinterpret_cast<unsigned short const*>(row) + at + j)) << (16 * (j & 1));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ void trim(uint4& v, int at, int width)
    {
        auto keep = [&](int j) { return at + j >= 0 && at + j < width; };
        auto word = [&](uint32_t w, int j) { return (keep(j) ? w & 0xffffu : 0u) | (keep(j + 1) ? w & 0xffff0000u : 0u); };
        v = make_uint4(word(v.x, 0), word(v.y, 2), word(v.z, 4), word(v.w, 6));
    }
};
template <>
struct Chunk<float>
{
    static constexpr int kElems = 4;
    static __device__ __forceinline__ float absMax(uint4 const& v)
    {
        return maxAbsNan(maxAbsNan(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z)), __uint_as_float(v.w), 0.f);
    }
    static __device__ __forceinline__ void unpack(uint4 const& v, float (&f)[4])
    {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 loadPart(float const* row, int at, int width)
    {
        auto value = [&](int j) { return at + j >= 0 && at + j < width ? __float_as_uint(ldGlobal(row + at + j)) : 0u; };
        return make_uint4(value(0), value(1), value(2), value(3));
    }
    static __device__ __forceinline__ void trim(uint4& v, int at, int width)
    {
        auto word = [&](uint32_t w, int j) { return at + j >= 0 && at + j < width ? w : 0u; };
        v = make_uint4(word(v.x, 0), word(v.y, 1), word(v.z, 2), word(v.w, 3));
    }
};

// A row is shared by WPR warps and stays in registers between the maximum and the quantisation, so it is read once: lane owns CPL
// 16-byte chunks. Bound by HBM: 3 bytes a value for FP16. Measured, of the copy rate: FP16 24576 x 4096 52.4 us (0.89; 63 us with one value
// per instruction), x 1024 14.3 us (0.82), FP32 24576 x 1024 19.4 us (1.0). Rows of eight warps and FP32 rows have the next row on its way
// while this one is quantised: FP32 12000 x 4096 43.0 -> 39.0 us, FP16 12000 x 8192 53.6 -> 51.2 us; FP16 rows of fewer warps lose by the
// registers it takes (24576 x 1024 14.3 -> 16.7 us).
template <typename T, int CPL, int WPR>
__global__ void __launch_bounds__(kThreads) quantizeRowsKernel(int64_t const rows, int32_t const width, T const* in,
    int64_t const inStride, int8_t* __restrict__ out, int64_t const outStride, float* __restrict__ scales)
{
    constexpr int E = Chunk<T>::kElems;
    constexpr int kRowsPerCta = kThreads / 32 / WPR;
    constexpr bool kAhead = sizeof(T) == 4 || WPR == 8;
    __shared__ float red[kRowsPerCta][2][WPR];
    int turn = 0;
    int const lane = threadIdx.x & 31;
    int const warp = threadIdx.x >> 5;
    int const rowInCta = warp / WPR;
    int const wInRow = warp % WPR;
    gridDependencyLaunch();
    gridDependencyWait();

    int64_t const step = static_cast<int64_t>(gridDim.x) * kRowsPerCta;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + rowInCta;
    auto load = [&](int64_t r, uint4 (&v)[CPL]) {
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const left = width - ((i * WPR + wInRow) * 32 + lane) * E;
            T const* const p = in + r * inStride + ((i * WPR + wInRow) * 32 + lane) * E;
            v[i] = left >= E ? ldgStream(p) : left > 0 ? Chunk<T>::loadPart(p, 0, left) : make_uint4(0, 0, 0, 0);
        }
    };
    uint4 ahead[CPL];
    if (kAhead && row < rows)
        load(row, ahead);
    for (; row < rows; row += step)
    {
        uint4 v[CPL];
        if (kAhead)
        {
#pragma unroll
            for (int i = 0; i < CPL; ++i)
                v[i] = ahead[i];
        }
        else
            load(row, v);
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < CPL; ++i)
            m = maxNan(m, Chunk<T>::absMax(v[i]));
        if (kAhead && row + step < rows)
            load(row + step, ahead);
        m = rowMax<WPR>(m, red[rowInCta], rowInCta, wInRow, lane, turn);
        RowScale const s = makeRowScale(m);
        if (wInRow == 0 && lane == 0)
            scales[row] = rowScaleValue(m);
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const left = width - ((i * WPR + wInRow) * 32 + lane) * E;
            int8_t* const p = out + row * outStride + ((i * WPR + wInRow) * 32 + lane) * E;
            if (left <= 0)
                continue;
            float f[E];
            Chunk<T>::unpack(v[i], f);
            uint32_t w[E / 4];
            quantRowChunk<E, sizeof(T) == 4>(f, s, w);
            if (left >= E)
            {
                if constexpr (E == 8)
                    stgStream8(p, make_uint2(w[0], w[1]));
                else
                    *reinterpret_cast<uint32_t*>(p) = w[0];
            }
            else
            {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (j < left)
                        p[j] = static_cast<int8_t>(w[j / 4] >> (8 * (j & 3)));
            }
        }
    }
}

// Rows that begin at any value: the 16-byte vectors that hold them are quantised as they lie, `mis` values behind the row's; what moves by `mis` is
// the results, a quarter or half as many bytes: a lane's vector and its neighbour's, together, hold the bytes it stores. Mostly issue slots (110
// instructions per vector and warp; 72 % of the slots used at 24576 x 4095 FP16, the rest waits for the row's loads and its maximum). FP16 24576 x 1001 19.3 us (17.5 us on 16 bytes), x 4095 79 us (52), FP32 12000 x 4097 49 us (39); with one value per
// lane and load 61, 115 and 59 us, with two overlapping vectors per lane for each it quantises 25, 88 and 59 us.
template <typename T, int CPL, int WPR>
__global__ void __launch_bounds__(kThreads, 4) quantizeRowsOddKernel(int64_t const rows, int32_t const width, T const* in,
    int64_t const inStride, int8_t* __restrict__ out, int64_t const outStride, float* __restrict__ scales)
{
    constexpr int E = Chunk<T>::kElems;
    constexpr int kWords = E / 4;
    constexpr int kRowsPerCta = kThreads / 32 / WPR;
    constexpr bool kAhead = sizeof(T) == 4 && WPR == 8; // 12000 x 4097 54.3 -> 48.8 us, FP16 5000 x 8190 32.2 -> 34.6 us
    __shared__ float red[kRowsPerCta][2][WPR];
    __shared__ uint32_t heads[kRowsPerCta][WPR][kWords]; // the results of the warps' first vectors
    int turn = 0;
    int const lane = threadIdx.x & 31;
    int const warp = threadIdx.x >> 5;
    int const rowInCta = warp / WPR;
    int const wInRow = warp % WPR;
    int const first = wInRow * CPL * 32 + lane; // of this lane's vectors, 32 apart
    gridDependencyLaunch();
    gridDependencyWait();

    T const* const end = in + (rows - 1) * inStride + width;
    int64_t const step = static_cast<int64_t>(gridDim.x) * kRowsPerCta;
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + rowInCta;
    auto misOf = [&](int64_t r) { return static_cast<int>((reinterpret_cast<uintptr_t>(in + r * inStride) & 15u) / sizeof(T)); };
    auto load = [&](int64_t r, uint4 (&v)[CPL]) {
        T const* const p = in + r * inStride;
        int const mis = misOf(r), nVec = (width + mis + E - 1) / E;
        T const* const q = p - mis;
        if (q >= in && q + nVec * E <= end) // whole vectors, with values of the rows beside this one or of the gap between them
        {
#pragma unroll
            for (int i = 0; i < CPL; ++i)
                v[i] = first + 32 * i < nVec ? ldgStream(q + (first + 32 * i) * E) : make_uint4(0, 0, 0, 0);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < CPL; ++i)
                v[i] = Chunk<T>::loadPart(p, (first + 32 * i) * E - mis, width);
        }
    };
    uint4 ahead[CPL];
    if (kAhead && row < rows)
        load(row, ahead);
    for (; row < rows; row += step)
    {
        uint4 v[CPL];
        if (kAhead)
        {
#pragma unroll
            for (int i = 0; i < CPL; ++i)
                v[i] = ahead[i];
        }
        else
            load(row, v);
        int const mis = misOf(row);
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const e0 = (first + 32 * i) * E - mis;
            if (e0 < 0 || e0 + E > width)
                Chunk<T>::trim(v[i], e0, width);
            m = maxNan(m, Chunk<T>::absMax(v[i]));
        }
        if (kAhead && row + step < rows)
            load(row + step, ahead);
        m = rowMax<WPR>(m, red[rowInCta], rowInCta, wInRow, lane, turn);
        RowScale const s = makeRowScale(m);
        if (wInRow == 0 && lane == 0)
            scales[row] = rowScaleValue(m);
        uint32_t w[CPL][kWords];
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            float f[E];
            Chunk<T>::unpack(v[i], f);
            quantRowChunk<E, sizeof(T) == 4>(f, s, w[i]);
        }
        if (WPR > 1)
        {
            if (lane == 0)
#pragma unroll
                for (int j = 0; j < kWords; ++j)
                    heads[rowInCta][wInRow][j] = w[0][j];
            asm volatile("bar.sync %0, %1;" ::"r"(1 + rowInCta), "n"(WPR * 32) : "memory"); // (the next writes are behind the next row's maximum)
        }
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            uint32_t t[2 * kWords];
#pragma unroll
            for (int j = 0; j < kWords; ++j)
            {
                t[j] = w[i][j];
                t[kWords + j] = __shfl_sync(0xffffffffu, lane == 0 && i + 1 < CPL ? w[i + 1 < CPL ? i + 1 : i][j] : w[i][j], (lane + 1) & 31);
                if (WPR > 1 && i + 1 == CPL && lane == 31)
                    t[kWords + j] = heads[rowInCta][wInRow + 1 < WPR ? wInRow + 1 : wInRow][j];
            }
            uint32_t u[kWords];
            if constexpr (kWords == 2)
            {
                uint32_t const a = (mis & 4) ? t[1] : t[0], b = (mis & 4) ? t[2] : t[1], c = (mis & 4) ? t[3] : t[2];
                u[0] = __funnelshift_r(a, b, (mis & 3) * 8);
                u[1] = __funnelshift_r(b, c, (mis & 3) * 8);
            }
            else
                u[0] = __funnelshift_r(t[0], t[1], mis * 8);
            int const at = (first + 32 * i) * E, left = width - at;
            int8_t* const o = out + row * outStride + at;
            if (left >= E)
            {
                if constexpr (kWords == 2)
                    stgStream8(o, make_uint2(u[0], u[1]));
                else
                    *reinterpret_cast<uint32_t*>(o) = u[0];
            }
            else if (left > 0)
            {
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (j < left)
                        o[j] = static_cast<int8_t>(u[j / 4] >> (8 * (j & 3)));
            }
        }
    }
}

// Rows longer than the registers of eight warps, or whose results are not aligned for wide stores: a CTA per row reads it twice (the second time from
// L1 or L2), one value per lane and load. FP32 6000 x 8192 64 us (floor 38 us), FP16 3000 x 14336 54 us (20 us), 3000 x 8200
// 32.2 us (11.4 us): the loads of single values, not the memory.
template <typename T>
__global__ void __launch_bounds__(kThreads) quantizeRowsLongKernel(int64_t const rows, int32_t const width, T const* in,
    int64_t const inStride, int8_t* __restrict__ out, int64_t const outStride, float* __restrict__ scales)
{
    __shared__ float red[2][kThreads / 32];
    int turn = 0;
    gridDependencyLaunch();
    gridDependencyWait();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
    {
        T const* const p = in + row * inStride;
        float m = 0.f;
#pragma unroll 8
        for (int i = threadIdx.x; i < width; i += kThreads)
            m = maxNan(m, fabsf(static_cast<float>(p[i])));
        m = rowMax<kThreads / 32>(m, red, 0, threadIdx.x >> 5, threadIdx.x & 31, turn);
        RowScale const s = makeRowScale(m);
        if (threadIdx.x == 0)
            scales[row] = rowScaleValue(m);
        for (int i0 = threadIdx.x; i0 < width; i0 += 8 * kThreads)
        {
            float v[8]; // all of them on their way before the first result is stored
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = i0 + j * kThreads < width ? static_cast<float>(p[i0 + j * kThreads]) : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i0 + j * kThreads < width)
                    out[row * outStride + i0 + j * kThreads] = quantRowValue<sizeof(T) == 4>(v[j], s);
        }
    }
}

template <typename T>
int32_t quantizeRows(cudaStream_t stream, int64_t rows, int32_t width, T const* in, int64_t inStride, int8_t* out, int64_t outStride, float* scales)
{
    constexpr int E = Chunk<T>::kElems;
    bool const odd = !aligned16(in) || (inStride % E != 0 && rows > 1);
    int const chunks = (width + (odd ? E - 1 : 0) + E - 1) / E; // vectors that a row may lie in
    bool const wide = (reinterpret_cast<uintptr_t>(out) | static_cast<uintptr_t>(outStride)) % E == 0;
    cudaError_t e = cudaErrorUnknown;
    if (!wide || chunks > 8 * 4 * 32 + (odd ? 1 : 0))
    {
        int64_t const most = static_cast<int64_t>(smCount()) * 8;
        e = launchDependent(quantizeRowsLongKernel<T>, dim3(static_cast<unsigned>(rows < most ? rows : most)), dim3(kThreads), 0, stream, rows, width, in,
            inStride, out, outStride, scales);
    }
    else
    {
        // Four chunks per lane, or two where there are fewer rows than places for them: 37 x 4096 FP16 2.2 -> 1.7 us, 24576 x 4096 52 -> 66 us.
        int const most = rows <= 2 * smCount() ? 2 : 4;
        int wpr = 1;
        while (chunks > 32 * most * wpr + (odd ? 1 : 0) && wpr < 8)
            wpr *= 2;
        int const cpl = (chunks + 32 * wpr - 1) / (32 * wpr); // up to five where a row of whole vectors has four
        int64_t const ctas = (rows + 8 / wpr - 1) / (8 / wpr);
        int64_t const places = static_cast<int64_t>(smCount()) * (sizeof(T) == 4 ? 4 : 8);
        unsigned const grid = static_cast<unsigned>(ctas < places ? ctas : places);
#define B200_QUANT_CASE(C, W)                                                                                          \
    if (cpl == C && wpr == W)                                                                                          \
        e = launchDependent(odd ? quantizeRowsOddKernel<T, C, W> : quantizeRowsKernel<T, C, W>, dim3(grid), dim3(kThreads), 0, stream, rows, width, in, \
            inStride, out, outStride, scales);
#define B200_QUANT_ODD_CASE(C, W)                                                                                      \
    if (odd && cpl == C && wpr == W)                                                                                   \
        e = launchDependent(quantizeRowsOddKernel<T, C, W>, dim3(grid), dim3(kThreads), 0, stream, rows, width, in, inStride, out, outStride, scales);
        B200_QUANT_CASE(1, 1)
        B200_QUANT_CASE(2, 1)
        B200_QUANT_CASE(3, 1)
        B200_QUANT_CASE(4, 1)
        B200_QUANT_CASE(2, 2)
        B200_QUANT_CASE(3, 2)
        B200_QUANT_CASE(4, 2)
        B200_QUANT_CASE(2, 4)
        B200_QUANT_CASE(3, 4)
        B200_QUANT_CASE(4, 4)
        B200_QUANT_CASE(2, 8)
        B200_QUANT_CASE(3, 8)
        B200_QUANT_CASE(4, 8)
        B200_QUANT_ODD_CASE(5, 1)
        B200_QUANT_ODD_CASE(5, 2)
        B200_QUANT_ODD_CASE(5, 4)
        B200_QUANT_ODD_CASE(5, 8)
#undef B200_QUANT_ODD_CASE
#undef B200_QUANT_CASE
    }
    if (e != cudaSuccess)
        B200_FAIL(BERT_B200_CUDA_ERROR, "quantizeRowsKernel: %s", cudaGetErrorString(e));
    return checkLaunch("quantizeRowsKernel");
}

} // namespace
} // namespace b200

using namespace b200;

extern "C" int32_t bert_b200_quantize_rows(void* stream, int32_t type_id, int64_t rows, int32_t width, void const* input, int64_t input_stride,
    int8_t* output, int64_t output_stride, float* row_scales)
{
    B200_REQUIRE(type_id == BERT_B200_FP16 || type_id == BERT_B200_FP32, "quantize_rows: type_id %d (FP16 or FP32)", type_id);
    B200_REQUIRE(rows >= 0 && width > 0 && width <= 1 << 30, "quantize_rows: bad sizes rows=%lld width=%d", static_cast<long long>(rows), width);
    B200_REQUIRE(input_stride >= width && output_stride >= width, "quantize_rows: a row stride is smaller than the row's %d values", width);
    if (rows == 0)
        return BERT_B200_OK;
    B200_REQUIRE(input && output && row_scales, "quantize_rows: null pointer");
    uintptr_t const elem = type_id == BERT_B200_FP16 ? 2 : 4;
    B200_REQUIRE(reinterpret_cast<uintptr_t>(input) % elem == 0 && reinterpret_cast<uintptr_t>(row_scales) % 4 == 0,
        "quantize_rows: input or row_scales is not aligned to its type");
    auto s = static_cast<cudaStream_t>(stream);
    if (type_id == BERT_B200_FP16)
        return quantizeRows(s, rows, width, static_cast<__half const*>(input), input_stride, output, output_stride, row_scales);
    return quantizeRows(s, rows, width, static_cast<float const*>(input), input_stride, output, output_stride, row_scales);
}
