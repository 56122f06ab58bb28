// Residual + bias + LayerNorm whose result is also quantised to INT8 with a scale per row (see row_quant.cuh): what a row-wise INT8 layer
// behind it multiplies. No counterpart in the reference, whose INT8 SkipLayerNorm takes one calibrated step per tensor
// (plugin/skipLayerNormPlugin/skipLayerNormKernel.cu:219-250).
//
// The same values as skipLnKernel (skip_ln.cu), to the bit: rows are shared by the same warps and their sums are taken in the same order.
#include "row_quant.cuh"

namespace b200
{
namespace
{

constexpr int kWarpsPerCta = 8;
constexpr int kThreads = kWarpsPerCta * 32;

// One value per warp of a row, in the order of the warps (`slots`: two lines used alternately, see rowSum in skip_ln.cu).
template <int WPR, typename F>
__device__ __forceinline__ float overWarps(float v, float (*slots)[WPR], int rowInCta, int wInRow, int lane, int& turn, F const& join)
{
    if (WPR == 1)
        return v;
    float* const slot = slots[turn];
    turn ^= 1;
    if (lane == 0)
        slot[wInRow] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(1 + rowInCta), "n"(WPR * 32) : "memory");
    float t = join(0.f, slot[0]);
#pragma unroll
    for (int w = 1; w < WPR; ++w)
        t = join(t, slot[w]);
    return t;
}

// A 16-byte chunk as pairs of FP32 numbers, and back.
template <typename T>
struct Pairs;
template <>
struct Pairs<__half>
{
    static constexpr int kElems = 8;
    static __device__ __forceinline__ void unpack(uint4 const& v, uint64_t (&f)[4])
    {
        __half2 const* h = reinterpret_cast<__half2 const*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            float2 const t = __half22float2(h[i]);
            f[i] = pack2(t.x, t.y);
        }
    }
    static __device__ __forceinline__ uint4 pack(float const (&f)[8])
    {
        return packHalf8(f);
    }
};
template <>
struct Pairs<float>
{
    static constexpr int kElems = 4;
    static __device__ __forceinline__ void unpack(uint4 const& v, uint64_t (&f)[2])
    {
        f[0] = pack2(__uint_as_float(v.x), __uint_as_float(v.y));
        f[1] = pack2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ uint4 pack(float const (&f)[4])
    {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};

template <int CPL>
constexpr int kCtasPerSm = CPL == 1 ? 3 : 2;

// One row is shared by WPR warps; each lane owns CPL 16-byte chunks and keeps them in registers through three reductions: sum, squares,
// largest magnitude. Arithmetic for pairs of values: with one value per instruction (36 of them each) the kernel was bound by issue slots.
template <typename T, int CPL, int WPR, bool HAS_BIAS>
__global__ void __launch_bounds__(kThreads, kCtasPerSm<CPL>) skipLnQuantKernel(int32_t const ld, int64_t const rows,
    T const* __restrict__ in, T const* __restrict__ skip, T const* __restrict__ beta, T const* __restrict__ gamma, T const* __restrict__ bias,
    T* __restrict__ out, float const eps, int8_t* __restrict__ outI8, float* __restrict__ rowScales)
{
    constexpr int E = Pairs<T>::kElems;
    constexpr int P = E / 2;
    constexpr int kRowsPerCta = kWarpsPerCta / WPR;
    __shared__ float red[kRowsPerCta][2][WPR];
    int turn = 0;

    int const lane = threadIdx.x & 31;
    int const warp = threadIdx.x >> 5;
    int const rowInCta = warp / WPR;
    int const wInRow = warp % WPR;
    int const chunksPerRow = ld / E;
    float const rld = 1.f / static_cast<float>(ld);
    gridDependencyLaunch();
    if (blockIdx.x == 0) // usually in DRAM; a prefetch yields no value, whoever may still be writing it
        for (int i = threadIdx.x * (128 / static_cast<int>(sizeof(T))); i < ld; i += kThreads * (128 / static_cast<int>(sizeof(T))))
        {
            prefetchL2(gamma + i);
            prefetchL2(beta + i);
            if (HAS_BIAS)
                prefetchL2(bias + i);
        }
    gridDependencyWait();

    int64_t const rowsRounded = (rows + kRowsPerCta - 1) / kRowsPerCta * kRowsPerCta;
    int64_t const rowStride = static_cast<int64_t>(gridDim.x) * kRowsPerCta;
    uint4 a[CPL], b[CPL];
    auto loadRow = [&](int64_t r) {
        bool const rOk = r < rows;
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const c = (i * WPR + wInRow) * 32 + lane;
            bool const ok = rOk && c < chunksPerRow;
            a[i] = ok ? ldgStream(in + r * ld + c * E) : make_uint4(0, 0, 0, 0);
            b[i] = ok && skip ? ldgStream(skip + r * ld + c * E) : make_uint4(0, 0, 0, 0);
        }
    };

    auto sum = [](float x, float y) { return x + y; };
    auto most = [](float x, float y) { return maxNan(x, y); };
    // Up to two chunks per lane: its columns' parameters stay in registers, converted once (24576 x 1024 35.6 -> 33.5 us at two CTAs per SM
    // instead of three); more chunks find them in L1 in every row.
    constexpr bool kKeep = CPL <= 2;
    uint64_t keptGamma[CPL][P], keptBeta[CPL][P], keptBias[CPL][P];
    if (kKeep)
    {
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const c = (i * WPR + wInRow) * 32 + lane;
            if (c < chunksPerRow)
            {
                Pairs<T>::unpack(ldgKeep(gamma + c * E), keptGamma[i]);
                Pairs<T>::unpack(ldgKeep(beta + c * E), keptBeta[i]);
                if (HAS_BIAS)
                    Pairs<T>::unpack(ldgKeep(bias + c * E), keptBias[i]);
            }
        }
    }
    loadRow(static_cast<int64_t>(blockIdx.x) * kRowsPerCta + rowInCta);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + rowInCta; row < rowsRounded; row += rowStride)
    {
        bool const rowOk = row < rows;
        uint64_t x[CPL][P];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const c = (i * WPR + wInRow) * 32 + lane;
            uint64_t t[P];
            Pairs<T>::unpack(a[i], x[i]);
            Pairs<T>::unpack(b[i], t);
#pragma unroll
            for (int j = 0; j < P; ++j)
                x[i][j] = add2(x[i][j], t[j]);
            if (HAS_BIAS && c < chunksPerRow)
            {
                if (!kKeep)
                    Pairs<T>::unpack(ldgKeep(bias + c * E), keptBias[i]);
#pragma unroll
                for (int j = 0; j < P; ++j)
                    x[i][j] = add2(x[i][j], keptBias[i][j]);
            }
#pragma unroll
            for (int j = 0; j < P; ++j)
            {
                float lo, hi;
                unpack2(x[i][j], lo, hi);
                s += lo;
                s += hi;
            }
        }
        // a / b are unpacked: the next row's loads go out now and land during the statistics and the stores of this row
        if (row + rowStride < rowsRounded)
            loadRow(row + rowStride);
        float const mu = overWarps<WPR>(warpSum(s), red[rowInCta], rowInCta, wInRow, lane, turn, sum) * rld;
        uint64_t const minusMu = pack2(-mu, -mu);
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const c = (i * WPR + wInRow) * 32 + lane;
            if (c < chunksPerRow)
            {
#pragma unroll
                for (int j = 0; j < P; ++j)
                {
                    x[i][j] = add2(x[i][j], minusMu);
                    float lo, hi;
                    unpack2(x[i][j], lo, hi);
                    q = fmaf(lo, lo, q);
                    q = fmaf(hi, hi, q);
                }
            }
        }
        float const var = overWarps<WPR>(warpSum(q), red[rowInCta], rowInCta, wInRow, lane, turn, sum) * rld;
        float const rsigma = rsqrtf(var + eps);
        uint64_t const rs2 = pack2(rsigma, rsigma);

        float largest = 0.f;
        float y[CPL][E];
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const c = (i * WPR + wInRow) * 32 + lane;
            if (rowOk && c < chunksPerRow)
            {
                if (!kKeep)
                {
                    Pairs<T>::unpack(ldgKeep(gamma + c * E), keptGamma[i]);
                    Pairs<T>::unpack(ldgKeep(beta + c * E), keptBeta[i]);
                }
#pragma unroll
                for (int j = 0; j < P; ++j)
                {
                    unpack2(fma2(mul2(keptGamma[i][j], x[i][j]), rs2, keptBeta[i][j]), y[i][2 * j], y[i][2 * j + 1]);
                    largest = maxAbsNan(largest, y[i][2 * j], y[i][2 * j + 1]);
                }
                if (out)
                    stgStream(out + row * ld + c * E, Pairs<T>::pack(y[i]));
            }
        }
        largest = overWarps<WPR>(warpMaxNan(largest), red[rowInCta], rowInCta, wInRow, lane, turn, most);
        RowScale const scale = makeRowScale(largest);
        if (rowOk && wInRow == 0 && lane == 0)
            rowScales[row] = rowScaleValue(largest);
#pragma unroll
        for (int i = 0; i < CPL; ++i)
        {
            int const c = (i * WPR + wInRow) * 32 + lane;
            if (rowOk && c < chunksPerRow)
            {
                uint32_t w[E / 4];
                quantRowChunk<E, true>(y[i], scale, w);
                if constexpr (E == 8)
                    stgStream8(outI8 + row * ld + c * E, make_uint2(w[0], w[1]));
                else
                    *reinterpret_cast<uint32_t*>(outI8 + row * ld + c * E) = w[0];
            }
        }
    }
}

// Any ld, scalar accesses, one warp per row; the row is revisited from L1 / L2 instead of registers.
template <typename T, bool HAS_BIAS>
__global__ void __launch_bounds__(kThreads) skipLnQuantScalarKernel(int32_t const ld, int64_t const rows, T const* in, T const* skip,
    T const* __restrict__ beta, T const* __restrict__ gamma, T const* __restrict__ bias, T* out, float const eps, int8_t* __restrict__ outI8,
    float* __restrict__ rowScales)
{
    int const lane = threadIdx.x & 31;
    int const warp = threadIdx.x >> 5;
    float const rld = 1.f / static_cast<float>(ld);
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarpsPerCta + warp; row < rows; row += static_cast<int64_t>(gridDim.x) * kWarpsPerCta)
    {
        T const* const a = in + row * ld;
        T const* const b = skip ? skip + row * ld : nullptr;
        auto value = [&](int i) {
            return static_cast<float>(a[i]) + (b ? static_cast<float>(b[i]) : 0.f) + (HAS_BIAS ? static_cast<float>(bias[i]) : 0.f);
        };
        float s = 0.f;
        for (int i = lane; i < ld; i += 32)
            s += value(i);
        float const mu = warpSum(s) * rld;
        float q = 0.f;
        for (int i = lane; i < ld; i += 32)
        {
            float const d = value(i) - mu;
            q += d * d;
        }
        float const rsigma = rsqrtf(warpSum(q) * rld + eps);
        auto result = [&](int i) { return static_cast<float>(gamma[i]) * (value(i) - mu) * rsigma + static_cast<float>(beta[i]); };
        float most = 0.f;
        for (int i = lane; i < ld; i += 32)
            most = maxNan(most, fabsf(result(i)));
        most = warpMaxNan(most);
        RowScale const scale = makeRowScale(most);
        if (lane == 0)
            rowScales[row] = rowScaleValue(most);
        for (int i = lane; i < ld; i += 32)
        {
            float const y = result(i); // read before it is written: `out` may be the input's rows
            outI8[row * ld + i] = quantRowValue<true>(y, scale);
            if (out)
                out[row * ld + i] = static_cast<T>(y);
        }
    }
}

template <typename T>
struct Args
{
    int32_t ld;
    int64_t rows;
    T const *in, *skip, *beta, *gamma, *bias;
    T* out;
    float eps;
    int8_t* outI8;
    float* rowScales;
};

// As many passes for every CTA (gridFor in skip_ln.cu).
inline int gridFor(int64_t groups, int ctasPerSm)
{
    int64_t const cap = static_cast<int64_t>(smCount()) * ctasPerSm;
    if (groups <= cap)
        return static_cast<int>(groups);
    int64_t const passes = (groups + cap - 1) / cap;
    return static_cast<int>((groups + passes - 1) / passes);
}

template <typename T, int CPL, int WPR>
int32_t launch(cudaStream_t s, Args<T> const& p)
{
    int const rowsPerCta = kWarpsPerCta / WPR;
    dim3 const grid(gridFor((p.rows + rowsPerCta - 1) / rowsPerCta, kCtasPerSm<CPL>));
    cudaError_t const e = p.bias
        ? launchDependent(skipLnQuantKernel<T, CPL, WPR, true>, grid, dim3(kThreads), 0, s, p.ld, p.rows, p.in, p.skip, p.beta, p.gamma, p.bias, p.out, p.eps, p.outI8, p.rowScales)
        : launchDependent(skipLnQuantKernel<T, CPL, WPR, false>, grid, dim3(kThreads), 0, s, p.ld, p.rows, p.in, p.skip, p.beta, p.gamma, p.bias, p.out, p.eps, p.outI8, p.rowScales);
    if (e != cudaSuccess)
        B200_FAIL(BERT_B200_CUDA_ERROR, "skipLnQuantKernel: %s", cudaGetErrorString(e));
    return checkLaunch("skipLnQuantKernel");
}

template <typename T>
int32_t dispatch(cudaStream_t s, Args<T> const& p)
{
    constexpr int E = 16 / sizeof(T);
    bool const vec = p.ld % E == 0 && p.ld / E <= 32 * 4 * 8 && aligned16(p.in) && aligned16(p.skip) && aligned16(p.out) && aligned16(p.beta)
        && aligned16(p.gamma) && aligned16(p.bias) && reinterpret_cast<uintptr_t>(p.outI8) % E == 0;
    if (!vec)
    {
        int const grid = gridFor((p.rows + kWarpsPerCta - 1) / kWarpsPerCta, 8);
        if (p.bias)
            skipLnQuantScalarKernel<T, true><<<grid, kThreads, 0, s>>>(p.ld, p.rows, p.in, p.skip, p.beta, p.gamma, p.bias, p.out, p.eps, p.outI8, p.rowScales);
        else
            skipLnQuantScalarKernel<T, false><<<grid, kThreads, 0, s>>>(p.ld, p.rows, p.in, p.skip, p.beta, p.gamma, p.bias, p.out, p.eps, p.outI8, p.rowScales);
        return checkLaunch("skipLnQuantScalarKernel");
    }
    // the warps per row of dispatchSkipLn (skip_ln.cu), so that the sums are the same
    int const chunks = p.ld / E;
    int wpr = 1;
    while (chunks > 32 * 4 * wpr)
        wpr *= 2;
    if (wpr == 1 && chunks > 32 * 3)
        wpr = 2;
    int const cpl = (chunks + 32 * wpr - 1) / (32 * wpr);
#define B200_CASE(C, W)                                                                                                \
    if (cpl == C && wpr == W)                                                                                          \
        return launch<T, C, W>(s, p);
    B200_CASE(1, 1)
    B200_CASE(2, 1)
    B200_CASE(3, 1)
    B200_CASE(2, 2)
    B200_CASE(3, 2)
    B200_CASE(4, 2)
    B200_CASE(3, 4)
    B200_CASE(4, 4)
    B200_CASE(3, 8)
    B200_CASE(4, 8)
#undef B200_CASE
    B200_FAIL(BERT_B200_NOT_SUPPORTED, "skip_layer_norm_quantize: no kernel for ld=%d", p.ld);
}

template <typename T>
int32_t run(cudaStream_t s, int32_t ld, int64_t n, void const* input, void const* skip, void const* beta, void const* gamma, void* output, int8_t* outI8,
    float* rowScales, void const* bias, float eps)
{
    return dispatch<T>(s, Args<T>{ld, n / ld, static_cast<T const*>(input), static_cast<T const*>(skip), static_cast<T const*>(beta), static_cast<T const*>(gamma),
                              static_cast<T const*>(bias), static_cast<T*>(output), eps, outI8, rowScales});
}

} // namespace
} // namespace b200

using namespace b200;

extern "C" int32_t bert_b200_skip_layer_norm_quantize(void* stream, int32_t type_id, int32_t ld, int64_t n, void const* input, void const* skip,
    void const* beta, void const* gamma, void* output, int8_t* out_i8, float* row_scales, void const* bias, float eps)
{
    B200_REQUIRE(type_id == BERT_B200_FP16 || type_id == BERT_B200_FP32, "skip_layer_norm_quantize: type_id %d (FP16 or FP32)", type_id);
    B200_REQUIRE(ld > 0 && ld <= 1 << 30 && n >= 0 && n % ld == 0, "skip_layer_norm_quantize: n=%lld is not a multiple of ld=%d", static_cast<long long>(n), ld);
    B200_REQUIRE(eps >= 0.f, "skip_layer_norm_quantize: eps must not be negative");
    if (n == 0)
        return BERT_B200_OK;
    B200_REQUIRE(input && beta && gamma && out_i8 && row_scales, "skip_layer_norm_quantize: null pointer");
    uintptr_t const values = reinterpret_cast<uintptr_t>(input) | reinterpret_cast<uintptr_t>(skip) | reinterpret_cast<uintptr_t>(beta)
        | reinterpret_cast<uintptr_t>(gamma) | reinterpret_cast<uintptr_t>(output) | reinterpret_cast<uintptr_t>(bias);
    B200_REQUIRE(values % (type_id == BERT_B200_FP16 ? 2 : 4) == 0 && reinterpret_cast<uintptr_t>(row_scales) % 4 == 0,
        "skip_layer_norm_quantize: a pointer is not aligned to its type");
    auto s = static_cast<cudaStream_t>(stream);
    return type_id == BERT_B200_FP16 ? run<__half>(s, ld, n, input, skip, beta, gamma, output, out_i8, row_scales, bias, eps)
                                     : run<float>(s, ld, n, input, skip, beta, gamma, output, out_i8, row_scales, bias, eps);
}
