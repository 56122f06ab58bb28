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
    T const* in, T const* skip, T const* beta, T const* gamma, T const* bias,
    T* out, float const eps, int8_t* __restrict__ outI8, float* __restrict__ rowScales)
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
    // Where the INT8 rows go does not choose the kernel (y has to have the bits that skip_layer_norm gives): rows at an odd address go out byte by byte.
    bool const wholeStores = reinterpret_cast<uintptr_t>(outI8) % E == 0;
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
                int8_t* const to = outI8 + row * ld + c * E;
                if (!wholeStores)
                {
#pragma unroll
                    for (int j = 0; j < E; ++j)
                        to[j] = static_cast<int8_t>(w[j / 4] >> (8 * (j & 3)));
                }
                else if constexpr (E == 8)
                    stgStream8(to, make_uint2(w[0], w[1]));
                else
                    *reinterpret_cast<uint32_t*>(to) = w[0];
            }
        }
    }
}

// Rows that cannot be read 16 bytes at a time: WPR warps per row, each with NV neighbouring values per lane, 32 apart, in registers, so that the sums
// can be those of one warp that goes along the row (skip_ln.cu's scalar kernel, to the bit): each warp goes on where the one before it ended.
// The next row's 16-byte vectors are on their way to shared memory meanwhile, where single values are read from; the parameters are
// there for the whole launch. Some 35 instructions per value; up to 1024 values (a warp per row) issue slots bound it, beyond that the order of the sums:
// the row's warps add one after the other, twice, and most of them wait (3000 x 4001 FP16: 42 % of the slots used, 13 warps per SM; of a warp's 8 cycles
// per instruction 2.0 for loads, 1.5 at barriers). FP16 24576 x 1001 44.8 us (x 1024 34.0 us; 116 us with the kernel below), FP32 12000 x 1001 33.9 us (81 us), FP16
// 3000 x 4001 43 us (74 us), 2957 x 2543 32.7 us, 37 x 1001 4.5 us (11.4 us). Aligned FP32 rows of 4100 to 8192 values come here too, since skip_layer_norm sums
// them in this order, one CTA per SM by their shared memory: 1500 x 4100 56 us, 1500 x 8192 64 us (floor 24.7 us; skip_layer_norm 297 us).
template <typename T>
struct alignas(2 * sizeof(T)) GammaBeta
{
    T gamma, beta;
};

template <typename T>
__host__ __device__ constexpr int oddRowBytes(int slots) // of a row in shared memory, and what its lanes may read behind it
{
    return (slots * static_cast<int>(sizeof(T)) + 31) / 16 * 16;
}

template <typename T, int NV, int WPR, bool HAS_BIAS>
__global__ void __launch_bounds__(kThreads, NV <= 8 ? 4 : NV <= 16 ? 3 : 2) skipLnQuantOddKernel(int32_t const ld, int64_t const rows, T const* in, T const* skip,
    T const* beta, T const* gamma, T const* bias, T* out, float const eps, int8_t* __restrict__ outI8,
    float* __restrict__ rowScales)
{
    constexpr int kRowsPerCta = kWarpsPerCta / WPR;
    constexpr int kSlots = NV * WPR * 32;
    constexpr int kSure = WPR == 1 && NV > 8 ? NV - 8 : 0; // of a lane's values, those that every row handled here has
    constexpr int kRowBytes = oddRowBytes<T>(kSlots);
    extern __shared__ __align__(16) uint8_t oddSmem[];
    __shared__ float chain[kRowsPerCta][32];
    __shared__ float red[kRowsPerCta][2][WPR];
    GammaBeta<T>* const params = reinterpret_cast<GammaBeta<T>*>(oddSmem);
    T* const biases = reinterpret_cast<T*>(params + kSlots);
    int const lane = threadIdx.x & 31;
    int const warp = threadIdx.x >> 5;
    int const rowInCta = warp / WPR;
    int const wInRow = warp % WPR;
    uint8_t* const bufA = reinterpret_cast<uint8_t*>(biases + kSlots) + rowInCta * 2 * kRowBytes;
    uint8_t* const bufB = bufA + kRowBytes;
    int turn = 0;
    int const first = wInRow * NV * 32 + lane;
    float const rld = 1.f / static_cast<float>(ld);
    auto barrier = [&]() {
        if (WPR == 1)
            __syncwarp();
        else
            asm volatile("bar.sync %0, %1;" ::"r"(1 + rowInCta), "n"(WPR * 32) : "memory");
    };
    auto misOf = [&](T const* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15u); };
    // The vectors that hold the row; of those that reach beyond the matrix only the row's values.
    auto copy = [&](uint8_t* buf, T const* base, int64_t r) {
        T const* const p = base + r * ld;
        uint8_t const* const q = reinterpret_cast<uint8_t const*>(p) - misOf(p);
        int const n = (misOf(p) + ld * static_cast<int>(sizeof(T)) + 15) / 16;
        uint8_t const *const begin = reinterpret_cast<uint8_t const*>(base), *const end = reinterpret_cast<uint8_t const*>(base + rows * ld);
        for (int i = wInRow * 32 + lane; i < n; i += WPR * 32)
            if (q + 16 * i >= begin && q + 16 * i + 16 <= end)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(buf + 16 * i))), "l"(q + 16 * i)
                             : "memory");
            else
                for (int j = 0; j < 16; j += static_cast<int>(sizeof(T)))
                {
                    T const* const x = reinterpret_cast<T const*>(q + 16 * i + j);
                    if (x >= p && x < p + ld)
                        *reinterpret_cast<T*>(buf + 16 * i + j) = *x;
                }
    };
    // add(s): s and this lane's values, in order
    auto along = [&](auto const& add) {
        if (WPR == 1)
            return add(0.f);
#pragma unroll 1
        for (int w = 0; w < WPR; ++w)
        {
            if (w == wInRow)
                chain[rowInCta][lane] = add(w == 0 ? 0.f : chain[rowInCta][lane]);
            barrier();
        }
        return chain[rowInCta][lane];
    };
    auto most = [](float x, float y) { return maxNan(x, y); };

    gridDependencyLaunch();
    gridDependencyWait();
    int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsPerCta + rowInCta;
    int64_t const step = static_cast<int64_t>(gridDim.x) * kRowsPerCta;
    if (row < rows)
    {
        copy(bufA, in, row);
        if (skip)
            copy(bufB, skip, row);
    }
    for (int i = threadIdx.x; i < kSlots; i += kThreads)
    {
        bool const ok = i < ld;
        T const zero = static_cast<T>(0.f);
        params[i] = GammaBeta<T>{ok ? gamma[i] : zero, ok ? beta[i] : zero};
        if (HAS_BIAS)
            biases[i] = ok ? bias[i] : zero;
    }
    __syncthreads();
    for (; row < rows; row += step)
    {
        asm volatile("cp.async.wait_all;" ::: "memory");
        barrier();
        T const* const a = reinterpret_cast<T const*>(bufA + misOf(in + row * ld)) + first;
        T const* const b = skip ? reinterpret_cast<T const*>(bufB + misOf(skip + row * ld)) + first : nullptr;
        // f(j, whether the row has this lane's value j); of several warps all but the last have all of theirs
        auto each = [&](auto const& f) {
            if (WPR > 1 && (wInRow + 1) * NV * 32 <= ld)
            {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    f(j, true);
            }
            else
            {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    f(j, j < kSure || first + 32 * j < ld);
            }
        };
        float x[NV / 8][8];
        each([&](int j, bool ok) { x[j / 8][j % 8] = ok ? static_cast<float>(a[32 * j]) : 0.f; });
        if (b)
            each([&](int j, bool ok) { x[j / 8][j % 8] += ok ? static_cast<float>(b[32 * j]) : 0.f; });
        if (HAS_BIAS)
#pragma unroll
            for (int j = 0; j < NV; ++j)
                x[j / 8][j % 8] += static_cast<float>(biases[first + 32 * j]);
        barrier(); // the row's buffers are read, `chain` as well
        if (row + step < rows)
        {
            copy(bufA, in, row + step);
            if (skip)
                copy(bufB, skip, row + step);
        }
        float const mu = __fmul_rn(warpSum(along([&](float s) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                s += x[j / 8][j % 8];
            return s;
        })), rld);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            x[j / 8][j % 8] -= mu;
        if (WPR > 1)
            barrier(); // `chain` has been read
        float const rsigma = rsqrtf(warpSum(along([&](float q) {
            each([&](int j, bool ok) {
                if (ok)
                    q = fmaf(x[j / 8][j % 8], x[j / 8][j % 8], q);
            });
            return q;
        })) * rld + eps);
        float largest = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
        {
            GammaBeta<T> const p = params[first + 32 * j]; // zeros behind the row: 0, or NaN where the row's own are
            x[j / 8][j % 8] = fmaf(static_cast<float>(p.gamma) * x[j / 8][j % 8], rsigma, static_cast<float>(p.beta));
            largest = maxNan(largest, fabsf(x[j / 8][j % 8]));
        }
        if (out)
        {
            T* const y = out + row * ld + first;
            each([&](int j, bool ok) {
                if (ok)
                    y[32 * j] = static_cast<T>(x[j / 8][j % 8]);
            });
        }
        largest = overWarps<WPR>(warpMaxNan(largest), red[rowInCta], rowInCta, wInRow, lane, turn, most);
        RowScale const scale = makeRowScale(largest);
        if (wInRow == 0 && lane == 0)
            rowScales[row] = rowScaleValue(largest);
        uint32_t w[NV / 8][2];
#pragma unroll
        for (int c = 0; c < NV / 8; ++c)
            quantRowChunk<8, true>(x[c], scale, w[c]);
        int8_t* const q = outI8 + row * ld + first;
        each([&](int j, bool ok) {
            if (ok)
                q[32 * j] = static_cast<int8_t>(w[j / 8][j / 4 & 1] >> (8 * (j & 3)));
        });
    }
}

// Longer rows, scalar accesses, one warp per row; the row is revisited from L1 / L2 instead of registers. 1500 x 12288 FP16 274 us, FP32 391 us (skip_layer_norm,
// in the same order, 228 us FP16).
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

template <typename T, int NV, int WPR>
int32_t launchOdd(cudaStream_t s, Args<T> const& p)
{
    static SmemOptIn optIn[2];
    constexpr int kSlots = 32 * NV * WPR, kRowsPerCta = kWarpsPerCta / WPR;
    constexpr int kSmem = kSlots * 3 * static_cast<int>(sizeof(T)) + kRowsPerCta * 2 * oddRowBytes<T>(kSlots);
    constexpr int kCtas = kSmem > 110 * 1024 ? 1 : kSmem > 73 * 1024 || NV > 16 ? 2 : NV > 8 ? 3 : 4;
    cudaError_t const e = launchDependentCluster(&optIn[p.bias ? 1 : 0],
        p.bias ? skipLnQuantOddKernel<T, NV, WPR, true> : skipLnQuantOddKernel<T, NV, WPR, false>,
        dim3(gridFor((p.rows + kRowsPerCta - 1) / kRowsPerCta, kCtas)), dim3(kThreads), kSmem, s, 1, p.ld, p.rows, p.in, p.skip, p.beta, p.gamma, p.bias,
        p.out, p.eps, p.outI8, p.rowScales);
    if (e != cudaSuccess)
        B200_FAIL(BERT_B200_CUDA_ERROR, "skipLnQuantOddKernel: %s", cudaGetErrorString(e));
    return checkLaunch("skipLnQuantOddKernel");
}

template <typename T>
int32_t dispatch(cudaStream_t s, Args<T> const& p)
{
    constexpr int E = 16 / sizeof(T);
    bool const vec = p.ld % E == 0 && p.ld / E <= 32 * 4 * 8 && aligned16(p.in) && aligned16(p.skip) && aligned16(p.out) && aligned16(p.beta)
        && aligned16(p.gamma) && aligned16(p.bias); // the conditions of dispatchSkipLn (skip_ln.cu)
    if (!vec && p.ld <= 32 * 32 * 8)
    {
        // as few warps as hold the row, 32 values per lane at most
#define B200_ODD_CASE(NV, W)                                                                                           \
    if (p.ld <= 32 * NV * W)                                                                                           \
        return launchOdd<T, NV, W>(s, p);
        B200_ODD_CASE(8, 1)
        B200_ODD_CASE(16, 1)
        B200_ODD_CASE(24, 1)
        B200_ODD_CASE(32, 1)
        B200_ODD_CASE(32, 2)
        B200_ODD_CASE(32, 4)
        B200_ODD_CASE(32, 8)
#undef B200_ODD_CASE
    }
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
