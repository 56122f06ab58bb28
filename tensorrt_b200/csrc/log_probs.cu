// Log probabilities of given tokens, entropy and the most likely tokens of each row of logits, in one pass over the logits.
//
// With M the row's maximum, c how often it occurs, s = sum of exp(x - M) over the other values and t = sum of (x - M) exp(x - M):
//   log p(x) = (x - M) - L,   L = ln c + ln1p(s / c),   entropy = L - t / (c + s).
// The maxima are kept out of s so that a row that is sure of a token keeps the digits of 1 - p: L is then as precise as s.
// No counterpart in the reference (its plugins end at the encoder's output).
//
// A CTA takes a row (a part of it, where it is long) into shared memory by asynchronous copies, every thread the 16-byte vectors that it
// will read itself, so the maximum is known before the first exponential and nothing is read twice; the next part's copies are on their
// way as soon as a thread has read its vectors for the last time. W warps do that; one more puts the results together (it keeps the likely
// tokens, a lane each, and writes what is asked for) while they are at the next part, from one of two hand-over places.
// The k most likely tokens: the k-th largest of 32 or 64 groups' maxima is a lower bound of the k-th largest value, so only what is at least that
// (a few more than k) is handed over. Where that is more than the list holds (hundreds of equal values) the last warp reads the part again.
// Short rows: one warp each, the same steps one after the other.
// Few rows may be shared by a cluster of CTAs each: their last warps hand what they found to the first CTA's through distributed shared memory. Such
// a cluster has one row only (clusterFor), so no place there is used twice.
//
// Of some 10000 warp instructions of a row of 30522 halves, 4000 are exponentials (34 per eight values: conversion, one multiply-add, ex2, two sums,
// clamp), 700 the maximum, 900 copies, the rest per row and warp. 0.63 of the issue slots are used with 24 warps per SM; a warp's other cycles go to
// dependent instructions, the CTA's barriers and shared memory. 3686 x 30522 FP16, top 10: 54.9 us, 4.1 TB/s (floor 34.9 us; 146 us with rows in registers, 102 us with
// everything in turn); FP32 888 rows without likely tokens 23.7 us, 4.6 TB/s. One row 5.7 us. Short rows: 0.64 of the slots (20000 x 2000 FP16, top 10, 51 us, floor
// 12.5 us), every step of a row behind the one before it in the same warp.
// Slow, though right: parts whose list overflows. Those are parts with fewer than topK values above one that hundreds share (masks of the type's lowest value,
// equal logits: 30522 values, top 5, one FP16 row with three tokens left 47 us instead of 6, 400 FP32 rows whose second half, a part, is masked 53 us instead of 14, 3686
// FP16 rows of equal values 530 us instead of 53; without likely tokens such values are only counted: 31 us instead of 13 for those 400 rows), and, for 17 to 20 tokens,
// up to 444 rows of 65 to 76 vectors, which leave some of the 32 pairs of groups empty (FP16 505 ... 608, FP32 256 ... 304 values: 12 ... 33 us instead of 4 ... 7).
#include "sm100.cuh"

namespace b200
{
namespace
{

constexpr int kMaxTop = 32;

struct LogProbsArgs
{
    int64_t rows;
    int32_t vocab;
    void const* logits;
    int64_t stride;
    int32_t numTokens;
    int32_t const* tokenIds;
    int32_t topK;
    float* logProbs;
    float* entropy;
    int32_t* topIds;
    float* topLogProbs;
    uint32_t* statusWord;
};

__device__ __forceinline__ float negInf()
{
    return __int_as_float(0xff800000);
}

__device__ __forceinline__ float exp2Approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whole numbers in the order of the values (-0 equals 0), and back.
__device__ __forceinline__ uint32_t orderOf(float x)
{
    int32_t const b = __float_as_int(x + 0.f);
    return static_cast<uint32_t>(b ^ ((b >> 31) & 0x7fffffff)) ^ 0x80000000u;
}
__device__ __forceinline__ float valueOf(uint32_t order)
{
    int32_t const o = static_cast<int32_t>(order ^ 0x80000000u);
    return __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
}
constexpr uint32_t kOrderNegInf = 0x007fffffu;

// Larger values first, of equal ones the lower id; never 0.
__device__ __forceinline__ uint64_t makeKey(float x, int32_t id)
{
    return static_cast<uint64_t>(orderOf(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ int32_t keyId(uint64_t k)
{
    return static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k));
}
__device__ __forceinline__ float keyValue(uint64_t k)
{
    return valueOf(static_cast<uint32_t>(k >> 32));
}

template <typename T>
struct Vec;
template <>
struct Vec<__half>
{
    static constexpr int kElems = 8;
    static __device__ __forceinline__ void unpack(uint4 const& v, float (&f)[8])
    {
        unpackHalf8(v, f);
    }
    // values below `floor` become it
    static __device__ __forceinline__ void unpackAbove(uint4 const& v, float floor, float (&f)[8])
    {
        __half2 const* h = reinterpret_cast<__half2 const*>(&v);
        __half2 const lo = __float2half2_rn(floor);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            float2 const t = __half22float2(__hmax2(h[i], lo));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
    static __device__ __forceinline__ float most(uint4 const& v)
    {
        __half2 const* h = reinterpret_cast<__half2 const*>(&v);
        __half2 const m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return maxNan(__low2float(m), __high2float(m));
    }
    // the maximum of many vectors
    struct Most
    {
        __half2 a = __half2half2(__ushort_as_half(0xfc00)), b = a;
        __device__ __forceinline__ void add(uint4 const& v)
        {
            __half2 const* h = reinterpret_cast<__half2 const*>(&v);
            a = __hmax2_nan(a, __hmax2_nan(h[0], h[1]));
            b = __hmax2_nan(b, __hmax2_nan(h[2], h[3]));
        }
        __device__ __forceinline__ float get() const
        {
            __half2 const m = __hmax2_nan(a, b);
            return maxNan(__low2float(m), __high2float(m));
        }
        __device__ __forceinline__ float getA() const // of one half of the values
        {
            return maxNan(__low2float(a), __high2float(a));
        }
        __device__ __forceinline__ float getB() const // of the other
        {
            return maxNan(__low2float(b), __high2float(b));
        }
    };
};
template <>
struct Vec<float>
{
    static constexpr int kElems = 4;
    static __device__ __forceinline__ void unpack(uint4 const& v, float (&f)[4])
    {
        f[0] = __uint_as_float(v.x);
        f[1] = __uint_as_float(v.y);
        f[2] = __uint_as_float(v.z);
        f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ void unpackAbove(uint4 const& v, float floor, float (&f)[4])
    {
        unpack(v, f);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            f[i] = fmaxf(f[i], floor);
    }
    static __device__ __forceinline__ float most(uint4 const& v)
    {
        return maxNan(maxNan(__uint_as_float(v.x), __uint_as_float(v.y)), maxNan(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    struct Most
    {
        float a = negInf(), b = negInf();
        __device__ __forceinline__ void add(uint4 const& v)
        {
            a = maxNan(a, maxNan(__uint_as_float(v.x), __uint_as_float(v.y)));
            b = maxNan(b, maxNan(__uint_as_float(v.z), __uint_as_float(v.w)));
        }
        __device__ __forceinline__ float get() const
        {
            return maxNan(a, b);
        }
        __device__ __forceinline__ float getA() const
        {
            return a;
        }
        __device__ __forceinline__ float getB() const
        {
            return b;
        }
    };
};

// Maximum, how often it occurs, sum and weighted sum of the others (see above). count == 0: nothing yet.
struct alignas(16) Stat
{
    float m, count, s, t;
};

__device__ __forceinline__ Stat merge(Stat const& a, Stat const& b)
{
    if (a.count == 0.f)
        return b;
    if (b.count == 0.f)
        return a;
    if (a.m == b.m)
        return Stat{a.m, a.count + b.count, a.s + b.s, a.t + b.t};
    Stat const& hi = a.m > b.m ? a : b;
    Stat const& lo = a.m > b.m ? b : a;
    float const d = fmaxf(lo.m - hi.m, -200.f); // exp(-200) is 0 in FP32
    float const w = expf(d), n = lo.s + lo.count;
    return Stat{hi.m, hi.count, fmaf(w, n, hi.s), fmaf(w, fmaf(d, n, lo.t), hi.t)};
}

// What the warps that read a part hand over.
template <int W>
struct Place
{
    static constexpr int kCap = W == 1 ? 128 : 256;
    uint64_t cand[kCap];
    float2 sums[W * 32]; // of each thread
    float m;            // the part's maximum; -infinity: nothing in it, NaN or +infinity: the row has no distribution
    int32_t ties;       // how often it occurs
    int32_t listed;     // candidates, also those beyond kCap
};

__device__ __forceinline__ void copyAsync16(uint4* dst, void const* src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copyAsync16(uint4* dst, void const* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))), "l"(src) : "memory");
}

// A row as 16-byte vectors: `p` its first value, `mis` values behind a 16-byte boundary, nVec vectors that hold some of its values.
template <typename T>
struct Row
{
    static constexpr int E = Vec<T>::kElems;
    T const* p;
    int mis, nVec;
    bool firstRow, lastRow;

    __device__ __forceinline__ Row(LogProbsArgs const& args, int64_t row)
        : p(static_cast<T const*>(args.logits) + row * args.stride)
        , mis(static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T)))
        , nVec((args.vocab + mis + E - 1) / E)
        , firstRow(row < E) // (a stride of one value is the least there is)
        , lastRow(args.rows - 1 - row < E)
    {
    }

    // The vectors [begin, end) of `n` from `first` on that can be copied as they are: whole vectors, with which values of the rows beside this
    // one may come along; where there may be none, at the ends of the matrix, the row's first and last vector by copyEdge.
    __device__ __forceinline__ int begin(int first) const
    {
        return firstRow && first == 0 ? 1 : 0;
    }
    __device__ __forceinline__ int end(int first, int n) const
    {
        return lastRow && first + n == nVec ? n - 1 : n;
    }
    __device__ __forceinline__ bool edge(int vec) const
    {
        return vec == 0 || vec == nVec - 1;
    }
    __device__ __forceinline__ T const* at(int first) const
    {
        return p - mis + static_cast<int64_t>(first) * E;
    }

    // Starts the copies of this thread's share of `n` vectors from `first` on, from its vector `i` on.
    template <int kThreads>
    __device__ __forceinline__ void copy(uint4* buf, int first, int n, int i, int tid, LogProbsArgs const& args) const
    {
        if (n == 0)
            return;
        T const* const q = at(first);
        int const lo = begin(first), hi = end(first, n);
#pragma unroll 4
        for (; i < hi; i += kThreads)
            if (i >= lo)
                copyAsync16(buf + i, q + static_cast<int64_t>(i) * E);
        if (tid == 0 && lo > 0 && hi > 0)
            copyEdge(buf, 0, args);
        if (hi < n && hi % kThreads == tid)
            copyEdge(buf + hi, nVec - 1, args);
    }

    // A vector that holds values of the row only in part, and beside them perhaps nothing that may be read.
    __device__ __forceinline__ void copyEdge(uint4* dst, int vec, LogProbsArgs const& args) const
    {
        int32_t const e0 = vec * E - mis;
        int const left = args.vocab - e0;
        if (e0 >= 0)
            copyAsync16(dst, p + e0, left < E ? left * static_cast<int>(sizeof(T)) : 16);
        else
            for (int j = 0; j < E; ++j)
                if (e0 + j >= 0 && j < left)
                    reinterpret_cast<T*>(dst)[j] = ldGlobal(p + e0 + j);
    }

    // What of the copied vector is not the row's becomes -infinity.
    __device__ __forceinline__ void trim(uint4* dst, int vec, int32_t vocab) const
    {
        int32_t const e0 = vec * E - mis;
        if (e0 < 0 || e0 + E > vocab)
            for (int j = 0; j < E; ++j)
                if (e0 + j < 0 || e0 + j >= vocab)
                    reinterpret_cast<T*>(dst)[j] = static_cast<T>(negInf());
    }
};

constexpr float kLog2e = 1.4426950408889634f;

// Sums over a thread's values of exp(x - m) and (x - m) exp(x - m), two of each.
struct Sums
{
    uint64_t s = pack2(0.f, 0.f), t = pack2(0.f, 0.f);
};

// For any m.
template <typename T>
__device__ __forceinline__ void addExponentials(uint4 const& v, float m, Sums& sums)
{
    constexpr int E = Vec<T>::kElems;
    float f[E];
    Vec<T>::unpack(v, f);
#pragma unroll
    for (int j = 0; j < E; j += 2)
    {
        float const a = fmaxf(f[j] - m, -200.f), b = fmaxf(f[j + 1] - m, -200.f); // masked values: 0 times a finite number
        uint64_t const e = pack2(exp2Approx(a * kLog2e), exp2Approx(b * kLog2e));
        sums.s = add2(sums.s, e);
        sums.t = fma2(e, pack2(a, b), sums.t);
    }
}

// For m of moderate size: sums of 2^u and u 2^u with u = x log2(e) - c, c = m log2(e) as rounded. u is
// rounded once, whatever m; how far c is from m log2(e), the same for all values, is put right in `finish`.
// Moderate: m - 100, rounded to FP16, stays more than 88 below m.
constexpr float kModerate = 4096.f;
template <typename T>
__device__ __forceinline__ void addPowers(uint4 const& v, float floor, uint64_t minusC, Sums& sums)
{
    constexpr int E = Vec<T>::kElems;
    uint64_t const log2e = pack2(kLog2e, kLog2e);
    float f[E];
    Vec<T>::unpackAbove(v, floor, f); // masked values: 0 times a finite number
#pragma unroll
    for (int j = 0; j < E; j += 2)
    {
        uint64_t const u = fma2(pack2(f[j], f[j + 1]), log2e, minusC);
        float a, b;
        unpack2(u, a, b);
        uint64_t const e = pack2(exp2Approx(a), exp2Approx(b));
        sums.s = add2(sums.s, e);
        sums.t = fma2(e, u, sums.t);
    }
}

// Barriers of the CTA: among the reading warps, and the two hand-over places' full and free ones (reading warps and the last one).
enum
{
    kBarRead = 1,
    kBarFull = 2,
    kBarFree = 4
};
template <int kThreads>
__device__ __forceinline__ void barSync(int id)
{
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
}
template <int kThreads>
__device__ __forceinline__ void barArrive(int id)
{
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
}

// Reads the part that lies in `buf` (n vectors, vector `first` of the row first) and leaves what it found in `place`. `claim` waits until the
// place is free; afterwards its counters are 0. `next` starts the copy that takes the place of a vector which has been read for the last time.
template <typename T, int W, typename F, typename G>
__device__ __forceinline__ void readPart(Place<W>& place, float* groupMax, float* threshold, uint4* buf, Row<T> const& row, int32_t vocab, int first, int n,
    int topK, int tid, F const& claim, G const& next)
{
    constexpr int kThreads = W * 32;
    constexpr int E = Vec<T>::kElems;
    int const lane = tid & 31, warp = tid >> 5;
    auto sync = [&]() {
        if (W == 1)
            __syncwarp();
        else
            barSync<kThreads>(kBarRead);
    };
    if (first == 0 && tid == 0)
        row.trim(buf, 0, vocab);
    if (first + n == row.nVec && (n - 1) % kThreads == tid)
        row.trim(buf + n - 1, row.nVec - 1, vocab);

    typename Vec<T>::Most most;
#pragma unroll 4
    for (int i = tid; i < n; i += kThreads)
        most.add(buf[i]);
    float const mine = most.get();
    // W > 1: the maxima of 64 groups of threads, two per lane
    float gm = mine, gm2 = negInf();
    if constexpr (W > 1)
    {
        constexpr int kGroup = kThreads / 64;
#pragma unroll
        for (int o = 1; o < kGroup; o *= 2)
            gm = maxNan(gm, __shfl_xor_sync(0xffffffffu, gm, o));
        if (lane % kGroup == 0)
            groupMax[tid / kGroup] = gm;
        claim();
        sync();
        gm = groupMax[lane];
        gm2 = groupMax[lane + 32];
    }
    float const m = warpMaxNan(maxNan(gm, gm2));
    bool const some = m < __int_as_float(0x7f800000) && m != negInf();
    if (tid == 0)
        place.m = m;
    float thr = m;
    if (some && topK > 0)
    {
        if constexpr (W == 1)
        {
            if (topK <= 12)
            {
                // the largest of the lanes' maxima is taken out topK - 1 times
                float rest = gm;
                for (int j = 1; j < topK; ++j)
                    if (__ffs(__ballot_sync(0xffffffffu, rest == warpMaxNan(rest))) - 1 == lane)
                        rest = negInf();
                thr = warpMaxNan(rest);
            }
            else
            {
                // The maxima of two halves of each lane's values, the topK-th of the 64 to 16 binary places: of 32 maxima the last would leave more
                // than the list holds (20000 x 2000 FP16, top 32: 442 -> 71 us; 7079 x 231 FP32 48 -> 13.5 us).
                uint32_t const a = orderOf(most.getA()), b = orderOf(most.getB());
                uint32_t at = 0;
                for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
                    if (__popc(__ballot_sync(0xffffffffu, a >= (at | bit))) + __popc(__ballot_sync(0xffffffffu, b >= (at | bit))) >= topK)
                        at |= bit;
                thr = valueOf(at > kOrderNegInf ? at : kOrderNegInf);
            }
        }
        else
        {
            // The groups' maxima in order, each warp places its share of them: 32 pairs of groups for few tokens (12 values are at least the
            // 10th of 32 maxima, 31 the 20th), all 64 for more (32: 44 values, with 32 maxima 110).
            if (topK <= 20)
            {
                gm = fmaxf(gm, gm2);
#pragma unroll
                for (int j = 0; j < 32 / W; ++j)
                {
                    int const at = warp * (32 / W) + j;
                    float const x = __shfl_sync(0xffffffffu, gm, at);
                    int const rank = __popc(__ballot_sync(0xffffffffu, gm > x || (gm == x && lane < at)));
                    if (rank == topK - 1 && lane == 0)
                        *threshold = x;
                }
            }
            else
            {
#pragma unroll
                for (int j = 0; j < 64 / W; ++j)
                {
                    int const at = warp * (64 / W) + j;
                    float const x = groupMax[at];
                    int const rank = __popc(__ballot_sync(0xffffffffu, gm > x || (gm == x && lane < at)))
                        + __popc(__ballot_sync(0xffffffffu, gm2 > x || (gm2 == x && lane + 32 < at)));
                    if (rank == topK - 1 && lane == 0)
                        *threshold = x;
                }
            }
        }
    }
    sync();
    if (some)
    {
        if (W > 1 && topK > 0)
            thr = *threshold;
        // Candidates are listed; the part's maxima are counted and no longer among the others.
        int ties = 0;
        auto look = [&](int i) {
            if (Vec<T>::most(buf[i]) < thr)
                return;
            T* const e = reinterpret_cast<T*>(buf + i);
            bool const list = topK > 0 && *static_cast<int32_t volatile*>(&place.listed) <= Place<W>::kCap; // beyond, only that it is so counts
            for (int j = 0; j < E; ++j)
            {
                float const x = static_cast<float>(e[j]);
                if (x >= thr && x != negInf())
                {
                    if (list)
                    {
                        int const slot = atomicAdd(&place.listed, 1);
                        if (slot < Place<W>::kCap)
                            place.cand[slot] = makeKey(x, (first + i) * E - row.mis + j);
                    }
                    if (x == m)
                    {
                        e[j] = static_cast<T>(negInf());
                        ++ties;
                    }
                }
            }
        };
        uint32_t hits = __ballot_sync(0xffffffffu, mine >= thr && mine != negInf()); // the threads that have such values
        // Short rows, of which many threads have some: every thread its own vectors.
        if (W == 1 && 2 * ((n + kThreads - 1) / kThreads) < __popc(hits))
            for (int i = tid; i < n; i += kThreads)
                look(i);
        else // the warp looks through two threads' vectors at a time, 16 lanes and one vector per lane for each (a part has at most 16 per thread)
            while (hits != 0)
            {
                uint32_t const rest = hits & (hits - 1); // without the first
                uint32_t const own = (lane & 16) ? rest : hits;
                hits = rest & (rest - 1);
                int const i = warp * 32 + __ffs(own) - 1 + (lane & 15) * kThreads;
                if (own != 0 && i < n)
                    look(i);
                if (W == 1 && own != 0 && i + 16 * kThreads < n)
                    look(i + 16 * kThreads);
            }
        if (ties > 0)
            atomicAdd(&place.ties, ties);
        __syncwarp();
    }
    Sums sums;
    float a, b, s, t;
    if (fabsf(m) < kModerate)
    {
        float const c = m * kLog2e;
        uint64_t const minusC = pack2(-c, -c);
        float const floor = m - 100.f; // exp(-100) is below what FP32 holds in normal numbers
#pragma unroll 4
        for (int i = tid; i < n; i += kThreads)
        {
            addPowers<T>(buf[i], floor, minusC, sums);
            next(i);
        }
        unpack2(sums.s, a, b);
        s = a + b;
        unpack2(sums.t, a, b);
        t = a + b;
        float const off = fmaf(m, kLog2e, -c), w = exp2Approx(-off); // u of m itself
        t = fmaf(-off, s, t) * (w * 0.69314718055994531f);
        s *= w;
    }
    else
    {
        for (int i = tid; i < n; i += kThreads)
        {
            if (some)
                addExponentials<T>(buf[i], m, sums);
            next(i);
        }
        unpack2(sums.s, a, b);
        s = a + b;
        unpack2(sums.t, a, b);
        t = a + b;
    }
    place.sums[tid] = make_float2(s, t);
}

// A row's results as one warp collects them.
struct Result
{
    Stat stat{negInf(), 0.f, 0.f, 0.f};
    uint64_t key = 0; // of this lane's place among the likely tokens, 0: none
    bool bad = false; // a NaN or +infinity has been seen

    // One key per lane (0: none; none that is there already) to the likely tokens.
    __device__ __forceinline__ void insert(uint64_t k, int topK, int lane)
    {
        uint32_t todo = __ballot_sync(0xffffffffu, k > __shfl_sync(0xffffffffu, key, topK - 1));
        if (__popc(todo) > 8)
        {
            // Sorted among each other, then the better of the i-th best here and the i-th worst there: twenty exchanges instead of a chain of
            // shuffles for each key (32 keys 1.9 us). The first keys need no second half, 16 of them ten exchanges.
#pragma unroll
            for (int size = 2; size <= 16; size *= 2)
                sortStep(k, size, lane);
            bool const first = __shfl_sync(0xffffffffu, key, 0) == 0;
            if (!first || __any_sync(0xffffffffu, lane >= 16 && k != 0))
                sortStep(k, 32, lane);
            if (first)
            {
                key = k;
                return;
            }
            uint64_t const other = __shfl_sync(0xffffffffu, k, 31 - lane);
            key = other > key ? other : key;
#pragma unroll
            for (int o = 16; o > 0; o /= 2)
                key = exchange(key, o, (lane & o) == 0);
            return;
        }
        for (; todo != 0; todo &= todo - 1)
        {
            uint64_t const x = __shfl_sync(0xffffffffu, k, __ffs(todo) - 1);
            int const at = __popc(__ballot_sync(0xffffffffu, key > x));
            uint64_t const before = __shfl_up_sync(0xffffffffu, key, 1);
            key = lane < at ? key : lane == at ? x : before;
        }
    }

    // Runs of `size` keys, each of which rises and falls, become sorted: largest first in every other one, and in the last step.
    static __device__ __forceinline__ void sortStep(uint64_t& k, int size, int lane)
    {
#pragma unroll
        for (int o = size / 2; o > 0; o /= 2)
            k = exchange(k, o, ((lane & o) == 0) == ((lane & size) == 0 || size == 32));
    }

    // The larger or the smaller of this lane's and that of the lane `o` away.
    static __device__ __forceinline__ uint64_t exchange(uint64_t k, int o, bool larger)
    {
        uint64_t const x = __shfl_xor_sync(0xffffffffu, k, o);
        return (k > x) == larger ? k : x;
    }

    // The key, or 0 if it is among the likely tokens already. All lanes call it.
    __device__ __forceinline__ uint64_t unlessThere(uint64_t k, int topK) const
    {
        for (int i = 0; i < topK; ++i)
            if (__shfl_sync(0xffffffffu, key, i) == k)
                k = 0;
        return k;
    }
};

// Adds what is in `place` to the result and empties the place.
template <typename T, int W>
__device__ __forceinline__ void takePlace(Result& res, Place<W>& place, Row<T> const& row, int32_t vocab, int first, int n, int topK, int lane)
{
    constexpr int E = Vec<T>::kElems;
    float const m = place.m;
    if (!(m < __int_as_float(0x7f800000)))
        res.bad = true;
    else if (m != negInf())
    {
        float s = 0.f, t = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w)
        {
            float2 const x = place.sums[w * 32 + lane];
            s += x.x;
            t += x.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
        {
            s += __shfl_xor_sync(0xffffffffu, s, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
        }
        res.stat = merge(res.stat, Stat{m, static_cast<float>(place.ties), s, t});
        int const listed = topK > 0 ? place.listed : 0;
        for (int i = 0; i < listed && i < Place<W>::kCap; i += 32)
            res.insert(i + lane < listed && i + lane < Place<W>::kCap ? place.cand[i + lane] : 0ull, topK, lane);
        if (listed > Place<W>::kCap)
        {
            // Not all were listed: the part is read again for what is above the last of those found so far, four vectors per lane at a time;
            // where one of 32 has such values (or may hold values that are not the row's) all of theirs are looked at.
            T const* const q = row.at(first);
            for (int i = lane; i - lane < n; i += 4 * 32)
            {
                uint4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (i + 32 * j < n && !row.edge(first + i + 32 * j))
                        v[j] = ldgStream(q + static_cast<int64_t>(i + 32 * j) * E);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    uint64_t const last = __shfl_sync(0xffffffffu, res.key, topK - 1);
                    int32_t const id = (first + i + 32 * j) * E - row.mis;
                    bool look = i + 32 * j < n;
                    if (look && last != 0ull && !row.edge(first + i + 32 * j))
                    {
                        float const most = Vec<T>::most(v[j]);
                        look = most > keyValue(last) || (most == keyValue(last) && id < keyId(last));
                    }
                    if (__any_sync(0xffffffffu, look))
                        for (int e = 0; e < E; ++e)
                        {
                            float const x = look && id + e >= 0 && id + e < vocab ? static_cast<float>(ldGlobal(row.p + id + e)) : negInf();
                            res.insert(res.unlessThere(x == negInf() ? 0ull : makeKey(x, id + e), topK), topK, lane);
                        }
                }
            }
        }
    }
    __syncwarp();
    if (lane == 0)
        place.ties = place.listed = 0;
}

// Writes a row's answers. `tokenLogit`: that of token `lane` of the first 32.
template <typename T>
__device__ __forceinline__ void writeRow(LogProbsArgs const& args, Result const& res, Row<T> const& row, int64_t r, float tokenLogit, int lane)
{
    Stat const& st = res.stat;
    bool const bad = res.bad;
    bool const none = !bad && st.count == 0.f;
    float const nan = __int_as_float(0x7fffffff);
    float const lse = none ? 0.f : logf(st.count) + log1pf(st.s / st.count);
    auto logProb = [&](float x) {
        return bad ? nan : none ? negInf() : (x - st.m) - lse;
    };
    if (lane < args.numTokens)
        args.logProbs[r * args.numTokens + lane] = logProb(tokenLogit);
    if (args.numTokens > 32)
    {
        // four of a lane at a time, the next four on their way with these ones' logits: 30522 tokens of a row 74 us, one by one 350 us
        constexpr int kAtOnce = 4;
        auto loadTokens = [&](int j0, int32_t (&token)[kAtOnce]) {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                token[i] = j0 + 32 * i < args.numTokens ? ldGlobal(args.tokenIds + r * args.numTokens + j0 + 32 * i) : -1;
        };
        int32_t token[kAtOnce];
        loadTokens(lane + 32, token);
        for (int j0 = lane + 32; j0 < args.numTokens; j0 += kAtOnce * 32)
        {
            float x[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                x[i] = token[i] >= 0 && token[i] < args.vocab ? static_cast<float>(ldGlobal(row.p + token[i])) : negInf();
            loadTokens(j0 + kAtOnce * 32, token);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (j0 + 32 * i < args.numTokens)
                    args.logProbs[r * args.numTokens + j0 + 32 * i] = logProb(x[i]);
        }
    }
    if (lane == 0 && args.entropy)
        args.entropy[r] = bad ? nan : none ? 0.f : lse - st.t / (st.count + st.s);
    if (lane < args.topK)
    {
        bool const have = !bad && res.key != 0;
        args.topIds[r * args.topK + lane] = have ? keyId(res.key) : -1;
        args.topLogProbs[r * args.topK + lane] = have ? logProb(keyValue(res.key)) : bad ? nan : negInf();
    }
}

// The logit of token `lane` of the first 32 asked for.
template <typename T>
__device__ __forceinline__ float loadToken(LogProbsArgs const& args, Row<T> const& row, int64_t r, int lane)
{
    if (lane < args.numTokens)
    {
        int32_t const token = ldGlobal(args.tokenIds + r * args.numTokens + lane);
        if (token >= 0 && token < args.vocab)
            return static_cast<float>(ldGlobal(row.p + token));
    }
    return negInf();
}

__device__ __forceinline__ void copiesWait()
{
    asm volatile("cp.async.wait_all;" ::: "memory"); // every thread reads its own copies (or, behind a warp's barrier, its warp's)
}

// Short rows: a warp each, kGroups of them per CTA. `partVecs`: vectors of a row, at most.
template <typename T, int kGroups>
__global__ void __launch_bounds__(32 * kGroups) logProbsWarpKernel(LogProbsArgs const args, int const partVecs)
{
    __shared__ Place<1> places[kGroups];
    extern __shared__ __align__(16) uint4 buffers[];
    int const lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    Place<1>& place = places[group];
    uint4* const buf = buffers + group * partVecs;
    int64_t const rowStep = static_cast<int64_t>(gridDim.x) * kGroups;
    if (lane == 0)
        place.ties = place.listed = 0;
    gridDependencyLaunch();
    gridDependencyWait();
    int64_t r = static_cast<int64_t>(blockIdx.x) * kGroups + group;
    if (r < args.rows)
    {
        Row<T> const row(args, r);
        row.template copy<32>(buf, 0, row.nVec, lane, lane, args);
    }
    for (; r < args.rows; r += rowStep)
    {
        Row<T> const row(args, r);
        float const tokenLogit = loadToken(args, row, r, lane);
        copiesWait();
        Result res;
        readPart<T, 1>(place, nullptr, nullptr, buf, row, args.vocab, 0, row.nVec, args.topK, lane, []() {}, [](int) {});
        if (r + rowStep < args.rows)
        {
            Row<T> const next(args, r + rowStep);
            next.template copy<32>(buf, 0, next.nVec, lane, lane, args);
        }
        __syncwarp();
        takePlace<T, 1>(res, place, row, args.vocab, 0, row.nVec, args.topK, lane);
        writeRow(args, res, row, r, tokenLogit, lane);
    }
}

// What the last warp of a cluster's other CTA hands to that of the first.
struct Joined
{
    Stat stat;
    uint64_t key[kMaxTop];
    uint32_t bad;
};

constexpr int kReadingWarps = 8;
constexpr int kCtasPerSm = 3;
constexpr int kPartVecs = 4096; // 64 KB, so that three CTAs fit an SM
constexpr int kMaxCluster = 4;

// Rows are dealt over CTAs, each of which has parts of `partVecs` vectors of them; or, with clusterSize > 1, there is a cluster for every row, of which a
// CTA takes every clusterSize-th part.
template <typename T, int W>
__global__ void __launch_bounds__((W + 1) * 32, kCtasPerSm) logProbsKernel(LogProbsArgs const args, int const clusterSize, int const partVecs)
{
    constexpr int kReaders = W * 32, kAll = kReaders + 32;
    constexpr int E = Vec<T>::kElems;
    __shared__ Place<W> places[2];
    __shared__ float groupMax[64], threshold;
    __shared__ Joined joined[kMaxCluster - 1]; // what the others found, in the first CTA
    __shared__ uint64_t joinFull;
    __shared__ uint32_t abortWord;
    extern __shared__ __align__(16) uint4 buf[];
    int const tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
    int const rank = static_cast<int>(blockIdx.x % clusterSize);
    int64_t const rowStep = gridDim.x / clusterSize;
    int const partStep = clusterSize * partVecs;
    if (tid < 2)
    {
        places[tid].ties = places[tid].listed = 0;
        abortWord = 0;
    }
    if (tid == 0)
        mbarInit(&joinFull, 32 * (clusterSize - 1) + (clusterSize == 1 ? 1 : 0));
    fenceBarrierInit();
    gridDependencyLaunch();
    if (clusterSize > 1)
        clusterSync();
    else
        __syncthreads();
    gridDependencyWait();

    int use = 0; // parts of this CTA so far
    if (warp < W)
    {
        int64_t r = blockIdx.x / clusterSize;
        int first = rank * partVecs;
        auto vectors = [&](Row<T> const& row, int from) {
            int const left = row.nVec - from;
            return left < partVecs ? left > 0 ? left : 0 : partVecs;
        };
        Row<T> row(args, r < args.rows ? r : 0);
        if (r < args.rows)
            row.template copy<kReaders>(buf, first, vectors(row, first), tid, tid, args);
        for (; r < args.rows; r += rowStep)
        {
            bool const rowsLeft = r + rowStep < args.rows;
            Row<T> const below(args, rowsLeft ? r + rowStep : r);
            int n = vectors(row, first);
            while (n > 0)
            {
                // what comes after this part
                bool const sameRow = first + partStep < row.nVec;
                Row<T> const then = sameRow ? row : below;
                int const thenFirst = sameRow ? first + partStep : 0; // (a CTA that has more than one row has all of their parts)
                int const thenN = sameRow || rowsLeft ? vectors(then, thenFirst) : 0;
                int const lo = then.begin(thenFirst), hi = thenN > 0 ? then.end(thenFirst, thenN) : 0;
                T const* const q = then.at(thenFirst);
                copiesWait();
                readPart<T, W>(
                    places[use & 1], groupMax, &threshold, buf, row, args.vocab, first, n, args.topK, tid,
                    [&]() {
                        if (use >= 2)
                            barSync<kAll>(kBarFree + (use & 1));
                    },
                    [&](int i) {
                        if (i >= lo && i < hi)
                            copyAsync16(buf + i, q + static_cast<int64_t>(i) * E);
                    });
                barArrive<kAll>(kBarFull + (use & 1));
                if (thenN > 0) // what lies beyond this part's vectors, and the edges
                    then.template copy<kReaders>(buf, thenFirst, thenN, n <= tid ? tid : tid + (n - 1 - tid) / kReaders * kReaders + kReaders, tid, args);
                ++use;
                first = thenFirst;
                n = sameRow ? thenN : 0;
            }
            row = below;
        }
        for (int i = use < 2 ? 0 : use - 2; i < use; ++i) // the places' last releases
            barSync<kAll>(kBarFree + (i & 1));
    }
    else
    {
        for (int64_t r = blockIdx.x / clusterSize; r < args.rows; r += rowStep)
        {
            Row<T> const row(args, r);
            float const tokenLogit = rank == 0 ? loadToken(args, row, r, lane) : negInf();
            Result res;
            for (int first = rank * partVecs; first < row.nVec; first += partStep, ++use)
            {
                int const n = row.nVec - first < partVecs ? row.nVec - first : partVecs;
                barSync<kAll>(kBarFull + (use & 1));
                takePlace<T, W>(res, places[use & 1], row, args.vocab, first, n, args.topK, lane);
                __syncwarp();
                barArrive<kAll>(kBarFree + (use & 1));
            }
            if (clusterSize > 1)
            {
                if (rank != 0)
                {
                    Joined& to = joined[rank - 1];
                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mapaShared(&to.key[lane], 0)), "l"(res.key) : "memory");
                    if (lane == 0)
                    {
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(mapaShared(&to.stat, 0)), "f"(res.stat.m),
                            "f"(res.stat.count), "f"(res.stat.s), "f"(res.stat.t)
                            : "memory");
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapaShared(&to.bad, 0)), "r"(res.bad ? 1u : 0u) : "memory");
                    }
                    mbarArriveCluster(mapaShared(&joinFull, 0));
                }
                else
                {
                    bool const ok = mbarWaitWarp(&joinFull, 0, &abortWord, kWaitTmaFull);
                    asm volatile("fence.acq_rel.cluster;" ::: "memory");
                    res.bad |= !ok;
                    for (int c = 1; c < clusterSize && ok; ++c) // their sums in order
                    {
                        Joined const& from = joined[c - 1];
                        res.stat = merge(res.stat, from.stat);
                        res.bad |= from.bad != 0;
                        if (args.topK > 0)
                            res.insert(from.key[lane], args.topK, lane);
                    }
                }
            }
            if (rank == 0)
                writeRow(args, res, row, r, tokenLogit, lane);
        }
        if (lane == 0 && abortWord != 0 && args.statusWord)
            atomicMax(args.statusWord, abortWord);
    }
    if (clusterSize > 1)
        clusterSync(); // the others may still write here, or signal
}

// Which kernel, and how many CTAs share a row.
//  - A warp per row for up to 64 vectors, for more where there are rows for many warps: FP16 20000 x 2000 42 us against 118 us with
//    a CTA per row, 12000 x 4320 28 / 60 us, 2000 x 6400 11.4 / 14.2 us, but 1200 x 6400 9.9 / 9.6 us, 600 x 4000 11.7 / 8.1 us and 100 x 2000 7.0 /
//    4.8 us; beyond 832 vectors, 2000 x 8000 16.5 / 15.8 us, top 10 25.5 / 20.8 us. Up to 224 a second
//    round of CTAs is enough: 1000 x 1440, top 10, 9.2 / 10.6 us, x 2000 10.8 / 10.3 us. Up to 160 also for more than 20 tokens, since the vectors
//    are then too few for 64 groups of threads to bound the 32nd value and most are listed: 1 x 832, top 32, 7.4 / 44 us, x 1440 8.1 / 7.2 us.
//  - One, two or four CTAs per row, whichever has the shortest way: a CTA's share of a row, what a part costs beside its vectors and what joining
//    costs (in vectors, from times of single rows), where all clusters find a place at once (2.75 CTAs per SM: more clusters of four
//    wait for one another), so that none has a second row. With one / two / four CTAs, top 5: FP32 1 x 120000 20.4 / 13.5 / 10.0 us, 100 x 120000
//    34.5 / 22.7 / 17.0 us, 200 x 120000 36 / 24.4 / 33.3 us, 100 x 30522 12.6 / 10.6 / 10.3 us, 140 x 30522 12.7 / 11.4 / 18.9 us; FP16 1 x 30522 5.7 / 6.4 /
//    6.9 us; beyond, FP32 500 x 30522 19.5 / 28.4 / 47.8 us.
inline int clusterFor(int64_t rows, int vecs, int64_t sms)
{
    constexpr int kPart = 600, kJoin = 2000;
    int best = 1;
    int bestCost = 0;
    for (int c = 1; c <= kMaxCluster && (c == 1 || rows * c <= sms * 11 / 4); c *= 2)
    {
        int const share = (vecs + c - 1) / c;
        int const cost = share + kPart * ((share + kPartVecs - 1) / kPartVecs) + kJoin * (c - 1);
        if (c == 1 || cost < bestCost)
        {
            best = c;
            bestCost = cost;
        }
    }
    return best;
}

template <typename T>
int32_t launchLogProbs(LogProbsArgs const& args, cudaStream_t stream)
{
    constexpr int E = Vec<T>::kElems;
    int const vecs = (args.vocab + E - 1) / E + 1; // a row may begin inside a vector
    int64_t const sms = smCount();
    cudaError_t e;
    if (vecs <= 64 || (vecs <= 160 && args.topK > 20) || (vecs <= 224 && args.rows > 3 * sms) || (vecs <= 640 && args.rows > 8 * sms)
        || (vecs <= 832 && args.rows > 12 * sms))
    {
        constexpr int kGroups = sizeof(T) == 4 ? 2 : 4; // warps per CTA: FP32 3000 x 1200 8.5 us with four, 7.1 us with two; FP16 12000 x 4000 27.1 / 27.8 us
        static SmemOptIn optIn;
        int64_t const most = sms * (64 / kGroups), ctas = (args.rows + kGroups - 1) / kGroups;
        e = launchDependentCluster(&optIn, logProbsWarpKernel<T, kGroups>, dim3(static_cast<unsigned>(ctas < most ? ctas : most)), dim3(32 * kGroups),
            static_cast<size_t>(vecs) * 16 * kGroups, stream, 1, args, vecs);
    }
    else
    {
        static SmemOptIn optIn;
        int const cluster = clusterFor(args.rows, vecs, sms);
        // Parts of the same length: after 4096 vectors a rest of 64 costs like many more (FP16 600 x 33280, top 5, 21.0 -> 19.1 us), and it has too few
        // threads at work to bound the 32nd value (66 -> 28.7 us).
        int const share = (vecs + cluster - 1) / cluster;
        int const parts = (share + kPartVecs - 1) / kPartVecs, partVecs = (share + parts - 1) / parts;
        int64_t const most = sms * kCtasPerSm, ctas = args.rows * cluster;
        e = launchDependentCluster(&optIn, logProbsKernel<T, kReadingWarps>, dim3(static_cast<unsigned>(cluster > 1 || ctas < most ? ctas : most)),
            dim3((kReadingWarps + 1) * 32), static_cast<size_t>(partVecs) * 16, stream, cluster, args, cluster, partVecs);
    }
    if (e != cudaSuccess)
        B200_FAIL(BERT_B200_CUDA_ERROR, "logProbsKernel: %s", cudaGetErrorString(e));
    return checkLaunch("logProbsKernel");
}

} // namespace
} // namespace b200

using namespace b200;

extern "C" int32_t bert_b200_token_log_probs(bert_b200_log_probs_params const* p, void* stream)
{
    B200_REQUIRE(p != nullptr, "token_log_probs: null params");
    B200_REQUIRE(p->type_id == BERT_B200_FP16 || p->type_id == BERT_B200_FP32, "token_log_probs: type_id %d (FP16 or FP32)", p->type_id);
    B200_REQUIRE(p->rows >= 0 && p->rows < (1ll << 31) / 8 && p->vocab > 0 && p->vocab <= 1 << 24, "token_log_probs: bad sizes rows=%lld vocab=%d (at most %d)",
        static_cast<long long>(p->rows), p->vocab, 1 << 24);
    B200_REQUIRE(p->logits_stride >= p->vocab, "token_log_probs: the logits' row stride is smaller than the vocabulary");
    B200_REQUIRE(p->num_tokens >= 0 && p->num_tokens <= 1 << 24 && p->top_k >= 0 && p->top_k <= kMaxTop, "token_log_probs: num_tokens=%d (0 to %d), top_k=%d (0 to %d)",
        p->num_tokens, 1 << 24, p->top_k, kMaxTop);
    B200_REQUIRE(p->num_tokens > 0 || p->top_k > 0 || p->entropy, "token_log_probs: nothing is asked for");
    if (p->rows == 0)
        return BERT_B200_OK;
    B200_REQUIRE(p->logits && (p->num_tokens == 0 || (p->token_ids && p->log_probs)) && (p->top_k == 0 || (p->top_ids && p->top_log_probs)),
        "token_log_probs: null pointer");
    uintptr_t const elem = p->type_id == BERT_B200_FP16 ? 2 : 4;
    uintptr_t const words = reinterpret_cast<uintptr_t>(p->status_word) | reinterpret_cast<uintptr_t>(p->token_ids) | reinterpret_cast<uintptr_t>(p->log_probs) | reinterpret_cast<uintptr_t>(p->entropy)
        | reinterpret_cast<uintptr_t>(p->top_ids) | reinterpret_cast<uintptr_t>(p->top_log_probs);
    B200_REQUIRE(reinterpret_cast<uintptr_t>(p->logits) % elem == 0 && words % 4 == 0, "token_log_probs: a pointer is not aligned to its type");
    LogProbsArgs const args{p->rows, p->vocab, p->logits, p->logits_stride, p->num_tokens, p->token_ids, p->top_k, p->log_probs, p->entropy, p->top_ids,
        p->top_log_probs, p->status_word};
    auto s = static_cast<cudaStream_t>(stream);
    return p->type_id == BERT_B200_FP16 ? launchLogProbs<__half>(args, s) : launchLogProbs<float>(args, s);
}
