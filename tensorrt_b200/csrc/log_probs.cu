// Log probabilities of given tokens, entropy and the most likely tokens of each row of logits, in one pass over the logits.
//
// With M the row's maximum, c how often it occurs, s = sum of exp(x - M) over the other values and t = sum of (x - M) exp(x - M):
//   log p(x) = (x - M) - L,   L = ln c + ln1p(s / c),   entropy = L - t / (c + s).
// The maxima are kept out of s so that a row that is sure of a token keeps the digits of 1 - p: L is then as precise as s.
// No counterpart in the reference (its plugins end at the encoder's output).
//
// A group of W warps takes a part of a row, NV 16-byte vectors per thread, into registers, so that the maximum is known before the first
// exponential and nothing is read twice. The k most likely tokens: the k-th largest of 32 groups' maxima is a lower bound of the k-th
// largest value, so only what is at least that (a few more than k) is listed and ranked, by value, then by the lower id. Rows where the
// list overflows (thousands of equal values) are selected one after the other from the L2 instead.
// Rows longer than a part: a cluster of CTAs takes the parts at once and joins them through distributed shared memory where that does not
// take SMs from other rows; otherwise a CTA takes them by turns.
#include "common.cuh"

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

// Larger values first, of equal ones (-0 equals 0) the lower id; never 0.
__device__ __forceinline__ uint64_t makeKey(float x, int32_t id)
{
    int32_t const b = __float_as_int(x + 0.f);
    uint32_t const order = static_cast<uint32_t>(b ^ ((b >> 31) & 0x7fffffff)) ^ 0x80000000u;
    return static_cast<uint64_t>(order) << 32 | (0xffffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ int32_t keyId(uint64_t k)
{
    return static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k));
}
__device__ __forceinline__ float keyValue(uint64_t k)
{
    int32_t const o = static_cast<int32_t>(static_cast<uint32_t>(k >> 32) ^ 0x80000000u);
    return __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
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
    static __device__ __forceinline__ float most(uint4 const& v)
    {
        __half2 const* h = reinterpret_cast<__half2 const*>(&v);
        __half2 const m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        return maxNan(__low2float(m), __high2float(m));
    }
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
    static __device__ __forceinline__ float most(uint4 const& v)
    {
        return maxNan(maxNan(__uint_as_float(v.x), __uint_as_float(v.y)), maxNan(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
};

template <typename T, typename F>
__device__ __forceinline__ int countIf(uint4 const& v, F const& f)
{
    float x[Vec<T>::kElems];
    Vec<T>::unpack(v, x);
    int n = 0;
#pragma unroll
    for (int j = 0; j < Vec<T>::kElems; ++j)
        n += f(x[j]) ? 1 : 0;
    return n;
}

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

template <int W>
struct Scratch
{
    static constexpr int kCap = W == 1 ? 256 : 512;
    uint64_t cand[kCap];
    uint64_t top[kMaxTop];
    uint64_t best[W];
    Stat stat;
    float groupMax[32];
    float2 sums[W];
    float threshold;
    int32_t ties, listed, topCount;
    int32_t bad; // a NaN or +infinity has been seen
};

template <int W>
__device__ __forceinline__ void groupSync()
{
    if (W == 1)
        __syncwarp();
    else
        __syncthreads();
}

// One part of a row: vectors [first, first + T * NV) of `nVec`; `p` is the row's first value, `mis` values behind a 16-byte boundary.
// Adds to sh.stat and sh.top.
template <typename T, int W, int NV>
__device__ __forceinline__ void takePart(Scratch<W>& sh, T const* p, int mis, int32_t vocab, int first, int nVec, int topK, int tid)
{
    constexpr int kThreads = W * 32;
    constexpr int E = Vec<T>::kElems;
    int const lane = tid & 31, warp = tid >> 5;
    uint4 v[NV];
    uint32_t const fill = sizeof(T) == 2 ? 0xfc00fc00u : 0xff800000u; // -infinity
    auto load = [&](int vec) {
        int32_t const e0 = vec * E - mis;
        if (e0 >= 0 && e0 + E <= vocab)
            return ldgStream(p + e0);
        uint4 r = make_uint4(fill, fill, fill, fill);
        T* const e = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (e0 + j >= 0 && e0 + j < vocab)
                e[j] = __ldg(p + e0 + j);
        return r;
    };
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i * kThreads < nVec) // the same for all threads
            v[i] = load(first + i * kThreads + tid);
    float mine = negInf();
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (first + i * kThreads < nVec)
            mine = maxNan(mine, Vec<T>::most(v[i]));
    float g = mine;
#pragma unroll
    for (int o = 1; o < W; o *= 2)
        g = maxNan(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (lane % W == 0)
        sh.groupMax[tid / W] = g;
    // the tokens found so far compete with this part's
    int const had = sh.topCount;
    if (tid < had)
        sh.cand[tid] = sh.top[tid];
    groupSync<W>();

    float const gm = sh.groupMax[lane];
    float const m = warpMaxNan(gm);
    bool const bad = !(m < __int_as_float(0x7f800000)); // NaN or +infinity
    bool const some = !bad && m != negInf();
    if (tid == 0)
        sh.bad |= bad ? 1 : 0;
    float s = 0.f, t = 0.f;
    if (some)
    {
        if (topK > 0 && warp == W - 1)
        {
            int rank = 0;
#pragma unroll
            for (int o = 1; o < 32; ++o)
            {
                float const x = __shfl_xor_sync(0xffffffffu, gm, o);
                rank += x > gm || (x == gm && (lane ^ o) < lane) ? 1 : 0;
            }
            float thr = __shfl_sync(0xffffffffu, gm, __ffs(__ballot_sync(0xffffffffu, rank == topK - 1)) - 1);
            if (had == topK)
                thr = fmaxf(thr, keyValue(sh.cand[topK - 1]));
            if (lane == 0)
                sh.threshold = thr;
        }
        if (mine == m)
        {
            // the row's maxima are listed and counted here, and no longer among the others
            int n = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (first + i * kThreads < nVec)
                    n += countIf<T>(v[i], [&](float x) { return x == m; });
            atomicAdd(&sh.ties, n);
            int at = topK > 0 ? atomicAdd(&sh.listed, n) : 0;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (first + i * kThreads < nVec)
                {
                    T* const e = reinterpret_cast<T*>(&v[i]);
#pragma unroll
                    for (int j = 0; j < E; ++j)
                        if (static_cast<float>(e[j]) == m)
                        {
                            e[j] = static_cast<T>(negInf());
                            if (topK > 0 && at < Scratch<W>::kCap)
                                sh.cand[at++] = makeKey(m, (first + i * kThreads + tid) * E - mis + j);
                        }
                }
        }
        uint64_t const negM = pack2(-m, -m), log2e = pack2(1.4426950408889634f, 1.4426950408889634f);
        uint64_t s2 = pack2(0.f, 0.f), t2 = s2;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (first + i * kThreads < nVec)
            {
                float f[E];
                Vec<T>::unpack(v[i], f);
#pragma unroll
                for (int j = 0; j < E; j += 2)
                {
                    float a, b;
                    unpack2(add2(pack2(f[j], f[j + 1]), negM), a, b);
                    a = fmaxf(a, -200.f); // masked values: 0 times a finite number
                    b = fmaxf(b, -200.f);
                    uint64_t const d = pack2(a, b);
                    unpack2(mul2(d, log2e), a, b);
                    uint64_t const e = pack2(exp2Approx(a), exp2Approx(b));
                    s2 = add2(s2, e);
                    t2 = fma2(e, d, t2);
                }
            }
        float a, b;
        unpack2(s2, a, b);
        s = a + b;
        unpack2(t2, a, b);
        t = a + b;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
    {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    if (lane == 0)
        sh.sums[warp] = make_float2(s, t);
    groupSync<W>();

    if (some)
    {
        if (topK > 0)
        {
            float const thr = sh.threshold;
            if (mine >= thr && mine != negInf())
            {
int n = 0;
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (first + i * kThreads < nVec)
                        n += countIf<T>(v[i], [&](float x) { return x >= thr && x != negInf(); });
                int at = atomicAdd(&sh.listed, n);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (first + i * kThreads < nVec)
                    {
                        float f[E];
                        Vec<T>::unpack(v[i], f);
#pragma unroll
                        for (int j = 0; j < E; ++j)
                            if (f[j] >= thr && f[j] != negInf() && at < Scratch<W>::kCap)
                                sh.cand[at++] = makeKey(f[j], (first + i * kThreads + tid) * E - mis + j);
                    }
            }
        }
        if (warp == 0)
        {
            float2 const x = lane < W ? sh.sums[lane] : make_float2(0.f, 0.f);
            s = x.x;
            t = x.y;
#pragma unroll
            for (int o = W / 2; o > 0; o >>= 1)
            {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                t += __shfl_xor_sync(0xffffffffu, t, o);
            }
            if (lane == 0)
                sh.stat = merge(sh.stat, Stat{m, static_cast<float>(sh.ties), s, t});
        }
    }
    groupSync<W>();

    if (some && topK > 0)
    {
        int const n = sh.listed;
        if (n <= Scratch<W>::kCap)
        {
            for (int i = tid; i < n; i += kThreads)
            {
                uint64_t const k = sh.cand[i];
                int rank = 0;
                for (int j = 0; j < n; ++j)
                    rank += sh.cand[j] > k ? 1 : 0;
                if (rank < topK)
                    sh.top[rank] = k;
            }
            if (tid == 0)
                sh.topCount = n < topK ? n : topK;
        }
        else
        {
            // more than the list holds: the largest key that is below the last one found, topK times
            uint64_t last = ~0ull;
            auto scan = [&]() {
                uint64_t best = tid < had && sh.cand[tid] < last ? sh.cand[tid] : 0ull;
                for (int i = 0; i < NV; ++i)
                    for (int j = 0; j < E; ++j)
                    {
                        int32_t const id = (first + i * kThreads + tid) * E - mis + j;
                        if (id < 0 || id >= vocab)
                            continue;
                        float const x = static_cast<float>(__ldg(p + id));
                        uint64_t const k = x == negInf() ? 0ull : makeKey(x, id);
                        best = k < last && k > best ? k : best;
                    }
                return best;
            };
            uint64_t best = scan();
            int found = 0;
            for (; found < topK; ++found)
            {
                uint64_t k = best;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                {
                    uint64_t const x = __shfl_xor_sync(0xffffffffu, k, o);
                    k = x > k ? x : k;
                }
                if (lane == 0)
                    sh.best[warp] = k;
                groupSync<W>();
                k = sh.best[0];
#pragma unroll
                for (int w = 1; w < W; ++w)
                    k = sh.best[w] > k ? sh.best[w] : k;
                groupSync<W>();
                if (k == 0ull)
                    break;
                if (tid == 0)
                    sh.top[found] = k;
                if (best == k)
                {
                    last = k;
                    best = scan();
                }
            }
            if (tid == 0)
                sh.topCount = found;
        }
    }
    if (tid == 0)
        sh.ties = 0;
    groupSync<W>();
    if (tid == 0)
        sh.listed = sh.topCount;
}

// kRows rows per CTA (one per warp) where W == 1; otherwise one row per cluster of `gridDim.x / rows` CTAs.
template <typename T, int W, int NV, int kRows>
__global__ void __launch_bounds__(W * 32 * kRows, W == 16 ? 2 : 1) logProbsKernel(LogProbsArgs const args, int const clusterSize)
{
    static_assert(W == 1 || kRows == 1, "several rows per CTA: one warp each");
    constexpr int kThreads = W * 32;
    constexpr int E = Vec<T>::kElems;
    __shared__ Scratch<W> scratch[kRows];
    int const tid = W == 1 ? static_cast<int>(threadIdx.x & 31) : static_cast<int>(threadIdx.x);
    Scratch<W>& sh = scratch[W == 1 ? threadIdx.x >> 5 : 0];
    int const rank = W == 1 ? 0 : static_cast<int>(blockIdx.x % clusterSize);
    int64_t const row = W == 1 ? static_cast<int64_t>(blockIdx.x) * kRows + (threadIdx.x >> 5) : static_cast<int64_t>(blockIdx.x / clusterSize);
    gridDependencyLaunch();
    if (tid == 0)
    {
        sh.stat = Stat{negInf(), 0.f, 0.f, 0.f};
        sh.ties = sh.listed = sh.topCount = sh.bad = 0;
    }
    gridDependencyWait();
    if (row >= args.rows) // whole warps of a CTA that has no other barrier
        return;
    groupSync<W>();
    T const* const p = static_cast<T const*>(args.logits) + row * args.stride;
    int const mis = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
    int const nVec = (args.vocab + mis + E - 1) / E;
    // the tokens asked for: their logits are on the way while the row is worked on
    int32_t token = -1;
    float tokenLogit = negInf();
    if (rank == 0 && tid < args.numTokens)
    {
        token = __ldg(args.tokenIds + row * args.numTokens + tid);
        if (token >= 0 && token < args.vocab)
            tokenLogit = static_cast<float>(__ldg(p + token));
    }
    for (int first = rank * kThreads * NV; first < nVec; first += clusterSize * kThreads * NV)
        takePart<T, W, NV>(sh, p, mis, args.vocab, first, nVec, args.topK, tid);

    if (W > 1 && clusterSize > 1)
    {
        clusterBarrier();
        if (rank == 0)
        {
            // what the other CTAs found, joined by this one: their sums in order, their tokens ranked together
            Stat st = sh.stat;
            int bad = sh.bad, n = sh.topCount;
            for (int i = tid; i < n; i += kThreads)
                sh.cand[i] = sh.top[i];
            for (int r = 1; r < clusterSize; ++r)
            {
                float4 const x = ldSharedCluster4(reinterpret_cast<float const*>(&sh.stat), r);
                st = merge(st, Stat{x.x, x.y, x.z, x.w});
                bad |= static_cast<int>(ldSharedCluster(reinterpret_cast<uint32_t const*>(&sh.bad), r));
                int const more = static_cast<int>(ldSharedCluster(reinterpret_cast<uint32_t const*>(&sh.topCount), r));
                if (tid < more)
                {
                    uint32_t const* const k = reinterpret_cast<uint32_t const*>(&sh.top[tid]);
                    sh.cand[n + tid] = static_cast<uint64_t>(ldSharedCluster(k + 1, r)) << 32 | ldSharedCluster(k, r);
                }
                n += more;
            }
            __syncthreads();
            if (tid == 0)
            {
                sh.stat = st;
                sh.bad = bad;
                sh.topCount = n < args.topK ? n : args.topK;
            }
            for (int i = tid; i < n; i += kThreads)
            {
                uint64_t const k = sh.cand[i];
                int place = 0;
                for (int j = 0; j < n; ++j)
                    place += sh.cand[j] > k ? 1 : 0;
                if (place < args.topK)
                    sh.top[place] = k;
            }
            __syncthreads();
        }
        clusterBarrier(); // the others' shared memory has been read
        if (rank != 0)
            return;
    }
    groupSync<W>();

    Stat const st = sh.stat;
    bool const bad = sh.bad != 0;
    bool const none = !bad && st.count == 0.f;
    float const nan = __int_as_float(0x7fffffff);
    float const lse = none ? 0.f : logf(st.count) + log1pf(st.s / st.count);
    auto logProb = [&](float x) {
        return bad ? nan : none ? negInf() : (x - st.m) - lse;
    };
    for (int j = tid; j < args.numTokens; j += kThreads)
    {
        if (j != tid)
        {
            token = __ldg(args.tokenIds + row * args.numTokens + j);
            tokenLogit = token >= 0 && token < args.vocab ? static_cast<float>(__ldg(p + token)) : negInf();
        }
        args.logProbs[row * args.numTokens + j] = logProb(tokenLogit);
    }
    if (tid == 0 && args.entropy)
        args.entropy[row] = bad ? nan : none ? 0.f : lse - st.t / (st.count + st.s);
    if (tid < args.topK)
    {
        bool const have = !bad && tid < sh.topCount;
        uint64_t const k = have ? sh.top[tid] : 0ull;
        args.topIds[row * args.topK + tid] = have ? keyId(k) : -1;
        args.topLogProbs[row * args.topK + tid] = have ? logProb(keyValue(k)) : bad ? nan : negInf();
    }
}

template <typename T>
int32_t launchLogProbs(LogProbsArgs const& args, cudaStream_t stream)
{
    constexpr int E = Vec<T>::kElems;
    int64_t const vecs = (static_cast<int64_t>(args.vocab) + E - 1) / E + 1; // a row may begin inside a vector
    cudaError_t e;
    if (vecs <= 32 * 4)
        e = launchDependent(logProbsKernel<T, 1, 4, 4>, dim3(static_cast<unsigned>((args.rows + 3) / 4)), dim3(128), 0, stream, args, 1);
    else if (vecs <= 256 * 4)
        e = launchDependent(logProbsKernel<T, 8, 4, 1>, dim3(static_cast<unsigned>(args.rows)), dim3(256), 0, stream, args, 1);
    else
    {
        int64_t const resident = static_cast<int64_t>(smCount()) * 2;
        int cluster = 1;
        while (cluster < 8 && args.rows * cluster * 2 <= resident && vecs > 512 * cluster)
            cluster *= 2;
        e = launchDependentCluster(nullptr, logProbsKernel<T, 16, 8, 1>, dim3(static_cast<unsigned>(args.rows * cluster)), dim3(512), 0, stream, cluster,
            args, cluster);
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
    B200_REQUIRE(p->num_tokens >= 0 && p->top_k >= 0 && p->top_k <= kMaxTop, "token_log_probs: num_tokens=%d, top_k=%d (0 to %d)", p->num_tokens, p->top_k,
        kMaxTop);
    B200_REQUIRE(p->num_tokens > 0 || p->top_k > 0 || p->entropy, "token_log_probs: nothing is asked for");
    if (p->rows == 0)
        return BERT_B200_OK;
    B200_REQUIRE(p->logits && (p->num_tokens == 0 || (p->token_ids && p->log_probs)) && (p->top_k == 0 || (p->top_ids && p->top_log_probs)),
        "token_log_probs: null pointer");
    uintptr_t const elem = p->type_id == BERT_B200_FP16 ? 2 : 4;
    uintptr_t const words = reinterpret_cast<uintptr_t>(p->token_ids) | reinterpret_cast<uintptr_t>(p->log_probs) | reinterpret_cast<uintptr_t>(p->entropy)
        | reinterpret_cast<uintptr_t>(p->top_ids) | reinterpret_cast<uintptr_t>(p->top_log_probs);
    B200_REQUIRE(reinterpret_cast<uintptr_t>(p->logits) % elem == 0 && words % 4 == 0, "token_log_probs: a pointer is not aligned to its type");
    LogProbsArgs const args{p->rows, p->vocab, p->logits, p->logits_stride, p->num_tokens, p->token_ids, p->top_k, p->log_probs, p->entropy, p->top_ids,
        p->top_log_probs};
    auto s = static_cast<cudaStream_t>(stream);
    return p->type_id == BERT_B200_FP16 ? launchLogProbs<__half>(args, s) : launchLogProbs<float>(args, s);
}
