// Fully connected layer on the sm_100a tensor cores: C = epilogue(A * Wt^T).
//
// Replaces the cublasLtMatmul call of the reference FC plugin (plugin/fcPlugin/fcPlugin.cpp:551-610)
// and the separate bias / GELU / quantise layers that follow it in the reference graph.
// The kernels themselves are in fc_tcgen05.cuh.
#include "fc_tcgen05.cuh"

#include <mutex>

namespace b200
{

int32_t fcF32(bert_b200_fc_params const& p, cudaStream_t stream);

EncodeTiledFn getEncodeTiled()
{
    static std::mutex mtx;
    static EncodeTiledFn fn = nullptr;
    std::lock_guard<std::mutex> lock(mtx);
    if (!fn)
    {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess
            && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

int32_t makeTensorMap(CUtensorMap* map, CUtensorMapDataType type, int rank, void const* base, uint64_t const* dims,
    uint64_t const* stridesBytes, uint32_t const* box, CUtensorMapSwizzle swizzle)
{
    EncodeTiledFn const fn = getEncodeTiled();
    if (!fn)
        B200_FAIL(BERT_B200_NOT_INITIALIZED, "cuTensorMapEncodeTiled is not available from this driver");
    cuuint64_t d[5];
    cuuint64_t s[4];
    cuuint32_t b[5];
    cuuint32_t es[5];
    for (int i = 0; i < rank; ++i)
    {
        d[i] = dims[i];
        b[i] = box[i];
        es[i] = 1;
        if (i > 0)
            s[i - 1] = stridesBytes[i - 1];
    }
    CUresult const r = fn(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), d, s, b, es,
        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        B200_FAIL(BERT_B200_BAD_PARAM, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(r));
    return BERT_B200_OK;
}

int32_t fcRun(bert_b200_fc_params const& p, cudaStream_t s, bool weightsReady)
{
    B200_REQUIRE(p.m >= 0 && p.n > 0 && p.k > 0, "fc: bad sizes m=%lld n=%lld k=%lld", static_cast<long long>(p.m),
        static_cast<long long>(p.n), static_cast<long long>(p.k));
    B200_REQUIRE(p.a && p.wt && p.c, "fc: null pointer");
    B200_REQUIRE(p.lda >= p.k && p.ldc >= p.n, "fc: lda/ldc smaller than the row length");
    B200_REQUIRE(p.activation == BERT_B200_ACT_NONE || p.activation == BERT_B200_ACT_GELU_ERF, "fc: unknown activation %d",
        p.activation);
    if (p.m == 0)
        return BERT_B200_OK;
    if (p.type_id == BERT_B200_FP32)
    {
        B200_REQUIRE(p.out_type_id == BERT_B200_FP32, "fc: FP32 input needs FP32 output");
        return fcF32(p, s);
    }
    B200_REQUIRE(p.type_id == BERT_B200_FP16 || p.type_id == BERT_B200_INT8, "fc: type_id %d", p.type_id);
    B200_REQUIRE(p.out_type_id != BERT_B200_INT8 || p.out_scale > 0.f, "fc: INT8 output needs out_scale > 0");
    B200_REQUIRE(p.m < (1ll << 31) && p.n < (1ll << 31) && p.k < (1ll << 31), "fc: sizes exceed the 32-bit TMA coordinates");
    int const elem = p.type_id == BERT_B200_FP16 ? 2 : 1;
    B200_REQUIRE((p.k * elem) % 16 == 0 && (p.lda * elem) % 16 == 0, "fc: row bytes of A / Wt must be a multiple of 16");
    B200_REQUIRE(aligned16(p.a) && aligned16(p.wt) && aligned16(p.c), "fc: A, Wt and C must be 16-byte aligned");
    B200_REQUIRE(p.n % 16 == 0, "fc: n=%lld must be a multiple of 16", static_cast<long long>(p.n));
    B200_REQUIRE(!p.bias || aligned16(p.bias), "fc: bias must be 16-byte aligned");
    int const outElem = p.out_type_id == BERT_B200_FP16 ? 2 : 1;
    B200_REQUIRE((p.ldc * outElem) % 16 == 0, "fc: row bytes of C must be a multiple of 16");
    FcPlan const plan = planFc(p);
    FcProblem const q = plainFc(p);
    bool const shortTile = p.m <= 64; // the narrow tiles also come with 64 rows (see the kernel)
#define B200_FC_TILE(IN, OUT)                                                                                          \
    switch (plan.blockN)                                                                                               \
    {                                                                                                                  \
    case 16: return shortTile ? launchFcTile<IN, 64, 16, OUT>(q, weightsReady, s) : launchFcTile<IN, 128, 16, OUT>(q, weightsReady, s); \
    case 32: return shortTile ? launchFcTile<IN, 64, 32, OUT>(q, weightsReady, s) : launchFcTile<IN, 128, 32, OUT>(q, weightsReady, s); \
    case 64: return launchFcTile<IN, 128, 64, OUT>(q, weightsReady, s);                                                \
    default: return launchFcTile<IN, 128, 128, OUT>(q, weightsReady, s);                                               \
    }
#define B200_FC_DISPATCH(IN, OUT)                                                                                      \
    if (plan.pair)                                                                                                     \
        switch (plan.blockN)                                                                                           \
        {                                                                                                              \
        case 128: return launchFcPair<IN, 128, OUT>(q, s);                                                             \
        case 160: return launchFcPair<IN, 160, OUT>(q, s);                                                             \
        case 192: return launchFcPair<IN, 192, OUT>(q, s);                                                             \
        case 224: return launchFcPair<IN, 224, OUT>(q, s);                                                             \
        default: return launchFcPair<IN, 256, OUT>(q, s);                                                              \
        }                                                                                                              \
    B200_FC_TILE(IN, OUT)
    if (p.type_id == BERT_B200_FP16)
    {
        B200_REQUIRE(p.out_type_id == BERT_B200_FP16, "fc: FP16 input needs FP16 output");
        B200_FC_DISPATCH(__half, __half)
    }
    if (p.out_type_id == BERT_B200_INT8)
    {
        B200_FC_DISPATCH(int8_t, int8_t)
    }
    B200_REQUIRE(p.out_type_id == BERT_B200_FP16, "fc: INT8 input needs INT8 or FP16 output");
    B200_FC_DISPATCH(int8_t, __half)
#undef B200_FC_TILE
#undef B200_FC_DISPATCH
}

} // namespace b200

extern "C" int32_t bert_b200_fc(bert_b200_fc_params const* params, void* stream)
{
    B200_REQUIRE(params != nullptr, "fc: null params");
    // Nothing is known about who writes the weights: a kernel two places ahead in the stream may still be at it.
    return b200::fcRun(*params, static_cast<cudaStream_t>(stream), false);
}
