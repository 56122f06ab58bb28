// INT8 product with a scale for each row of A (each token) and each output channel, on the kernels of fc_tcgen05.cuh.
// No counterpart in the reference, whose INT8 layers take one calibrated step per tensor.
#include "fc_tcgen05.cuh"

namespace b200
{

int32_t fcRowwiseRun(bert_b200_fc_rowwise_params const& r, cudaStream_t s, bool weightsReady)
{
    B200_REQUIRE(r.m >= 0 && r.n > 0 && r.k > 0, "fc_rowwise: bad sizes m=%lld n=%lld k=%lld", static_cast<long long>(r.m),
        static_cast<long long>(r.n), static_cast<long long>(r.k));
    B200_REQUIRE(r.out_type_id == BERT_B200_FP16 || r.out_type_id == BERT_B200_FP32, "fc_rowwise: out_type_id %d (FP16 or FP32)", r.out_type_id);
    B200_REQUIRE(r.activation == BERT_B200_ACT_NONE || r.activation == BERT_B200_ACT_GELU_ERF, "fc_rowwise: unknown activation %d", r.activation);
    B200_REQUIRE(r.k <= 131071, "fc_rowwise: k=%lld products of 128 * 128 may exceed the 32-bit sums (131071 at most)", static_cast<long long>(r.k));
    B200_REQUIRE(r.m < (1ll << 31) && r.n < (1ll << 31), "fc_rowwise: sizes exceed the 32-bit TMA coordinates");
    B200_REQUIRE(r.lda >= r.k && r.ldw >= r.k && r.ldc >= r.n, "fc_rowwise: lda / ldw / ldc smaller than the row length");
    if (r.m == 0)
        return BERT_B200_OK;
    B200_REQUIRE(r.a && r.a_scales && r.wt && r.wt_scales && r.c, "fc_rowwise: null pointer");
    int64_t const outElem = r.out_type_id == BERT_B200_FP16 ? 2 : 4;
    B200_REQUIRE(r.lda < (1ll << 40) && r.ldw < (1ll << 40) && r.ldc < (1ll << 40) / outElem, "fc_rowwise: row strides exceed the 40 bits of a tensor map");
    B200_REQUIRE(r.lda % 16 == 0 && r.ldw % 16 == 0 && r.ldc * outElem % 16 == 0, "fc_rowwise: row strides of A, Wt and C must be multiples of 16 bytes");
    B200_REQUIRE(aligned16(r.a) && aligned16(r.wt) && aligned16(r.c), "fc_rowwise: A, Wt and C must be 16-byte aligned");
    B200_REQUIRE((reinterpret_cast<uintptr_t>(r.a_scales) | reinterpret_cast<uintptr_t>(r.wt_scales) | reinterpret_cast<uintptr_t>(r.bias)) % 4 == 0,
        "fc_rowwise: a_scales, wt_scales or bias is not aligned to its type");
    FcProblem p{};
    p.type_id = BERT_B200_INT8;
    p.out_type_id = r.out_type_id;
    p.m = r.m;
    p.n = r.n;
    p.k = r.k;
    p.a = r.a;
    p.lda = r.lda;
    p.wt = r.wt;
    p.c = r.c;
    p.ldc = r.ldc;
    p.bias = r.bias;
    p.activation = r.activation;
    p.status_word = r.status_word;
    p.ldw = r.ldw;
    p.rowScale = r.a_scales;
    p.colScale = r.wt_scales;
    FcPlan const plan = planFc(p);
    bool const shortTile = p.m <= 64;
#define B200_FC_DISPATCH(OUT)                                                                                          \
    if (plan.pair)                                                                                                     \
        switch (plan.blockN)                                                                                           \
        {                                                                                                              \
        case 128: return launchFcPair<int8_t, 128, OUT, true>(p, s);                                                   \
        case 160: return launchFcPair<int8_t, 160, OUT, true>(p, s);                                                   \
        case 192: return launchFcPair<int8_t, 192, OUT, true>(p, s);                                                   \
        case 224: return launchFcPair<int8_t, 224, OUT, true>(p, s);                                                   \
        default: return launchFcPair<int8_t, 256, OUT, true>(p, s);                                                    \
        }                                                                                                              \
    switch (plan.blockN)                                                                                               \
    {                                                                                                                  \
    case 16:                                                                                                           \
        return shortTile ? launchFcTile<int8_t, 64, 16, OUT, true>(p, weightsReady, s)                                 \
                         : launchFcTile<int8_t, 128, 16, OUT, true>(p, weightsReady, s);                               \
    case 32:                                                                                                           \
        return shortTile ? launchFcTile<int8_t, 64, 32, OUT, true>(p, weightsReady, s)                                 \
                         : launchFcTile<int8_t, 128, 32, OUT, true>(p, weightsReady, s);                               \
    case 64: return launchFcTile<int8_t, 128, 64, OUT, true>(p, weightsReady, s);                                      \
    default: return launchFcTile<int8_t, 128, 128, OUT, true>(p, weightsReady, s);                                     \
    }
    if (p.out_type_id == BERT_B200_FP16)
    {
        B200_FC_DISPATCH(__half)
    }
    B200_FC_DISPATCH(float)
#undef B200_FC_DISPATCH
}

} // namespace b200

extern "C" int32_t bert_b200_fc_rowwise(bert_b200_fc_rowwise_params const* params, void* stream)
{
    B200_REQUIRE(params != nullptr, "fc_rowwise: null params");
    return b200::fcRowwiseRun(*params, static_cast<cudaStream_t>(stream), false);
}
