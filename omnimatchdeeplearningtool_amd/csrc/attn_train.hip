// attn_train.hip — attention for training on fp16 / bf16 data: the entries of the
// plain view (attn_train_kernels.hpp holds the kernels).
//
// The reference trains MultiHeadAttention through autograd nodes of the
// unfused chain (src/engine/om.engine.vit.ixx:150-239: qkvSplitHeads,
// tensorBatchedMatmul, tensorSoftmaxLastDim, tensorBatchedMatmul, mergeHeads),
// which keep the S x S probabilities. If causal, query i sees keys j <= i +
// nSeqK - nSeqQ.
#include "attn_train_kernels.hpp"
#include "../../include/omhip.h"

using namespace omhip;

extern "C" {

int omHipAttentionTrainForwardHalf(int nDtype, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV, long long nLdQ,
                                   long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                                   const int* pKeyLens, int bCausal, uint16_t* pOut, float* pLse, int nBatch, int nSeqQ,
                                   int nSeqK, int nHeads, int nKVHeads, int nHeadDim, float fScale) {
    const char* name = "omHipAttentionTrainForwardHalf";
    clearError();
    const int rc = checkSizes(name, nDtype, nLdQ, nStrideQ, nLdKV, nStrideKV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads,
                              nHeadDim, fScale, false);
    if (rc < 0) return -1;
    if (rc || nSeqQ == 0) return 0;
    AttnTrainParams p{};
    if (forwardArguments(p, name, pQ, pK, pV, nLdQ, nStrideQ, nLdKV, nStrideKV, pQueryLens, pKeyLens, bCausal, pOut, pLse, nBatch,
                         nSeqQ, nSeqK, nHeads, nKVHeads, nHeadDim, fScale) ||
        forwardParts(p, (nSeqK + kTileKeys - 1) / kTileKeys))
        return -1;
    return nDtype == 1 ? forward<true, kAtPlain>(p) : forward<false, kAtPlain>(p);
}

int omHipAttentionBackwardHalf(int nDtype, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV, long long nLdQ,
                               long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                               const int* pKeyLens, int bCausal, const uint16_t* pOut, const float* pLse,
                               const uint16_t* pGradOut, uint16_t* pGradQ, uint16_t* pGradK, uint16_t* pGradV, int nBatch,
                               int nSeqQ, int nSeqK, int nHeads, int nKVHeads, int nHeadDim, float fScale) {
    const char* name = "omHipAttentionBackwardHalf";
    clearError();
    const int rc = checkSizes(name, nDtype, nLdQ, nStrideQ, nLdKV, nStrideKV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads,
                              nHeadDim, fScale, true);
    if (rc < 0) return -1;
    if (rc || (nSeqQ == 0 && nSeqK == 0)) return 0;
    AttnTrainParams p{};
    if (backwardArguments(p, name, pQ, pK, pV, nLdQ, nStrideQ, nLdKV, nStrideKV, pQueryLens, pKeyLens, bCausal, pOut, pLse,
                          pGradOut, pGradQ, pGradK, pGradV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads, nHeadDim, fScale))
        return -1;
    const size_t keyBlocks = (size_t)nBatch * nKVHeads * ((nSeqK + kBlockQ - 1) / kBlockQ);
    p.parts = walkParts((long long)keyBlocks, p.SqP / kTileKeys * (nHeads / nKVHeads), (nHeadDim <= 64 ? 4LL : 2LL) * cuCount());
    p.partRows = (nSeqK + kBlockQ - 1) / kBlockQ * kBlockQ;
    if (backwardParts(p, (nSeqK + kTileKeys - 1) / kTileKeys, p.parts > 1 ? keyBlocks * p.parts * kBlockQ * nHeadDim : 0, 0,
                      nullptr))
        return -1;
    return nDtype == 1 ? backward<true, kAtPlain>(p) : backward<false, kAtPlain>(p);
}

}  // extern "C"
