// attn_window.hip — attention in a sliding window with a few first tokens that
// stay visible: the entries of the window view (attn_train_kernels.hpp holds
// the kernels of long sequences).
//
// An image of nQ queries and nK keys has its query i at p = i + nK - nQ and
// sees key j where |p - j| < nWindow or j < nFirst, and j <= p if causal. Blocks
// of queries walk over the tiles of their windows and of the first keys alone;
// blocks of keys over the queries whose windows reach them, the first keys'
// over all, by several workgroups.
#include "attn_train_kernels.hpp"
#include "../../include/omhip.h"

namespace omhip {

namespace {

constexpr int kMaxSeq = 1 << 29;   // positions, and sums of one and a window, stay below 2^31

// Sizes past checkSizes: what a window adds; 0 or -1.
int checkWindow(const char* name, int nSeqQ, int nSeqK, int nWindow, int nFirst) {
    if (nSeqQ > kMaxSeq || nSeqK > kMaxSeq) return fail("%s: a sequence exceeds 2^29 tokens", name);
    if (nWindow < 1) return fail("%s: a window holds one position at least", name);
    if (nFirst < 0) return fail("%s: negative number of first tokens", name);
    return 0;
}

// Tiles of 64 rows that a block of 128 sees through a window, of `most`.
int windowTiles(int window, int causal, int most) {
    return (int)std::min<long long>(most, ((long long)window * (causal ? 1 : 2) + kBlockQ) / kTileKeys + 1);
}

}  // namespace

}  // namespace omhip

using namespace omhip;

extern "C" {

int omHipAttentionWindowForwardHalf(int nDtype, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV, long long nLdQ,
                                    long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                                    const int* pKeyLens, int bCausal, int nWindow, int nFirst, uint16_t* pOut, float* pLse,
                                    int nBatch, int nSeqQ, int nSeqK, int nHeads, int nKVHeads, int nHeadDim, float fScale) {
    const char* name = "omHipAttentionWindowForwardHalf";
    clearError();
    const int rc = checkSizes(name, nDtype, nLdQ, nStrideQ, nLdKV, nStrideKV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads,
                              nHeadDim, fScale, false);
    if (rc < 0 || checkWindow(name, nSeqQ, nSeqK, nWindow, nFirst)) return -1;
    if (rc || nSeqQ == 0) return 0;
    AttnWindowParams p{};
    if (forwardArguments(p, name, pQ, pK, pV, nLdQ, nStrideQ, nLdKV, nStrideKV, pQueryLens, pKeyLens, bCausal, pOut, pLse, nBatch,
                         nSeqQ, nSeqK, nHeads, nKVHeads, nHeadDim, fScale))
        return -1;
    p.window = std::min(nWindow, std::max(nSeqQ, nSeqK));
    p.first = std::min(nFirst, nSeqK);
    const int all = (nSeqK + kTileKeys - 1) / kTileKeys;
    if (forwardParts(p, std::min(all, windowTiles(p.window, p.causal, all) + (p.first + kTileKeys - 1) / kTileKeys))) return -1;
    return nDtype == 1 ? forward<true, kAtWindow>(p) : forward<false, kAtWindow>(p);
}

int omHipAttentionWindowBackwardHalf(int nDtype, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV, long long nLdQ,
                                     long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                                     const int* pKeyLens, int bCausal, int nWindow, int nFirst, const uint16_t* pOut,
                                     const float* pLse, const uint16_t* pGradOut, uint16_t* pGradQ, uint16_t* pGradK,
                                     uint16_t* pGradV, int nBatch, int nSeqQ, int nSeqK, int nHeads, int nKVHeads, int nHeadDim,
                                     float fScale) {
    const char* name = "omHipAttentionWindowBackwardHalf";
    clearError();
    const int rc = checkSizes(name, nDtype, nLdQ, nStrideQ, nLdKV, nStrideKV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads,
                              nHeadDim, fScale, true);
    if (rc < 0 || checkWindow(name, nSeqQ, nSeqK, nWindow, nFirst)) return -1;
    if (rc || (nSeqQ == 0 && nSeqK == 0)) return 0;
    AttnWindowParams p{};
    if (backwardArguments(p, name, pQ, pK, pV, nLdQ, nStrideQ, nLdKV, nStrideKV, pQueryLens, pKeyLens, bCausal, pOut, pLse,
                          pGradOut, pGradQ, pGradK, pGradV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads, nHeadDim, fScale))
        return -1;
    p.window = std::min(nWindow, std::max(nSeqQ, nSeqK));
    p.first = std::min(nFirst, nSeqK);
    const int group = nHeads / nKVHeads, perCu = nHeadDim <= 64 ? 4 : 2;
    const int allQ = p.SqP / kTileKeys, allK = (nSeqK + kTileKeys - 1) / kTileKeys;
    const long long blocks = (nSeqK + kBlockQ - 1) / kBlockQ, heads = (long long)nBatch * nKVHeads;
    const int walk = windowTiles(p.window, p.causal, allQ) * group;   // of a block of keys
    p.parts = walkParts(heads * blocks, walk, perCu);
    // The first keys' blocks walk over every query after them: as many parts as make those as long as the others' walks,
    // and no more than fill the card.
    p.sinkBlocks = (p.first + kBlockQ - 1) / kBlockQ;
    p.sinkParts = p.parts;
    if (p.sinkBlocks > 0) {
        const long long equal = (long long)allQ * group / std::max(4, walk / p.parts);
        const long long most = 8LL * cuCount() / (heads * p.sinkBlocks);
        p.sinkParts = (int)std::clamp<long long>(std::min(equal, most), p.parts, std::max(p.parts, 64));
    }
    const long long units = (long long)p.sinkBlocks * p.sinkParts + (blocks - p.sinkBlocks) * p.parts;
    p.partUnits = (int)(p.parts > 1 ? units : p.sinkParts > 1 ? (long long)p.sinkBlocks * p.sinkParts : 0);
    if (backwardParts(p, std::min(allK, windowTiles(p.window, p.causal, allK) + (p.first + kTileKeys - 1) / kTileKeys),
                      (size_t)heads * p.partUnits * kBlockQ * nHeadDim, 0, nullptr))
        return -1;
    return nDtype == 1 ? backward<true, kAtWindow>(p) : backward<false, kAtWindow>(p);
}

}  // extern "C"
