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

constexpr int kMaxSinks = 256;     // first keys that get workgroups of their own

// Workgroups that share a block's walk of `tiles` 64-row tiles, all blocks' walks alike: those with which the last one ends
// first where `resident` a CU run at once. A walk's start and end are as long as four tiles, the join of parts as eight.
int evenParts(long long blocks, int tiles, int resident) {
    const long long room = (long long)resident * cuCount();
    int best = 1;
    long long least = 0;
    for (int parts = 1; parts <= std::min(16, std::max(1, tiles / 4)); ++parts) {
        const long long rounds = (blocks * parts + room - 1) / room;
        const long long time = rounds * ((tiles + parts - 1) / parts + 4) + (parts > 1 ? 8 : 0);
        if (parts == 1 || time < least) best = parts, least = time;
    }
    return best;
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
    const int group = nHeads / nKVHeads, resident = nHeadDim <= 64 ? 2 : 1;
    const int allQ = p.SqP / kTileKeys, allK = (nSeqK + kTileKeys - 1) / kTileKeys;
    const long long blocks = (nSeqK + kBlockQ - 1) / kBlockQ, heads = (long long)nBatch * nKVHeads;
    const int walk = windowTiles(p.window, p.causal, allQ);   // of a block of keys, for each query head
    p.parts = evenParts(heads * blocks, walk * group, resident);
    // The first keys: by workgroups of their own, unless they are so many that their blocks may as well walk over everything,
    // or the window is as wide as the sequences.
    if (p.first > kMaxSinks) {
        p.sinkBlocks = (p.first + kBlockQ - 1) / kBlockQ;
        p.parts = walkParts(heads * blocks, allQ * group, 2 * resident);
    } else if (p.first > 0 && p.window < std::max(nSeqQ, nSeqK)) {
        const long long groups = heads * ((p.first + 31) / 32);
        p.sinkParts = (int)std::clamp<long long>(std::min<long long>((long long)resident * cuCount() / groups,
                                                                     ((long long)std::max(1, allQ - walk) * group + 3) / 4), 1, 64);
    }
    p.partRows = p.parts > 1 ? (int)blocks * kBlockQ : p.sinkParts > 0 ? p.first : 0;
    const size_t sinks = (size_t)heads * p.sinkParts * ((p.first + 31) / 32 * 32) * nHeadDim;
    float* more = nullptr;
    if (backwardParts(p, std::min(allK, windowTiles(p.window, p.causal, allK) + (p.first + kTileKeys - 1) / kTileKeys),
                      (size_t)heads * p.parts * p.partRows * nHeadDim, 2 * sinks, &more))
        return -1;
    p.sinkDk = more;
    p.sinkDv = more + sinks;
    return nDtype == 1 ? backward<true, kAtWindow>(p) : backward<false, kAtWindow>(p);
}

}  // extern "C"
