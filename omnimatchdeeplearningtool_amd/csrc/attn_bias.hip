// attn_bias.hip — attention with a learned bias by relative position, forward
// and backward: the entries of the bias view (attn_train_kernels.hpp holds the
// attention kernels), and the sums of the table's gradient.
//
// S = scale Q K^T + bias, bias_ij = table[bucketOf[pos_i - pos_j + zero]][head]:
// a table of learned biases, and a map from the difference of two positions to
// its rows. One map serves sequences (position i; buckets that grow with the
// distance) and grids of patches (position y (2 width - 1) + x, whose differences
// tell both distances). dtable is the sum of dS over the pairs of a bucket:
//  * the dQ kernel, which has dS in registers, adds each to its wave's sums by
//    offset in LDS, and leaves its workgroup's;
//  * attn_bias_table_kernel adds those of a head, then the offsets of each
//    bucket. All in a fixed order, but for lanes of a wave that add to one
//    address at once (attn_train_kernels.hpp).
#include "attn_train_kernels.hpp"
#include "../../include/omhip.h"

#include <climits>

namespace omhip {

namespace {

constexpr int kMaxBuckets = 16384;   // attn_bias_table_kernel's sums take 128 KB of LDS
constexpr int kMaxSeq = 1 << 29;     // positions stay below 2^31

// A workgroup adds 64 offsets' sums of a head over its `units` rows of bins, a sixteenth a wave, into offsetSums; the head's
// last one to arrive adds the offsets of each bucket, by one wave, into gradTable. What passes between workgroups is written and
// read coherently past the XCDs' L2s and has landed before the counter goes up. Two launches measured 9.6 us where this one
// measures 7.2 (12 heads, 128 units, 731 offsets). units 0: no pair, and so zeros.
__global__ __launch_bounds__(1024) void attn_bias_table_kernel(AttnBiasParams p, int units) {
    __shared__ double part[16][64];
    __shared__ int last;
    extern __shared__ double bucketSums[];   // [nBuckets]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o = (int)blockIdx.x * 64 + lane, head = (int)blockIdx.y;
    const __amdgpu_buffer_rsrc_t sums = bufferRsrc(p.offsetSums + (long long)head * p.nOffsets, units > 0 ? (uint32_t)p.nOffsets * 4u : 0u);
    if (units > 0) {
        const int first = (int)((long long)units * wave / 16), end = (int)((long long)units * (wave + 1) / 16);
        double s = 0.;
        if (o < p.nOffsets) {
            const float* from = p.bins + (long long)head * units * p.nOffsets + o;
#pragma unroll 8
            for (int u = first; u < end; ++u) s += (double)from[(long long)u * p.nOffsets];
        }
        part[wave][lane] = s;
        __syncthreads();
        if (wave == 0) {
            s = 0.;
#pragma unroll
            for (int k = 0; k < 16; ++k) s += part[k][lane];
            bufStore1Agent(sums, (uint32_t)o * 4u, 0, (float)s);   // past the last offset: out of range, not written
            __builtin_amdgcn_s_waitcnt(0);                         // the sums have landed
            if (lane == 0)
                last = __hip_atomic_fetch_add(p.arrivals + head, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        }
        __syncthreads();
        if (!last) return;
    }
    for (int b = (int)threadIdx.x; b < p.nBuckets; b += 1024) bucketSums[b] = 0.;
    __syncthreads();
    if (wave == 0 && units > 0) {
        constexpr int N = 8;   // loads under way
        for (int o0 = lane; o0 < p.nOffsets; o0 += 64 * N) {
            int b[N];
            float v[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int i = o0 + 64 * k;
                b[k] = i < p.nOffsets ? p.bucketOf[i] : -1;
                v[k] = bufLoad1Agent(sums, (uint32_t)i * 4u, 0);
            }
#pragma unroll
            for (int k = 0; k < N; ++k)
                if ((uint32_t)b[k] < (uint32_t)p.nBuckets) atAdd(bucketSums + b[k], (double)v[k]);
        }
        __builtin_amdgcn_s_waitcnt(0);
    }
    __syncthreads();
    for (int b = (int)threadIdx.x; b < p.nBuckets; b += 1024) p.gradTable[(long long)b * p.H + head] = (float)bucketSums[b];
    if (threadIdx.x == 0 && units > 0) __hip_atomic_store(p.arrivals + head, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
}

int tableGradient(AttnBiasParams& p, int units) {
    if (units > 0) {
        p.arrivals = static_cast<unsigned*>(workspace((size_t)p.H * sizeof(unsigned), kWsCounters));
        if (!p.arrivals) return -1;   // workspace() recorded the cause
    }
    OMHIP_CHECK(OMHIP_SET_MAX_DYNAMIC_LDS_ONCE(attn_bias_table_kernel, kMaxBuckets * sizeof(double)));
    hipLaunchKernelGGL(attn_bias_table_kernel, dim3(units > 0 ? (p.nOffsets + 63) / 64 : 1, p.H), dim3(1024),
                       (size_t)p.nBuckets * sizeof(double), stream(), p, units);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

// What a bias asks of its arguments; 0 or -1.
int biasArguments(AttnBiasParams& p, const char* name, const float* pTable, const int* pBuckets, const int* pQueryPos,
                  const int* pKeyPos, int nBuckets, int nOffsets, int nZero, int nSeqQ, int nSeqK, int nHeads) {
    if (nSeqQ > kMaxSeq || nSeqK > kMaxSeq) return fail("%s: a sequence exceeds 2^29 tokens", name);
    if (nBuckets < 1 || nBuckets > kMaxBuckets) return fail("%s: %d buckets (supported: 1 to %d)", name, nBuckets, kMaxBuckets);
    if (nOffsets < 1 || nOffsets > kMaxOffsets) return fail("%s: %d offsets (supported: 1 to %d)", name, nOffsets, kMaxOffsets);
    if (nZero < -(1 << 30) || nZero > 1 << 30) return fail("%s: the map's zero is past +-2^30", name);   // its ends' differences fit 32 bits
    if (nHeads > 65535) return fail("%s: more than 65535 heads", name);
    if (!pTable || !pBuckets) return fail("%s: null pointer", name);
    if (!pQueryPos != !pKeyPos && nSeqQ > 0 && nSeqK > 0) return fail("%s: positions of queries and keys go together", name);
    if (!aligned4(pTable) || !aligned4(pBuckets) || !aligned4(pQueryPos) || !aligned4(pKeyPos))
        return fail("%s: a pointer is not aligned to its elements", name);
    p.table = pTable; p.bucketOf = pBuckets;
    p.qPos = pQueryPos; p.kPos = pKeyPos;
    p.nBuckets = nBuckets; p.nOffsets = nOffsets; p.zero = nZero;
    return 0;
}

}  // namespace

}  // namespace omhip

using namespace omhip;

extern "C" {

int omHipAttentionBiasForwardHalf(int nDtype, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV, long long nLdQ,
                                  long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                                  const int* pKeyLens, int bCausal, const float* pTable, const int* pBuckets,
                                  const int* pQueryPos, const int* pKeyPos, int nBuckets, int nOffsets, int nZero, uint16_t* pOut,
                                  float* pLse, int nBatch, int nSeqQ, int nSeqK, int nHeads, int nKVHeads, int nHeadDim,
                                  float fScale) {
    const char* name = "omHipAttentionBiasForwardHalf";
    clearError();
    const int rc = checkSizes(name, nDtype, nLdQ, nStrideQ, nLdKV, nStrideKV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads,
                              nHeadDim, fScale, false);
    AttnBiasParams p{};
    if (rc < 0 ||
        biasArguments(p, name, pTable, pBuckets, pQueryPos, pKeyPos, nBuckets, nOffsets, nZero, nSeqQ, nSeqK, nHeads))
        return -1;
    if (rc || nSeqQ == 0) return 0;
    if (forwardArguments(p, name, pQ, pK, pV, nLdQ, nStrideQ, nLdKV, nStrideKV, pQueryLens, pKeyLens, bCausal, pOut, pLse, nBatch,
                         nSeqQ, nSeqK, nHeads, nKVHeads, nHeadDim, fScale) ||
        forwardParts(p, (nSeqK + kTileKeys - 1) / kTileKeys))
        return -1;
    return nDtype == 1 ? forward<true, kAtBias>(p) : forward<false, kAtBias>(p);
}

int omHipAttentionBiasBackwardHalf(int nDtype, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV, long long nLdQ,
                                   long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                                   const int* pKeyLens, int bCausal, const float* pTable, const int* pBuckets,
                                   const int* pQueryPos, const int* pKeyPos, int nBuckets, int nOffsets, int nZero,
                                   const uint16_t* pOut, const float* pLse, const uint16_t* pGradOut, uint16_t* pGradQ,
                                   uint16_t* pGradK, uint16_t* pGradV, float* pGradTable, int nBatch, int nSeqQ, int nSeqK,
                                   int nHeads, int nKVHeads, int nHeadDim, float fScale) {
    const char* name = "omHipAttentionBiasBackwardHalf";
    clearError();
    const int rc = checkSizes(name, nDtype, nLdQ, nStrideQ, nLdKV, nStrideKV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads,
                              nHeadDim, fScale, true);
    AttnBiasParams p{};
    if (rc < 0 ||
        biasArguments(p, name, pTable, pBuckets, pQueryPos, pKeyPos, nBuckets, nOffsets, nZero, nSeqQ, nSeqK, nHeads))
        return -1;
    if (!pGradTable) return fail("%s: null pointer", name);
    if (!aligned4(pGradTable)) return fail("%s: a pointer is not aligned to its elements", name);
    p.gradTable = pGradTable;
    p.H = nHeads;
    if (rc || (nSeqQ == 0 && nSeqK == 0)) return tableGradient(p, 0);
    if (backwardArguments(p, name, pQ, pK, pV, nLdQ, nStrideQ, nLdKV, nStrideKV, pQueryLens, pKeyLens, bCausal, pOut, pLse,
                          pGradOut, pGradQ, pGradK, pGradV, nBatch, nSeqQ, nSeqK, nHeads, nKVHeads, nHeadDim, fScale))
        return -1;
    const long long blocksQ = (nSeqQ + kBlockQ - 1) / kBlockQ, blocksK = (nSeqK + kBlockQ - 1) / kBlockQ;
    const int tiles = (nSeqK + kTileKeys - 1) / kTileKeys;
    // two workgroups a CU at any head dimension. Whole backward, us, with two (one, three, four): causal 2 x 2048, 8 heads of 32: 74
    // (89, 73, 75), of 64: 94 (106, 95, 98), of 128: 167 (172, 178, 189); 1 x 4096, 4 of 32: 73 (91, 72, 75). Without a mask walks are
    // alike and one is enough: 4 x 1024, 8 of 64: 84 (78, 90, 92), 2 x 1000, 8 on 4 of 96: 85 (76, 85, 85).
    p.parts = walkParts((long long)nBatch * nKVHeads * blocksK, p.SqP / kTileKeys * (nHeads / nKVHeads), 2LL * cuCount());
    p.partRows = (nSeqK + kBlockQ - 1) / kBlockQ * kBlockQ;
    // A workgroup of dQ keeps its sums over the images that it takes: so many groups of images that the grid has eight
    // workgroups a CU. Whole backward, us, with 2, 4, 8 and 16 a CU: 1024 x 49, 4 heads of 32: 85, 70, 72, 75; 2000 x 49, 6 of 64: 329, 316,
    // 289, 286; 64 x 197, 12 of 64: 120, 125, 120, 120; 64 x 257, 16 of 96: 532, 535, 523, 542.
    const int parts = walkParts((long long)nBatch * nHeads * blocksQ, tiles, 2LL * cuCount());
    const long long each = std::max(1LL, nHeads * blocksQ * parts);   // workgroups of a group
    p.imageGroups = (int)std::clamp<long long>(8LL * cuCount() / each, 1, nBatch);
    const long long units = nSeqQ > 0 ? p.imageGroups * blocksQ * parts : 0;
    if (units > INT_MAX) return fail("%s: too many blocks of queries", name);
    const size_t sumFloats = (size_t)nHeads * nOffsets, tableFloats = (size_t)nHeads * (nOffsets + 2 * kMapEnd);
    float* more = nullptr;
    if (backwardParts(p, tiles, p.parts > 1 ? (size_t)nBatch * nKVHeads * blocksK * p.parts * kBlockQ * nHeadDim : 0,
                      nSeqQ > 0 ? tableFloats + sumFloats * (1 + (size_t)units) : 0, &more))
        return -1;
    p.tables = more;
    p.offsetSums = more + tableFloats;
    p.bins = p.offsetSums + sumFloats;
    if (nDtype == 1 ? backward<true, kAtBias>(p) : backward<false, kAtBias>(p)) return -1;
    return tableGradient(p, (int)units);
}

}  // extern "C"
