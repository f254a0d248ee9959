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

// ---------------------------------------------------------------- few queries: a sequence's next tokens
// At most 64 workgroups share a key head's keys, whose parts the last one reads alone. One query, us, with 16, 32, 64 and 128: a cache
// of 16384, 8 heads of 64: 14, 13, 18, 28; of 65536, 8 on 2 of 128: 42, 27, 22, 26; of 131072, 4 of 64: 64, 37, 30, 35.
constexpr int kTokenKeys = 32, kMaxTokenParts = 64;

struct TokenParams : AttnWindowParams {
    int rows;             // queries of a key head, Sq * H / Hkv, at most 32
    int parts;            // workgroups of a key head
    float* partial;       // [B * Hkv, parts, rows, D + 4]: contexts, then their log-sum-exp
    unsigned* arrivals;   // [B * Hkv], zero at rest
};

// The queries of all heads that read a key head are the 32 columns of one MFMA operand, so its keys are read once. A wave
// takes 32 keys in sight at a time, S^T = K Q^T, running softmax, O^T += V^T P^T as in the forward kernel; nothing is shared
// between waves before their contexts are joined in LDS, and the workgroups' by the last one to arrive, with accesses coherent
// past the XCDs' L2s (partials have landed before the counter goes up). Bound by latency: the keys in sight of a cache are a
// few 100 KB, which enough workgroups read at once. Measured: 16 caches of up to 8192 tokens, 16 heads on 4 of 128, window
// 1024, 4 first keys: 12 us (the forward kernel and its join 27.5); one of 4096, 8 heads of 64, window 256: 7.2 (10.0).
template <bool BF16, int KD>
__global__ __launch_bounds__(256, 2) void attn_window_token_kernel(TokenParams p) {
    using T = AtTile<KD>;
    constexpr float kShift = BF16 ? 0.f : 6.f;   // as in the forward kernel
    constexpr int N = kTokenKeys * T::RS, CHUNKS = T::RS / 4;
    __shared__ __attribute__((aligned(256))) uint16_t tiles[4 * 2 * N];   // a wave's K and V, then its contexts [32, RS] in fp32
    __shared__ float tops[4][32], totals[4][32];
    __shared__ int last;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = lane & 31, h = lane >> 5;
    const int part = (int)(blockIdx.x % (uint32_t)p.parts);
    const uint32_t bh = blockIdx.x / (uint32_t)p.parts;
    const int b = (int)(bh / (uint32_t)p.Hkv), kvHead = (int)(bh % (uint32_t)p.Hkv), group = p.H / p.Hkv;
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk), off = nK - nQ;
    const int token = l / group, head = kvHead * group + l % group;
    const bool some = l < p.rows && token < nQ;

    // tiles in sight: of the first keys, then of the window from the first query's on
    const int sinkTiles = (min(p.first, nK) + kTokenKeys - 1) / kTokenKeys;
    const int t0 = max(0, off - p.window + 1) / kTokenKeys, t1 = nQ > 0 ? (nK + kTokenKeys - 1) / kTokenKeys : 0;
    const AtWalk walk = sinkTiles >= t0 ? AtWalk{t1, 0, 0} : AtWalk{max(0, sinkTiles + t1 - t0), sinkTiles, t0 - sinkTiles};
    const int end = (int)((long long)walk.n * (part + 1) / p.parts);
    int i = (int)((long long)walk.n * part / p.parts) + wave;

    uint16_t *kt = tiles + wave * 2 * N, *vt = kt + N;
    const long long kv = (long long)b * p.skv + (long long)kvHead * p.D;
    auto fetch = [&](int key0) {
        T::start(p.k + kv + (long long)key0 * p.ldkv, nK - key0, p.ldkv, p.D, kt, lane);
        T::start(p.v + kv + (long long)key0 * p.ldkv, nK - key0, p.ldkv, p.D, vt, lane);
    };
    if (i < end) fetch(walk.tile<kAtWindow>(i) * kTokenKeys);
    const float c = fmaxf(fabsf(p.scale * kAtLog2e), FLT_MIN);
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    const uint16_t* row = p.q + (long long)b * p.sq + (long long)token * p.ldq + (long long)head * p.D;
    at_u32x4 qf[T::NS];
#pragma unroll
    for (int s = 0; s < T::NS; ++s) {
        qf[s] = T::direct(row, some, s, h, p.D);
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[s][e] ^= flip;
    }
    const typename T::Lane at(lane);
    const AtReach<kAtWindow> reach{nK, 0, off, 0, 0, 0, p.window, p.first, p.causal != 0};
    at_f32x16 o[KD];
#pragma unroll
    for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m = -INFINITY, sum = 0.f;
    for (; i < end; i += 4) {
        const int key0 = walk.tile<kAtWindow>(i) * kTokenKeys;
        __builtin_amdgcn_s_waitcnt(0);
        at_f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int st = 0; st < T::NS; ++st) s = atMfma<BF16>(at.natural(kt, 0, st), qf[st], s);
        AtSeen seen = reach.seen(token, key0, h);
        if (!some) seen.bits[0] = 0u;
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = seen.pick<kAtWindow>(8 * (r / 4) + r % 4, s[r], -INFINITY);
            top = fmaxf(top, s[r]);
        }
        top = atMaxHalves(top);
        const float next = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next) * c);
        const float base = next == -INFINITY ? 0.f : kShift - next * c;
        sum *= alpha;
        m = next;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, base));
            sum += s[r];
        }
#pragma unroll
        for (int dt = 0; dt < KD; ++dt) {
#pragma unroll
            for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
#pragma unroll
            for (int u = 0; u < 2; ++u) o[dt] = atMfma<BF16>(at.transposed(vt, 16 * u, dt), atPack8<BF16>(s, u), o[dt]);
        }
        __builtin_amdgcn_s_waitcnt(0);   // the tile is read
        if (i + 4 < end) fetch(walk.tile<kAtWindow>(i + 4) * kTokenKeys);
    }
    sum = atSumHalves(sum);
    if (h == 0) {
        tops[wave][l] = m;
        totals[wave][l] = sum;
    }
    float* own = reinterpret_cast<float*>(kt);   // chunk c of 4 values of column l in slot c ^ l: a read or write hits all banks
#pragma unroll
    for (int dt = 0; dt < KD; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<at_f32x4*>(own + l * T::RS + ((8 * dt + r / 2 + h) ^ (l & (CHUNKS - 1))) * 4) =
                at_f32x4{o[dt][r], o[dt][r + 1], o[dt][r + 2], o[dt][r + 3]};
    __syncthreads();

    const int chunks = p.D / 4, work = p.rows * chunks;
    auto result = [&](int column, int chunk, const at_f32x4& v, float lse) {   // a column's context and log-sum-exp
        const int i = column / group, j = kvHead * group + column % group;
        uint16_t* to = p.out + (((long long)b * p.Sq + i) * p.H + j) * p.D + chunk * 4;
        *reinterpret_cast<at_u32x2*>(to) = at_u32x2{atPack2<BF16>(v[0], v[1]), atPack2<BF16>(v[2], v[3])};
        if (chunk == 0) p.lse[((long long)b * p.H + j) * p.Sq + i] = lse;
    };
    const int pitch = p.D + 4;
    const uint32_t partBytes = (uint32_t)(p.rows * pitch) * 4u;
    const __amdgpu_buffer_rsrc_t partials = bufferRsrc(p.partial + (long long)bh * p.parts * p.rows * pitch, p.parts > 1 ? partBytes * p.parts : 0u);
    for (int x = (int)threadIdx.x; x < work; x += 256) {
        const int column = x / chunks, chunk = x % chunks;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, tops[w][column]);
        float total = 0.f;
        at_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = tops[w][column] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((tops[w][column] - top) * c);
            total += f * totals[w][column];
            v += f * *reinterpret_cast<const at_f32x4*>(reinterpret_cast<const float*>(tiles + w * 2 * N) + column * T::RS +
                                                        (chunk ^ (column & (CHUNKS - 1))) * 4);
        }
        const bool empty = total == 0.f;
        v = empty ? at_f32x4{0.f, 0.f, 0.f, 0.f} : v * (1.f / total);   // not by 0: a NaN of V is in the sums of hidden columns too
        const float lse = empty ? -INFINITY : top * (c * kAtLn2) + (__logf(total) - kShift * kAtLn2);
        if (p.parts == 1) {
            result(column, chunk, v, lse);
        } else {
            const uint32_t to = (uint32_t)((part * p.rows + column) * pitch + chunk * 4) * 4u;
            bufStore4Agent(partials, to, 0, v);
            if (chunk == 0) bufStore1Agent(partials, to + (uint32_t)p.D * 4u, 0, lse);
        }
    }
    if (p.parts == 1) return;
    __builtin_amdgcn_s_waitcnt(0);   // this wave's partials have landed
    __syncthreads();                 // every wave's have
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(p.arrivals + bh, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(p.parts - 1);
    __syncthreads();
    if (!last) return;
    for (int x = (int)threadIdx.x; x < work; x += 256) {   // as attn_train_join_kernel, eight parts' loads at a time
        const int column = x / chunks, chunk = x % chunks;
        float top = -INFINITY, total = 0.f;
        at_f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int first = 0; first < p.parts; first += 8) {
            float lse[8], most = top;
            f32x4 part8[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {   // past the last part: out of range, no access
                const uint32_t from = (uint32_t)(((first + k) * p.rows + column) * pitch) * 4u;
                part8[k] = bufLoad4Agent(partials, first + k < p.parts ? from + (uint32_t)chunk * 16u : kOOB, 0);
                lse[k] = bufLoad1Agent(partials, first + k < p.parts ? from + (uint32_t)p.D * 4u : kOOB, 0);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (first + k >= p.parts) lse[k] = -INFINITY;
                most = fmaxf(most, lse[k]);
            }
            const float from0 = most == -INFINITY ? 0.f : most, alpha = top == -INFINITY ? 0.f : __expf(top - from0);
            total *= alpha;
            v *= alpha;
            top = most;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float w = __expf(lse[k] - from0);
                total += w;
                v += w * part8[k];
            }
        }
        const bool empty = total == 0.f;
        v = empty ? at_f32x4{0.f, 0.f, 0.f, 0.f} : v * (1.f / total);
        result(column, chunk, v, empty ? -INFINITY : (top == -INFINITY ? 0.f : top) + __logf(total));
    }
    if (threadIdx.x == 0) __hip_atomic_store(p.arrivals + bh, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
}

template <bool BF16>
int launchToken(const TokenParams& p) {
    const dim3 grid((uint32_t)(p.B * p.Hkv) * (uint32_t)p.parts);
    switch ((p.D + 31) / 32) {
        case 1: hipLaunchKernelGGL((attn_window_token_kernel<BF16, 1>), grid, dim3(256), 0, stream(), p); break;
        case 2: hipLaunchKernelGGL((attn_window_token_kernel<BF16, 2>), grid, dim3(256), 0, stream(), p); break;
        case 3: hipLaunchKernelGGL((attn_window_token_kernel<BF16, 3>), grid, dim3(256), 0, stream(), p); break;
        default: hipLaunchKernelGGL((attn_window_token_kernel<BF16, 4>), grid, dim3(256), 0, stream(), p); break;
    }
    OMHIP_CHECK_LAUNCH();
    return 0;
}

// Queries of few tokens: workgroups share a key head's keys in sight, 32 a wave, as far as they all run at once (16 caches of up to
// 8192, 16 heads on 4 of 128, window 1024: 8 a key head 11.9 us, one 15.0; 8 of 8192, 8 of 128, all keys in sight: 44 and 76).
int tokens(const AttnWindowParams& p, int nDtype) {
    TokenParams t{};
    static_cast<AttnWindowParams&>(t) = p;
    t.rows = p.Sq * (p.H / p.Hkv);
    const long long heads = (long long)p.B * p.Hkv, resident = (long long)(p.D <= 64 ? 4 : 2) * cuCount();
    const long long seen = std::min<long long>(p.Sk, (long long)p.window + p.Sq + p.first) / kTokenKeys + 2;   // tiles
    t.parts = (int)std::clamp<long long>(std::min((seen + 3) / 4, (resident + heads - 1) / heads), 1, kMaxTokenParts);
    if (t.parts > 1) {
        t.partial = static_cast<float*>(workspace((size_t)heads * t.parts * t.rows * (p.D + 4) * sizeof(float), kWsOperand));
        t.arrivals = static_cast<unsigned*>(workspace((size_t)heads * sizeof(unsigned), kWsCounters));
        if (!t.partial || !t.arrivals) return -1;   // workspace() recorded the cause
    }
    return nDtype == 1 ? launchToken<true>(t) : launchToken<false>(t);
}

// ---------------------------------------------------------------- sizes
// Sizes past checkSizes: what a window adds; 0 or -1.
int checkWindow(const char* name, int nSeqQ, int nSeqK, int nWindow, int nFirst) {
    if (nSeqQ > kMaxSeq || nSeqK > kMaxSeq) return fail("%s: a sequence exceeds 2^29 tokens", name);
    if (nWindow < 1) return fail("%s: a window holds one position at least", name);
    if (nFirst < 0) return fail("%s: negative number of first tokens", name);
    return 0;
}

// First keys that get workgroups of their own; more go with their blocks' walks over everything. Backward with workgroups of their
// own (whole walks), us, of first keys of        32         256         300         512         1024
//   2 x 4096, 16 heads on 4 of 128, window 512   194 (330)  236 (347)   257 (350)   292 (366)   443 (399)
//   1 x 8192, 8 of 64, window 256                 55 (137)   69 (142)    76 (144)    88 (149)   118 (164)
//   4 x 2048, 8 of 64, window 128 both ways       51 (67)    74 (74)     77 (81)     87 (89)    126 (122)
//   16 x 1024, 4 of 32, window 64                 32 (38)    43 (44)     47 (47)     53 (52)     67 (55)
constexpr int kMaxSinks = 256;

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
    if ((long long)nSeqQ * (nHeads / nKVHeads) <= 32) return tokens(p, nDtype);
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
    const int group = nHeads / nKVHeads;
    const long long room = (nHeadDim <= 64 ? 2LL : 1LL) * cuCount();   // workgroups of dK and dV that run at once
    const int allQ = p.SqP / kTileKeys, allK = (nSeqK + kTileKeys - 1) / kTileKeys;
    const long long blocks = (nSeqK + kBlockQ - 1) / kBlockQ, heads = (long long)nBatch * nKVHeads;
    const int walk = windowTiles(p.window, p.causal, allQ);   // of a block of keys, for each query head
    p.parts = walkParts(heads * blocks, walk * group, room);
    // The first keys: by workgroups of their own, unless they are so many that their blocks may as well walk over everything
    // (or more than a launch's 2^32 - 1 threads take), the window is as wide as the sequences, or there are no queries (and no
    // workspace).
    const long long groups = heads * ((p.first + 31) / 32);
    if (p.first > kMaxSinks || groups * 256 > 0xffffffffLL) {
        p.sinkBlocks = (p.first + kBlockQ - 1) / kBlockQ;
        p.parts = walkParts(heads * blocks, allQ * group, 2 * room);
    } else if (p.first > 0 && nSeqQ > 0 && p.window < std::max(nSeqQ, nSeqK)) {
        p.sinkParts = (int)std::clamp<long long>(std::min<long long>(room / groups,
                                                                     ((long long)std::max(1, allQ - walk) * group + 3) / 4), 1, 64);
    }
    p.partRows = p.parts > 1 ? (int)blocks * kBlockQ : p.sinkParts > 0 ? p.first : 0;
    const size_t sinks = (size_t)heads * p.sinkParts * ((p.first + 31) / 32 * 32) * nHeadDim;
    float* more = nullptr;
    if (backwardParts(p, std::min(allK, windowTiles(p.window, p.causal, allK) + (p.first + kTileKeys - 1) / kTileKeys),
                      (size_t)heads * p.parts * p.partRows * nHeadDim, 2 * sinks, &more))
        return -1;
    if (p.sinkParts > 0 && p.parts == 1) {
        p.arrivals = static_cast<unsigned*>(workspace((size_t)heads * ((p.first + 31) / 32) * sizeof(unsigned), kWsCounters));
        if (!p.arrivals) return -1;   // workspace() recorded the cause
    }
    p.sinkDk = more;
    p.sinkDv = more + sinks;
    return nDtype == 1 ? backward<true, kAtWindow>(p) : backward<false, kAtWindow>(p);
}

}  // extern "C"
