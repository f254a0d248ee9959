// attn_train_kernels.hpp — the kernels of attention for training: a forward pass
// that keeps each row's log-sum-exp, and the backward pass that computes the
// probabilities again from it.
//
// With S = scale Q K^T (+ a bias) over the keys that a query sees, P = exp(S -
// lse), lse = log sum exp S:
//   O  = P V                    dV = P^T dO
//   dP = dO V^T                 dS = P (dP - delta),  delta_i = sum_d dO_id O_id
//   dQ = scale dS K             dK = scale dS^T Q
// A key head's dK and dV are the sums over the query heads that read it. All
// sums are in fp32 in a fixed order; the products take P and dS rounded to the
// data's type, as operands of the matrix cores.
//
// Query i sees key j where j < the image's key length and, if causal,
// j <= i's position. A query that sees none, or whose scores are all -inf, has
// O = 0 and lse = -inf and passes no gradient. What else a query sees, and
// where it stands, is the kernels' view (AtView): attn_train.hip, attn_window.hip
// and attn_bias.hip hold the entries of one each.
#pragma once

#include "attn_share.hpp"
#include "attn_tile.hpp"
#include "buffer_io.hpp"
#include "omhip_internal.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace omhip {

namespace {

constexpr int kWaves = 4;         // of a workgroup that holds queries; pairs of waves of one that holds keys
constexpr int kTileKeys = 64;    // keys per LDS tile
constexpr int kBlockQ = 32 * kWaves;

struct AttnTrainParams {
    const uint16_t *q, *k, *v;
    long long ldq, sq, ldkv, skv;   // elements between tokens, between images
    const int *qLens, *kLens;
    int B, Sq, Sk, H, Hkv, D, causal;
    float scale;
    // forward: the context [B, Sq, H, D] and log-sum-exp [B, H, Sq]; backward: their saved values
    uint16_t* out;
    float* lse;
    // backward
    const uint16_t* gradOut;
    uint16_t *dq, *dk, *dv;
    float* stats;                   // [B, H, SqP / 32]: shift of 32 rows, then their delta
    int SqP;                        // Sq rounded up to whole tiles
    // workgroups that share a block's walk, and their fp32 results where there are several
    int keyParts;                   // forward, dQ: of a block of queries
    float *rowPart, *lsePart;       // [B, Sq, H, keyParts, D] contexts or dQ, [B, H, Sq, keyParts] log-sum-exps
    int parts;                      // dK, dV: of a block of keys
    float *dkPart, *dvPart;         // [B, Hkv, parts, partRows, D], in those workgroups' order
    int partRows;                   // blocks * kBlockQ; of a window with one part, the first keys
    uint32_t heads, blocks;         // grid: heads x blocks workgroups
};

// What a query sees beside the keys of its image below the causal mask's border.
enum AtView {
    kAtPlain,    // all of them; query i stands at i + Sk - Sq
    kAtWindow,   // those in a window around it, and the image's first few
    kAtBias,     // all of them, with a bias by the distance of two positions
};
// In the last two an image's last query stands at its last key, i + nK - nQ for query i.

struct AttnWindowParams : AttnTrainParams {
    int window, first;         // key j where |position - j| < window or j < first
    // dK, dV of the first keys: blocks that walk over all queries (where they are many), or else
    // sinkParts workgroups for each 32 of them that take the queries which the blocks' walks leave out
    int sinkBlocks, sinkParts;
    float *sinkDk, *sinkDv;    // [B, Hkv, sinkParts, first keys rounded to 32, D]
    unsigned* arrivals;        // [B * Hkv * (first + 31) / 32], zero at rest; null where the join adds the sinks' parts
};

constexpr float kNoBias = -1e30f;   // a bias at or below hides the key

struct AttnBiasParams : AttnTrainParams {
    const float* table;        // [nBuckets, H]
    const int* bucketOf;       // [nOffsets]: of a query's position - a key's + zero, taken into 0 .. nOffsets - 1
    const int *qPos, *kPos;    // [Sq], [Sk]; null: as above, and j
    int nBuckets, nOffsets, zero;
    int imageGroups;           // dQ: workgroups that share a head's block of queries over the images
    float* tables;             // [H, nOffsets + 2 kMapEnd] biases by offset times log2 e, which dQ leaves for dK, dV
    float* bins;               // [H, imageGroups * blocks * keyParts, nOffsets] sums of dS by offset
    float* offsetSums;         // [H, nOffsets]
    unsigned* arrivals;        // [H], zero at rest
    float* gradTable;          // [nBuckets, H]
};

template <int VIEW>
using AtParams = std::conditional_t<VIEW == kAtWindow, AttnWindowParams,
                                    std::conditional_t<VIEW == kAtBias, AttnBiasParams, AttnTrainParams>>;

// The tiles of keys that a block of queries walks over: 0 .. n - 1, of a window from the (skipFrom)th on `skip` later.
struct AtWalk {
    int n, skipFrom, skip;
    template <int VIEW>
    __device__ __forceinline__ int tile(int i) const {
        if constexpr (VIEW == kAtWindow) return i < skipFrom ? i : i + skip;
        return i;
    }
};

// Bits below n, of n from anywhere.
__device__ __forceinline__ uint32_t atBitsBelow(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// The keys that the lane's query sees, of a tile's key0 + 4 h ...: r below `end`; of a window a bit each, 0 .. 31 and 32 .. 63.
struct AtSeen {
    int end;
    uint32_t bits[2];
    // x where r is seen, else `hidden`. From a bit two operations (sign-extended, then one of two by bits); bounds took four.
    template <int VIEW>
    __device__ __forceinline__ float pick(int r, float x, float hidden) const {
        if constexpr (VIEW == kAtWindow) {
            const uint32_t all = (uint32_t)((int)(bits[r / 32] << (31 - r % 32)) >> 31);
            return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & all) | (__builtin_bit_cast(uint32_t, hidden) & ~all));
        }
        return r < end ? x : hidden;
    }
};

// A wave's 32 queries q0 ... of an image: what they see.
template <int VIEW>
struct AtReach {
    int nK, q0, off, end, begin, sinks, window, first;   // no key from `end` on, of a window none of sinks .. begin - 1
    bool causal;
    __device__ __forceinline__ bool tile(int key0) const {   // some key of the tile, as far as this tells
        if constexpr (VIEW == kAtWindow) return key0 < end && (key0 < sinks || key0 + kTileKeys > begin);
        return key0 < end;
    }
    __device__ __forceinline__ bool edge(int key0) const {   // some query does not see some of the tile's keys
        bool e = key0 + kTileKeys > nK || (causal && key0 + kTileKeys - 1 > q0 + off);
        if constexpr (VIEW == kAtWindow) e = e || key0 + kTileKeys > q0 + off + window || key0 < q0 + 32 + off - window;
        return e;
    }
    __device__ __forceinline__ AtSeen seen(int query, int key0, int h) const {
        const int at = key0 + 4 * h;
        if constexpr (VIEW == kAtWindow) {
            const int p = query + off, most = causal ? min(nK, p + 1) : nK;
            const int end = min(most, p + window) - at, begin = p - window + 1 - at, sink = min(first, most) - at;
            return {end,
                    {(atBitsBelow(end) & ~atBitsBelow(begin)) | atBitsBelow(sink),
                     (atBitsBelow(end - 32) & ~atBitsBelow(begin - 32)) | atBitsBelow(sink - 32)}};
        }
        return {(causal ? min(nK, query + off + 1) : nK) - at, {0u, 0u}};
    }
};

// What a block of queries first .. last sees of a window, as tiles and for the wave's own 32 queries. kEnd: the keys of the
// image below the block's causal border, 0 where the block has no query.
__device__ __forceinline__ void atWindow(const AttnWindowParams& p, int first, int last, int kEnd, AtReach<kAtWindow>& r, AtWalk& w) {
    const int begin = max(0, first + r.off - p.window + 1), end = min(kEnd, last + r.off + p.window);
    const int sinkTiles = (max(min(p.first, kEnd), 0) + kTileKeys - 1) / kTileKeys;
    const int t0 = begin / kTileKeys, t1 = max(t0, (max(end, 0) + kTileKeys - 1) / kTileKeys);
    if (sinkTiles >= t0)
        w = {max(sinkTiles, t1), 0, 0};
    else
        w = {sinkTiles + t1 - t0, sinkTiles, t0 - sinkTiles};
    r.begin = max(0, r.q0 + r.off - p.window + 1);
    r.sinks = min(p.first, r.end);
    r.end = max(min(r.end, r.q0 + 31 + r.off + p.window), r.sinks);
    r.window = p.window;
    r.first = p.first;
}

// The least and the largest of a wave's values.
__device__ __forceinline__ void atRange(int v, int& least, int& most) {
    int lo = v, hi = v;
#define OMHIP_AT_STEP(ctrl)                                                            \
    lo = min(lo, __builtin_amdgcn_update_dpp(lo, lo, ctrl, 0xf, 0xf, false));          \
    hi = max(hi, __builtin_amdgcn_update_dpp(hi, hi, ctrl, 0xf, 0xf, false));
    OMHIP_AT_STEP(0x111) OMHIP_AT_STEP(0x112) OMHIP_AT_STEP(0x114) OMHIP_AT_STEP(0x118)   // row_shr: lane 15 of each row of 16
    OMHIP_AT_STEP(0x142) OMHIP_AT_STEP(0x143)                                             // row_bcast 15, 31: lane 63
#undef OMHIP_AT_STEP
    least = __builtin_amdgcn_readlane(lo, 63);
    most = __builtin_amdgcn_readlane(hi, 63);
}

// Arrays by offset in LDS have 64 entries more at either end, one of a lane each at least, for differences past the map:
// lanes that add to one address are served one after another. A lane's entry is its offset taken into -64 + lane .. nOffsets +
// lane, which leaves what is inside the map where it is, and the rest in the ends' entries.
constexpr int kMapEnd = 64;
__device__ __forceinline__ int atEntry(const AttnBiasParams& p, int q, int k, int lane) {
    const int d = __builtin_elementwise_sub_sat(q, k);   // a difference past 32 bits is past the map too
    int e;   // min(max(d, low), high): the compiler does not know that low is below high
    asm("v_med3_i32 %0, %1, %2, %3" : "=v"(e) : "v"(d), "v"(lane - kMapEnd - p.zero), "v"(p.nOffsets + lane - p.zero));
    return e + p.zero;
}

// A head's biases by offset and the ends', times log2 e, into `to` by a workgroup: -inf where the table hides the key, 0 where the
// offset has no bucket. Four entries of a thread are under way at once: one by one, every entry would wait for its bucket and
// then for its bias (ViT-B/16 b64, 14 x 14 grid: forward 35.9 -> 34.6 us).
template <int THREADS, class F>
__device__ __forceinline__ void atFillBiases(const AttnBiasParams& p, int head, F&& to) {
    constexpr int N = 4;
    const int each = p.nOffsets + 2 * kMapEnd;
    for (int i0 = (int)threadIdx.x; i0 < each; i0 += N * THREADS) {
        int b[N];
        float v[N];
#pragma unroll
        for (int k = 0; k < N; ++k) b[k] = p.bucketOf[min(max(i0 + k * THREADS - kMapEnd, 0), p.nOffsets - 1)];
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = p.table[(long long)((uint32_t)b[k] < (uint32_t)p.nBuckets ? b[k] : 0) * p.H + head];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if ((uint32_t)b[k] >= (uint32_t)p.nBuckets) v[k] = 0.f;
            if (i0 + k * THREADS < each) to(i0 + k * THREADS, v[k] <= kNoBias ? -INFINITY : v[k] * kAtLog2e);
        }
    }
}

// Where the offsets of a block of pairs lie: all past one end of the map (one bias for all), or anywhere.
enum AtOffsets { kAtLow, kAtHigh, kAtMap };
__device__ __forceinline__ AtOffsets atOffsets(const AttnBiasParams& p, int qLeast, int qMost, int kLeast, int kMost) {
    if (__builtin_elementwise_sub_sat(qMost, kLeast) <= -p.zero) return kAtLow;
    return __builtin_elementwise_sub_sat(qLeast, kMost) >= p.nOffsets - 1 - p.zero ? kAtHigh : kAtMap;
}

// f(i, entry) of 4 N pairs: the lane's own token, and the other side's 8 (i / 4) + i % 4 of `theirs`.
template <bool QUERY, int N = 4, class F>
__device__ __forceinline__ void atForEntries(const AttnBiasParams& p, int own, const int* theirs, int lane, F&& f) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const at_i32x4 pos = *reinterpret_cast<const at_i32x4*>(theirs + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) f(4 * j + e, atEntry(p, QUERY ? own : pos[e], QUERY ? pos[e] : own, lane));
    }
}

// A wave's sums of dS by offset. They are of type T: an LDS add of doubles takes 9 cycles of a CU, one of floats 177 (64 lanes,
// no two on one address), so floats are for maps that leave no room for doubles (mostWide). A wave's instructions are done in order; the
// lanes of one on the same address are served in an order of the hardware's, which has repeated in every run but which nothing
// promises.
// Written out: before an atomic of its own the compiler waits for every copy into LDS under way. The wave waits for its adds
// (__builtin_amdgcn_s_waitcnt) before the barrier behind which they are read.
__device__ __forceinline__ uint32_t atLdsAddress(const void* at) {
    return (uint32_t)reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)at);
}
__device__ __forceinline__ void atAdd(double* at, double v) { asm volatile("ds_add_f64 %0, %1" : : "v"(atLdsAddress(at)), "v"(v)); }
__device__ __forceinline__ void atAdd(float* at, float v) { asm volatile("ds_add_f32 %0, %1" : : "v"(atLdsAddress(at)), "v"(v)); }

// Values from LDS, waited for here: for arrays that the compiler cannot tell from those which copies are under way to.
__device__ __forceinline__ float atReadOne(const float* at) {
    float v;
    asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(atLdsAddress(at)));
    return v;
}
__device__ __forceinline__ void atReadEight(const uint32_t (&from)[8], float (&v)[8]) {
    asm volatile("ds_read_b32 %0, %8\n\tds_read_b32 %1, %9\n\tds_read_b32 %2, %10\n\tds_read_b32 %3, %11\n\t"
                 "ds_read_b32 %4, %12\n\tds_read_b32 %5, %13\n\tds_read_b32 %6, %14\n\tds_read_b32 %7, %15\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(from[0]), "v"(from[1]), "v"(from[2]), "v"(from[3]), "v"(from[4]), "v"(from[5]), "v"(from[6]),
                   "v"(from[7]));
}

// Stores a wave's 32 rows of a transposed result (the lane's column is row l; its registers hold head dimensions 32 dt +
// 8 (r / 4) + 4 h + r % 4) times f, or zeros, as halves. Rows are turned around in `stage`, 32 rows of the wave's own in
// LDS, and leave as whole chunks of 16 bytes, 64 / CH rows an instruction: stored from the registers, every instruction
// would touch 32 rows for 16 bytes each. rows: how many of the 32 exist.
template <bool BF16, int KD>
__device__ __forceinline__ void storeRows(uint16_t* to, long long ld, int rows, const at_f32x16 (&acc)[KD], float f, bool zero,
                                          uint16_t* stage, int lane, int D) {
    using T = AtTile<KD>;
    const int l = lane & 31, h = lane >> 5;
#pragma unroll
    for (int dt = 0; dt < KD; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<at_u32x2*>(stage + l * T::RS + ((4 * dt + r / 4) ^ T::swizzle(l)) * 8 + 4 * h) =
                zero ? at_u32x2{0u, 0u}
                     : at_u32x2{atPack2<BF16>(acc[dt][r] * f, acc[dt][r + 1] * f),
                                atPack2<BF16>(acc[dt][r + 2] * f, acc[dt][r + 3] * f)};
    __builtin_amdgcn_wave_barrier();   // the wave's own LDS operations complete in order
#pragma unroll
    for (int i = 0; i < T::CH / 2; ++i) {
        const int id = i * 64 + lane, row = id / T::CH, c = id % T::CH;
        const at_u32x4 v = *reinterpret_cast<const at_u32x4*>(stage + row * T::RS + (c ^ T::swizzle(row)) * 8);
        if (row < rows && c * 8 < D) *reinterpret_cast<at_u32x4*>(to + (long long)row * ld + c * 8) = v;
    }
}

template <int KD>
__device__ __forceinline__ void storeColumnF32(float* row, const at_f32x16 (&acc)[KD], float f, int h, int D,
                                               bool zero) {
#pragma unroll
    for (int dt = 0; dt < KD; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = 32 * dt + 2 * r + 4 * h;
            if (d < D)
                *reinterpret_cast<at_f32x4*>(row + d) =
                    zero ? at_f32x4{0.f, 0.f, 0.f, 0.f}
                         : at_f32x4{acc[dt][r] * f, acc[dt][r + 1] * f, acc[dt][r + 2] * f, acc[dt][r + 3] * f};
        }
}

// Positions of `count` tokens from `first` on into LDS, by one wave; they are there after the next wait and barrier. Past
// `tokens` they are 0. Without positions token t stands at t + off.
__device__ __forceinline__ void atCopyPositions(const int* positions, int first, int count, int tokens, int off, int lane, int* to) {
    if (!positions) {
        if (lane < count) to[lane] = first + lane + off;
    } else if (lane < count) {
        const uint32_t bytes = (uint32_t)max(0, min(count, tokens - first)) * 4u;
        atCopy4(atView(positions + first, bytes), reinterpret_cast<float*>(to), (uint32_t)lane * 4u);
    }
}
// The position of a lane's own token and the range of the wave's; past `tokens` they go on from the last one's (on one place,
// their lanes' adds of nothing to one sum would be served one after another).
__device__ __forceinline__ int atOwnPosition(const int* positions, int token, int tokens, int off, int& least, int& most) {
    const int t = min(token, tokens - 1);
    const int v = !positions ? token + off : t >= 0 ? __builtin_elementwise_add_sat(positions[t], token - t) : 0;
    atRange(v, least, most);
    return v;
}

// ---------------------------------------------------------------- forward
// A workgroup holds 128 queries of a head, 32 a wave, and walks the keys 64 at
// a time: S^T = K Q^T (the lane's column is its query), the softmax with a
// running reference m of the row's maximum, O^T += V^T P^T.
//  * p = exp2(c s - c m + shift), c = |scale| log2 e (a negative scale flips Q's
//    signs as it is loaded). m only moves when a tile's maximum exceeds it by
//    more than 8 / c, so the sums are rescaled a few times a row instead of
//    every tile; p is at most 2^(8 + shift).
//  * shift: fp16 keeps 2^-14 .. 2^16 at full precision, so its p is raised by
//    2^6 (at most 2^14); bf16 needs none.
//  * the next tile's K and V land in the other pair of buffers meanwhile.
// 32 x 32 x 16 MFMAs with 32 queries a wave: an LDS fragment feeds 32 columns, half of what 16 x 16 tiles would read.
// Measured: 2 images x 4096 tokens, 16 query heads on 4 of 128, causal, bf16: 141-160 us by card (0.86-0.98 PFLOP/s of the
// visible pairs; a large library product reaches 1.27 here), matrix cores busy 56 % of CU cycles at 1.94 GHz, no bank
// conflicts: bound by the two waves of a SIMD that share its issue between MFMAs (1024 cycles a tile) and exponentials (1050).
// ViT-B/16 b64 (197 tokens, 768 heads of 64, fp16): 23.6-25.5 us, 3.1-3.3 TB/s over its compulsory bytes; four tiles a walk,
// so its start and end (copies in, results out), which nothing overlaps, are half of it.
template <bool BF16, int KD, int VIEW, int W>
__global__ __launch_bounds__(64 * W, 2) void attn_train_forward_kernel(AtParams<VIEW> p) {
    using T = AtTile<KD>;
    constexpr int BLOCK = 32 * W;   // queries of the workgroup
    constexpr float kShift = BF16 ? 0.f : 6.f;
    __shared__ __attribute__((aligned(256))) uint16_t k0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t k1[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v1[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(16))) int at0[VIEW == kAtBias ? kTileKeys : 4];   // positions of the keys
    __shared__ __attribute__((aligned(16))) int at1[VIEW == kAtBias ? kTileKeys : 4];
    extern __shared__ float biasesLds[];   // [nOffsets] and the ends
    const float* biases = biasesLds + kMapEnd;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = lane & 31, h = lane >> 5;
    uint32_t bh, qb;
    atPlace(blockIdx.x, p.heads, p.blocks * p.keyParts, p.causal, bh, qb);
    const int part = (int)(qb % (uint32_t)p.keyParts);
    qb = p.blocks - 1 - qb / (uint32_t)p.keyParts;   // causal: the longest walks first
    const int b = (int)(bh / (uint32_t)p.H), head = (int)(bh % (uint32_t)p.H);
    const int kvHead = head / (p.H / p.Hkv);
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk);
    const int off = VIEW == kAtPlain ? p.Sk - p.Sq : nK - nQ;
    const int q0 = (int)qb * BLOCK + wave * 32;   // the wave's first query
    const int query = q0 + l;
    const uint16_t* kBase = p.k + (long long)b * p.skv + (long long)kvHead * p.D;
    const uint16_t* vBase = p.v + (long long)b * p.skv + (long long)kvHead * p.D;

    // keys seen by the workgroup's and by the wave's queries
    const int blockLast = min((int)qb * BLOCK + BLOCK, nQ) - 1;
    int kEnd = blockLast >= (int)qb * BLOCK ? nK : 0;
    if (p.causal) kEnd = min(kEnd, blockLast + off + 1);
    int waveEnd = q0 < nQ ? kEnd : 0;
    if (p.causal) waveEnd = min(waveEnd, q0 + 32 + off);
    AtReach<VIEW> reach{nK, q0, off, waveEnd, 0, 0, 0, 0, p.causal != 0};
    AtWalk walk{kEnd > 0 ? (kEnd + kTileKeys - 1) / kTileKeys : 0, 0, 0};
    if constexpr (VIEW == kAtWindow) atWindow(p, (int)qb * BLOCK, blockLast, kEnd, reach, walk);
    const int tBegin = (int)((long long)walk.n * part / p.keyParts), nt = (int)((long long)walk.n * (part + 1) / p.keyParts);

    // of a score; with a bias, scores are scaled before it is added and c is 1
    const float scaled = p.scale * kAtLog2e;
    const float c = VIEW == kAtBias ? 1.f : fmaxf(fabsf(scaled), FLT_MIN);
    const uint32_t flip = VIEW != kAtBias && p.scale < 0.f ? 0x80008000u : 0u;
    const typename T::Lane at(lane);
    typename T::template Copy<kTileKeys, W> copy;
    const uint32_t ld2 = (uint32_t)p.ldkv * 2u;
    copy.init(wave, lane, ld2, p.D);
    auto fetch = [&](int t, uint16_t* kd, uint16_t* vd, int* kp) {
        const int key0 = walk.tile<VIEW>(t) * kTileKeys;
        if constexpr (VIEW == kAtBias)
            if (wave == 0) atCopyPositions(p.kPos, key0, kTileKeys, nK, 0, lane, kp);
        const long long at = (long long)key0 * p.ldkv;
        copy.run(kBase + at, nK - key0, ld2, p.D, kd, wave);
        copy.run(vBase + at, nK - key0, ld2, p.D, vd, wave);
    };

    // the wave's queries through its part of the second pair of buffers, which tile 1 is copied to after the first barrier
    uint16_t* stage = (wave < 2 ? k1 : v1) + (wave & 1) * 32 * T::RS;
    T::start(p.q + (long long)b * p.sq + (long long)q0 * p.ldq + (long long)head * p.D, nQ - q0, p.ldq, p.D, stage, lane);
    if (nt > tBegin) fetch(tBegin, k0, v0, at0);
    int position = 0, qLeast = 0, qMost = 0;   // the lane's query's, the wave's
    if constexpr (VIEW == kAtBias) {
        atFillBiases<64 * W>(p, head, [&](int i, float v) { biasesLds[i] = v; });
        position = atOwnPosition(p.qPos, query, nQ, off, qLeast, qMost);
    }
    __builtin_amdgcn_s_waitcnt(0);
    at_u32x4 qf[T::NS];
    T::take(at, stage, qf);
#pragma unroll
    for (int s = 0; s < T::NS; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[s][e] ^= flip;

    at_f32x16 o[KD];
#pragma unroll
    for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    float m = -INFINITY, sum = 0.f;
    const float margin = fminf(8.f / c, FLT_MAX);

    auto tile = [&](int key0, const uint16_t* kd, const uint16_t* vd, const int* kp) {
        at_f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
            for (int st = 0; st < T::NS; ++st) s[kb] = atMfma<BF16>(at.natural(kd, 32 * kb, st), qf[st], s[kb]);
        }
        atPipeline<2 * T::NS, 1, 4>();
        if constexpr (VIEW == kAtBias) {
            int kLeast, kMost;
            atRange(kp[lane], kLeast, kMost);
            const AtOffsets kind = atOffsets(p, qLeast, qMost, kLeast, kMost);
            if (kind == kAtMap) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    atForEntries<true>(p, position, kp + 32 * kb + 4 * h, lane,
                                       [&](int i, int o) { s[kb][i] = __builtin_fmaf(s[kb][i], scaled, biases[o]); });
            } else {
                const float one = biases[kind == kAtLow ? 0 : p.nOffsets - 1];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = __builtin_fmaf(s[kb][r], scaled, one);
            }
        }
        if (reach.edge(key0)) {
            const AtSeen seen = reach.seen(query, key0, h);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[kb][r] = seen.pick<VIEW>(32 * kb + 8 * (r / 4) + r % 4, s[kb][r], -INFINITY);
        }
        float top = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
        top = atMaxHalves(top);
        if (__any(top > m + margin)) {   // also where m is -inf and the row sees its first key
            const float next = fmaxf(m, top);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - next) * c);
            sum *= alpha;
#pragma unroll
            for (int dt = 0; dt < KD; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
            m = next;
        }
        const float base = m == -INFINITY ? 0.f : kShift - m * c;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
#pragma unroll
            for (int r = 8 * (u & 1); r < 8 * (u & 1) + 8; ++r) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u / 2][r], c, base));
                s[u / 2][r] = e;
                sum += e;
            }
            const at_u32x4 pf = atPack8<BF16>(s[u / 2], u & 1);
#pragma unroll
            for (int dt = 0; dt < KD; ++dt) o[dt] = atMfma<BF16>(at.transposed(vd, 16 * u, dt), pf, o[dt]);
        }
        // the weights of step u + 1 are computed, and its fragments read, under the MFMAs of step u
        atReads<2 * KD>();
        atValu<20>();
        atTrans<8>();
        atValu<20>();
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int dt = 0; dt < KD; ++dt) {
                atMfmas<1>();
                if (u < 3) {
                    atReads<2>();
                    atTrans<8 / KD>();
                    atValu<20 / KD>();
                }
            }
    };

    // Copies of tile t + 1 start once every wave is done with tile t - 1, whose buffers they fill, and are waited for at
    // the top of the next trip. Whole pairs of trips, then what is left: a way out of the middle would cost every trip
    // copies of the sums.
    auto trip = [&](int t, const uint16_t* kd, const uint16_t* vd, const int* kp, uint16_t* kNext, uint16_t* vNext, int* kpNext) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1, kNext, vNext, kpNext);
        const int key0 = walk.tile<VIEW>(t) * kTileKeys;
        if (reach.tile(key0)) tile(key0, kd, vd, kp);
    };
    int t = tBegin;
    for (; t + 1 < nt; t += 2) {
        trip(t, k0, v0, at0, k1, v1, at1);
        trip(t + 1, k1, v1, at1, k0, v0, at0);
    }
    if (t < nt) trip(t, k0, v0, at0, k1, v1, at1);

    sum = atSumHalves(sum);
    const bool empty = !(query < nQ) || sum == 0.f;
    const float inv = empty ? 0.f : 1.f / sum;
    // the hardware's logarithm: a few 2^-24 of log2(sum), as the sum itself
    const float lse = empty ? -INFINITY : m * (c * kAtLn2) + (__logf(sum) - kShift * kAtLn2);
    const long long row = ((long long)b * p.Sq + query) * p.H + head;
    const long long stat = ((long long)b * p.H + head) * p.Sq + query;
    if (p.keyParts > 1) {
        if (query >= p.Sq) return;
        if (h == 0) p.lsePart[stat * p.keyParts + part] = lse;
        storeColumnF32<KD>(p.rowPart + (row * p.keyParts + part) * p.D, o, inv, h, p.D, empty);
    } else {
        if (h == 0 && query < p.Sq) p.lse[stat] = lse;
        __syncthreads();   // every wave is done with the tiles
        storeRows<BF16, KD>(p.out + (((long long)b * p.Sq + q0) * p.H + head) * p.D, (long long)p.H * p.D, p.Sq - q0, o, inv,
                            empty, (wave < 2 ? k0 : v0) + (wave & 1) * 32 * T::RS, lane, p.D);
    }
}

// The parts' contexts, each the mean of its keys: out = sum_i exp(lse_i - lse) out_i, eight values of a row a thread.
template <bool BF16>
__global__ __launch_bounds__(256) void attn_train_join_kernel(AttnTrainParams p) {
    const int chunks = p.D / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;   // (b, q, head, chunk)
    if (i >= (long long)p.B * p.Sq * p.H * chunks) return;
    const int c = (int)(i % chunks);
    const long long row = i / chunks;
    const int head = (int)(row % p.H);
    const long long bq = row / p.H;
    const int q = (int)(bq % p.Sq), b = (int)(bq / p.Sq);
    const long long stat = ((long long)b * p.H + head) * p.Sq + q;
    const float* lse = p.lsePart + stat * p.keyParts;
    const float* from = p.rowPart + row * p.keyParts * p.D + c * 8;
    float top = -INFINITY;
    for (int k = 0; k < p.keyParts; ++k) top = fmaxf(top, lse[k]);
    const float from0 = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    at_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int k = 0; k < p.keyParts; ++k) {
        const float w = __expf(lse[k] - from0);
        total += w;
#pragma unroll
        for (int e = 0; e < 2; ++e) s[e] += w * *reinterpret_cast<const at_f32x4*>(from + (long long)k * p.D + 4 * e);
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;   // 0: no part has a key
    if (c == 0) p.lse[stat] = total == 0.f ? -INFINITY : from0 + __logf(total);
    *reinterpret_cast<at_u32x4*>(p.out + row * p.D + c * 8) =
        at_u32x4{atPack2<BF16>(s[0][0] * inv, s[0][1] * inv), atPack2<BF16>(s[0][2] * inv, s[0][3] * inv),
                 atPack2<BF16>(s[1][0] * inv, s[1][1] * inv), atPack2<BF16>(s[1][2] * inv, s[1][3] * inv)};
}

// ---------------------------------------------------------------- backward
// P of the dK / dV kernel is taken raised by 2^15 in fp16 (it is at most 1, and loses bits below 2^-14): part of the
// row statistics' shift.
template <bool BF16>
constexpr float kRaise = BF16 ? 0.f : 15.f;

// dS as halves. bf16 has fp32's range; fp16 loses dS below 2^-14 (a probability of 1 / 4096 times a gradient of
// 2^-10 is there) and has no value past 65504. A lane's dS all go into one column of the sum (its query's dQ, its
// key's dK), so the lane scales them by a power of two of its own, which starts where its first non-zero ones come
// to about 2^9 and is lowered, with the sums so far, whenever they would pass 2^15; it is divided out of the column
// at the end. Powers of two: no rounding of its own.
template <bool BF16, int KD>
struct DsScale {
    float f = BF16 ? 1.f : 0.f;   // 0: no dS yet
    // x: |dS| of the lane's column at most, in both half-waves
    __device__ __forceinline__ void update(float x, at_f32x16 (&acc)[KD]) {
        if constexpr (BF16) return;
        if (__any(x * f >= 32768.f || (f == 0.f && x > 0.f))) {
            if (x * f >= 32768.f || (f == 0.f && x > 0.f)) {
                // 2^9 / 2^(exponent of x), kept within floats' range; infinities and NaN of x stay what they are
                const int e = (int)((__builtin_bit_cast(uint32_t, x) >> 23) & 255u) - 127;
                const float next = __builtin_bit_cast(float, (uint32_t)(min(max(9 - e, -60), 60) + 127) << 23);
                const float r = f == 0.f ? 0.f : next / f;
                f = next;
#pragma unroll
                for (int t = 0; t < KD; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[t][i] *= r;
            }
        }
    }
    __device__ __forceinline__ float undo() const { return f == 0.f ? 1.f : 1.f / f; }
};

// ---------------------------------------------------------------- backward: dQ
// As the forward pass, a wave holds 32 queries as columns and the workgroup walks the keys: S^T = K Q^T,
// dP^T = V dO^T, dQ^T += K^T dS^T. It also makes and leaves the rows' statistics, shift = -lse log2 e and delta =
// sum_d dO O, for the dK / dV kernel that follows; rows that pass no gradient (past the query length, past Sq, or
// without a key) get shift = -inf, which makes their probabilities 0.
// dQ and dK / dV are two kernels that each compute S and dP, 7 products where one pass would need 5: sums of a row's dQ
// over workgroups would have to be added atomically, in an order that changes, or written whole for every block of keys.
// Measured (sizes as for the forward pass): 211-242 us by card (0.85-0.98 PFLOP/s), matrix cores busy 54 %; ViT-B/16 b64 37.
template <bool BF16, int KD, int VIEW, class Sum, int W>
__global__ __launch_bounds__(64 * W, 2) void attn_train_dq_kernel(AtParams<VIEW> p) {
    using T = AtTile<KD>;
    constexpr int BLOCK = 32 * W;   // queries of the workgroup
    __shared__ __attribute__((aligned(256))) uint16_t k0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t k1[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v1[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(16))) int at0[VIEW == kAtBias ? kTileKeys : 4];   // positions of the keys
    __shared__ __attribute__((aligned(16))) int at1[VIEW == kAtBias ? kTileKeys : 4];
    extern __shared__ float biasesLds[];   // [nOffsets] and the ends, rounded to 64, then each wave's sums of dS
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t bh, qb;
    atPlace(blockIdx.x, p.heads, p.blocks * p.keyParts, p.causal, bh, qb);
    const int part = (int)(qb % (uint32_t)p.keyParts);
    qb = p.blocks - 1 - qb / (uint32_t)p.keyParts;   // causal: the longest walks first
    const int group = (int)(bh / (uint32_t)p.H), head = (int)(bh % (uint32_t)p.H);   // group: the image, or of images
    const int kvHead = head / (p.H / p.Hkv);
    const int q0 = (int)qb * BLOCK + wave * 32;
    Sum* sums = nullptr;
    if constexpr (VIEW == kAtBias) {
        const int each = p.nOffsets + 2 * kMapEnd;
        Sum* all = reinterpret_cast<Sum*>(biasesLds + (each + 63) / 64 * 64);
        float* leave = group == 0 && qb == 0 && part == 0 ? p.tables + (long long)head * each : nullptr;
        atFillBiases<64 * W>(p, head, [&](int i, float v) {
            biasesLds[i] = v;
            if (leave) leave[i] = v;
        });
        for (int i = (int)threadIdx.x; i < W * each; i += 64 * W) all[i] = 0;   // added to after the first barrier
        sums = all + wave * each + kMapEnd;
    }
    // One image. The arrays in dynamic LDS apart from the others (restrict): the compiler would wait for the copies under way
    // before it touches them.
    auto image = [&](int b, const float* __restrict__ biases, Sum* __restrict__ sums) __attribute__((always_inline)) {
        int lane = threadIdx.x & 63;
        if constexpr (VIEW == kAtBias) asm volatile("" : "+v"(lane));   // else the lane's addresses are kept in 60 registers over the loop
        const int l = lane & 31, h = lane >> 5, query = q0 + l;
        const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk);
        const int off = VIEW == kAtPlain ? p.Sk - p.Sq : nK - nQ;
        const uint16_t* kBase = p.k + (long long)b * p.skv + (long long)kvHead * p.D;
        const uint16_t* vBase = p.v + (long long)b * p.skv + (long long)kvHead * p.D;

        const int blockLast = min((int)qb * BLOCK + BLOCK, nQ) - 1;
        int kEnd = blockLast >= (int)qb * BLOCK ? nK : 0;
        if (p.causal) kEnd = min(kEnd, blockLast + off + 1);
        int waveEnd = q0 < nQ ? kEnd : 0;
        if (p.causal) waveEnd = min(waveEnd, q0 + 32 + off);
        AtReach<VIEW> reach{nK, q0, off, waveEnd, 0, 0, 0, 0, p.causal != 0};
        AtWalk walk{kEnd > 0 ? (kEnd + kTileKeys - 1) / kTileKeys : 0, 0, 0};
        if constexpr (VIEW == kAtWindow) atWindow(p, (int)qb * BLOCK, blockLast, kEnd, reach, walk);
        const int tBegin = (int)((long long)walk.n * part / p.keyParts), nt = (int)((long long)walk.n * (part + 1) / p.keyParts);

        const float c = p.scale * kAtLog2e;
        const typename T::Lane at(lane);
        typename T::template Copy<kTileKeys, W> copy;
        const uint32_t ld2 = (uint32_t)p.ldkv * 2u;
        copy.init(wave, lane, ld2, p.D);
        auto fetch = [&](int t, uint16_t* kd, uint16_t* vd, int* kp) {
            const int key0 = walk.tile<VIEW>(t) * kTileKeys;
            if constexpr (VIEW == kAtBias)
                if (wave == 0) atCopyPositions(p.kPos, key0, kTileKeys, nK, 0, lane, kp);
            const long long o = (long long)key0 * p.ldkv;
            copy.run(kBase + o, nK - key0, ld2, p.D, kd, wave);
            copy.run(vBase + o, nK - key0, ld2, p.D, vd, wave);
        };
        // Q and dO of the wave's queries, and delta. Head dimensions up to 64: by whole rows, Q through its part of the second
        // pair of buffers, which tile 1 is copied to after the first barrier, dO through rows of its own; larger ones straight
        // into fragments, 32 rows for 16 bytes an instruction: rows of dO's own would leave one workgroup a CU, and a head
        // dimension of 128 is at 256 registers and 12-20 bytes of scratch without the chunks of dO and O for delta. (dO through
        // the first pair of buffers, free until the first tile is fetched, has not been measured.)
        constexpr bool kStaged = KD <= 2;
        __shared__ __attribute__((aligned(256))) uint16_t gStage[kStaged ? BLOCK * T::RS : 8];
        __shared__ float rowDelta[W][32];
        const uint16_t* qRows = p.q + (long long)b * p.sq + (long long)q0 * p.ldq + (long long)head * p.D;
        const uint16_t* gRows = p.gradOut + (((long long)b * p.Sq + q0) * p.H + head) * p.D;
        const uint16_t* oRows = p.out + (((long long)b * p.Sq + q0) * p.H + head) * p.D;
        const long long ldo = (long long)p.H * p.D;
        const long long image = (long long)b * p.H + head;
        const float lse = query < nQ ? p.lse[image * p.Sq + query] : -INFINITY;
        auto dot = [&](const at_u32x4& x, const at_u32x4& y, float d) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x0, x1, y0, y1;
                atUnpack2<BF16>(x[e], x0, x1);
                atUnpack2<BF16>(y[e], y0, y1);
                d = __builtin_fmaf(x0, y0, d);
                d = __builtin_fmaf(x1, y1, d);
            }
            return d;
        };
        at_u32x4 qf[T::NS], gf[T::NS];
        float delta = 0.f;
        if constexpr (kStaged) {
            uint16_t *qStage = (wave < 2 ? k1 : v1) + (wave & 1) * 32 * T::RS, *dStage = gStage + wave * 32 * T::RS;
            T::start(qRows, nQ - q0, p.ldq, p.D, qStage, lane);
            T::start(gRows, nQ - q0, ldo, p.D, dStage, lane);
            if (nt > tBegin) fetch(tBegin, k0, v0, at0);
            constexpr int N = T::CH / 2;   // instructions of 64 / CH rows, a whole chunk a lane
            at_u32x4 g[N], o[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = (i * 64 + lane) / T::CH, d = (i * 64 + lane) % T::CH * 8;
                const bool in = q0 + row < nQ && d < p.D;
                g[i] = in ? *reinterpret_cast<const at_u32x4*>(gRows + row * ldo + d) : at_u32x4{0u, 0u, 0u, 0u};
                o[i] = in ? *reinterpret_cast<const at_u32x4*>(oRows + row * ldo + d) : at_u32x4{0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float d = dot(g[i], o[i], 0.f);
#pragma unroll
                for (int s = T::CH / 2; s > 0; s >>= 1) d += __shfl_xor(d, s, 64);
                if (lane % T::CH == 0) rowDelta[wave][(i * 64 + lane) / T::CH] = d;
            }
            __builtin_amdgcn_wave_barrier();   // the wave's own LDS operations complete in order
            delta = rowDelta[wave][l];
            __builtin_amdgcn_s_waitcnt(0);
            T::take(at, qStage, qf);
            T::take(at, dStage, gf);
        } else {
            if (nt > tBegin) fetch(tBegin, k0, v0, at0);
#pragma unroll
            for (int s = 0; s < T::NS; ++s) {
                qf[s] = T::direct(qRows + l * p.ldq, query < nQ, s, h, p.D);
                gf[s] = T::direct(gRows + l * ldo, query < nQ, s, h, p.D);
                delta = dot(gf[s], T::direct(oRows + l * ldo, query < nQ, s, h, p.D), delta);
            }
            delta = atSumHalves(delta);
        }
        float shift = -INFINITY;
        if (lse == -INFINITY)
            delta = 0.f;
        else
            shift = -lse * kAtLog2e;
        if (h == 0 && part == 0 && query < p.SqP) {
            float* to = p.stats + 2 * (image * p.SqP + q0) + l;
            to[0] = shift + kRaise<BF16>;
            to[32] = delta;
        }
        int position = 0, qLeast = 0, qMost = 0;   // the lane's query's, the wave's
        if constexpr (VIEW == kAtBias) position = atOwnPosition(p.qPos, query, nQ, off, qLeast, qMost);
        at_f32x16 dq[KD];
#pragma unroll
        for (int t = 0; t < KD; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) dq[t][r] = 0.f;
        DsScale<BF16, KD> scale;

        auto tile = [&](auto edgeTag, auto mapTag, int key0, const uint16_t* kd, const uint16_t* vd, const int* kp, float one, Sum* end) {
            constexpr bool EDGE = decltype(edgeTag)::value;   // some query does not see some of the keys
            constexpr bool MAP = VIEW == kAtBias && decltype(mapTag)::value;   // biases by pair, else one for the tile
            const AtSeen seen = reach.seen(query, key0, h);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                if (EDGE && kb == 1 && key0 + 32 >= reach.end) break;   // the wave's queries see none of these
                at_f32x16 s, dp, bias;
                // biases are under way while the scores are computed; larger heads have no registers for them until then
                constexpr bool kAhead = MAP && KD <= 2;
                if constexpr (kAhead) {
                    atForEntries<true>(p, position, kp + 32 * kb + 4 * h, lane, [&](int i, int o) { bias[i] = biases[o]; });
                    __builtin_amdgcn_sched_barrier(0);   // the order below is for the fragments' reads
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
                for (int st = 0; st < T::NS; ++st) {
                    s = atMfma<BF16>(at.natural(kd, 32 * kb, st), qf[st], s);
                    dp = atMfma<BF16>(at.natural(vd, 32 * kb, st), gf[st], dp);
                }
                atPipeline<2 * T::NS, 1, 4>();
                float most = 0.f;
                auto weigh = [&](int r, float b) {
                    float x = __builtin_fmaf(s[r], c, shift);
                    if constexpr (VIEW == kAtBias) x = __builtin_fmaf(s[r], c, b) + shift;
                    float e = __builtin_amdgcn_exp2f(x);
                    if constexpr (EDGE) e = seen.pick<VIEW>(32 * kb + 8 * (r / 4) + r % 4, e, 0.f);
                    s[r] = e * (dp[r] - delta);
                    if constexpr (!BF16) most = fmaxf(most, fabsf(s[r]));
                };
                if constexpr (MAP) {
                    atForEntries<true>(p, position, kp + 32 * kb + 4 * h, lane, [&](int i, int o) {
                        weigh(i, kAhead ? bias[i] : biases[o]);
                        atAdd(sums + o, (Sum)s[i]);
                    });
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) weigh(r, one);
                    if constexpr (VIEW == kAtBias) {
                        float sum = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) sum += s[r];
                        atAdd(end, (Sum)sum);
                    }
                }
                if constexpr (!BF16) {
                    scale.update(atMaxHalves(most), dq);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] *= scale.f;
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const at_u32x4 df = atPack8<BF16>(s, u);
#pragma unroll
                    for (int dt = 0; dt < KD; ++dt) dq[dt] = atMfma<BF16>(at.transposed(kd, 32 * kb + 16 * u, dt), df, dq[dt]);
                }
                atPipeline<2 * KD, 2, KD < 3 ? KD : 3>();
            }
        };
        auto step = [&](int t, const uint16_t* kd, const uint16_t* vd, const int* kp) {
            const int key0 = walk.tile<VIEW>(t) * kTileKeys;
            if (!reach.tile(key0)) return;
            if constexpr (VIEW == kAtBias) {
                int kLeast, kMost;
                atRange(kp[lane], kLeast, kMost);
                const AtOffsets kind = atOffsets(p, qLeast, qMost, kLeast, kMost);
                if (kind != kAtMap && !reach.edge(key0))
                    return tile(std::false_type{}, std::false_type{}, key0, kd, vd, kp, biases[kind == kAtLow ? 0 : p.nOffsets - 1],
                                sums + (kind == kAtLow ? lane - kMapEnd : p.nOffsets + lane));
            }
            if (reach.edge(key0))   // of a bias by pair, at the map's ends too
                tile(std::true_type{}, std::true_type{}, key0, kd, vd, kp, 0.f, nullptr);
            else
                tile(std::false_type{}, std::true_type{}, key0, kd, vd, kp, 0.f, nullptr);
        };
        auto trip = [&](int t, const uint16_t* kd, const uint16_t* vd, const int* kp, uint16_t* kNext, uint16_t* vNext, int* kpNext) {   // as in the forward pass
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (t + 1 < nt) fetch(t + 1, kNext, vNext, kpNext);
            step(t, kd, vd, kp);
        };
        int t = tBegin;
        for (; t + 1 < nt; t += 2) {
            trip(t, k0, v0, at0, k1, v1, at1);
            trip(t + 1, k1, v1, at1, k0, v0, at0);
        }
        if (t < nt) trip(t, k0, v0, at0, k1, v1, at1);
        const float f = p.scale * scale.undo();
        const bool none = shift == -INFINITY;
        if (p.keyParts > 1) {
            if (query < p.Sq)
                storeColumnF32<KD>(p.rowPart + ((((long long)b * p.Sq + query) * p.H + head) * p.keyParts + part) * p.D, dq, f, h,
                                   p.D, none);
        } else {
            __syncthreads();   // every wave is done with the tiles
            storeRows<BF16, KD>(p.dq + (long long)b * p.sq + (long long)q0 * p.ldq + (long long)head * p.D, p.ldq, p.Sq - q0, dq, f,
                                none, (wave < 2 ? k0 : v0) + (wave & 1) * 32 * T::RS, lane, p.D);
        }
    };
    if constexpr (VIEW == kAtBias) {
        for (int b = group; b < p.B; b += p.imageGroups) {
            image(b, biasesLds + kMapEnd, sums);
            __builtin_amdgcn_s_waitcnt(0);   // the wave's adds
            __syncthreads();                 // the buffers and statistics are the next image's
        }
    } else {
        image(group, nullptr, nullptr);
    }
    if constexpr (VIEW == kAtBias) {
        // the ends' entries, then the waves, in order
        const int lane = threadIdx.x & 63;
        Sum low = sums[lane - kMapEnd], high = sums[p.nOffsets + lane];
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) {
            low += __shfl_xor(low, m, 64);
            high += __shfl_xor(high, m, 64);
        }
        if (lane == 0) {
            sums[0] += low;
            sums[p.nOffsets - 1] += high;
        }
        __syncthreads();
        float* to = p.bins + ((((long long)head * p.imageGroups + group) * p.blocks + qb) * p.keyParts + part) * p.nOffsets;
        const int each = p.nOffsets + 2 * kMapEnd;
        const Sum* first = sums - wave * each;
        for (int o = (int)threadIdx.x; o < p.nOffsets; o += 64 * W)
            to[o] = (float)(W == 2 ? first[o] + first[o + each] : (first[o] + first[o + each]) + (first[o + 2 * each] + first[o + 3 * each]));
    }
}

// The parts' sums of dQ, eight values of a row a thread.
template <bool BF16>
__global__ __launch_bounds__(256) void attn_train_dq_join_kernel(AttnTrainParams p) {
    const int chunks = p.D / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;   // (b, q, head, chunk)
    if (i >= (long long)p.B * p.Sq * p.H * chunks) return;
    const int c = (int)(i % chunks);
    const long long row = i / chunks;
    const int head = (int)(row % p.H);
    const long long bq = row / p.H;
    const int q = (int)(bq % p.Sq), b = (int)(bq / p.Sq);
    const float* from = p.rowPart + row * p.keyParts * p.D + c * 8;
    at_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int k = 0; k < p.keyParts; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) s[e] += *reinterpret_cast<const at_f32x4*>(from + (long long)k * p.D + 4 * e);
    *reinterpret_cast<at_u32x4*>(p.dq + (long long)b * p.sq + (long long)q * p.ldq + (long long)head * p.D + c * 8) =
        at_u32x4{atPack2<BF16>(s[0][0], s[0][1]), atPack2<BF16>(s[0][2], s[0][3]), atPack2<BF16>(s[1][0], s[1][1]),
                 atPack2<BF16>(s[1][2], s[1][3])};
}

// ---------------------------------------------------------------- backward: dK and dV
// A workgroup holds 128 keys of a key head and walks the queries of every head that reads them, 32 at a time. Four
// pairs of waves hold 32 keys each, as columns; of a pair (both waves are on one SIMD),
//  * the first computes S = Q K^T, P and dV^T += dO^T P, and leaves P (fp32, in its registers' order) in LDS;
//  * the second, one tile behind, computes dP = dO V^T, dS from that P, and dK^T += Q^T dS.
// One wave doing both needs 128 + 64 registers for its sums and K, V fragments at a head dimension of 128, so only one
// fits a SIMD and every LDS read and exponential of it is waited out: 465-489 us at 2 x 4096 x 16 heads on 4 of 128,
// causal, against 289-319 us (0.86-0.95 PFLOP/s, matrix cores busy 51 %) for two waves that fill each other's gaps. ViT-B/16
// b64: 41 us. Q and dO tiles are in three buffers: the next one's copy, the first waves' and the second waves'.
// Where the blocks of keys are few for the card, `parts` workgroups take a share of a block's walk each and leave fp32
// sums, which attn_train_dkv_join_kernel adds in order.
constexpr int kTileQ = 32;

// LDS of the kernel. Each buffer is an array of its own, so that the compiler sees that a copy into one does not touch
// the others and lets reads of them go ahead of it.
struct DkvBuffers {
    uint16_t *q[3], *g[3];
    float* stats[3];     // shift, delta, of a bias the positions
    float* weights;      // P by tile parity and pair
    float* biases;       // by offset, of a key head's first, third ... query head and of its second ...
};

// Tiles t0 .. t1 - 1 of an image's queries that see a key of a block.
struct DkvTiles {
    int t0, t1;
};
template <int VIEW, int BLOCK = kBlockQ>
__device__ __forceinline__ DkvTiles dkvTiles(const AtParams<VIEW>& p, int block, int nQ, int nK, int off) {
    const int first = block * BLOCK;
    DkvTiles t{p.causal ? max(0, first - off) / kTileQ : 0, first < nK ? (nQ + kTileQ - 1) / kTileQ : 0};
    if constexpr (VIEW == kAtWindow) {
        if (block >= p.sinkBlocks) {
            if (!p.causal) t.t0 = max(0, first - off - p.window + 1) / kTileQ;
            t.t1 = min(t.t1, (max(0, first + BLOCK - 1 - off + p.window) + kTileQ - 1) / kTileQ);
        }
    }
    return t;
}

// A wave's work in attn_train_dkv_kernel.
template <bool BF16, int KD, int VIEW, int PAIRS, bool SECOND>
__device__ __forceinline__ void dkvWalk(const AtParams<VIEW>& p, const DkvBuffers& lds, int wave, int lane) {
    using T = AtTile<KD>;
    constexpr float kLower = BF16 ? 1.f : 1.f / 32768.f;   // takes kRaise out
    const int l = lane & 31, h = lane >> 5, pair = wave % PAIRS;
    uint32_t bh, block;
    // causal, or first keys with longer walks: the first keys' walks are longest
    atPlace(blockIdx.x, p.heads, p.blocks * p.parts, p.causal || VIEW == kAtWindow, bh, block);
    const int part = (int)(block % (uint32_t)p.parts);
    block /= (uint32_t)p.parts;
    const int b = (int)(bh / (uint32_t)p.Hkv), kvHead = (int)(bh % (uint32_t)p.Hkv);
    const int group = p.H / p.Hkv;
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk);
    const int off = VIEW == kAtPlain ? p.Sk - p.Sq : nK - nQ;
    const int key0 = (int)block * 32 * PAIRS + pair * 32;
    const int key = key0 + l;

    // query tiles that see a key of the workgroup: t0 .. t1 of each head of the group; this part's share of them
    const auto [t0, t1] = dkvTiles<VIEW, 32 * PAIRS>(p, (int)block, nQ, nK, off);
    const int per = max(0, t1 - t0), total = per * group;
    const int begin = (int)((long long)total * part / p.parts), n = (int)((long long)total * (part + 1) / p.parts) - begin;

    const typename T::Lane at(lane);
    // K or V of the wave's keys through LDS that nothing is copied to, and no weights go to, before the first barrier
    constexpr int kStage = 32 * T::RS;
    uint16_t* stage = reinterpret_cast<uint16_t*>(lds.weights) + (KD <= 2 ? wave : pair) * kStage;
    if (KD > 2 && SECOND) stage = pair == 0 ? lds.q[1] : pair == 1 ? lds.q[2] : pair == 2 ? lds.g[1] : lds.g[2];
    const long long first = (long long)b * p.skv + (long long)key0 * p.ldkv + (long long)kvHead * p.D;
    T::start((SECOND ? p.v : p.k) + first, nK - key0, p.ldkv, p.D, stage, lane);
    const float c = p.scale * kAtLog2e;
    constexpr int kCopyWaves = T::CH * kTileQ / 64 < 2 * PAIRS ? T::CH * kTileQ / 64 : 2 * PAIRS;   // a head dimension of 32 has 2 instructions
    typename T::template Copy<kTileQ, kCopyWaves> copyQ, copyG;
    const uint32_t ldq2 = (uint32_t)p.ldq * 2u, ldg2 = (uint32_t)(p.H * p.D) * 2u;
    copyQ.init(wave, lane, ldq2, p.D);
    copyG.init(wave, lane, ldg2, p.D);
    int fetchHead = per > 0 ? kvHead * group + begin / per : 0, fetchT = per > 0 ? t0 + begin % per : 0;
    bool fresh = true;   // the next tile is the first of its head, or of the walk
    auto fetch = [&](uint16_t* qd, uint16_t* gd, float* sd) {   // the next tile of the walk
        const long long first = (long long)fetchT * kTileQ;
        if constexpr (VIEW == kAtBias) {
            if (wave == 2 * PAIRS - 2)
                atCopyPositions(p.qPos, (int)first, kTileQ, nQ, off, lane, reinterpret_cast<int*>(sd + 2 * kTileQ));
            if (fresh) {
                const int each = p.nOffsets + 2 * kMapEnd, rounded = (each + 63) / 64 * 64;
                const __amdgpu_buffer_rsrc_t from = atView(p.tables + (long long)fetchHead * each, (uint32_t)each * 4u);
                for (int i = wave * 64; i < each; i += 128 * PAIRS)
                    atCopy4(from, lds.biases + ((fetchHead - kvHead * group) & 1) * rounded + i, (uint32_t)(i + lane) * 4u);
            }
            fresh = false;
        }
        const int rows = nQ - fetchT * kTileQ;
        if (wave < kCopyWaves) {
            copyQ.run(p.q + (long long)b * p.sq + first * p.ldq + (long long)fetchHead * p.D, rows, ldq2, p.D, qd, wave);
            copyG.run(p.gradOut + (((long long)b * p.Sq + first) * p.H + fetchHead) * p.D, rows, ldg2, p.D, gd, wave);
        }
        if (wave == 2 * PAIRS - 1)   // rows past the query length hold -inf and 0
            atCopy4(atView(p.stats + 2 * (((long long)b * p.H + fetchHead) * p.SqP + first), 2 * kTileQ * 4), sd, lane * 4);
        if (++fetchT == t1) {
            fetchT = t0;
            ++fetchHead;
            fresh = true;
        }
    };
    at_f32x16 acc[KD];
#pragma unroll
    for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    DsScale<BF16, KD> scale;

    int position = 0, kLeast = 0, kMost = 0;   // the lane's key's, the wave's
    if constexpr (VIEW == kAtBias && !SECOND) position = atOwnPosition(p.kPos, key, nK, 0, kLeast, kMost);
    if (n > 0) fetch(lds.q[0], lds.g[0], lds.stats[0]);
    __builtin_amdgcn_s_waitcnt(0);
    at_u32x4 own[T::NS];   // K, or V
    T::take(at, stage, own);

    // nat: the tile whose product with the wave's own fragments makes S or dP; tr: the one that the sums take
    auto work = [&](int first, const uint16_t* nat, const uint16_t* tr, const float* sd, float* wd, const float* biases) {
        at_f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int st = 0; st < T::NS; ++st) s = atMfma<BF16>(at.natural(nat, 0, st), own[st], s);
        atPipeline<T::NS, 1, T::NS < 4 ? T::NS : 4>();
        if constexpr (!SECOND) {
            if constexpr (VIEW == kAtBias) {
                const int* qp = reinterpret_cast<const int*>(sd + 2 * kTileQ);
                int qLeast, qMost;
                atRange(qp[l], qLeast, qMost);
                const AtOffsets kind = atOffsets(p, qLeast, qMost, kLeast, kMost);
                if (kind == kAtMap) {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        uint32_t from[8];
                        float b[8];
                        atForEntries<false, 2>(p, position, qp + 16 * u + 4 * h, lane,
                                               [&](int i, int o) { from[i] = atLdsAddress(biases + o); });
                        atReadEight(from, b);
#pragma unroll
                        for (int i = 0; i < 8; ++i) s[8 * u + i] = __builtin_fmaf(s[8 * u + i], c, b[i]);
                    }
                } else {
                    const float b = atReadOne(biases + (kind == kAtLow ? 0 : p.nOffsets - 1));
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], c, b);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const at_f32x4 shift = *reinterpret_cast<const at_f32x4*>(sd + 8 * j + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[4 * j + e] = __builtin_amdgcn_exp2f(VIEW == kAtBias ? s[4 * j + e] + shift[e] : __builtin_fmaf(s[4 * j + e], c, shift[e]));
            }
            if constexpr (VIEW == kAtWindow) {
                // rows that see the lane's key: from firstSeen on and below endSeen, a first key's with no end
                const int at0 = first + off;
                if ((p.causal && at0 < key0 + 31) || at0 + 31 >= key0 + p.window || (!p.causal && at0 < key0 + 32 - p.window)) {
                    const bool sink = key < p.first;
                    const int row = key - at0 - 4 * h;
                    const int firstSeen = p.causal ? row : sink ? 0 : row - p.window + 1, endSeen = sink ? kTileQ : row + p.window;
                    const AtSeen seen{0, {atBitsBelow(endSeen) & ~atBitsBelow(firstSeen), 0u}};
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = seen.pick<kAtWindow>(8 * (r / 4) + r % 4, s[r], 0.f);
                }
            } else if (p.causal && first + off < key0 + 31) {
                const int firstSeen = key - off - first - 4 * h;   // rows from here on see the lane's key
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (8 * (r / 4) + r % 4 < firstSeen) s[r] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<at_f32x4*>(wd + j * 256 + lane * 4) =
                    at_f32x4{s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]};
        } else {
            float most = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const at_f32x4 w = *reinterpret_cast<const at_f32x4*>(wd + j * 256 + lane * 4);
                const at_f32x4 delta = *reinterpret_cast<const at_f32x4*>(sd + kTileQ + 8 * j + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * j + e] = w[e] * (s[4 * j + e] - delta[e]);
                    if constexpr (!BF16) most = fmaxf(most, fabsf(s[4 * j + e]));
                }
            }
            if constexpr (!BF16) {
                scale.update(atMaxHalves(most), acc);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] *= scale.f;
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const at_u32x4 f = atPack8<BF16>(s, u);
#pragma unroll
            for (int dt = 0; dt < KD; ++dt) acc[dt] = atMfma<BF16>(at.transposed(tr, 16 * u, dt), f, acc[dt]);
        }
        if constexpr (SECOND && BF16) {   // one stretch of code with the product above
            atReads<8>();   // weights, delta
            atValu<20>();
        }
        atPipeline<2 * KD, 2, KD < 3 ? KD : 3>();
    };

    // Trip i: the first waves take tile i from the buffers i % 3, the second ones tile i - 1 from those before, and tile
    // i + 1 is copied into those after. Every wave makes trips 0 .. n, and so the same number of barriers. A tile whose
    // queries see none of the wave's keys (the first few of a causal walk) has weights 0; leaving it out would cost
    // every trip copies of the sums.
    int t = per > 0 ? t0 + begin % per : 0;   // the wave's next tile
    const float* biases = lds.biases + kMapEnd;   // of the tile's head
    if constexpr (VIEW == kAtBias && !SECOND)
        if (per > 0 && (begin / per & 1)) biases += (p.nOffsets + 2 * kMapEnd + 63) / 64 * 64;
    auto meet = [&](int i, auto bufTag) {
        constexpr int NEXT = (decltype(bufTag)::value + 1) % 3;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (i + 1 < n) fetch(lds.q[NEXT], lds.g[NEXT], lds.stats[NEXT]);
    };
    auto trip = [&](int i, auto bufTag) {
        constexpr int BUF = decltype(bufTag)::value, MINE = SECOND ? (BUF + 2) % 3 : BUF;
        meet(i, bufTag);
        float* wd = lds.weights + (((SECOND ? ~i : i) & 1) * PAIRS + pair) * (kTileQ * 32);
        if constexpr (SECOND)
            work(t * kTileQ, lds.g[MINE], lds.q[MINE], lds.stats[MINE], wd, nullptr);
        else
            work(t * kTileQ, lds.q[MINE], lds.g[MINE], lds.stats[MINE], wd, biases);
        if (++t == t1) {
            t = t0;
            if constexpr (VIEW == kAtBias && !SECOND) {
                const int rounded = (p.nOffsets + 2 * kMapEnd + 63) / 64 * 64;
                biases = lds.biases + kMapEnd + (biases == lds.biases + kMapEnd ? rounded : 0);
            }
        }
    };
    if (n > 0) {
        if constexpr (SECOND) meet(0, std::integral_constant<int, 0>{});
        // whole rounds of the three buffers, then what is left: a way out of the middle of a round would cost every
        // trip copies of the sums
        using F = std::integral_constant<int, SECOND ? 1 : 0>;
        using S = std::integral_constant<int, SECOND ? 2 : 1>;
        using L = std::integral_constant<int, SECOND ? 0 : 2>;
        int i = SECOND ? 1 : 0;
        const int last = SECOND ? n : n - 1;
        if (key0 >= nK) {   // a pair without keys copies and meets the others
            for (; i + 2 <= last; i += 3) {
                meet(i, F{});
                meet(i + 1, S{});
                meet(i + 2, L{});
            }
            if (i <= last) meet(i, F{});
            if (i + 1 <= last) meet(i + 1, S{});
            i = last + 1;
        }
        for (; i + 2 <= last; i += 3) {
            trip(i, F{});
            trip(i + 1, S{});
            trip(i + 2, L{});
        }
        if (i <= last) trip(i, F{});
        if (i + 1 <= last) trip(i + 1, S{});
        if constexpr (!SECOND) __syncthreads();   // the second waves' last trip begins; nothing is copied any more
    }
    const float f = SECOND ? p.scale * kLower * scale.undo() : kLower;
    bool part32 = p.parts > 1;   // fp32 sums for attn_train_dkv_join_kernel
    if constexpr (VIEW == kAtWindow) part32 = part32 || key < p.partRows;
    if (part32) {
        const long long row = ((long long)bh * p.parts + part) * p.partRows + key;
        storeColumnF32<KD>((SECOND ? p.dkPart : p.dvPart) + row * p.D, acc, f, h, p.D, false);
    }
    if (p.parts == 1) {
        __syncthreads();   // every wave is done with the tiles and the weights
        storeRows<BF16, KD>((SECOND ? p.dk : p.dv) + first, p.ldkv, p.Sk - key0, acc, f, key >= nK, stage, lane, p.D);
    }
}

template <bool BF16, int KD, int VIEW, int PAIRS>
__global__ __launch_bounds__(128 * PAIRS, 2) void attn_train_dkv_kernel(AtParams<VIEW> p) {
    constexpr int N = kTileQ * AtTile<KD>::RS;
    __shared__ __attribute__((aligned(256))) uint16_t q0[N];
    __shared__ __attribute__((aligned(256))) uint16_t q1[N];
    __shared__ __attribute__((aligned(256))) uint16_t q2[N];
    __shared__ __attribute__((aligned(256))) uint16_t g0[N];
    __shared__ __attribute__((aligned(256))) uint16_t g1[N];
    __shared__ __attribute__((aligned(256))) uint16_t g2[N];
    __shared__ __attribute__((aligned(256))) float s0[(VIEW == kAtBias ? 3 : 2) * kTileQ];
    __shared__ __attribute__((aligned(256))) float s1[(VIEW == kAtBias ? 3 : 2) * kTileQ];
    __shared__ __attribute__((aligned(256))) float s2[(VIEW == kAtBias ? 3 : 2) * kTileQ];
    __shared__ __attribute__((aligned(16))) float weights[2 * PAIRS * kTileQ * 32];   // behind the tiles: their offsets fit a read's 16 bits
    // [nOffsets] and the ends, rounded to 64, twice where a key head has several query heads
    extern __shared__ float biases[];
    const DkvBuffers lds{{q0, q1, q2}, {g0, g1, g2}, {s0, s1, s2}, weights, biases};
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < PAIRS)
        dkvWalk<BF16, KD, VIEW, PAIRS, false>(p, lds, wave, lane);
    else
        dkvWalk<BF16, KD, VIEW, PAIRS, true>(p, lds, wave, lane);
}

// The parts' sums of dK (blockIdx.y 0) or dV (1), eight values of a key a thread, of the first `keys`.
template <bool BF16, int VIEW>
__global__ __launch_bounds__(256) void attn_train_dkv_join_kernel(AtParams<VIEW> p, int keys) {
    const int chunks = p.D / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;   // (b, key, kvHead, chunk)
    if (i >= (long long)p.B * keys * p.Hkv * chunks) return;
    const int c = (int)(i % chunks);
    const long long bkh = i / chunks;
    const int kvHead = (int)(bkh % p.Hkv);
    const int key = (int)(bkh / p.Hkv % keys), b = (int)(bkh / p.Hkv / keys);
    const long long bh = (long long)b * p.Hkv + kvHead;
    at_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    auto add = [&](const float* from, long long rows, int parts) {
        from += (bh * parts * rows + key) * p.D + c * 8;
#pragma unroll 4
        for (int part = 0; part < parts; ++part)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                s[e] += *reinterpret_cast<const at_f32x4*>(from + (long long)part * rows * p.D + 4 * e);
    };
    add(blockIdx.y ? p.dvPart : p.dkPart, p.partRows, p.parts);
    if constexpr (VIEW == kAtWindow)
        if (p.sinkParts > 0 && key < p.first) add(blockIdx.y ? p.sinkDv : p.sinkDk, (p.first + 31) / 32 * 32, p.sinkParts);
    at_u32x4 v = {atPack2<BF16>(s[0][0], s[0][1]), atPack2<BF16>(s[0][2], s[0][3]), atPack2<BF16>(s[1][0], s[1][1]),
                  atPack2<BF16>(s[1][2], s[1][3])};
    if (key >= atLength(p.kLens, b, p.Sk)) v = at_u32x4{0u, 0u, 0u, 0u};
    uint16_t* to = (blockIdx.y ? p.dv : p.dk) + (long long)b * p.skv + (long long)key * p.ldkv + (long long)kvHead * p.D;
    *reinterpret_cast<at_u32x4*>(to + c * 8) = v;
}

// ---------------------------------------------------------------- backward: dK and dV of a window's first keys
// Every query after a first key sees it, the other keys of its block only those in their windows: the block's walk leaves out
// the far queries' tiles, which these workgroups take for 32 keys at a time. A wave has tiles of its own: S = Q K^T, dP = dO
// V^T, dV^T += dO^T P, dK^T += Q^T dS, with K, V and both sums in its registers; the next tile's Q and dO land in the wave's
// other buffers meanwhile. The waves' sums are added in order and left in fp32, a part a workgroup; where the blocks' walks are
// not shared, the last workgroup of 32 keys to arrive adds them and the block's own sum and writes dK and dV (parts are
// written and read coherently past the XCDs' L2s and have landed before the counter goes up), else the join does.
// Walks of whole blocks over all queries kept three of four waves at work that no key asked for: 2 x 4096 x 16 heads on 4 of
// 128, window 512, 4 first keys: dK, dV and join 165 us, with these workgroups 120 (99 + 21; a wave's 3 or 4 tiles are as long as
// its start and end).
template <bool BF16, int KD>
__global__ __launch_bounds__(256, KD <= 2 ? 2 : 1) void attn_window_sinks_kernel(AttnWindowParams p) {
    using T = AtTile<KD>;
    constexpr float kLower = BF16 ? 1.f : 1.f / 32768.f;   // takes kRaise out
    constexpr int N = kTileQ * T::RS;
    __shared__ __attribute__((aligned(256))) uint16_t q0[4 * N];
    __shared__ __attribute__((aligned(256))) uint16_t g0[4 * N];
    __shared__ __attribute__((aligned(256))) uint16_t q1[4 * N];
    __shared__ __attribute__((aligned(256))) uint16_t g1[4 * N];
    __shared__ __attribute__((aligned(256))) float s0[4 * 2 * kTileQ];
    __shared__ __attribute__((aligned(256))) float s1[4 * 2 * kTileQ];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = lane & 31, h = lane >> 5;
    const int groups = (p.first + 31) / 32, part = (int)(blockIdx.x % (uint32_t)p.sinkParts);
    const int keyGroup = (int)(blockIdx.x / (uint32_t)p.sinkParts) % groups;
    const uint32_t bh = blockIdx.x / (uint32_t)(p.sinkParts * groups);
    const int b = (int)(bh / (uint32_t)p.Hkv), kvHead = (int)(bh % (uint32_t)p.Hkv);
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk), off = nK - nQ;
    const int key0 = keyGroup * 32;
    const bool sees = key0 + l < min(p.first, nK);

    // the far tiles of each head: before t0 (not causal) and from t1 on
    const auto [t0, t1] = dkvTiles<kAtWindow>(p, key0 / kBlockQ, nQ, nK, off);
    const int end = max(t0, t1), before = p.causal ? 0 : t0, per = key0 < nK ? before + max(0, (nQ + kTileQ - 1) / kTileQ - end) : 0;
    const int total = per * (p.H / p.Hkv);

    const typename T::Lane at(lane);
    typename T::template Copy<kTileQ, 1> copyQ, copyG;
    const uint32_t ldq2 = (uint32_t)p.ldq * 2u, ldg2 = (uint32_t)(p.H * p.D) * 2u;
    copyQ.init(0, lane, ldq2, p.D);
    copyG.init(0, lane, ldg2, p.D);
    auto fetch = [&](int i, uint16_t* qd, uint16_t* gd, float* sd) {
        const int head = kvHead * (p.H / p.Hkv) + i / per, x = i % per, t = x < before ? x : x - before + end;
        const long long first = (long long)t * kTileQ;
        copyQ.run(p.q + (long long)b * p.sq + first * p.ldq + (long long)head * p.D, nQ - (int)first, ldq2, p.D, qd + wave * N, 0);
        copyG.run(p.gradOut + (((long long)b * p.Sq + first) * p.H + head) * p.D, nQ - (int)first, ldg2, p.D, gd + wave * N, 0);
        atCopy4(atView(p.stats + 2 * (((long long)b * p.H + head) * p.SqP + first), 2 * kTileQ * 4), sd + wave * 2 * kTileQ, lane * 4);
    };
    const long long firstKey = (long long)b * p.skv + (long long)key0 * p.ldkv + (long long)kvHead * p.D;
    T::start(p.k + firstKey, nK - key0, p.ldkv, p.D, q1 + wave * N, lane);
    T::start(p.v + firstKey, nK - key0, p.ldkv, p.D, g1 + wave * N, lane);
    const int step = 4 * p.sinkParts;
    int i = part * 4 + wave;
    if (i < total) fetch(i, q0, g0, s0);
    __builtin_amdgcn_s_waitcnt(0);
    at_u32x4 kf[T::NS], vf[T::NS];
    T::take(at, q1 + wave * N, kf);
    T::take(at, g1 + wave * N, vf);
    __builtin_amdgcn_s_waitcnt(0);   // read before the next copies land there

    const float c = p.scale * kAtLog2e;
    at_f32x16 dk[KD], dv[KD];
#pragma unroll
    for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) dk[t][r] = dv[t][r] = 0.f;
    DsScale<BF16, KD> scale;
    auto tile = [&](const uint16_t* qt, const uint16_t* gt, const float* sd) {
        at_f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
        for (int st = 0; st < T::NS; ++st) {
            s = atMfma<BF16>(at.natural(qt, 0, st), kf[st], s);
            dp = atMfma<BF16>(at.natural(gt, 0, st), vf[st], dp);
        }
        atPipeline<2 * T::NS, 1, 4>();
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const at_f32x4 shift = *reinterpret_cast<const at_f32x4*>(sd + 8 * j + 4 * h);
            const at_f32x4 delta = *reinterpret_cast<const at_f32x4*>(sd + kTileQ + 8 * j + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * j + e;
                s[r] = sees ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, shift[e])) : 0.f;
                dp[r] = s[r] * (dp[r] - delta[e]);
                if constexpr (!BF16) most = fmaxf(most, fabsf(dp[r]));
            }
        }
        if constexpr (!BF16) {
            scale.update(atMaxHalves(most), dk);
#pragma unroll
            for (int r = 0; r < 16; ++r) dp[r] *= scale.f;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const at_u32x4 pf = atPack8<BF16>(s, u), df = atPack8<BF16>(dp, u);
#pragma unroll
            for (int dt = 0; dt < KD; ++dt) {
                dv[dt] = atMfma<BF16>(at.transposed(gt, 16 * u, dt), pf, dv[dt]);
                dk[dt] = atMfma<BF16>(at.transposed(qt, 16 * u, dt), df, dk[dt]);
            }
        }
        atPipeline<4 * KD, 2, KD < 3 ? KD : 3>();
    };
    auto trip = [&](int i, const uint16_t* qt, const uint16_t* gt, const float* st, uint16_t* qNext, uint16_t* gNext, float* sNext) {
        if (i + step < total) fetch(i + step, qNext, gNext, sNext);
        tile(qt + wave * N, gt + wave * N, st + wave * 2 * kTileQ);
        __builtin_amdgcn_s_waitcnt(0);   // the next tile is here, this one read
    };
    for (; i + step < total; i += 2 * step) {
        trip(i, q0, g0, s0, q1, g1, s1);
        trip(i + step, q1, g1, s1, q0, g0, s0);
    }
    if (i < total) trip(i, q0, g0, s0, q1, g1, s1);

    // the waves' sums, in order, then the rows that are first keys
    const float fk = p.scale * kLower * scale.undo();
    constexpr int R = T::RS + 4;   // floats a row: the lanes' rows in different banks
    float *sumK = reinterpret_cast<float*>(q0), *sumV = reinterpret_cast<float*>(g0);   // [32, R]
    for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave != w || key0 + l >= p.first) continue;
#pragma unroll
        for (int dt = 0; dt < KD; ++dt)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int o = l * R + 32 * dt + 2 * r + 4 * h;
                at_f32x4 x = {dk[dt][r] * fk, dk[dt][r + 1] * fk, dk[dt][r + 2] * fk, dk[dt][r + 3] * fk};
                at_f32x4 y = {dv[dt][r] * kLower, dv[dt][r + 1] * kLower, dv[dt][r + 2] * kLower, dv[dt][r + 3] * kLower};
                if (w > 0) {
                    x += *reinterpret_cast<const at_f32x4*>(sumK + o);
                    y += *reinterpret_cast<const at_f32x4*>(sumV + o);
                }
                *reinterpret_cast<at_f32x4*>(sumK + o) = x;
                *reinterpret_cast<at_f32x4*>(sumV + o) = y;
            }
    }
    __syncthreads();
    const int rows = min(32, p.first - key0), quads = p.D / 4;
    const long long own = (long long)bh * p.sinkParts * groups * 32 * p.D;   // the key head's parts
    const uint32_t pitch = (uint32_t)(groups * 32 * p.D) * 4u, bytes = pitch * (uint32_t)p.sinkParts;
    const __amdgpu_buffer_rsrc_t partK = bufferRsrc(p.sinkDk + own, bytes), partV = bufferRsrc(p.sinkDv + own, bytes);
    for (int x = (int)threadIdx.x; x < rows * quads; x += 256) {
        const int row = x / quads, d = x % quads * 4;
        const uint32_t to = (uint32_t)part * pitch + (uint32_t)((key0 + row) * p.D + d) * 4u;
        bufStore4Agent(partK, to, 0, *reinterpret_cast<const at_f32x4*>(sumK + row * R + d));
        bufStore4Agent(partV, to, 0, *reinterpret_cast<const at_f32x4*>(sumV + row * R + d));
    }
    if (!p.arrivals) return;
    __shared__ int last;
    __builtin_amdgcn_s_waitcnt(0);   // this wave's parts have landed
    __syncthreads();                 // every wave's have
    unsigned* arrival = p.arrivals + bh * (uint32_t)groups + keyGroup;
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(arrival, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(p.sinkParts - 1);
    __syncthreads();
    if (!last) return;
    for (int x = (int)threadIdx.x; x < rows * quads; x += 256) {
        const int row = x / quads, d = x % quads * 4;
        const uint32_t from = (uint32_t)((key0 + row) * p.D + d) * 4u;
        const long long block = ((long long)bh * p.partRows + key0 + row) * p.D + d;   // the block's walk, of the launch before
        at_f32x4 k = *reinterpret_cast<const at_f32x4*>(p.dkPart + block), v = *reinterpret_cast<const at_f32x4*>(p.dvPart + block);
        for (int first = 0; first < p.sinkParts; first += 8) {
            f32x4 a[8], c8[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {   // past the last part: out of range, zeros
                const uint32_t at8 = first + i < p.sinkParts ? from + (uint32_t)(first + i) * pitch : kOOB;
                a[i] = bufLoad4Agent(partK, at8, 0);
                c8[i] = bufLoad4Agent(partV, at8, 0);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                k += a[i];
                v += c8[i];
            }
        }
        if (key0 + row >= nK) k = v = at_f32x4{0.f, 0.f, 0.f, 0.f};
        const long long to = firstKey + (long long)row * p.ldkv + d;
        *reinterpret_cast<at_u32x2*>(p.dk + to) = at_u32x2{atPack2<BF16>(k[0], k[1]), atPack2<BF16>(k[2], k[3])};
        *reinterpret_cast<at_u32x2*>(p.dv + to) = at_u32x2{atPack2<BF16>(v[0], v[1]), atPack2<BF16>(v[2], v[3])};
    }
    if (threadIdx.x == 0) __hip_atomic_store(arrival, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next launch
}

// ---------------------------------------------------------------- launches
constexpr int kMaxOffsets = 4096;   // of a bias's map

// The longest map whose sums in doubles fit a dQ workgroup's LDS beside its biases (rounded to 64) and static arrays: the tiles
// and positions of two buffers, dO's rows, delta. Four waves: 3697 offsets at a head dimension of 32, 3015 at 64, 2560 at 128;
// two waves: any map. Beyond, sums are floats.
template <int KD, int W>
constexpr int mostWide() {
    constexpr int rs = AtTile<KD>::RS, fixed = 4 * kTileKeys * rs * 2 + 2 * kTileKeys * 4 + (KD <= 2 ? 32 * W * rs * 2 : 0) + 32 * W * 4;
    constexpr int kLds = 160 << 10, kPadding = 256;   // of the static arrays' alignment
    return std::min(kMaxOffsets, (kLds - fixed - kPadding - 63 * 4) / (4 + 8 * W) - 2 * kMapEnd);
}

size_t biasLds(const AttnBiasParams& p, int tables) {
    return (size_t)((p.nOffsets + 2 * kMapEnd + 63) / 64 * 64) * sizeof(float) * tables;
}
template <int VIEW>
size_t dynamicLds(const AtParams<VIEW>& p, int tables) {
    if constexpr (VIEW == kAtBias) return biasLds(p, tables);
    return 0;
}
#define OMHIP_AT_LDS(kernel, view, tables) \
    if constexpr (view == kAtBias) OMHIP_CHECK(OMHIP_SET_MAX_DYNAMIC_LDS_ONCE(kernel, (kMaxOffsets + 2 * kMapEnd) * 4 * tables))

// Workgroups of a bias for sequences of up to 64 tokens and head dimensions of up to 64 (windows of an image) have half as many
// waves: of four, two would hold no token. 1024 windows of 7 x 7, 4 heads of 32: backward
// 75 us, with four waves 100.
template <int KD, int VIEW>
constexpr bool kShort = VIEW == kAtBias && KD <= 2;

template <bool BF16, int KD, int VIEW, int W>
int launchForwardKernel(const AtParams<VIEW>& p) {
    OMHIP_AT_LDS((attn_train_forward_kernel<BF16, KD, VIEW, W>), VIEW, 1);
    hipLaunchKernelGGL((attn_train_forward_kernel<BF16, KD, VIEW, W>), dim3(p.heads * p.blocks * p.keyParts), dim3(64 * W),
                       dynamicLds<VIEW>(p, 1), stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <bool BF16, int KD, int VIEW>
int launchForward(AtParams<VIEW>& p) {
    p.heads = (uint32_t)(p.B * p.H);
    p.blocks = (uint32_t)((p.Sq + kBlockQ - 1) / kBlockQ);
    if constexpr (kShort<KD, VIEW>) {
        if (p.Sq <= kBlockQ / 2 ? launchForwardKernel<BF16, KD, VIEW, kWaves / 2>(p) : launchForwardKernel<BF16, KD, VIEW, kWaves>(p))
            return -1;
    } else if (launchForwardKernel<BF16, KD, VIEW, kWaves>(p)) {
        return -1;
    }
    if (p.keyParts > 1) {
        const long long n = (long long)p.B * p.Sq * p.H * (p.D / 8);
        hipLaunchKernelGGL((attn_train_join_kernel<BF16>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
    }
    return 0;
}

template <bool BF16, int KD, int VIEW, class Sum, int W>
int launchDqKernel(const AtParams<VIEW>& p) {
    size_t lds = 0;
    if constexpr (VIEW == kAtBias) {
        constexpr int most = sizeof(Sum) == 8 ? mostWide<KD, W>() : kMaxOffsets;
        lds = biasLds(p, 1) + W * (size_t)(p.nOffsets + 2 * kMapEnd) * sizeof(Sum);
        OMHIP_CHECK(OMHIP_SET_MAX_DYNAMIC_LDS_ONCE((attn_train_dq_kernel<BF16, KD, VIEW, Sum, W>),
                                                   (most + 2 * kMapEnd) * (sizeof(float) + W * sizeof(Sum)) + 63 * sizeof(float)));
    }
    hipLaunchKernelGGL((attn_train_dq_kernel<BF16, KD, VIEW, Sum, W>), dim3(p.heads * p.blocks * p.keyParts), dim3(64 * W), lds,
                       stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <bool BF16, int KD, int VIEW, int W>
int launchDqSums(const AtParams<VIEW>& p) {
    if constexpr (VIEW == kAtBias) {
        if constexpr (mostWide<KD, W>() < kMaxOffsets)
            if (p.nOffsets > mostWide<KD, W>()) return launchDqKernel<BF16, KD, VIEW, float, W>(p);
        return launchDqKernel<BF16, KD, VIEW, double, W>(p);
    } else {
        return launchDqKernel<BF16, KD, VIEW, float, W>(p);
    }
}

template <bool BF16, int KD, int VIEW>
int launchDq(const AtParams<VIEW>& p) {
    if constexpr (kShort<KD, VIEW>)
        if (p.Sq <= kBlockQ / 2) return launchDqSums<BF16, KD, VIEW, kWaves / 2>(p);
    return launchDqSums<BF16, KD, VIEW, kWaves>(p);
}

template <bool BF16, int KD, int VIEW, int PAIRS>
int launchDkvKernel(const AtParams<VIEW>& p) {
    OMHIP_AT_LDS((attn_train_dkv_kernel<BF16, KD, VIEW, PAIRS>), VIEW, 2);
    hipLaunchKernelGGL((attn_train_dkv_kernel<BF16, KD, VIEW, PAIRS>), dim3(p.heads * p.blocks * p.parts), dim3(128 * PAIRS),
                       dynamicLds<VIEW>(p, p.H > p.Hkv ? 2 : 1), stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <bool BF16, int KD, int VIEW>
int launchBackward(AtParams<VIEW>& p) {
    if (p.Sq > 0) {
        p.heads = (uint32_t)(p.B * p.H);
        if constexpr (VIEW == kAtBias) p.heads = (uint32_t)(p.imageGroups * p.H);
        p.blocks = (uint32_t)((p.Sq + kBlockQ - 1) / kBlockQ);
        if (launchDq<BF16, KD, VIEW>(p)) return -1;
        if (p.keyParts > 1) {
            const long long n = (long long)p.B * p.Sq * p.H * (p.D / 8);
            hipLaunchKernelGGL((attn_train_dq_join_kernel<BF16>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream(), p);
            OMHIP_CHECK_LAUNCH();
        }
    }
    if (p.Sk > 0) {
        p.heads = (uint32_t)(p.B * p.Hkv);
        p.blocks = (uint32_t)((p.Sk + kBlockQ - 1) / kBlockQ);
        if constexpr (kShort<KD, VIEW>) {
            if (p.Sk <= kBlockQ / 2 ? launchDkvKernel<BF16, KD, VIEW, kWaves / 2>(p) : launchDkvKernel<BF16, KD, VIEW, kWaves>(p))
                return -1;
        } else if (launchDkvKernel<BF16, KD, VIEW, kWaves>(p)) {
            return -1;
        }
        int keys = p.parts > 1 ? p.Sk : 0;   // with fp32 sums
        if constexpr (VIEW == kAtWindow) {
            if (p.sinkParts > 0) {
                hipLaunchKernelGGL((attn_window_sinks_kernel<BF16, KD>), dim3(p.heads * ((p.first + 31) / 32) * p.sinkParts),
                                   dim3(256), 0, stream(), p);
                OMHIP_CHECK_LAUNCH();
            }
        }
        if (keys > 0) {
            const long long n = (long long)p.B * keys * p.Hkv * (p.D / 8);
            hipLaunchKernelGGL((attn_train_dkv_join_kernel<BF16, VIEW>), dim3((unsigned)((n + 255) / 256), 2), dim3(256), 0,
                               stream(), p, keys);
            OMHIP_CHECK_LAUNCH();
        }
    }
    return 0;
}

template <bool BF16, int VIEW>
int forward(AtParams<VIEW>& p) {
    switch ((p.D + 31) / 32) {
        case 1: return launchForward<BF16, 1, VIEW>(p);
        case 2: return launchForward<BF16, 2, VIEW>(p);
        case 3: return launchForward<BF16, 3, VIEW>(p);
        default: return launchForward<BF16, 4, VIEW>(p);
    }
}

template <bool BF16, int VIEW>
int backward(AtParams<VIEW>& p) {
    switch ((p.D + 31) / 32) {
        case 1: return launchBackward<BF16, 1, VIEW>(p);
        case 2: return launchBackward<BF16, 2, VIEW>(p);
        case 3: return launchBackward<BF16, 3, VIEW>(p);
        default: return launchBackward<BF16, 4, VIEW>(p);
    }
}

// ---------------------------------------------------------------- checks
// Whether the images' rows of `width` elements lie apart, image after image or token after token (gradients are written
// there).
bool imagesApart(int nBatch, int nSeq, long long nLd, long long nStride, long long nWidth) {
    return nBatch <= 1 || nSeq == 0 || nStride >= (nSeq - 1) * nLd + nWidth ||
           (nStride >= nWidth && nLd >= (nBatch - 1) * nStride + nWidth);
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What both directions ask of their sizes; 0, 1 (nothing to do) or -1.
int checkSizes(const char* name, int nDtype, long long nLdQ, long long nStrideQ, long long nLdKV, long long nStrideKV,
               int nBatch, int nSeqQ, int nSeqK, int nHeads, int nKVHeads, int nHeadDim, float fScale, bool backward) {
    if (nDtype != 0 && nDtype != 1) return fail("%s: dtype must be 0 (fp16) or 1 (bf16)", name);
    if (nBatch < 0 || nSeqQ < 0 || nSeqK < 0) return fail("%s: negative size", name);
    if (nHeads < 1 || nKVHeads < 1 || nHeads % nKVHeads != 0)
        return fail("%s: %d query heads are not a multiple of %d key heads", name, nHeads, nKVHeads);
    if (nHeadDim < 8 || nHeadDim > 128 || nHeadDim % 8 != 0)
        return fail("%s: head dimension %d (supported: multiples of 8 up to 128)", name, nHeadDim);
    if (!std::isfinite(fScale)) return fail("%s: scale must be finite", name);
    if (nLdQ < (long long)nHeads * nHeadDim || nLdKV < (long long)nKVHeads * nHeadDim)
        return fail("%s: a row stride is below the heads' width", name);
    if (nLdQ >= kAtMaxLd || nLdKV >= kAtMaxLd) return fail("%s: a row stride reaches 2^23 elements", name);
    if ((nLdQ | nStrideQ | nLdKV | nStrideKV) & 7) return fail("%s: strides must be multiples of 8 elements", name);
    if (nStrideQ < 0 || nStrideKV < 0) return fail("%s: negative stride", name);
    // grid and row counters
    if (nSeqQ > (1 << 30) || nSeqK > (1 << 30)) return fail("%s: a sequence exceeds 2^30 tokens", name);
    const long long heads = (long long)nBatch * nHeads;   // below 2^51 (row strides); at most 2^24 tiles each
    if (heads > 0x3fffffffLL || heads * ((std::max(nSeqQ, nSeqK) + 63LL) / 64) > 0x3fffffffLL)
        return fail("%s: too many (image, head, token) triples", name);
    // a launch takes 2^32 - 1 threads in a dimension, and silently drops the bits above: 256 threads for a block of
    // queries, 512 for one of keys (shared walks, which multiply them, are for grids of a few per CU)
    if (heads * ((nSeqQ + kBlockQ - 1LL) / kBlockQ) * 256 > 0xffffffffLL)
        return fail("%s: too many (image, head, block of %d queries) triples", name, kBlockQ);
    if (backward && (long long)nBatch * nKVHeads * ((nSeqK + kBlockQ - 1LL) / kBlockQ) * 512 > 0xffffffffLL)
        return fail("%s: too many (image, key head, block of %d keys) triples", name, kBlockQ);
    return nBatch == 0 ? 1 : 0;
}

// The arguments of a forward call whose sizes are checked and not empty; 0 or -1.
int forwardArguments(AttnTrainParams& p, const char* name, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV,
                     long long nLdQ, long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                     const int* pKeyLens, int bCausal, uint16_t* pOut, float* pLse, int nBatch, int nSeqQ, int nSeqK, int nHeads,
                     int nKVHeads, int nHeadDim, float fScale) {
    if (!pQ || !pOut || !pLse || (nSeqK > 0 && (!pK || !pV))) return fail("%s: null pointer", name);
    if (!aligned16(pQ) || !aligned16(pK) || !aligned16(pV) || !aligned16(pOut))
        return fail("%s: data must be 16-byte aligned", name);
    if (!aligned4(pLse) || !aligned4(pQueryLens) || !aligned4(pKeyLens))
        return fail("%s: a pointer is not aligned to its elements", name);
    p.q = pQ; p.k = pK; p.v = pV;
    p.ldq = nLdQ; p.sq = nStrideQ; p.ldkv = nLdKV; p.skv = nStrideKV;
    p.qLens = pQueryLens; p.kLens = pKeyLens;
    p.B = nBatch; p.Sq = nSeqQ; p.Sk = nSeqK; p.H = nHeads; p.Hkv = nKVHeads; p.D = nHeadDim;
    p.causal = bCausal != 0;
    p.scale = fScale;
    p.out = pOut; p.lse = pLse;
    return 0;
}

// The parts of the forward walks of `tiles` tiles and their workspace; 0 or -1.
int forwardParts(AttnTrainParams& p, int tiles) {
    p.keyParts = walkParts((long long)p.B * p.H * ((p.Sq + kBlockQ - 1) / kBlockQ), tiles, 2LL * cuCount());
    if (p.keyParts > 1) {
        const size_t rows = (size_t)p.B * p.H * p.Sq * p.keyParts;
        p.rowPart = static_cast<float*>(workspace(rows * (p.D + 1) * sizeof(float), kWsOperand));
        if (!p.rowPart) return -1;   // workspace() recorded the cause
        p.lsePart = p.rowPart + rows * p.D;
    }
    return 0;
}

// The same of a backward call.
int backwardArguments(AttnTrainParams& p, const char* name, const uint16_t* pQ, const uint16_t* pK, const uint16_t* pV,
                      long long nLdQ, long long nStrideQ, long long nLdKV, long long nStrideKV, const int* pQueryLens,
                      const int* pKeyLens, int bCausal, const uint16_t* pOut, const float* pLse, const uint16_t* pGradOut,
                      uint16_t* pGradQ, uint16_t* pGradK, uint16_t* pGradV, int nBatch, int nSeqQ, int nSeqK, int nHeads,
                      int nKVHeads, int nHeadDim, float fScale) {
    if ((nSeqQ > 0 && (!pQ || !pOut || !pLse || !pGradOut || !pGradQ)) || (nSeqK > 0 && (!pK || !pV || !pGradK || !pGradV)))
        return fail("%s: null pointer", name);
    for (const void* x : {(const void*)pQ, (const void*)pK, (const void*)pV, (const void*)pOut, (const void*)pGradOut,
                          (const void*)pGradQ, (const void*)pGradK, (const void*)pGradV})
        if (!aligned16(x)) return fail("%s: data must be 16-byte aligned", name);
    if (!aligned4(pLse) || !aligned4(pQueryLens) || !aligned4(pKeyLens))
        return fail("%s: a pointer is not aligned to its elements", name);
    if (!imagesApart(nBatch, nSeqQ, nLdQ, nStrideQ, (long long)nHeads * nHeadDim) ||
        !imagesApart(nBatch, nSeqK, nLdKV, nStrideKV, (long long)nKVHeads * nHeadDim))
        return fail("%s: the images' gradients would overlap at these strides", name);
    p.q = pQ; p.k = pK; p.v = pV;
    p.ldq = nLdQ; p.sq = nStrideQ; p.ldkv = nLdKV; p.skv = nStrideKV;
    p.qLens = pQueryLens; p.kLens = pKeyLens;
    p.B = nBatch; p.Sq = nSeqQ; p.Sk = nSeqK; p.H = nHeads; p.Hkv = nKVHeads; p.D = nHeadDim;
    p.causal = bCausal != 0;
    p.scale = fScale;
    p.out = const_cast<uint16_t*>(pOut); p.lse = const_cast<float*>(pLse);
    p.gradOut = pGradOut;
    p.dq = pGradQ; p.dk = pGradK; p.dv = pGradV;
    p.SqP = (nSeqQ + kTileKeys - 1) / kTileKeys * kTileKeys;
    return 0;
}

// The parts of dQ's walks of `tiles` tiles, and the workspace of row statistics, of those parts, of dK and dV's `sums` floats
// each and, where `more` is given, of so many others; 0 or -1.
int backwardParts(AttnTrainParams& p, int tiles, size_t sums, size_t others, float** more) {
    const size_t rows = (size_t)p.B * p.H * p.SqP;
    p.keyParts = walkParts((long long)p.B * p.H * ((p.Sq + kBlockQ - 1) / kBlockQ), tiles, 2LL * cuCount());
    const size_t rowSums = p.keyParts > 1 ? (size_t)p.B * p.H * p.Sq * p.keyParts * p.D : 0;
    if (rows) {
        p.stats = static_cast<float*>(workspace(((rows + sums) * 2 + rowSums + others) * sizeof(float), kWsOperand));
        if (!p.stats) return -1;   // workspace() recorded the cause
        p.dkPart = p.stats + 2 * rows;
        p.dvPart = p.dkPart + sums;
        p.rowPart = p.dvPart + sums;
        if (more) *more = p.rowPart + rowSums;
    }
    return 0;
}

}  // namespace

}  // namespace omhip
