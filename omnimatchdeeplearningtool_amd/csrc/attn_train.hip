// attn_train.hip — attention for training on fp16 / bf16 data: a forward pass
// that keeps each row's log-sum-exp, and the backward pass that computes the
// probabilities again from it.
//
// The reference trains MultiHeadAttention through autograd nodes of the
// unfused chain (src/engine/om.engine.vit.ixx:150-239: qkvSplitHeads,
// tensorBatchedMatmul, tensorSoftmaxLastDim, tensorBatchedMatmul, mergeHeads),
// which keep the S x S probabilities. With S = scale Q K^T over the keys that
// a query sees, P = exp(S - lse), lse = log sum exp S:
//   O  = P V                    dV = P^T dO
//   dP = dO V^T                 dS = P (dP - delta),  delta_i = sum_d dO_id O_id
//   dQ = scale dS K             dK = scale dS^T Q
// A key head's dK and dV are the sums over the query heads that read it. All
// sums are in fp32 in a fixed order; the products take P and dS rounded to the
// data's type, as operands of the matrix cores.
//
// Query i sees key j where j < the image's key length and, if causal,
// j <= i + nSeqK - nSeqQ. A query that sees none, or whose scores are all
// -inf, has O = 0 and lse = -inf and passes no gradient.
#include "attn_tile.hpp"
#include "omhip_internal.hpp"
#include "../../include/omhip.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

namespace omhip {

namespace {

constexpr int kWaves = 4;
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
    float *dkPart, *dvPart;         // [B, Hkv, parts, blocks * kBlockQ, D]
    uint32_t heads, blocks;         // grid: heads x blocks workgroups
};

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
template <bool BF16, int KD>
__global__ __launch_bounds__(256, 2) void attn_train_forward_kernel(AttnTrainParams p) {
    using T = AtTile<KD>;
    constexpr float kShift = BF16 ? 0.f : 6.f;
    __shared__ __attribute__((aligned(256))) uint16_t k0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t k1[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v1[kTileKeys * T::RS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = lane & 31, h = lane >> 5;
    uint32_t bh, qb;
    atPlace(blockIdx.x, p.heads, p.blocks * p.keyParts, p.causal, bh, qb);
    const int part = (int)(qb % (uint32_t)p.keyParts);
    qb = p.blocks - 1 - qb / (uint32_t)p.keyParts;   // causal: the longest walks first
    const int b = (int)(bh / (uint32_t)p.H), head = (int)(bh % (uint32_t)p.H);
    const int kvHead = head / (p.H / p.Hkv);
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk);
    const int off = p.Sk - p.Sq;
    const int q0 = (int)qb * kBlockQ + wave * 32;   // the wave's first query
    const int query = q0 + l;
    const uint16_t* kBase = p.k + (long long)b * p.skv + (long long)kvHead * p.D;
    const uint16_t* vBase = p.v + (long long)b * p.skv + (long long)kvHead * p.D;

    // keys seen by the workgroup's and by the wave's queries
    const int blockLast = min((int)qb * kBlockQ + kBlockQ, nQ) - 1;
    int kEnd = blockLast >= (int)qb * kBlockQ ? nK : 0;
    if (p.causal) kEnd = min(kEnd, blockLast + off + 1);
    int waveEnd = q0 < nQ ? kEnd : 0;
    if (p.causal) waveEnd = min(waveEnd, q0 + 32 + off);
    const int tiles = kEnd > 0 ? (kEnd + kTileKeys - 1) / kTileKeys : 0;
    const int tBegin = (int)((long long)tiles * part / p.keyParts), nt = (int)((long long)tiles * (part + 1) / p.keyParts);

    const float c = fmaxf(fabsf(p.scale) * kAtLog2e, FLT_MIN);
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    const typename T::Lane at(lane);
    typename T::template Copy<kTileKeys, kWaves> copy;
    const uint32_t ld2 = (uint32_t)p.ldkv * 2u;
    copy.init(wave, lane, ld2, p.D);
    auto fetch = [&](int t, uint16_t* kd, uint16_t* vd) {
        const long long at = (long long)t * kTileKeys * p.ldkv;
        copy.run(kBase + at, nK - t * kTileKeys, ld2, p.D, kd, wave);
        copy.run(vBase + at, nK - t * kTileKeys, ld2, p.D, vd, wave);
    };

    // the wave's queries through its part of the second pair of buffers, which tile 1 is copied to after the first barrier
    uint16_t* stage = (wave < 2 ? k1 : v1) + (wave & 1) * 32 * T::RS;
    T::start(p.q + (long long)b * p.sq + (long long)q0 * p.ldq + (long long)head * p.D, nQ - q0, p.ldq, p.D, stage, lane);
    if (nt > tBegin) fetch(tBegin, k0, v0);
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

    auto tile = [&](int t, const uint16_t* kd, const uint16_t* vd) {
        at_f32x16 s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
            for (int st = 0; st < T::NS; ++st) s[kb] = atMfma<BF16>(at.natural(kd, 32 * kb, st), qf[st], s[kb]);
        }
        atPipeline<2 * T::NS, 1, 4>();
        const int key0 = t * kTileKeys;
        if (key0 + kTileKeys > nK || (p.causal && key0 + kTileKeys - 1 > q0 + off)) {
            const int seen = (p.causal ? min(nK, query + off + 1) : nK) - key0 - 4 * h;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * kb + 8 * (r / 4) + r % 4 >= seen) s[kb][r] = -INFINITY;
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
    auto trip = [&](int t, const uint16_t* kd, const uint16_t* vd, uint16_t* kNext, uint16_t* vNext) {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1, kNext, vNext);
        if (t * kTileKeys < waveEnd) tile(t, kd, vd);
    };
    int t = tBegin;
    for (; t + 1 < nt; t += 2) {
        trip(t, k0, v0, k1, v1);
        trip(t + 1, k1, v1, k0, v0);
    }
    if (t < nt) trip(t, k0, v0, k1, v1);

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
template <bool BF16, int KD>
__global__ __launch_bounds__(256, 2) void attn_train_dq_kernel(AttnTrainParams p) {
    using T = AtTile<KD>;
    __shared__ __attribute__((aligned(256))) uint16_t k0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v0[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t k1[kTileKeys * T::RS];
    __shared__ __attribute__((aligned(256))) uint16_t v1[kTileKeys * T::RS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = lane & 31, h = lane >> 5;
    uint32_t bh, qb;
    atPlace(blockIdx.x, p.heads, p.blocks * p.keyParts, p.causal, bh, qb);
    const int part = (int)(qb % (uint32_t)p.keyParts);
    qb = p.blocks - 1 - qb / (uint32_t)p.keyParts;   // causal: the longest walks first
    const int b = (int)(bh / (uint32_t)p.H), head = (int)(bh % (uint32_t)p.H);
    const int kvHead = head / (p.H / p.Hkv);
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk);
    const int off = p.Sk - p.Sq;
    const int q0 = (int)qb * kBlockQ + wave * 32;
    const int query = q0 + l;
    const uint16_t* kBase = p.k + (long long)b * p.skv + (long long)kvHead * p.D;
    const uint16_t* vBase = p.v + (long long)b * p.skv + (long long)kvHead * p.D;

    const int blockLast = min((int)qb * kBlockQ + kBlockQ, nQ) - 1;
    int kEnd = blockLast >= (int)qb * kBlockQ ? nK : 0;
    if (p.causal) kEnd = min(kEnd, blockLast + off + 1);
    int waveEnd = q0 < nQ ? kEnd : 0;
    if (p.causal) waveEnd = min(waveEnd, q0 + 32 + off);
    const int tiles = kEnd > 0 ? (kEnd + kTileKeys - 1) / kTileKeys : 0;
    const int tBegin = (int)((long long)tiles * part / p.keyParts), nt = (int)((long long)tiles * (part + 1) / p.keyParts);

    const float c = p.scale * kAtLog2e;
    const typename T::Lane at(lane);
    typename T::template Copy<kTileKeys, kWaves> copy;
    const uint32_t ld2 = (uint32_t)p.ldkv * 2u;
    copy.init(wave, lane, ld2, p.D);
    auto fetch = [&](int t, uint16_t* kd, uint16_t* vd) {
        const long long o = (long long)t * kTileKeys * p.ldkv;
        copy.run(kBase + o, nK - t * kTileKeys, ld2, p.D, kd, wave);
        copy.run(vBase + o, nK - t * kTileKeys, ld2, p.D, vd, wave);
    };
    // Q and dO of the wave's queries, and delta. Head dimensions up to 64: by whole rows, Q through its part of the second
    // pair of buffers, which tile 1 is copied to after the first barrier, dO through rows of its own; larger ones straight
    // into fragments, 32 rows for 16 bytes an instruction: rows of dO's own would leave one workgroup a CU, and a head
    // dimension of 128 is at 256 registers and 12-20 bytes of scratch without the chunks of dO and O for delta. (dO through
    // the first pair of buffers, free until the first tile is fetched, has not been measured.)
    constexpr bool kStaged = KD <= 2;
    __shared__ __attribute__((aligned(256))) uint16_t gStage[kStaged ? kBlockQ * T::RS : 8];
    __shared__ float rowDelta[kWaves][32];
    const uint16_t* qRows = p.q + (long long)b * p.sq + (long long)q0 * p.ldq + (long long)head * p.D;
    const uint16_t* gRows = p.gradOut + (((long long)b * p.Sq + q0) * p.H + head) * p.D;
    const uint16_t* oRows = p.out + (((long long)b * p.Sq + q0) * p.H + head) * p.D;
    const long long ldo = (long long)p.H * p.D;
    const float lse = query < nQ ? p.lse[(long long)bh * p.Sq + query] : -INFINITY;
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
        if (nt > tBegin) fetch(tBegin, k0, v0);
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
        if (nt > tBegin) fetch(tBegin, k0, v0);
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
        float* to = p.stats + 2 * ((long long)bh * p.SqP + q0) + l;
        to[0] = shift + kRaise<BF16>;
        to[32] = delta;
    }
    at_f32x16 dq[KD];
#pragma unroll
    for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) dq[t][r] = 0.f;
    DsScale<BF16, KD> scale;

    auto tile = [&](auto edgeTag, int key0, const uint16_t* kd, const uint16_t* vd) {
        constexpr bool EDGE = decltype(edgeTag)::value;   // some query does not see some of the keys
        const int seen = (p.causal ? min(nK, query + off + 1) : nK) - key0 - 4 * h;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            if (EDGE && kb == 1 && key0 + 32 >= waveEnd) break;   // the wave's queries see none of these
            at_f32x16 s, dp;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = dp[r] = 0.f;
#pragma unroll
            for (int st = 0; st < T::NS; ++st) {
                s = atMfma<BF16>(at.natural(kd, 32 * kb, st), qf[st], s);
                dp = atMfma<BF16>(at.natural(vd, 32 * kb, st), gf[st], dp);
            }
            atPipeline<2 * T::NS, 1, 4>();
            float most = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, shift));
                if (EDGE && 32 * kb + 8 * (r / 4) + r % 4 >= seen) e = 0.f;
                s[r] = e * (dp[r] - delta);
                if constexpr (!BF16) most = fmaxf(most, fabsf(s[r]));
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
    auto step = [&](int t, const uint16_t* kd, const uint16_t* vd) {
        const int key0 = t * kTileKeys;
        if (key0 >= waveEnd) return;
        if (key0 + kTileKeys > nK || (p.causal && key0 + kTileKeys - 1 > q0 + off))
            tile(std::true_type{}, key0, kd, vd);
        else
            tile(std::false_type{}, key0, kd, vd);
    };
    auto trip = [&](int t, const uint16_t* kd, const uint16_t* vd, uint16_t* kNext, uint16_t* vNext) {   // as in the forward pass
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (t + 1 < nt) fetch(t + 1, kNext, vNext);
        step(t, kd, vd);
    };
    int t = tBegin;
    for (; t + 1 < nt; t += 2) {
        trip(t, k0, v0, k1, v1);
        trip(t + 1, k1, v1, k0, v0);
    }
    if (t < nt) trip(t, k0, v0, k1, v1);
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
    float* stats[3];     // shift, delta
    float* weights;      // P by tile parity and pair
};

// A wave's work in attn_train_dkv_kernel.
template <bool BF16, int KD, bool SECOND>
__device__ __forceinline__ void dkvWalk(const AttnTrainParams& p, const DkvBuffers& lds, int wave, int lane) {
    using T = AtTile<KD>;
    constexpr float kLower = BF16 ? 1.f : 1.f / 32768.f;   // takes kRaise out
    const int l = lane & 31, h = lane >> 5, pair = wave & 3;
    uint32_t bh, block;
    atPlace(blockIdx.x, p.heads, p.blocks * p.parts, p.causal, bh, block);   // causal: the first keys' walks are longest
    const int part = (int)(block % (uint32_t)p.parts);
    block /= (uint32_t)p.parts;
    const int b = (int)(bh / (uint32_t)p.Hkv), kvHead = (int)(bh % (uint32_t)p.Hkv);
    const int group = p.H / p.Hkv;
    const int nQ = atLength(p.qLens, b, p.Sq), nK = atLength(p.kLens, b, p.Sk);
    const int off = p.Sk - p.Sq;
    const int key0 = (int)block * kBlockQ + pair * 32;
    const int key = key0 + l;

    // query tiles that see a key of the workgroup: t0 .. t1 of each head of the group; this part's share of them
    const int t0 = p.causal ? max(0, (int)block * kBlockQ - off) / kTileQ : 0;
    const int t1 = (int)block * kBlockQ < nK ? (nQ + kTileQ - 1) / kTileQ : 0;
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
    constexpr int kCopyWaves = T::CH * kTileQ / 64 < 8 ? T::CH * kTileQ / 64 : 8;   // a head dimension of 32 has 2 instructions
    typename T::template Copy<kTileQ, kCopyWaves> copyQ, copyG;
    const uint32_t ldq2 = (uint32_t)p.ldq * 2u, ldg2 = (uint32_t)(p.H * p.D) * 2u;
    copyQ.init(wave, lane, ldq2, p.D);
    copyG.init(wave, lane, ldg2, p.D);
    int fetchHead = per > 0 ? kvHead * group + begin / per : 0, fetchT = per > 0 ? t0 + begin % per : 0;
    auto fetch = [&](uint16_t* qd, uint16_t* gd, float* sd) {   // the next tile of the walk
        const long long first = (long long)fetchT * kTileQ;
        const int rows = nQ - fetchT * kTileQ;
        if (wave < kCopyWaves) {
            copyQ.run(p.q + (long long)b * p.sq + first * p.ldq + (long long)fetchHead * p.D, rows, ldq2, p.D, qd, wave);
            copyG.run(p.gradOut + (((long long)b * p.Sq + first) * p.H + fetchHead) * p.D, rows, ldg2, p.D, gd, wave);
        }
        if (wave == 7)   // rows past the query length hold -inf and 0
            atCopy4(atView(p.stats + 2 * (((long long)b * p.H + fetchHead) * p.SqP + first), 2 * kTileQ * 4), sd, lane * 4);
        if (++fetchT == t1) {
            fetchT = t0;
            ++fetchHead;
        }
    };
    at_f32x16 acc[KD];
#pragma unroll
    for (int t = 0; t < KD; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    DsScale<BF16, KD> scale;

    if (n > 0) fetch(lds.q[0], lds.g[0], lds.stats[0]);
    __builtin_amdgcn_s_waitcnt(0);
    at_u32x4 own[T::NS];   // K, or V
    T::take(at, stage, own);

    // nat: the tile whose product with the wave's own fragments makes S or dP; tr: the one that the sums take
    auto work = [&](int first, const uint16_t* nat, const uint16_t* tr, const float* sd, float* wd) {
        at_f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int st = 0; st < T::NS; ++st) s = atMfma<BF16>(at.natural(nat, 0, st), own[st], s);
        atPipeline<T::NS, 1, T::NS < 4 ? T::NS : 4>();
        if constexpr (!SECOND) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const at_f32x4 shift = *reinterpret_cast<const at_f32x4*>(sd + 8 * j + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    s[4 * j + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * j + e], c, shift[e]));
            }
            if (p.causal && first + off < key0 + 31) {
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
    auto meet = [&](int i, auto bufTag) {
        constexpr int NEXT = (decltype(bufTag)::value + 1) % 3;
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (i + 1 < n) fetch(lds.q[NEXT], lds.g[NEXT], lds.stats[NEXT]);
    };
    auto trip = [&](int i, auto bufTag) {
        constexpr int BUF = decltype(bufTag)::value, MINE = SECOND ? (BUF + 2) % 3 : BUF;
        meet(i, bufTag);
        float* wd = lds.weights + (((SECOND ? ~i : i) & 1) * 4 + pair) * (kTileQ * 32);
        if constexpr (SECOND)
            work(t * kTileQ, lds.g[MINE], lds.q[MINE], lds.stats[MINE], wd);
        else
            work(t * kTileQ, lds.q[MINE], lds.g[MINE], lds.stats[MINE], wd);
        if (++t == t1) t = t0;
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
    if (p.parts > 1) {
        const long long row = ((long long)bh * p.parts + part) * ((long long)p.blocks * kBlockQ) + key;
        storeColumnF32<KD>((SECOND ? p.dkPart : p.dvPart) + row * p.D, acc, f, h, p.D, false);
    } else {
        __syncthreads();   // every wave is done with the tiles and the weights
        storeRows<BF16, KD>((SECOND ? p.dk : p.dv) + first, p.ldkv, p.Sk - key0, acc, f, key >= nK, stage, lane, p.D);
    }
}

template <bool BF16, int KD>
__global__ __launch_bounds__(512, 2) void attn_train_dkv_kernel(AttnTrainParams p) {
    constexpr int N = kTileQ * AtTile<KD>::RS;
    __shared__ __attribute__((aligned(256))) uint16_t q0[N];
    __shared__ __attribute__((aligned(256))) uint16_t q1[N];
    __shared__ __attribute__((aligned(256))) uint16_t q2[N];
    __shared__ __attribute__((aligned(256))) uint16_t g0[N];
    __shared__ __attribute__((aligned(256))) uint16_t g1[N];
    __shared__ __attribute__((aligned(256))) uint16_t g2[N];
    __shared__ __attribute__((aligned(256))) float s0[2 * kTileQ];
    __shared__ __attribute__((aligned(256))) float s1[2 * kTileQ];
    __shared__ __attribute__((aligned(256))) float s2[2 * kTileQ];
    __shared__ __attribute__((aligned(16))) float weights[2 * 4 * kTileQ * 32];   // behind the tiles: their offsets fit a read's 16 bits
    const DkvBuffers lds{{q0, q1, q2}, {g0, g1, g2}, {s0, s1, s2}, weights};
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave < 4)
        dkvWalk<BF16, KD, false>(p, lds, wave, lane);
    else
        dkvWalk<BF16, KD, true>(p, lds, wave, lane);
}

// The parts' sums of dK (blockIdx.y 0) or dV (1), eight values of a key a thread.
template <bool BF16>
__global__ __launch_bounds__(256) void attn_train_dkv_join_kernel(AttnTrainParams p) {
    const int chunks = p.D / 8;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;   // (b, key, kvHead, chunk)
    if (i >= (long long)p.B * p.Sk * p.Hkv * chunks) return;
    const int c = (int)(i % chunks);
    const long long bkh = i / chunks;
    const int kvHead = (int)(bkh % p.Hkv);
    const int key = (int)(bkh / p.Hkv % p.Sk), b = (int)(bkh / p.Hkv / p.Sk);
    const long long keys = (long long)p.blocks * kBlockQ;
    const float* from = (blockIdx.y ? p.dvPart : p.dkPart) +
                        (((long long)b * p.Hkv + kvHead) * p.parts * keys + key) * p.D + c * 8;
    at_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int part = 0; part < p.parts; ++part)
#pragma unroll
        for (int e = 0; e < 2; ++e)
            s[e] += *reinterpret_cast<const at_f32x4*>(from + (long long)part * keys * p.D + 4 * e);
    at_u32x4 v = {atPack2<BF16>(s[0][0], s[0][1]), atPack2<BF16>(s[0][2], s[0][3]), atPack2<BF16>(s[1][0], s[1][1]),
                  atPack2<BF16>(s[1][2], s[1][3])};
    if (key >= atLength(p.kLens, b, p.Sk)) v = at_u32x4{0u, 0u, 0u, 0u};
    uint16_t* to = (blockIdx.y ? p.dv : p.dk) + (long long)b * p.skv + (long long)key * p.ldkv + (long long)kvHead * p.D;
    *reinterpret_cast<at_u32x4*>(to + c * 8) = v;
}

// ---------------------------------------------------------------- checks and launches
template <bool BF16, int KD>
int launchForward(AttnTrainParams& p) {
    p.heads = (uint32_t)(p.B * p.H);
    p.blocks = (uint32_t)((p.Sq + kBlockQ - 1) / kBlockQ);
    hipLaunchKernelGGL((attn_train_forward_kernel<BF16, KD>), dim3(p.heads * p.blocks * p.keyParts), dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    if (p.keyParts > 1) {
        const long long n = (long long)p.B * p.Sq * p.H * (p.D / 8);
        hipLaunchKernelGGL((attn_train_join_kernel<BF16>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
    }
    return 0;
}

template <bool BF16, int KD>
int launchBackward(AttnTrainParams& p) {
    if (p.Sq > 0) {
        p.heads = (uint32_t)(p.B * p.H);
        p.blocks = (uint32_t)((p.Sq + kBlockQ - 1) / kBlockQ);
        hipLaunchKernelGGL((attn_train_dq_kernel<BF16, KD>), dim3(p.heads * p.blocks * p.keyParts), dim3(256), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
        if (p.keyParts > 1) {
            const long long n = (long long)p.B * p.Sq * p.H * (p.D / 8);
            hipLaunchKernelGGL((attn_train_dq_join_kernel<BF16>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream(), p);
            OMHIP_CHECK_LAUNCH();
        }
    }
    if (p.Sk > 0) {
        p.heads = (uint32_t)(p.B * p.Hkv);
        p.blocks = (uint32_t)((p.Sk + kBlockQ - 1) / kBlockQ);
        hipLaunchKernelGGL((attn_train_dkv_kernel<BF16, KD>), dim3(p.heads * p.blocks * p.parts), dim3(512), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
        if (p.parts > 1) {
            const long long n = (long long)p.B * p.Sk * p.Hkv * (p.D / 8);
            hipLaunchKernelGGL((attn_train_dkv_join_kernel<BF16>), dim3((unsigned)((n + 255) / 256), 2), dim3(256), 0,
                               stream(), p);
            OMHIP_CHECK_LAUNCH();
        }
    }
    return 0;
}

template <bool BF16>
int forward(AttnTrainParams& p) {
    switch ((p.D + 31) / 32) {
        case 1: return launchForward<BF16, 1>(p);
        case 2: return launchForward<BF16, 2>(p);
        case 3: return launchForward<BF16, 3>(p);
        default: return launchForward<BF16, 4>(p);
    }
}

template <bool BF16>
int backward(AttnTrainParams& p) {
    switch ((p.D + 31) / 32) {
        case 1: return launchBackward<BF16, 1>(p);
        case 2: return launchBackward<BF16, 2>(p);
        case 3: return launchBackward<BF16, 3>(p);
        default: return launchBackward<BF16, 4>(p);
    }
}

// Workgroups that share a block's walk of `tiles` 64-row tiles: as many as give every CU `perCu` workgroups and no more
// (one workgroup past that starts a second round: 1 x 2048 x 5 heads of 128 causal backward 75.3 us, rounded up 89.4), of
// four tiles at least. Two of them, the long walk of one block and the short one of another, make a causal grid even; dK / dV
// of head dimensions up to 64 hold two workgroups a CU at once and ask for four. (Parts cost fp32 sums of every row: 2 x
// 4096 x 16 heads on 4 of 128 backward 499 us with two a CU, 516 with four, about 730 unshared.)
int walkParts(long long blocks, int tiles, int perCu) {
    if (blocks == 0 || tiles == 0) return 1;
    return (int)std::clamp<long long>((long long)perCu * cuCount() / blocks, 1, std::max(1, tiles / 4));
}

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

}  // namespace

}  // namespace omhip

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
    if (!pQ || !pOut || !pLse || (nSeqK > 0 && (!pK || !pV))) return fail("%s: null pointer", name);
    if (!aligned16(pQ) || !aligned16(pK) || !aligned16(pV) || !aligned16(pOut))
        return fail("%s: data must be 16-byte aligned", name);
    if (!aligned4(pLse) || !aligned4(pQueryLens) || !aligned4(pKeyLens))
        return fail("%s: a pointer is not aligned to its elements", name);
    AttnTrainParams p{};
    p.q = pQ; p.k = pK; p.v = pV;
    p.ldq = nLdQ; p.sq = nStrideQ; p.ldkv = nLdKV; p.skv = nStrideKV;
    p.qLens = pQueryLens; p.kLens = pKeyLens;
    p.B = nBatch; p.Sq = nSeqQ; p.Sk = nSeqK; p.H = nHeads; p.Hkv = nKVHeads; p.D = nHeadDim;
    p.causal = bCausal != 0;
    p.scale = fScale;
    p.out = pOut; p.lse = pLse;
    p.keyParts = walkParts((long long)nBatch * nHeads * ((nSeqQ + kBlockQ - 1) / kBlockQ), (nSeqK + kTileKeys - 1) / kTileKeys, 2);
    if (p.keyParts > 1) {
        const size_t rows = (size_t)nBatch * nHeads * nSeqQ * p.keyParts;
        p.rowPart = static_cast<float*>(workspace(rows * (nHeadDim + 1) * sizeof(float), kWsOperand));
        if (!p.rowPart) return -1;   // workspace() recorded the cause
        p.lsePart = p.rowPart + rows * nHeadDim;
    }
    return nDtype == 1 ? forward<true>(p) : forward<false>(p);
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
    AttnTrainParams p{};
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
    const size_t rows = (size_t)nBatch * nHeads * p.SqP;
    const size_t keyBlocks = (size_t)nBatch * nKVHeads * ((nSeqK + kBlockQ - 1) / kBlockQ);
    p.parts = walkParts((long long)keyBlocks, p.SqP / kTileKeys * (nHeads / nKVHeads), nHeadDim <= 64 ? 4 : 2);
    const long long queryBlocks = (long long)nBatch * nHeads * ((nSeqQ + kBlockQ - 1) / kBlockQ);
    p.keyParts = walkParts(queryBlocks, (nSeqK + kTileKeys - 1) / kTileKeys, 2);
    const size_t rowSums = p.keyParts > 1 ? (size_t)nBatch * nHeads * nSeqQ * p.keyParts * nHeadDim : 0;
    const size_t sums = p.parts > 1 ? keyBlocks * p.parts * kBlockQ * nHeadDim : 0;
    if (rows) {
        p.stats = static_cast<float*>(workspace(((rows + sums) * 2 + rowSums) * sizeof(float), kWsOperand));
        if (!p.stats) return -1;   // workspace() recorded the cause
        p.dkPart = p.stats + 2 * rows;
        p.dvPart = p.dkPart + sums;
        p.rowPart = p.dvPart + sums;
    }
    return nDtype == 1 ? backward<true>(p) : backward<false>(p);
}

}  // extern "C"
