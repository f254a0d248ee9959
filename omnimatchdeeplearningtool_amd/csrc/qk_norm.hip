// qk_norm.hip — norms of queries and keys for each head with the rotation by
// their positions in the same pass, and the gradients.
//
//   z = x inv w,  inv = 1 / sqrt(mean(x^2) + eps)   over a head's values
//   y = rotate(z):  pairs (a, b) of the first nRotary values -> (a c - b s, b c + a s),
//       c, s = cos, sin of the row of the token's position
// and with g = rotate^T(gy), xhat = x inv:
//   dx = inv (g w - xhat mean(g w xhat))            dw = sum of g xhat over tokens and heads
// x is read once and y written once; the backward pass reads x and gy and
// computes inv again (the row is at hand) rather than keep it. All in fp32.
#include "fastdiv.hpp"
#include "omhip_internal.hpp"
#include "vec_io.hpp"
#include "../../include/omhip.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace omhip {

namespace {

struct QkSide {                      // queries or keys
    const void *x, *g;               // input; backward: the output's gradient
    void* out;                       // output; backward: the input's gradient
    long long ldX, strideX, ldG, strideG, ldOut, strideOut;
    const float* weight;             // [D] or null
    float* gradWeight;               // [D] or null
    FastDiv heads;
    uint32_t rows, blocks;           // (image, token, head) triples; workgroups
};

struct QkNormParams {
    QkSide side[2];
    const float *cos, *sin;          // [table, rotary / 2]
    const int* positions;            // [images * seq] or null
    float* partials;                 // backward: [blocks of both sides, D]
    FastDiv seq;
    int D, rotary, table, interleaved;
    int unitsLog2;                   // lanes a row, a power of two
    float eps;
    bool streaming;
};

// W values from p on as fp32 and back; p's alignment is 16 bytes or, of 4 halves, 8.
template <int DT, int W>
struct Chunk {
    using Elem = typename Vec8<DT>::Elem;
    typedef Elem Piece __attribute__((ext_vector_type(W), aligned(DT != 2 && W == 4 ? 8 : 16)));
    static __device__ __forceinline__ void load(const Elem* p, float (&v)[W]) {
        const Piece e = *reinterpret_cast<const Piece*>(p);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = Vec8<DT>::toFloat(e[i]);
    }
    template <bool STREAM>
    static __device__ __forceinline__ void store(Elem* p, const float (&v)[W]) {
        Piece e;
#pragma unroll
        for (int i = 0; i < W; ++i) e[i] = Vec8<DT>::fromFloat(v[i]);
        Vec8<DT>::template put<STREAM>(reinterpret_cast<Piece*>(p), e);
    }
};
template <int W>
__device__ __forceinline__ void loadFloats(const float* p, float (&v)[W]) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
        const auto f = *reinterpret_cast<const Vec8<2>::Float4*>(p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i + e] = f[e];
    }
}

// A lane of a row holds two chunks of W values, whose pairs are its own: of the rotated part chunk u of either half or,
// interleaved, 2 W values in a row; of the rest 2 W values in a row. So a rotation never leaves the lane.
template <int W>
struct Place {
    int a, b;         // first columns
    bool in, turned;
    __device__ __forceinline__ Place(const QkNormParams& p, int unit) {
        in = unit * 2 * W < p.D;
        turned = unit * 2 * W < p.rotary;
        a = turned && !p.interleaved ? unit * W : unit * 2 * W;
        b = turned && !p.interleaved ? p.rotary / 2 + a : a + W;
    }
};

// (a, b) turned by the angles of a row of the table, or back (SIGN -1).
template <int W, int SIGN>
__device__ __forceinline__ void turn(const QkNormParams& p, long long at, float (&a)[W], float (&b)[W]) {
    float c[W], s[W];
    loadFloats<W>(p.cos + at, c);
    loadFloats<W>(p.sin + at, s);
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float& x = 2 * i < W ? a[2 * i] : b[2 * i - W];
            float& y = 2 * i < W ? a[2 * i + 1] : b[2 * i + 1 - W];
            const float u = x, v = y, t = SIGN * s[i];
            x = u * c[i] - v * t;
            y = v * c[i] + u * t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float u = a[i], v = b[i], t = SIGN * s[i];
            a[i] = u * c[i] - v * t;
            b[i] = v * c[i] + u * t;
        }
    }
}

// The sum over a row's lanes, in each of them.
__device__ __forceinline__ float sumOfRow(float v, int unitsLog2) {
    for (int s = (1 << unitsLog2) / 2; s > 0; s >>= 1) v += __shfl_xor(v, s, 64);
    return v;
}

// Rows of one side, as many at a time as a workgroup's lanes hold.
template <int DT, int W, bool BACKWARD>
__global__ __launch_bounds__(256) void qk_norm_kernel(QkNormParams p) {
    using C = Chunk<DT, W>;
    using Elem = typename C::Elem;
    const bool keys = blockIdx.x >= p.side[0].blocks;
    const QkSide& side = p.side[keys];
    const uint32_t block = keys ? blockIdx.x - p.side[0].blocks : blockIdx.x;
    const uint32_t unit = threadIdx.x & ((1u << p.unitsLog2) - 1), group = threadIdx.x >> p.unitsLog2;
    const uint32_t groups = 256u >> p.unitsLog2;
    const Place<W> at(p, (int)unit);
    float wa[W], wb[W];
#pragma unroll
    for (int i = 0; i < W; ++i) wa[i] = wb[i] = 1.f;
    if (side.weight && at.in) {
        loadFloats<W>(side.weight + at.a, wa);
        loadFloats<W>(side.weight + at.b, wb);
    }
    float da[W], db[W];   // the weight's gradient
#pragma unroll
    for (int i = 0; i < W; ++i) da[i] = db[i] = 0.f;

    // Every lane of a row stays to the sums; lanes past the head dimension hold zeros.
    forStores(p.streaming, [&](auto streamTag) {
        constexpr bool STREAM = decltype(streamTag)::value;
        for (uint32_t row = block * groups + group; row < side.rows; row += side.blocks * groups) {
            const uint32_t token = side.heads.div(row), head = row - token * side.heads.d;
            const uint32_t image = p.seq.div(token), t = token - image * p.seq.d;
            const long long column = (long long)head * p.D;
            const Elem* x = static_cast<const Elem*>(side.x) + image * side.strideX + t * side.ldX + column;
            Elem* out = static_cast<Elem*>(side.out) + image * side.strideOut + t * side.ldOut + column;
            const int position = !p.positions ? (int)t : p.positions[token];
            const bool turned = at.turned && (uint32_t)position < (uint32_t)p.table;
            const long long angles = (long long)position * (p.rotary / 2) + (int)unit * W;
            float a[W], b[W], ga[W], gb[W];
#pragma unroll
            for (int i = 0; i < W; ++i) a[i] = b[i] = ga[i] = gb[i] = 0.f;
            if (at.in) {
                C::load(x + at.a, a);
                C::load(x + at.b, b);
                if constexpr (BACKWARD) {
                    const Elem* g = static_cast<const Elem*>(side.g) + image * side.strideG + t * side.ldG + column;
                    C::load(g + at.a, ga);
                    C::load(g + at.b, gb);
                }
            }
            float squares = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) squares += a[i] * a[i] + b[i] * b[i];
            const float inv = rsqrtf(sumOfRow(squares, p.unitsLog2) / (float)p.D + p.eps);
            if constexpr (!BACKWARD) {
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a[i] = a[i] * inv * wa[i];
                    b[i] = b[i] * inv * wb[i];
                }
                if (turned) turn<W, 1>(p, angles, a, b);
            } else {
                if (turned) turn<W, -1>(p, angles, ga, gb);
                float dot = 0.f;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a[i] *= inv;   // xhat
                    b[i] *= inv;
                    da[i] += ga[i] * a[i];
                    db[i] += gb[i] * b[i];
                    ga[i] *= wa[i];
                    gb[i] *= wb[i];
                    dot += ga[i] * a[i] + gb[i] * b[i];
                }
                const float mean = sumOfRow(dot, p.unitsLog2) / (float)p.D;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a[i] = inv * (ga[i] - a[i] * mean);
                    b[i] = inv * (gb[i] - b[i] * mean);
                }
            }
            if (at.in) {
                C::template store<STREAM>(out + at.a, a);
                C::template store<STREAM>(out + at.b, b);
            }
        }
    });

    if constexpr (BACKWARD) {
        if (!side.gradWeight) return;
        // the groups' sums, added in order, a column a thread
        extern __shared__ float sums[];   // [groups, D]
        if (at.in) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
                sums[group * p.D + at.a + i] = da[i];
                sums[group * p.D + at.b + i] = db[i];
            }
        }
        __syncthreads();
        for (int c = (int)threadIdx.x; c < p.D; c += 256) {
            float s = 0.f;
            for (uint32_t k = 0; k < groups; ++k) s += sums[k * p.D + c];
            p.partials[(long long)blockIdx.x * p.D + c] = s;
        }
    }
}

// gradWeight of a side (blockIdx.y): the workgroups' sums of 32 columns, 32 runs of workgroups added in order.
__global__ __launch_bounds__(1024) void qk_norm_join_kernel(QkNormParams p) {
    __shared__ float part[32][32];
    const QkSide& side = p.side[blockIdx.y];
    if (!side.gradWeight) return;
    const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + lane;
    const uint32_t before = blockIdx.y ? p.side[0].blocks : 0u;
    const uint32_t first = (uint32_t)((uint64_t)side.blocks * run / 32), last = (uint32_t)((uint64_t)side.blocks * (run + 1) / 32);
    float s = 0.f;
    if (c < p.D) {
#pragma unroll 16
        for (uint32_t k = first; k < last; ++k) s += p.partials[(long long)(before + k) * p.D + c];
    }
    part[run][lane] = s;
    __syncthreads();
    if (run == 0 && c < p.D) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += part[k][lane];
        side.gradWeight[c] = s;
    }
}

template <int DT, int W>
int launch(const QkNormParams& p, bool backward) {
    const uint32_t blocks = p.side[0].blocks + p.side[1].blocks;
    if (blocks > 0) {
        if (backward)
            hipLaunchKernelGGL((qk_norm_kernel<DT, W, true>), dim3(blocks), dim3(256),
                               (size_t)(256 >> p.unitsLog2) * p.D * sizeof(float), stream(), p);
        else
            hipLaunchKernelGGL((qk_norm_kernel<DT, W, false>), dim3(blocks), dim3(256), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
    }
    if (backward && (p.side[0].gradWeight || p.side[1].gradWeight)) {
        hipLaunchKernelGGL(qk_norm_join_kernel, dim3((unsigned)((p.D + 31) / 32), 2), dim3(1024), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
    }
    return 0;
}

// Rows lie apart, image after image or token after token: what is written there does not overlap.
bool rowsApart(int nBatch, int nSeq, long long nLd, long long nStride, long long nWidth) {
    return nBatch <= 1 || nSeq == 0 || nStride >= (nSeq - 1) * nLd + nWidth ||
           (nStride >= nWidth && nLd >= (nBatch - 1) * nStride + nWidth);
}

struct QkArray {
    const void* p;
    long long ld, stride;
};

int run(const char* name, int nDtype, const QkArray (&x)[2], const QkArray (&g)[2], const QkArray (&out)[2],
        const float* const (&weight)[2], float* const (&gradWeight)[2], const float* pCos, const float* pSin,
        const int* pPositions, int nBatch, int nSeq, const int (&heads)[2], int nHeadDim, int nRotary, int nTable, float fEps,
        int bInterleaved, bool backward) {
    clearError();
    if (nDtype < 0 || nDtype > 2) return fail("%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", name);
    if (nBatch < 0 || nSeq < 0 || heads[0] < 0 || heads[1] < 0) return fail("%s: negative size", name);
    if (nHeadDim < 8 || nHeadDim > 256 || nHeadDim % 8 != 0)
        return fail("%s: head dimension %d (supported: multiples of 8 up to 256)", name, nHeadDim);
    if (nRotary < 0 || nRotary > nHeadDim || nRotary % 8 != 0)
        return fail("%s: %d rotated values (supported: multiples of 8 up to the head dimension)", name, nRotary);
    if (nTable < 0) return fail("%s: negative size", name);
    if (!(fEps >= 0.f) || !std::isfinite(fEps)) return fail("%s: eps must be finite and not negative", name);
    const auto aligned = [](const void* p, unsigned mask) { return (reinterpret_cast<uintptr_t>(p) & mask) == 0; };
    const long long tokens = (long long)nBatch * nSeq;
    const bool angles = nRotary > 0 && nTable > 0;
    if (tokens > 0 && angles && (!pCos || !pSin)) return fail("%s: null pointer", name);
    if (!aligned(pCos, 3) || !aligned(pSin, 3) || !aligned(pPositions, 3) || !aligned(weight[0], 3) || !aligned(weight[1], 3) ||
        !aligned(gradWeight[0], 3) || !aligned(gradWeight[1], 3))
        return fail("%s: a pointer is not aligned to its elements", name);
    for (int k = 0; k < 2; ++k) {
        if (heads[k] == 0) continue;
        const long long width = (long long)heads[k] * nHeadDim;
        if (tokens > 0x7fffffffLL || tokens * heads[k] > 0x7fffffffLL) return fail("%s: too many rows", name);
        for (const QkArray* a : {&x[k], &g[k], &out[k]}) {
            if (a == &g[k] && !backward) continue;
            if (tokens > 0 && !a->p) return fail("%s: null pointer", name);
            if (!aligned(a->p, 15)) return fail("%s: data must be 16-byte aligned", name);
            if (a->ld < width) return fail("%s: a row stride is below the heads' width", name);
            if (a->stride < 0) return fail("%s: negative stride", name);
            if ((a->ld | a->stride) & 7) return fail("%s: strides must be multiples of 8 elements", name);
            if (a->ld >= (1LL << 40) || a->stride >= (1LL << 60) / std::max(1, nBatch)) return fail("%s: a stride is too large", name);
        }
        if (!rowsApart(nBatch, nSeq, out[k].ld, out[k].stride, width)) return fail("%s: rows of the results would overlap", name);
        for (const QkArray* a : {&x[k], &g[k]})   // a row is written once it is read, so in place means row for row
            if (tokens > 0 && a->p == out[k].p && (a->ld != out[k].ld || a->stride != out[k].stride) && (a == &x[k] || backward))
                return fail("%s: results in place of an input with other strides", name);
    }
    const int w = nHeadDim % 16 == 0 && nRotary % 16 == 0 ? 8 : 4;
    QkNormParams p{};
    p.cos = pCos; p.sin = pSin;
    p.positions = pPositions;
    p.seq = FastDiv::make((uint32_t)std::max(1, nSeq));
    p.D = nHeadDim; p.rotary = nRotary; p.table = nTable; p.interleaved = bInterleaved != 0;
    p.eps = fEps;
    while ((2 * w << p.unitsLog2) < nHeadDim) ++p.unitsLog2;
    long long bytes = 0;
    for (int k = 0; k < 2; ++k) {
        QkSide& s = p.side[k];
        s.x = x[k].p; s.g = g[k].p; s.out = const_cast<void*>(out[k].p);
        s.ldX = x[k].ld; s.strideX = x[k].stride;
        s.ldG = g[k].ld; s.strideG = g[k].stride;
        s.ldOut = out[k].ld; s.strideOut = out[k].stride;
        s.weight = weight[k];
        s.gradWeight = gradWeight[k];
        s.heads = FastDiv::make((uint32_t)std::max(1, heads[k]));
        s.rows = (uint32_t)(heads[k] == 0 ? 0 : tokens * heads[k]);
        const uint32_t groups = 256u >> p.unitsLog2;
        s.blocks = std::min((s.rows + groups - 1) / groups, (uint32_t)(8 * cuCount()));
        bytes += (long long)s.rows * nHeadDim * (nDtype == 2 ? 4 : 2);
    }
    p.streaming = bytes >= kStreamBytes;
    if (backward && (gradWeight[0] || gradWeight[1]) && p.side[0].blocks + p.side[1].blocks > 0) {
        p.partials = static_cast<float*>(
            workspace((size_t)(p.side[0].blocks + p.side[1].blocks) * nHeadDim * sizeof(float), kWsPartials));
        if (!p.partials) return -1;   // workspace() recorded the cause
    }
    switch (nDtype * 2 + (w == 8)) {
        case 0: return launch<0, 4>(p, backward);
        case 1: return launch<0, 8>(p, backward);
        case 2: return launch<1, 4>(p, backward);
        case 3: return launch<1, 8>(p, backward);
        case 4: return launch<2, 4>(p, backward);
        default: return launch<2, 8>(p, backward);
    }
}

}  // namespace

}  // namespace omhip

using namespace omhip;

extern "C" {

int omHipQkNormRotary(int nDtype, const void* pQ, const void* pK, long long nLdQ, long long nStrideQ, long long nLdK,
                      long long nStrideK, const float* pWeightQ, const float* pWeightK, const float* pCos, const float* pSin,
                      const int* pPositions, void* pOutQ, void* pOutK, long long nLdOutQ, long long nStrideOutQ,
                      long long nLdOutK, long long nStrideOutK, int nBatch, int nSeq, int nHeads, int nKVHeads, int nHeadDim,
                      int nRotary, int nTable, float fEps, int bInterleaved) {
    return run("omHipQkNormRotary", nDtype, {{pQ, nLdQ, nStrideQ}, {pK, nLdK, nStrideK}}, {},
               {{pOutQ, nLdOutQ, nStrideOutQ}, {pOutK, nLdOutK, nStrideOutK}}, {pWeightQ, pWeightK}, {nullptr, nullptr}, pCos,
               pSin, pPositions, nBatch, nSeq, {nHeads, nKVHeads}, nHeadDim, nRotary, nTable, fEps, bInterleaved, false);
}

int omHipQkNormRotaryBackward(int nDtype, const void* pGradOutQ, const void* pGradOutK, long long nLdGradQ,
                              long long nStrideGradQ, long long nLdGradK, long long nStrideGradK, const void* pQ, const void* pK,
                              long long nLdQ, long long nStrideQ, long long nLdK, long long nStrideK, const float* pWeightQ,
                              const float* pWeightK, const float* pCos, const float* pSin, const int* pPositions, void* pGradQ,
                              void* pGradK, float* pGradWeightQ, float* pGradWeightK, int nBatch, int nSeq, int nHeads,
                              int nKVHeads, int nHeadDim, int nRotary, int nTable, float fEps, int bInterleaved) {
    return run("omHipQkNormRotaryBackward", nDtype, {{pQ, nLdQ, nStrideQ}, {pK, nLdK, nStrideK}},
               {{pGradOutQ, nLdGradQ, nStrideGradQ}, {pGradOutK, nLdGradK, nStrideGradK}},
               {{pGradQ, nLdQ, nStrideQ}, {pGradK, nLdK, nStrideK}}, {pWeightQ, pWeightK}, {pGradWeightQ, pGradWeightK}, pCos,
               pSin, pPositions, nBatch, nSeq, {nHeads, nKVHeads}, nHeadDim, nRotary, nTable, fEps, bInterleaved, true);
}

}  // extern "C"
