// dropout.hip — dropout whose mask comes from a counter-based generator and is
// never stored: the backward pass draws the same bits again.
//
// The reference's dropout keeps a float mask as large as its input
// (omCudaDropout, cuda_kernels.cu:2266-2337). Here the bits of a value are a
// function of (seed, step, stream, row, column):
//   Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw, "Parallel
//   random numbers: as easy as 1, 2, 3", SC11) with key (seed low, seed high)
//   and counter (group, stream, step low, step high); group = row *
//   ceil(nCols / 8) + column / 8. Its 128 bits are 16 for each of the group's
//   8 columns: column j takes half j % 2 (low first) of word j / 2.
// A value is kept where its 16 bits are at least T = round(65536 p) and scaled
// by 65536 / (65536 - T), the inverse of the probability that the bits really
// have: 16 bits move p by at most 2^-17 and keep the mean exact, and cost a
// half of the generator's work per value that 32 would.
#include "fastdiv.hpp"
#include "omhip_internal.hpp"
#include "vec_io.hpp"
#include "../../include/omhip.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace omhip {

namespace {

struct DropoutParams {
    const void* x;           // forward: input; backward: the output's gradient
    const float* bias;       // [nCols] or null
    const void* residual;    // or null
    void* out;
    float* partials;         // backward with a bias gradient: [chunks, nCols]
    const uint64_t* rng;     // device: seed, step
    uint32_t stream, threshold;
    float scale;
    int rows, cols;
    FastDiv perRow;          // groups of 8 columns in a row
    uint32_t groups;
    int rowsPerChunk;
    bool streaming;          // streaming stores
};

// Ten rounds of Philox4x32 on counter c with key k.
struct Bits {
    uint32_t w[4];
    __device__ __forceinline__ bool keep(int j, uint32_t threshold) const {
        return ((j & 1) ? w[j >> 1] >> 16 : w[j >> 1] & 0xffffu) >= threshold;
    }
};
__device__ __forceinline__ Bits philox(uint32_t group, uint32_t stream, uint64_t seed, uint64_t step) {
    uint32_t c0 = group, c1 = stream, c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(b >> 32) ^ c1 ^ k0, n2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        c0 = n0;
        c2 = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// One group of 8 columns a thread: out = keep ? (x + bias) scale : 0, + residual. The backward pass is the same
// without bias and residual.
template <int DT, bool EVEN>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutParams p) {
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= p.groups) return;
    const uint32_t r = p.perRow.div(g), c = (g - r * p.perRow.d) * 8u;
    const int n = min(8, p.cols - (int)c);
    const long long at = (long long)r * p.cols + c;
    float x[8], res[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    Vec8<DT>::template load<EVEN>(p.x, at, n, x);
    if (p.residual) Vec8<DT>::template load<EVEN>(p.residual, at, n, res);
    if (p.bias) {
        float b[8];
        Vec8<2>::load<EVEN>(p.bias, c, n, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += b[i];
    }
    const Bits bits = philox(g, p.stream, p.rng[0], p.rng[1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bits.keep(i, p.threshold) ? __builtin_fmaf(x[i], p.scale, res[i]) : res[i];
    forStores(p.streaming, [&](auto streamTag) {
        Vec8<DT>::template store<EVEN, decltype(streamTag)::value>(p.out, at, n, x);
    });
}

// Backward with the bias gradient: a workgroup takes TC groups of columns and a chunk of rows, 256 / TC rows at a
// time, and adds each column's kept gradients (unrounded) in row order; the threads of a column group are added in
// order at the end and leave one row of partial sums a chunk.
template <int DT, int TC, bool EVEN>
__global__ __launch_bounds__(256) void dropout_bias_kernel(DropoutParams p) {
    constexpr int TR = 256 / TC;
    __shared__ float part[TR][TC * 8 + 1];
    const int tc = threadIdx.x % TC, tr = threadIdx.x / TC;
    const uint32_t cg = blockIdx.x * TC + tc;
    const int c = (int)cg * 8, n = min(8, p.cols - c);
    const uint64_t seed = p.rng[0], step = p.rng[1];
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const long long first = (long long)blockIdx.y * p.rowsPerChunk;
    const int last = (int)min((long long)p.rows, first + p.rowsPerChunk);
    if (n > 0) {
        // four rows at a time, so that as many loads are under way
        auto rows = [&](auto rowsTag, auto streamTag, int r) {
            constexpr int ROWS = decltype(rowsTag)::value;
            float x[ROWS][8];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) Vec8<DT>::template load<EVEN>(p.x, (long long)(r + k * TR) * p.cols + c, n, x[k]);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                const Bits bits = philox((uint32_t)(r + k * TR) * p.perRow.d + cg, p.stream, seed, step);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[k][i] = bits.keep(i, p.threshold) ? x[k][i] * p.scale : 0.f;
                    sum[i] += x[k][i];
                }
                Vec8<DT>::template store<EVEN, decltype(streamTag)::value>(p.out, (long long)(r + k * TR) * p.cols + c, n,
                                                                           x[k]);
            }
        };
        forStores(p.streaming, [&](auto stream) {
            int r = (int)first + tr;
            for (; r < last - 3 * TR; r += 4 * TR) rows(std::integral_constant<int, 4>{}, stream, r);
            for (; r < last; r += TR) rows(std::integral_constant<int, 1>{}, stream, r);
        });
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[tr][tc * 8 + i] = sum[i];
    __syncthreads();
    for (int j = threadIdx.x; j < TC * 8; j += 256) {
        const int col = (int)blockIdx.x * TC * 8 + j;
        if (col >= p.cols) break;
        float s = 0.f;
        for (int i = 0; i < TR; ++i) s += part[i][j];
        p.partials[(long long)blockIdx.y * p.cols + col] = s;
    }
}

// gradBias[c] = the chunks' partial sums: 32 interleaved runs of them a column, then those pairwise. (8 runs took 20 us
// for 512 chunks of 1024 columns: loads waited out one by one.) Workgroups count through both dimensions of the grid: 2^22
// of them, 2^27 columns, are 2^32 threads, and a grid keeps 32 bits of its threads in a dimension.
__global__ __launch_bounds__(1024) void dropout_bias_sum_kernel(const float* partials, float* gradBias, int chunks, uint32_t cols) {
    __shared__ float part[32][33];
    const int tc = threadIdx.x & 31, tr = threadIdx.x >> 5;
    const uint32_t c = (blockIdx.y * gridDim.x + blockIdx.x) * 32u + tc;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int i = tr; i < chunks; i += 32) s += partials[(long long)i * cols + c];
    }
    part[tr][tc] = s;
#pragma unroll
    for (int half = 16; half > 0; half /= 2) {
        __syncthreads();
        if (tr < half) part[tr][tc] += part[tr + half][tc];
    }
    if (tr == 0 && c < cols) gradBias[c] = part[0][tc];
}

template <int DT>
int launchDropout(const DropoutParams& p) {
    const dim3 grid((p.groups + 255u) / 256u);
    if (p.cols % 8 == 0)
        hipLaunchKernelGGL((dropout_kernel<DT, true>), grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL((dropout_kernel<DT, false>), grid, dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <int DT, int TC>
int launchDropoutBias(const DropoutParams& p, int chunks) {
    const dim3 grid((p.perRow.d + TC - 1) / TC, chunks);
    if (p.cols % 8 == 0)
        hipLaunchKernelGGL((dropout_bias_kernel<DT, TC, true>), grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL((dropout_bias_kernel<DT, TC, false>), grid, dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <int DT>
int backwardWithBias(DropoutParams& p, float* pGradBias) {
    // column groups a workgroup takes: 32 (512 bytes of a row of halves), less where the row has less
    const uint32_t d = p.perRow.d;
    const int tc = d > 16 ? 32 : d > 4 ? 16 : 4, tiles = (int)((d + tc - 1) / tc);
    // chunks of rows: eight workgroups a CU, and eight rows a thread at least
    const int rowsAtOnce = 256 / tc;
    const int most = (p.rows + 8 * rowsAtOnce - 1) / (8 * rowsAtOnce);
    int chunks = std::clamp(8 * cuCount() / tiles, 1, std::min(most, 65535));
    p.rowsPerChunk = (p.rows + chunks - 1) / chunks;
    chunks = (p.rows + p.rowsPerChunk - 1) / p.rowsPerChunk;
    p.partials = static_cast<float*>(workspace((size_t)chunks * p.cols * sizeof(float), kWsPartials));
    if (!p.partials) return -1;   // workspace() recorded the cause
    const int rc = tc == 32 ? launchDropoutBias<DT, 32>(p, chunks)
                 : tc == 16 ? launchDropoutBias<DT, 16>(p, chunks)
                            : launchDropoutBias<DT, 4>(p, chunks);
    if (rc) return rc;
    const uint32_t blocks = ((uint32_t)p.cols + 31u) / 32u, width = std::min(blocks, 1u << 16);
    hipLaunchKernelGGL(dropout_bias_sum_kernel, dim3(width, (blocks + width - 1) / width), dim3(1024), 0, stream(), p.partials,
                       pGradBias, chunks, (uint32_t)p.cols);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

// Checks and parameters that both directions share; 0, 1 (nothing to do) or -1.
int dropoutParams(const char* name, int nDtype, int nRows, int nCols, float fProb, const void* pRng, int nStream,
                  DropoutParams& p) {
    if (nDtype < 0 || nDtype > 2) return fail("%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", name);
    if (nRows < 0 || nCols < 0) return fail("%s: negative size", name);
    if (!(fProb >= 0.f && fProb <= 1.f)) return fail("%s: probability %g is not within 0 .. 1", name, (double)fProb);
    if (nRows == 0 || nCols == 0) return 1;
    const long long groups = (long long)nRows * ((nCols + 7LL) / 8);
    // row counters run up to four rows a thread past the last one
    if (groups > 0x7fff0000LL) return fail("%s: %d rows of %d columns exceed 2^31 - 2^16 groups of 8", name, nRows, nCols);
    if (!pRng || (reinterpret_cast<uintptr_t>(pRng) & 7u)) return fail("%s: the generator's state must be 8-byte aligned", name);
    p.rng = static_cast<const uint64_t*>(pRng);
    p.stream = (uint32_t)nStream;
    p.threshold = (uint32_t)std::floor((double)fProb * 65536.0 + 0.5);
    p.scale = p.threshold < 65536u ? (float)(65536.0 / (65536.0 - p.threshold)) : 0.f;
    p.rows = nRows;
    p.cols = nCols;
    p.perRow = FastDiv::make((uint32_t)((nCols + 7LL) / 8));
    p.groups = (uint32_t)groups;
    p.streaming = (long long)nRows * nCols * (nDtype == 2 ? 4 : 2) >= kStreamBytes;
    return 0;
}

bool elementAligned(const void* p, int nDtype) { return (reinterpret_cast<uintptr_t>(p) & (nDtype == 2 ? 3u : 1u)) == 0; }

}  // namespace

}  // namespace omhip

using namespace omhip;

extern "C" {

int omHipDropout(int nDtype, const void* pX, const float* pBias, const void* pResidual, void* pOut, int nRows, int nCols,
                 float fProb, const uint64_t* pRng, int nStream) {
    const char* name = "omHipDropout";
    clearError();
    DropoutParams p{};
    const int rc = dropoutParams(name, nDtype, nRows, nCols, fProb, pRng, nStream, p);
    if (rc) return rc < 0 ? -1 : 0;
    if (!pX || !pOut) return fail("%s: null pointer", name);
    if (!elementAligned(pX, nDtype) || !elementAligned(pOut, nDtype) || !elementAligned(pResidual, nDtype) ||
        !elementAligned(pBias, 2))
        return fail("%s: a pointer is not aligned to its elements", name);
    p.x = pX; p.bias = pBias; p.residual = pResidual; p.out = pOut;
    return nDtype == 0 ? launchDropout<0>(p) : nDtype == 1 ? launchDropout<1>(p) : launchDropout<2>(p);
}

int omHipDropoutBackward(int nDtype, const void* pGradOut, void* pGradX, float* pGradBias, int nRows, int nCols, float fProb,
                         const uint64_t* pRng, int nStream) {
    const char* name = "omHipDropoutBackward";
    clearError();
    DropoutParams p{};
    const int rc = dropoutParams(name, nDtype, nRows, nCols, fProb, pRng, nStream, p);
    if (rc < 0) return -1;
    if (rc) return pGradBias && nCols > 0 ? byteFill(pGradBias, 0, (size_t)nCols * sizeof(float)) : 0;   // no rows
    if (!pGradOut || !pGradX) return fail("%s: null pointer", name);
    if (!elementAligned(pGradOut, nDtype) || !elementAligned(pGradX, nDtype) || !elementAligned(pGradBias, 2))
        return fail("%s: a pointer is not aligned to its elements", name);
    p.x = pGradOut; p.out = pGradX;
    if (pGradBias)
        return nDtype == 0 ? backwardWithBias<0>(p, pGradBias)
             : nDtype == 1 ? backwardWithBias<1>(p, pGradBias)
                           : backwardWithBias<2>(p, pGradBias);
    return nDtype == 0 ? launchDropout<0>(p) : nDtype == 1 ? launchDropout<1>(p) : launchDropout<2>(p);
}

}  // extern "C"
