// group_norm.hip — group normalisation with an activation on channels-last
// data [image, pixel, channel] (the layout of transformer tokens), forward and
// backward.
//
// The reference normalises groups of an NCHW tensor and runs the activation as
// its own pass (omCudaGroupNorm, cuda_kernels.cu:3205-3490). Over the pixels
// and the C / G channels of group g of image n:
//   xhat = (x - mean) inv, inv = 1 / sqrt(var + eps); z = xhat gamma + beta; y = act(z)
//   backward, dz = dy act'(z): dbeta = sum dz, dgamma = sum dz xhat over images and pixels,
//   dx = inv (gamma dz - mean_g(gamma dz) - xhat mean_g(gamma dz xhat))
//
// Both directions are bound by memory: one pass that leaves per-channel sums of
// a chunk of an image's pixels, one small launch that joins them, one pass that
// writes the result. A thread holds 8 neighbouring channels of a row (16 bytes
// of halves), so every access is a stretch of whole rows.
//
// Variance: a thread adds x - k and (x - k)^2 with k its own first value of the
// channel, turns them into (count, mean, sum of squared differences from the
// mean), and those are joined pairwise, M = Ma + Mb + (mb - ma)^2 na nb / n
// (T. F. Chan, G. H. Golub, R. J. LeVeque, "Updating formulae and a pairwise
// algorithm for computing sample variances", 1979): a mean far above the
// spread costs no digits. The order is fixed; nothing is added atomically.
#include "fastdiv.hpp"
#include "omhip_internal.hpp"
#include "vec_io.hpp"
#include "../../include/omhip.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace omhip {

namespace {

struct GroupNormParams {
    const void *x, *y, *gradY;
    void* out;                      // y or dx
    const float *gamma, *beta;      // null: 1, 0
    float *mean, *inv;              // [N, G]
    float2* partial;                // [N, chunks, C]: forward (mean, M), backward (sum dz, sum dz xhat)
    float2* means;                  // backward, [N, G]: the group means of gamma dz and gamma dz xhat
    float *gradGamma, *gradBeta;    // or null
    int N, P, C, G, per;            // per: channels of a group
    FastDiv byPer;
    int chunks, rowsPerChunk;
    bool stream;                    // streaming stores
    int width;                      // channels of a workgroup: 8 TC, or as many whole groups as those hold (small)
    int small;                      // an image's rows and whole groups in a workgroup
    float eps;
};

enum { kActNone = 0, kActRelu = 1, kActSilu = 2 };

// (count, mean, sum of squared differences) of a and b together. An empty a (count and mean 0) makes d the whole of b's
// mean, whose square may pass fp32's range: the count is multiplied in first.
struct Moments {
    float n, mean, m2;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (b.n == 0.f) return a;
    const float d = b.mean - a.mean, f = b.n / n;
    return {n, __builtin_fmaf(d, f, a.mean), a.m2 + b.m2 + d * (a.n * f) * d};
}

// Rows of a chunk.
__device__ __forceinline__ int chunkRows(const GroupNormParams& p, int chunk) {
    return min(p.P - chunk * p.rowsPerChunk, p.rowsPerChunk);
}

// Where a thread of a pass works: 8 channels from c on (n of them exist), rows tr, tr + TR, ... of its chunk.
template <int TC>
struct Place {
    static constexpr int TR = 256 / TC;
    int c, n, tr, first, rows, image, chunk;
    long long base;   // element of the image's first row
    __device__ __forceinline__ explicit Place(const GroupNormParams& p) {
        c = (int)blockIdx.x * p.width + (int)threadIdx.x % TC * 8;
        n = min(8, min(p.C, ((int)blockIdx.x + 1) * p.width) - c);
        tr = threadIdx.x / TC;
        chunk = blockIdx.y;
        image = blockIdx.z;
        first = chunk * p.rowsPerChunk;
        rows = chunkRows(p, chunk);
        base = (long long)image * p.P * p.C;
    }
    __device__ __forceinline__ long long at(const GroupNormParams& p, int r) const {
        return base + (long long)(first + r) * p.C + c;
    }
};

// Calls f(rows, r) for the thread's rows r, r + TR, ..., four at a time, so that as many loads are under way, then the
// rest one by one. (The loads of a row after a store could not be moved before it: the output may be the input.)
template <class W, class F>
__device__ __forceinline__ void forRows(const W& w, F&& f) {
    int r = w.tr;
    for (; r + 3 * W::TR < w.rows; r += 4 * W::TR) f(std::integral_constant<int, 4>{}, r);
    for (; r < w.rows; r += W::TR) f(std::integral_constant<int, 1>{}, r);
}

// What a thread needs of its channels.
template <bool EVEN>
struct Channels {
    float mean[8], inv[8], gamma[8], beta[8];
    // m, v: means and inverse deviations of the image's groups from `first` on
    __device__ __forceinline__ void load(const GroupNormParams& p, int c, int n, const float* m, const float* v, int first = 0) {
        // the first and the last channel's group
        const int g0 = (int)p.byPer.div((uint32_t)c) - first, g1 = (int)p.byPer.div((uint32_t)(c + n - 1)) - first;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            gamma[i] = 1.f;
            beta[i] = 0.f;
        }
        if (p.gamma) Vec8<2>::load<EVEN>(p.gamma, c, n, gamma);
        if (p.beta) Vec8<2>::load<EVEN>(p.beta, c, n, beta);
        if (g0 == g1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                mean[i] = m[g0];
                inv[i] = v[g0];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int g = i < n ? (int)p.byPer.div((uint32_t)(c + i)) - first : g0;
                mean[i] = m[g];
                inv[i] = v[g];
            }
        }
    }
};

// The hardware's exponential and reciprocal: off by about (|z| + 4) 2^-24 of itself (the exponent's rounding); 0 may stand for
// it below z = -87, where it is less than 2^-125.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == kActRelu) return z > 0.f ? z : 0.f;
    if constexpr (ACT == kActSilu) return z * sigmoid(z);
    return z;
}

// dz of dy. ReLU's gate is the saved output, so no rounding of z decides it.
template <int ACT>
__device__ __forceinline__ float gradient(float dy, float z, float y) {
    if constexpr (ACT == kActRelu) return y > 0.f ? dy : 0.f;
    if constexpr (ACT == kActSilu) {
        const float s = sigmoid(z);
        return dy * s * __builtin_fmaf(z, 1.f - s, 1.f);
    }
    return dy;
}

// ---------------------------------------------------------------- forward
// (mean, sum of squared differences) of the workgroup's channels over its chunk of rows: part[i][tc] for channel i of
// column group tc (its first TC entries, once the workgroup has met).
template <int DT, int TC, bool EVEN>
__device__ __forceinline__ void chunkMoments(const GroupNormParams& p, const Place<TC>& w, float2 (&part)[8][256]) {
    using W = Place<TC>;
    float shift[8], s[8], q[8];
    float count = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) shift[i] = s[i] = q[i] = 0.f;
    if (w.n > 0) {
        if (w.tr < w.rows) Vec8<DT>::template load<EVEN>(p.x, w.at(p, w.tr), w.n, shift);
        forRows<W>(w, [&](auto rowsTag, int r) {
            constexpr int ROWS = decltype(rowsTag)::value;
            float x[ROWS][8];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) Vec8<DT>::template load<EVEN>(p.x, w.at(p, r + k * W::TR), w.n, x[k]);
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = x[k][i] - shift[i];
                    s[i] += d;
                    q[i] = __builtin_fmaf(d, d, q[i]);
                }
            count += (float)ROWS;
        });
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float m = count > 0.f ? s[i] / count : 0.f;
        const float m2 = __builtin_fmaf(-m, s[i], q[i]);
        part[i][threadIdx.x] = {shift[i] + m, m2 < 0.f ? 0.f : m2};   // NaN, of infinite data, stays
    }
    // row threads tr and tr + half together, half = TR / 2 .. 1; thread tr then stands for rows tr, tr + half, ...
#pragma unroll
    for (int half = W::TR / 2; half > 0; half /= 2) {
        __syncthreads();
        if (w.tr < half) {
            auto rowsOf = [&](int tr) { return (float)(tr < w.rows ? (w.rows - tr + 2 * half - 1) / (2 * half) : 0); };
            const float na = rowsOf(w.tr), nb = rowsOf(w.tr + half);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 a = part[i][threadIdx.x], b = part[i][threadIdx.x + half * TC];
                const Moments j = join({na, a.x, a.y}, {nb, b.x, b.y});
                part[i][threadIdx.x] = {j.mean, j.m2};
            }
        }
    }
}

template <int TC>
__device__ __forceinline__ void leavePart(const GroupNormParams& p, const Place<TC>& w, const float2 (&part)[8][256]) {
    if (w.tr == 0 && w.n > 0) {
        float2* to = p.partial + ((long long)w.image * p.chunks + w.chunk) * p.C + w.c;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < w.n) to[i] = part[i][threadIdx.x];
    }
}

template <int DT, int TC, bool EVEN>
__global__ __launch_bounds__(256) void group_norm_moments_kernel(GroupNormParams p) {
    __shared__ float2 part[8][256];
    const Place<TC> w(p);
    chunkMoments<DT, TC, EVEN>(p, w, part);
    leavePart(p, w, part);
}

// (mean, inv) of an (image, group). Its entries are shared by as many waves as leave a lane eight of them, 16 at most, and
// a lane loads eight before it joins them: all but the last chunk have the same count of rows, which makes the joins' factors
// constants, so that no join waits for a division. (A wave a group, entry after entry, took longer than everything else where
// groups are few and wide: 12000 pixels x 2048 channels in one group, forward, bf16: 1235 us, now 73; 16384 x 256 in one: 593,
// now 35.5; the sums of 32 groups of 8 channels in 16 chunks take the same time either way.)
__global__ __launch_bounds__(1024) void group_norm_join_kernel(GroupNormParams p) {
    __shared__ Moments part[16];
    const int g = blockIdx.x, image = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const float2* from = p.partial + (long long)image * p.chunks * p.C + (long long)g * p.per;
    const uint32_t n = (uint32_t)p.chunks * (uint32_t)p.per, threads = blockDim.x;
    Moments t{0.f, 0.f, 0.f};
    for (uint32_t first = threadIdx.x; first < n; first += 8u * threads) {
        const int m = (int)min(8u, (n - first + threads - 1u) / threads);   // entries first, first + threads, ...
        float2 v[8];
        uint32_t chunk[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t e = i < m ? first + (uint32_t)i * threads : first;
            chunk[i] = p.byPer.div(e);
            v[i] = from[(long long)chunk[i] * p.C + (e - chunk[i] * (uint32_t)p.per)];
        }
        const float rows = (float)chunkRows(p, (int)chunk[0]);
        if (chunk[0] + 1u < (uint32_t)p.chunks && p.byPer.div(first + (uint32_t)(m - 1) * threads) + 1u == (uint32_t)p.chunks) {
#pragma unroll
            for (int i = 0; i < 8; ++i)   // the last chunk is among them
                if (i < m) t = join(t, {(float)chunkRows(p, (int)chunk[i]), v[i].x, v[i].y});
        } else {
            Moments u{rows * (float)m, v[0].x, v[0].y};
#pragma unroll
            for (int i = 1; i < 8; ++i)
                if (i < m) {
                    const float d = v[i].x - u.mean;
                    u.mean = __builtin_fmaf(d, 1.f / (float)(i + 1), u.mean);
                    u.m2 += v[i].y + d * (rows * ((float)i / (float)(i + 1))) * d;
                }
            t = join(t, u);
        }
    }
    auto joinLanes = [&] {
#pragma unroll
        for (int s = 32; s > 0; s >>= 1)
            t = join(t, {__shfl_down(t.n, s, 64), __shfl_down(t.mean, s, 64), __shfl_down(t.m2, s, 64)});
    };
    joinLanes();
    if (waves > 1) {
        if (lane == 0) part[wave] = t;
        __syncthreads();
        if (wave > 0) return;
        t = lane < waves ? part[lane] : Moments{0.f, 0.f, 0.f};
        joinLanes();
    }
    if (threadIdx.x == 0) {
        p.mean[(long long)image * p.G + g] = t.mean;
        p.inv[(long long)image * p.G + g] = 1.f / sqrtf(t.m2 / t.n + p.eps);
    }
}

// Waves that share a group's entries, `each` entries a lane.
int joinWaves(const GroupNormParams& p, int each) {
    return (int)std::clamp<long long>((long long)p.chunks * p.per / (64 * each), 1, 16);
}

// y of the workgroup's rows
template <int DT, int TC, int ACT, bool EVEN>
__device__ __forceinline__ void applyRows(const GroupNormParams& p, const Place<TC>& w, Channels<EVEN>& ch) {
    using W = Place<TC>;
#pragma unroll
    for (int i = 0; i < 8; ++i) ch.inv[i] *= ch.gamma[i];
    forStores(p.stream, [&](auto streamTag) {
        forRows<W>(w, [&](auto rowsTag, int r) {
            constexpr int ROWS = decltype(rowsTag)::value;
            float x[ROWS][8];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) Vec8<DT>::template load<EVEN>(p.x, w.at(p, r + k * W::TR), w.n, x[k]);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[k][i] = activate<ACT>(__builtin_fmaf(x[k][i] - ch.mean[i], ch.inv[i], ch.beta[i]));
                Vec8<DT>::template store<EVEN, decltype(streamTag)::value>(p.out, w.at(p, r + k * W::TR), w.n, x[k]);
            }
        });
    });
}

template <int DT, int TC, int ACT, bool EVEN>
__global__ __launch_bounds__(256) void group_norm_apply_kernel(GroupNormParams p) {
    const Place<TC> w(p);
    if (w.n <= 0) return;
    Channels<EVEN> ch;
    ch.load(p, w.c, w.n, p.mean + (long long)w.image * p.G, p.inv + (long long)w.image * p.G);
    applyRows<DT, TC, ACT, EVEN>(p, w, ch);
}

// An image of few pixels in one launch: a workgroup has all rows of its channels, and its channels are whole groups.
// Per-group values by the group's number within the workgroup; p.mean and p.inv receive them too.
template <int DT, int TC, int ACT, bool EVEN>
__global__ __launch_bounds__(256) void group_norm_small_kernel(GroupNormParams p) {
    __shared__ float2 part[8][256];
    __shared__ float mean[TC * 8], inv[TC * 8];
    const Place<TC> w(p);
    chunkMoments<DT, TC, EVEN>(p, w, part);
    __syncthreads();
    const int c0 = (int)blockIdx.x * p.width, g0 = c0 / p.per, groups = min(p.C - c0, p.width) / p.per;
    const int lane = threadIdx.x & 63;
    for (int g = (int)threadIdx.x >> 6; g < groups; g += 4) {   // a wave a group
        Moments t{0.f, 0.f, 0.f};
        for (int k = lane; k < p.per; k += 64) {
            const int c = g * p.per + k;
            const float2 v = part[c & 7][c >> 3];
            t = join(t, {(float)p.P, v.x, v.y});
        }
#pragma unroll
        for (int s = 32; s > 0; s >>= 1)
            t = join(t, {__shfl_down(t.n, s, 64), __shfl_down(t.mean, s, 64), __shfl_down(t.m2, s, 64)});
        if (lane == 0) {
            const float v = 1.f / sqrtf(t.m2 / t.n + p.eps);
            mean[g] = p.mean[(long long)w.image * p.G + g0 + g] = t.mean;
            inv[g] = p.inv[(long long)w.image * p.G + g0 + g] = v;
        }
    }
    __syncthreads();
    if (w.n <= 0) return;
    Channels<EVEN> ch;
    ch.load(p, w.c, w.n, mean, inv, g0);
    applyRows<DT, TC, ACT, EVEN>(p, w, ch);
}

// ---------------------------------------------------------------- backward
// xhat and dz of 8 channels of a row
template <int DT, int ACT, bool EVEN>
struct Row {
    float xhat[8], dz[8], y[ACT == kActRelu ? 8 : 1];
    __device__ __forceinline__ void load(const GroupNormParams& p, long long at, int n) {
        Vec8<DT>::template load<EVEN>(p.x, at, n, xhat);
        Vec8<DT>::template load<EVEN>(p.gradY, at, n, dz);
        if constexpr (ACT == kActRelu) Vec8<DT>::template load<EVEN>(p.y, at, n, y);
    }
    __device__ __forceinline__ void work(const Channels<EVEN>& ch) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xhat[i] = (xhat[i] - ch.mean[i]) * ch.inv[i];
            dz[i] = gradient<ACT>(dz[i], __builtin_fmaf(xhat[i], ch.gamma[i], ch.beta[i]), y[ACT == kActRelu ? i : 0]);
        }
    }
};

// (sum of dz, sum of dz xhat) of the workgroup's channels over its chunk of rows, as chunkMoments leaves its values
template <int DT, int TC, int ACT, bool EVEN>
__device__ __forceinline__ void chunkSums(const GroupNormParams& p, const Place<TC>& w, float2 (&part)[8][256]) {
    using W = Place<TC>;
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
    if (w.n > 0) {
        Channels<EVEN> ch;
        ch.load(p, w.c, w.n, p.mean + (long long)w.image * p.G, p.inv + (long long)w.image * p.G);
        forRows<W>(w, [&](auto rowsTag, int r) {
            constexpr int ROWS = decltype(rowsTag)::value;
            Row<DT, ACT, EVEN> row[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) row[k].load(p, w.at(p, r + k * W::TR), w.n);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                row[k].work(ch);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[i] += row[k].dz[i];
                    b[i] = __builtin_fmaf(row[k].dz[i], row[k].xhat[i], b[i]);
                }
            }
        });
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i][threadIdx.x] = {a[i], b[i]};
#pragma unroll
    for (int half = W::TR / 2; half > 0; half /= 2) {
        __syncthreads();
        if (w.tr < half)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 u = part[i][threadIdx.x], v = part[i][threadIdx.x + half * TC];
                part[i][threadIdx.x] = {u.x + v.x, u.y + v.y};
            }
    }
}

template <int DT, int TC, int ACT, bool EVEN>
__global__ __launch_bounds__(256) void group_norm_sums_kernel(GroupNormParams p) {
    __shared__ float2 part[8][256];
    const Place<TC> w(p);
    chunkSums<DT, TC, ACT, EVEN>(p, w, part);
    leavePart(p, w, part);
}

// The first workgroups: the means of gamma dz and gamma dz xhat of 16 >> share groups, 1 << share waves each (12000 x 2048 in
// one group, bf16: 472 us with a wave a group, now 146; SHARED: share is not 0, a choice at run time alone cost 8 x 1024 x 320
// in 32 groups 1 us of 17.4). The others: dgamma and dbeta of 32 channels, 32 interleaved runs over images and chunks a channel
// (with 8 runs, the loads' latency took 58 us at 32 x 28 x 28 x 512). Workgroups count through both dimensions of the grid: 2^26
// groups are 2^32 threads, and a grid keeps 32 bits of its threads in a dimension. What lies past the last channel finds
// nothing to do.
template <bool SHARED>
__global__ __launch_bounds__(1024) void group_norm_join_backward_kernel(GroupNormParams p, uint32_t groupBlocks, uint32_t shareBits) {
    __shared__ float2 part[1024];
    const uint32_t share = SHARED ? shareBits : 0u;
    const int t = threadIdx.x;
    float2 s{0.f, 0.f};
    const uint32_t groups = (uint32_t)(p.N * p.G), block = blockIdx.y * gridDim.x + blockIdx.x;
    if (block < groupBlocks) {
        const uint32_t wave = (uint32_t)t >> 6, id = (block * 16u + wave) >> share, threads = 64u << share;
        if (id < groups) {
            const uint32_t image = id / (uint32_t)p.G, g = id - image * (uint32_t)p.G;
            const float2* from = p.partial + (long long)image * p.chunks * p.C + (long long)g * p.per;
            const uint32_t n = (uint32_t)p.chunks * (uint32_t)p.per;
#pragma unroll 4
            for (uint32_t e = (uint32_t)t & (threads - 1u); e < n; e += threads) {
                const uint32_t chunk = p.byPer.div(e), k = e - chunk * (uint32_t)p.per;
                const float2 v = from[(long long)chunk * p.C + k];
                const float gamma = p.gamma ? p.gamma[g * p.per + k] : 1.f;
                s.x = __builtin_fmaf(gamma, v.x, s.x);
                s.y = __builtin_fmaf(gamma, v.y, s.y);
            }
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) {
            s.x += __shfl_down(s.x, d, 64);
            s.y += __shfl_down(s.y, d, 64);
        }
        if constexpr (SHARED) {
            if ((t & 63) == 0) part[wave] = s;
            __syncthreads();
            for (uint32_t i = 1; i < 1u << share && wave + i < 16u; ++i) {   // all of them for a group's first wave, which leaves the sum
                s.x += part[wave + i].x;
                s.y += part[wave + i].y;
            }
        }
        const float f = 1.f / ((float)p.P * (float)p.per);
        if (((uint32_t)t & (threads - 1u)) == 0 && id < groups) p.means[id] = {s.x * f, s.y * f};
        return;
    }
    const int c = (int)(block - groupBlocks) * 32 + (t & 31);
    if (c < p.C) {
#pragma unroll 8
        for (long long e = t >> 5; e < (long long)p.N * p.chunks; e += 32) {
            const float2 v = p.partial[e * p.C + c];
            s.x += v.x;
            s.y += v.y;
        }
    }
    part[t] = s;
#pragma unroll
    for (int half = 512; half >= 32; half /= 2) {   // down to a sum a channel
        __syncthreads();
        if (t < half) part[t] = {part[t].x + part[t + half].x, part[t].y + part[t + half].y};
    }
    if (t < 32 && c < p.C) {
        if (p.gradBeta) p.gradBeta[c] = part[t].x;
        if (p.gradGamma) p.gradGamma[c] = part[t].y;
    }
}

// dx of the workgroup's rows; means: those of the image's groups from `first` on
template <int DT, int TC, int ACT, bool EVEN>
__device__ __forceinline__ void gradientRows(const GroupNormParams& p, const Place<TC>& w, const float2* means, int first = 0) {
    using W = Place<TC>;
    Channels<EVEN> ch;
    ch.load(p, w.c, w.n, p.mean + (long long)w.image * p.G, p.inv + (long long)w.image * p.G);
    float2 m[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i] = means[(int)p.byPer.div((uint32_t)(i < w.n ? w.c + i : w.c)) - first];
    forStores(p.stream, [&](auto streamTag) {
        forRows<W>(w, [&](auto rowsTag, int r) {
            constexpr int ROWS = decltype(rowsTag)::value;
            Row<DT, ACT, EVEN> row[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k) row[k].load(p, w.at(p, r + k * W::TR), w.n);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                row[k].work(ch);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    row[k].dz[i] = ch.inv[i] * (__builtin_fmaf(row[k].dz[i], ch.gamma[i], -m[i].x) - row[k].xhat[i] * m[i].y);
                Vec8<DT>::template store<EVEN, decltype(streamTag)::value>(p.out, w.at(p, r + k * W::TR), w.n, row[k].dz);
            }
        });
    });
}

template <int DT, int TC, int ACT, bool EVEN>
__global__ __launch_bounds__(256) void group_norm_gradient_kernel(GroupNormParams p) {
    const Place<TC> w(p);
    if (w.n > 0) gradientRows<DT, TC, ACT, EVEN>(p, w, p.means + (long long)w.image * p.G);
}

// As group_norm_small_kernel. dgamma and dbeta of one image are its sums; of several, the sums are left for the join.
template <int DT, int TC, int ACT, bool EVEN>
__global__ __launch_bounds__(256) void group_norm_small_backward_kernel(GroupNormParams p) {
    __shared__ float2 part[8][256];
    __shared__ float2 means[TC * 8];
    const Place<TC> w(p);
    chunkSums<DT, TC, ACT, EVEN>(p, w, part);
    if (p.N > 1) {
        leavePart(p, w, part);
    } else if (w.tr == 0 && w.n > 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < w.n) {
                const float2 v = part[i][threadIdx.x];
                if (p.gradBeta) p.gradBeta[w.c + i] = v.x;
                if (p.gradGamma) p.gradGamma[w.c + i] = v.y;
            }
    }
    __syncthreads();
    const int c0 = (int)blockIdx.x * p.width, g0 = c0 / p.per, groups = min(p.C - c0, p.width) / p.per;
    const int lane = threadIdx.x & 63;
    for (int g = (int)threadIdx.x >> 6; g < groups; g += 4) {   // a wave a group
        float2 s{0.f, 0.f};
        for (int k = lane; k < p.per; k += 64) {
            const int c = g * p.per + k;
            const float2 v = part[c & 7][c >> 3];
            const float gamma = p.gamma ? p.gamma[c0 + c] : 1.f;
            s.x = __builtin_fmaf(gamma, v.x, s.x);
            s.y = __builtin_fmaf(gamma, v.y, s.y);
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) {
            s.x += __shfl_down(s.x, d, 64);
            s.y += __shfl_down(s.y, d, 64);
        }
        const float f = 1.f / ((float)p.P * (float)p.per);
        if (lane == 0) means[g] = {s.x * f, s.y * f};
    }
    __syncthreads();
    if (w.n > 0) gradientRows<DT, TC, ACT, EVEN>(p, w, means, g0);
}

// ---------------------------------------------------------------- launches
template <int DT, int TC, int ACT, bool EVEN>
int launchForward(const GroupNormParams& p) {
    const dim3 grid((p.C + p.width - 1) / p.width, p.chunks, p.N);
    if (p.small) {
        hipLaunchKernelGGL((group_norm_small_kernel<DT, TC, ACT, EVEN>), grid, dim3(256), 0, stream(), p);
        OMHIP_CHECK_LAUNCH();
        return 0;
    }
    hipLaunchKernelGGL((group_norm_moments_kernel<DT, TC, EVEN>), grid, dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    hipLaunchKernelGGL(group_norm_join_kernel, dim3(p.G, p.N), dim3(64 * joinWaves(p, 8)), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    hipLaunchKernelGGL((group_norm_apply_kernel<DT, TC, ACT, EVEN>), grid, dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <int DT, int TC, int ACT, bool EVEN>
int launchBackward(const GroupNormParams& p) {
    const dim3 grid((p.C + p.width - 1) / p.width, p.chunks, p.N);
    int share = 0;   // 16 entries a lane (8: 16384 x 64 in 8 groups 14.4 us, a wave a group 13.4)
    while (2 << share <= joinWaves(p, 16)) ++share;
    const int groupBlocks = p.small ? 0 : (int)((((long long)p.N * p.G << share) + 15) / 16);
    const int channelBlocks = (p.gradGamma || p.gradBeta) && !(p.small && p.N == 1) ? (p.C + 31) / 32 : 0;
    if (p.small)
        hipLaunchKernelGGL((group_norm_small_backward_kernel<DT, TC, ACT, EVEN>), grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL((group_norm_sums_kernel<DT, TC, ACT, EVEN>), grid, dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    if (groupBlocks + channelBlocks > 0) {
        const int blocks = groupBlocks + channelBlocks, width = std::min(blocks, 1 << 16);
        hipLaunchKernelGGL(share ? group_norm_join_backward_kernel<true> : group_norm_join_backward_kernel<false>,
                           dim3(width, (blocks + width - 1) / width), dim3(1024), 0, stream(), p, (uint32_t)groupBlocks,
                           (uint32_t)share);
        OMHIP_CHECK_LAUNCH();
    }
    if (p.small) return 0;
    hipLaunchKernelGGL((group_norm_gradient_kernel<DT, TC, ACT, EVEN>), grid, dim3(256), 0, stream(), p);
    OMHIP_CHECK_LAUNCH();
    return 0;
}

template <int DT, int TC, bool EVEN>
int byAct(const GroupNormParams& p, int act, bool backward) {
    if (backward)
        return act == kActNone ? launchBackward<DT, TC, kActNone, EVEN>(p)
             : act == kActRelu ? launchBackward<DT, TC, kActRelu, EVEN>(p)
                               : launchBackward<DT, TC, kActSilu, EVEN>(p);
    return act == kActNone ? launchForward<DT, TC, kActNone, EVEN>(p)
         : act == kActRelu ? launchForward<DT, TC, kActRelu, EVEN>(p)
                           : launchForward<DT, TC, kActSilu, EVEN>(p);
}

template <int DT, int TC>
int byRows(const GroupNormParams& p, int act, bool backward) {
    return p.C % 8 == 0 && p.width % 8 == 0 ? byAct<DT, TC, true>(p, act, backward) : byAct<DT, TC, false>(p, act, backward);
}

template <int DT>
int byWidth(const GroupNormParams& p, int tc, int act, bool backward) {
    return tc == 64 ? byRows<DT, 64>(p, act, backward) : tc == 32 ? byRows<DT, 32>(p, act, backward)
                                                                  : byRows<DT, 8>(p, act, backward);
}

size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// Checks, chunks and workspace that both directions share; 0, 1 (nothing to do) or -1.
int groupNormParams(const char* name, int nDtype, int nBatch, int nPixels, int nChannels, int nGroups, int nAct, float* pMean,
                    float* pInvStd, GroupNormParams& p, int& tc) {
    if (nDtype < 0 || nDtype > 2) return fail("%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", name);
    if (nAct < kActNone || nAct > kActSilu) return fail("%s: activation must be 0 (none), 1 (ReLU) or 2 (SiLU)", name);
    if (nBatch < 0 || nPixels < 0 || nChannels < 0) return fail("%s: negative size", name);
    if (nGroups < 1 || nChannels % nGroups != 0)
        return fail("%s: %d channels do not form %d groups", name, nChannels, nGroups);
    if (nBatch == 0 || nPixels == 0 || nChannels == 0) return 1;
    if (nBatch > 65535) return fail("%s: more than 65535 images", name);
    if (nPixels > (1 << 30)) return fail("%s: more than 2^30 pixels", name);
    if (nChannels > (1 << 18)) return fail("%s: more than 2^18 channels", name);
    if ((long long)nBatch * nGroups > 0x3fffffffLL) return fail("%s: too many (image, group) pairs", name);
    p.N = nBatch; p.P = nPixels; p.C = nChannels; p.G = nGroups; p.per = nChannels / nGroups;
    p.byPer = FastDiv::make((uint32_t)p.per);
    // channels a workgroup takes: 512 (1 KB of a row of halves), less where the row has less
    const int vecs = (int)((nChannels + 7LL) / 8);
    tc = vecs > 32 ? 64 : vecs > 8 ? 32 : 8;
    const int tiles = (vecs + tc - 1) / tc;
    // chunks of pixels: two workgroups a CU (8 / 4 / 2: 56 x 56 x 256 forward 39.9 / 34.4 / 34.1 us, 28 x 28 x 512
    // backward 43.7 / 41.2 / 37.4: what a workgroup does before and after its rows), and four rows a thread at least
    const int most = (int)((nPixels + 4LL * (256 / tc) - 1) / (4 * (256 / tc)));
    int chunks = (int)std::clamp<long long>((2LL * cuCount() + (long long)tiles * nBatch - 1) / ((long long)tiles * nBatch), 1,
                                            std::min(most, 4096));   // chunks x channels stay below 2^31
    p.width = 8 * tc;
    p.stream = (long long)nBatch * nPixels * nChannels * (nDtype == 2 ? 4 : 2) >= kStreamBytes;
    // Images of few pixels take one launch of workgroups that hold whole groups and all rows, where those are short walks
    // (8 rows a thread, 2 where the workgroups are fewer than the CUs) and not so many that narrow rows cost more than
    // launches. One launch against three, bf16 SiLU, forward and backward: 64 x 196 x 512 13.3 / 19.9 against 17.7 / 23.0
    // us, 2 x 64 x 1024 7.4 / 8.9 against 10.8 / 12.4; beyond the rule 8 x 256 x 320 (48 workgroups, 8 rows) 18.6 / 29.1
    // against 12.0 / 13.9, 64 x 49 x 2048 (2048 workgroups) 17.9 / 24.8 against 17.6 / 21.9.
    const int smallTc = p.per <= 64 ? 8 : p.per <= 256 ? 32 : 64;
    const int wholeGroups = std::max(1, 8 * smallTc / p.per) * p.per;
    const long long smallBlocks = (long long)nBatch * ((nChannels + wholeGroups - 1) / wholeGroups);
    const int mostRows = (smallBlocks < cuCount() ? 2 : 8) * (256 / smallTc);
    p.small = p.per <= 512 && nPixels <= mostRows && smallBlocks <= 4LL * cuCount();
    if (p.small) {
        tc = smallTc;
        chunks = 1;
        p.width = wholeGroups;
    }
    p.rowsPerChunk = (nPixels + chunks - 1) / chunks;
    p.chunks = (nPixels + p.rowsPerChunk - 1) / p.rowsPerChunk;
    const size_t groups = (size_t)nBatch * nGroups;
    const size_t bPartial = up256((size_t)nBatch * p.chunks * nChannels * sizeof(float2));
    char* ws = static_cast<char*>(workspace(bPartial + up256(groups * sizeof(float2)) * 2, kWsOperand));
    if (!ws) return -1;   // workspace() recorded the cause
    p.partial = reinterpret_cast<float2*>(ws);
    p.means = reinterpret_cast<float2*>(ws + bPartial);
    float* own = reinterpret_cast<float*>(ws + bPartial + up256(groups * sizeof(float2)));
    p.mean = pMean ? pMean : own;
    p.inv = pInvStd ? pInvStd : own + groups;
    return 0;
}

bool elementAligned(const void* p, int nDtype) { return (reinterpret_cast<uintptr_t>(p) & (nDtype == 2 ? 3u : 1u)) == 0; }

}  // namespace

}  // namespace omhip

using namespace omhip;

extern "C" {

int omHipGroupNormNhwc(int nDtype, const void* pX, const float* pGamma, const float* pBeta, void* pY, float* pMean,
                       float* pInvStd, int nBatch, int nPixels, int nChannels, int nGroups, float fEps, int nAct) {
    const char* name = "omHipGroupNormNhwc";
    clearError();
    if (!(fEps >= 0.f)) return fail("%s: eps must not be negative", name);
    for (const void* x : {(const void*)pGamma, (const void*)pBeta, (const void*)pMean, (const void*)pInvStd})
        if (!elementAligned(x, 2)) return fail("%s: a pointer is not aligned to its elements", name);
    if (nDtype >= 0 && nDtype <= 2 && (!elementAligned(pX, nDtype) || !elementAligned(pY, nDtype)))
        return fail("%s: a pointer is not aligned to its elements", name);
    if (nBatch > 0 && nPixels > 0 && nChannels > 0 && (!pX || !pY)) return fail("%s: null pointer", name);
    GroupNormParams p{};
    int tc = 0;
    const int rc = groupNormParams(name, nDtype, nBatch, nPixels, nChannels, nGroups, nAct, pMean, pInvStd, p, tc);
    if (rc) return rc < 0 ? -1 : 0;
    p.x = pX; p.out = pY; p.gamma = pGamma; p.beta = pBeta; p.eps = fEps;
    return nDtype == 0 ? byWidth<0>(p, tc, nAct, false) : nDtype == 1 ? byWidth<1>(p, tc, nAct, false)
                                                                     : byWidth<2>(p, tc, nAct, false);
}

int omHipGroupNormNhwcBackward(int nDtype, const void* pGradY, const void* pX, const void* pY, const float* pMean,
                               const float* pInvStd, const float* pGamma, const float* pBeta, void* pGradX, float* pGradGamma,
                               float* pGradBeta, int nBatch, int nPixels, int nChannels, int nGroups, int nAct) {
    const char* name = "omHipGroupNormNhwcBackward";
    clearError();
    for (const void* x : {(const void*)pGamma, (const void*)pBeta, (const void*)pMean, (const void*)pInvStd,
                          (const void*)pGradGamma, (const void*)pGradBeta})
        if (!elementAligned(x, 2)) return fail("%s: a pointer is not aligned to its elements", name);
    if (nDtype >= 0 && nDtype <= 2)
        for (const void* x : {pGradY, pX, pY, (const void*)pGradX})
            if (!elementAligned(x, nDtype)) return fail("%s: a pointer is not aligned to its elements", name);
    if (nBatch > 0 && nPixels > 0 && nChannels > 0) {
        if (!pGradY || !pX || !pMean || !pInvStd || !pGradX) return fail("%s: null pointer", name);
        if (nAct == kActRelu && !pY) return fail("%s: ReLU needs the saved output", name);
    }
    GroupNormParams p{};
    int tc = 0;
    const int rc = groupNormParams(name, nDtype, nBatch, nPixels, nChannels, nGroups, nAct, const_cast<float*>(pMean),
                                   const_cast<float*>(pInvStd), p, tc);
    if (rc < 0) return -1;
    if (rc) {   // nothing to sum
        for (float* g : {pGradGamma, pGradBeta})
            if (g && nChannels > 0 && byteFill(g, 0, (size_t)nChannels * sizeof(float))) return -1;
        return 0;
    }
    p.x = pX; p.y = pY; p.gradY = pGradY; p.out = pGradX; p.gamma = pGamma; p.beta = pBeta;
    p.gradGamma = pGradGamma; p.gradBeta = pGradBeta;
    return nDtype == 0 ? byWidth<0>(p, tc, nAct, true) : nDtype == 1 ? byWidth<1>(p, tc, nAct, true)
                                                                    : byWidth<2>(p, tc, nAct, true);
}

}  // extern "C"
