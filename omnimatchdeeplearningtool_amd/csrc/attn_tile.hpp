// attn_tile.hpp — tiles of the attention kernels for training: rows of halves
// in LDS, the MFMA fragments read from them, and the walk over blocks.
//
// A tile is R rows (keys or queries of one head) of RS halves in LDS, copied
// straight from memory (buffer_load ... lds). RS is the head dimension padded
// to 32, or to 128 past 64; columns past the head dimension and rows past the
// sequence read as zeros. v_mfma_f32_32x32x16 takes from a tile either
//  * natural fragments (the tile's rows are the product's rows, the sum runs
//    over the head dimension): lane (l, h) = (lane % 32, lane / 32) reads the
//    16 bytes of row l, columns 16 s + 8 h ..., or
//  * transposed ones (the product's rows are columns of the tile, the sum
//    runs over its rows): two ds_read_b64_tr_b16, which give the lane column
//    32 t + l of rows 4 h + j and 8 + 4 h + j, j = 0..3.
// The result of a product has column l and rows 8 (r / 4) + 4 h + r % 4 in the
// lane's register r. Registers 8 u .. 8 u + 7, rounded to halves, are thus the
// second operand of a product that sums over those rows, in the order in which
// the transposed fragment of rows 16 u .. 16 u + 15 has them: scores go from
// one product into the next without leaving the lane.
//
// Chunk c (16 bytes) of row r lies in slot c ^ f(r): f is one-to-one over the
// rows that share a chunk's banks (16 lanes of a natural read hit 16 slots of
// 256 bytes), and its high bits are the low bits of the row, so the four rows
// of a transposed read lie in four different 64-byte groups.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace omhip {

typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t at_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t at_u32x2 __attribute__((ext_vector_type(2)));
typedef short at_i16x4 __attribute__((ext_vector_type(4)));
typedef int at_i32x4 __attribute__((ext_vector_type(4)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));
typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* AtLdsPtr;

constexpr uint32_t kAtOOB = 0x7f000000u;     // an offset past every view of a tile
constexpr long long kAtMaxLd = 1LL << 23;    // 64 rows of halves stay below 2^30 bytes
constexpr float kAtLog2e = 1.4426950408889634f;
constexpr float kAtLn2 = 0.6931471805599453f;

template <bool BF16>
__device__ __forceinline__ at_f32x16 atMfma(const at_u32x4& a, const at_u32x4& b, const at_f32x16& c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(at_bf16x8, a), __builtin_bit_cast(at_bf16x8, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(at_f16x8, a), __builtin_bit_cast(at_f16x8, b), c,
                                                      0, 0, 0);
}

// Two floats rounded to nearest even into the half type, low then high.
template <bool BF16>
__device__ __forceinline__ uint32_t atPack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if constexpr (BF16) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
    }
}

template <bool BF16>
__device__ __forceinline__ void atUnpack2(uint32_t v, float& a, float& b) {
    if constexpr (BF16) {
        a = __builtin_bit_cast(float, v << 16);
        b = __builtin_bit_cast(float, v & 0xffff0000u);
    } else {
        a = (float)__builtin_bit_cast(_Float16, (uint16_t)v);
        b = (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16));
    }
}

// Registers 8 u .. 8 u + 7 of a product as the operand of the next one.
template <bool BF16>
__device__ __forceinline__ at_u32x4 atPack8(const at_f32x16& s, int u) {
    return at_u32x4{atPack2<BF16>(s[8 * u], s[8 * u + 1]), atPack2<BF16>(s[8 * u + 2], s[8 * u + 3]),
                    atPack2<BF16>(s[8 * u + 4], s[8 * u + 5]), atPack2<BF16>(s[8 * u + 6], s[8 * u + 7])};
}

// A buffer view of `bytes` bytes from `base` on: loads past it give zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t atView(const void* base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
}
// Memory -> LDS, 16 or 4 bytes a lane, lane after lane from dst on.
__device__ __forceinline__ void atCopy16(__amdgpu_buffer_rsrc_t r, uint16_t* dst, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (AtLdsPtr)dst, 16, voff, 0, 0, 0);
}
__device__ __forceinline__ void atCopy4(__amdgpu_buffer_rsrc_t r, float* dst, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (AtLdsPtr)dst, 4, voff, 0, 0, 0);
}

// Order of a stretch of straight code, a kind of instruction at a time (__builtin_amdgcn_sched_group_barrier). Left
// alone, the scheduler reads each fragment right before the MFMA that takes it and the wave waits out every read.
template <int N>
__device__ __forceinline__ void atMfmas() { if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(0x008, N, 0); }
template <int N>
__device__ __forceinline__ void atReads() { if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(0x100, N, 0); }
template <int N>
__device__ __forceinline__ void atValu() { if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(0x002, N, 0); }
template <int N>
__device__ __forceinline__ void atTrans() { if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(0x400, N, 0); }
// N MFMAs that take `reads` LDS reads, READS a MFMA: `ahead` of them first, then one MFMA and READS reads in turn.
template <int N, int READS, int AHEAD>
__device__ __forceinline__ void atPipeline() {
    atReads<AHEAD * READS>();
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
        atMfmas<1>();
        atReads<READS>();
    }
    atMfmas<AHEAD>();
}

// The two half-waves' values of a column (lanes l and l + 32), in the same order in both.
__device__ __forceinline__ void atBothHalves(float v, float& lower, float& upper) {
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    lower = __builtin_bit_cast(float, (uint32_t)r[0]);
    upper = __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float atMaxHalves(float v) {
    float a, b;
    atBothHalves(v, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float atSumHalves(float v) {
    float a, b;
    atBothHalves(v, a, b);
    return a + b;
}

__device__ __forceinline__ at_u32x2 atReadTransposed(const char* at) {
    return __builtin_bit_cast(at_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) at_i16x4*)at));
}

// KD: 32-column blocks of the padded head dimension.
template <int KD>
struct AtTile {
    static constexpr int RS = KD == 3 ? 128 : 32 * KD;   // halves per LDS row
    static constexpr int CH = RS / 8;                    // 16-byte chunks per row
    static constexpr int NS = 2 * KD;                    // MFMA steps over the head dimension

    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (CH == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        if constexpr (CH == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
        return (r >> 2) & 3;
    }

    // ---- memory -> LDS. Instruction i of wave w copies 64 consecutive chunks
    // of the tile; voff(i) is the lane's byte offset from the tile's first row.
    template <int ROWS, int NW>
    struct Copy {
        static constexpr int N = ROWS * CH / 64 / NW;
        static_assert(N * 64 * NW == ROWS * CH, "tile must split evenly over the waves");
        uint32_t voff[N];
        __device__ __forceinline__ void init(int wave, int lane, uint32_t ld2, int D) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int id = (wave * N + i) * 64 + lane;
                const int r = id / CH, c = (id % CH) ^ swizzle(r);
                voff[i] = c * 8 < D ? (uint32_t)r * ld2 + (uint32_t)c * 16u : kAtOOB;
            }
        }
        // rows: valid rows from `row0` on (rows past them, and columns past D, become zeros)
        __device__ __forceinline__ void run(const uint16_t* row0, int rows, uint32_t ld2, int D, uint16_t* dst,
                                            int wave) const {
            const uint32_t bytes = rows > 0 ? (uint32_t)((rows < ROWS ? rows : ROWS) - 1) * ld2 + 2u * D : 0u;
            const __amdgpu_buffer_rsrc_t rs = atView(row0, bytes);
#pragma unroll
            for (int i = 0; i < N; ++i) atCopy16(rs, dst + (wave * N + i) * 512, voff[i]);
        }
    };

    // ---- LDS -> fragments. The lane's byte offsets in a tile, made once: the compiler would make them again before
    // every read.
    struct Lane {
        uint32_t nat[NS], tr[KD][2];
        __device__ __forceinline__ explicit Lane(int lane) {
            const int l = lane & 31, h = lane >> 5, a = lane & 15, g = (lane >> 4) & 1;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                nat[s] = (uint32_t)(l * RS + ((2 * s + h) ^ swizzle(l)) * 8) * 2u;
                asm volatile("" : "+v"(nat[s]));
            }
#pragma unroll
            for (int t = 0; t < KD; ++t)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int r = 8 * j + 4 * h + (a >> 2), c = 4 * t + 2 * g + ((a & 3) >> 1);
                    tr[t][j] = (uint32_t)(r * RS + (c ^ swizzle(r)) * 8 + 4 * (a & 1)) * 2u;
                    asm volatile("" : "+v"(tr[t][j]));
                }
        }
        // rows row0 .. row0 + 31 (a multiple of 32), columns 16 s ...
        __device__ __forceinline__ at_u32x4 natural(const uint16_t* tile, int row0, int s) const {
            return *reinterpret_cast<const at_u32x4*>(reinterpret_cast<const char*>(tile) + nat[s] + row0 * RS * 2);
        }
        // columns 32 t ... of rows row0 .. row0 + 15 (a multiple of 16)
        __device__ __forceinline__ at_u32x4 transposed(const uint16_t* tile, int row0, int t) const {
            at_u32x2 p[2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
                p[j] = atReadTransposed(reinterpret_cast<const char*>(tile) + tr[t][j] + row0 * RS * 2);
            return at_u32x4{p[0][0], p[0][1], p[1][0], p[1][1]};
        }
    };

    // ---- memory -> fragments of a wave's 32 rows, through 32 rows of LDS of its own: whole rows an instruction. Loaded
    // straight into the fragments' lanes, every instruction would touch 32 rows for 32 bytes each. start() and, once the
    // wave's copies have landed, take().
    static __device__ __forceinline__ void start(const uint16_t* row0, int rows, long long ld, int D, uint16_t* stage, int lane) {
        Copy<32, 1> c;
        c.init(0, lane, (uint32_t)ld * 2u, D);
        c.run(row0, rows, (uint32_t)ld * 2u, D, stage, 0);
    }
    static __device__ __forceinline__ void take(const Lane& at, const uint16_t* stage, at_u32x4 (&f)[NS]) {
#pragma unroll
        for (int s = 0; s < NS; ++s) f[s] = at.natural(stage, 0, s);
    }
    // The same straight from memory, of row `rowPtr` ...: columns 16 s + 8 h ...
    static __device__ __forceinline__ at_u32x4 direct(const uint16_t* rowPtr, bool valid, int s, int h, int D) {
        const int c = 16 * s + 8 * h;
        return valid && c < D ? *reinterpret_cast<const at_u32x4*>(rowPtr + c) : at_u32x4{0u, 0u, 0u, 0u};
    }
};

// Workgroup id -> (head, block) of `heads` heads with `blocks` blocks each. Consecutive ids go to the 8 XCDs in turn;
// both orders keep a head's blocks on one XCD where they can, so that what they share stays in one L2.
//  * blocks of equal length: the blocks of 8 heads at a time;
//  * a causal mask (byLength): all heads' first blocks, which the callers make the longest, then their second ones.
//    Head after head, the last heads' long blocks would start late and run alone.
__device__ __forceinline__ void atPlace(uint32_t id, uint32_t heads, uint32_t blocks, bool byLength, uint32_t& head,
                                        uint32_t& block) {
    const uint32_t whole = heads / 8 * 8 * blocks;   // ids of the whole groups of 8 heads
    if (byLength) {
        head = id % heads;
        block = id / heads;
    } else if (id < whole) {
        const uint32_t xcd = id & 7, i = id >> 3;
        head = i / blocks * 8 + xcd;
        block = i % blocks;
    } else {
        head = heads / 8 * 8 + (id - whole) / blocks;
        block = (id - whole) % blocks;
    }
}

__device__ __forceinline__ int atLength(const int* lens, int b, int most) {
    if (!lens) return most;
    const int n = lens[b];
    return n < 0 ? 0 : n > most ? most : n;
}

}  // namespace omhip
