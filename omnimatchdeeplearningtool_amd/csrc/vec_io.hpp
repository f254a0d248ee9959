// vec_io.hpp — eight consecutive values of a row as fp32, whatever type holds
// them: 0 binary16, 1 bfloat16, 2 fp32 (the C entries' nDtype). A whole group
// is one 16-byte (fp32: two) access of any alignment, a row's last group as
// many single ones as it has values.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace omhip {

// An output of this many bytes is more than the L2s (8 x 4 MB) hold beside its inputs: it leaves with streaming stores
// (67 MB of dropout gradients 28.4 -> 24.6 us, 51 MB of normalised values 34.0 -> 32.3, 26 MB of their gradients 37.1 ->
// 35.8; 19 MB of dropout 11.9 -> 12.0, so smaller ones stay).
constexpr long long kStreamBytes = 24LL << 20;

// f(true_type or false_type): whole loops for either kind of store (a choice at each store costs half of the gain).
template <class F>
__device__ __forceinline__ void forStores(bool stream, F&& f) {
    if (stream)
        f(std::true_type{});
    else
        f(std::false_type{});
}

template <int DT>
struct Vec8 {
    using Elem = std::conditional_t<DT == 2, float, uint16_t>;

    static __device__ __forceinline__ float toFloat(Elem e) {
        if constexpr (DT == 0) return (float)__builtin_bit_cast(_Float16, e);
        if constexpr (DT == 1) return __builtin_bit_cast(float, (uint32_t)e << 16);
        if constexpr (DT == 2) return e;
    }
    static __device__ __forceinline__ Elem fromFloat(float v) {   // round to nearest even
        if constexpr (DT == 0) return __builtin_bit_cast(uint16_t, (_Float16)v);
        if constexpr (DT == 1) return __builtin_bit_cast(uint16_t, (__bf16)v);
        if constexpr (DT == 2) return v;
    }
    typedef uint32_t Word4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));

    static __device__ __forceinline__ void loadWhole(const Elem* p, float (&v)[8]) {
        if constexpr (DT == 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Float4 f = *reinterpret_cast<const Float4*>(p + 4 * k);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[4 * k + i] = f[i];
            }
        } else {
            const Word4 w = *reinterpret_cast<const Word4*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = toFloat((uint16_t)w[i]);
                v[2 * i + 1] = toFloat((uint16_t)(w[i] >> 16));
            }
        }
    }
    template <bool STREAM, class V>
    static __device__ __forceinline__ void put(V* p, const V& v) {
        if constexpr (STREAM)
            __builtin_nontemporal_store(v, p);
        else
            *p = v;
    }
    template <bool STREAM>
    static __device__ __forceinline__ void storeWhole(Elem* p, const float (&v)[8]) {
        if constexpr (DT == 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
                put<STREAM>(reinterpret_cast<Float4*>(p + 4 * k), Float4{v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]});
        } else {
            Word4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)fromFloat(v[2 * i]) | (uint32_t)fromFloat(v[2 * i + 1]) << 16;
            put<STREAM>(reinterpret_cast<Word4*>(p), w);
        }
    }
    // n: values of the group (1 .. 8); the others read as 0 and are not written. EVEN: rows are whole groups (n is 8),
    // known when the kernel is compiled: with the choice left to each access the compiler splits the wide ones.
    template <bool EVEN>
    static __device__ __forceinline__ void load(const void* base, long long at, int n, float (&v)[8]) {
        const Elem* p = static_cast<const Elem*>(base) + at;
        if (EVEN || n == 8) {
            loadWhole(p, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < n ? toFloat(p[i]) : 0.f;
        }
    }
    template <bool EVEN, bool STREAM>
    static __device__ __forceinline__ void store(void* base, long long at, int n, const float (&v)[8]) {
        Elem* p = static_cast<Elem*>(base) + at;
        if (EVEN || n == 8) {
            storeWhole<STREAM>(p, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = fromFloat(v[i]);
        }
    }
};

}  // namespace omhip
