// vec_io.hpp — eight consecutive values of a row as fp32, whatever type holds
// them: 0 binary16, 1 bfloat16, 2 fp32 (the C entries' nDtype). A whole group
// is one 16-byte (fp32: two) access of any alignment, a row's last group as
// many single ones as it has values.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace omhip {

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
    // n: values of the group (1 .. 8); the others read as 0 and are not written
    static __device__ __forceinline__ void load(const void* base, long long at, int n, float (&v)[8]) {
        const Elem* p = static_cast<const Elem*>(base) + at;
        Elem e[8];
        if (n == 8) {
            __builtin_memcpy(e, p, sizeof(e));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : Elem(0);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = toFloat(e[i]);
    }
    static __device__ __forceinline__ void store(void* base, long long at, int n, const float (&v)[8]) {
        Elem* p = static_cast<Elem*>(base) + at;
        Elem e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = fromFloat(v[i]);
        if (n == 8) {
            __builtin_memcpy(p, e, sizeof(e));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[i] = e[i];
        }
    }
};

}  // namespace omhip
