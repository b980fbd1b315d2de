// elements.cuh -- the element types of the codebook operators (fp32, bf16, fp16): arithmetic is fp32,
// with one rounding (to nearest) at the store.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <type_traits>

#include "hds_common.cuh"

namespace hds {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(f16 x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ f16 from_float<f16>(float x) { return __float2half_rn(x); }

// Two elements in a word, the first in its lower half; one conversion instruction for both.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float low, float high) {
    if constexpr (std::is_same<T, bf16>::value) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(low, high);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// V elements moved as one vector (V = 8, 4, 2 or 1): 32 bytes at most, one 256-bit access of sm_100.
template <typename T, int V>
struct Vec {
    static constexpr int BYTES = V * (int)sizeof(T);
    static constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
    uint32_t w[WORDS];

    __device__ __forceinline__ float get(int k) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[k]);
        } else {
            const uint16_t h = (uint16_t)(w[k / 2] >> (16 * (k % 2)));
            return to_float(*reinterpret_cast<const T*>(&h));
        }
    }
    // The vector of V floats, each rounded to nearest.
    static __device__ __forceinline__ Vec pack(const float* x) {
        Vec r;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < V; k++) r.w[k] = __float_as_uint(x[k]);
        } else if constexpr (V == 1) {
            const T v = from_float<T>(x[0]);
            r.w[0] = *reinterpret_cast<const uint16_t*>(&v);
        } else {
#pragma unroll
            for (int k = 0; k < V; k += 2) r.w[k / 2] = pack_pair<T>(x[k], x[k + 1]);
        }
        return r;
    }
};

// Loads of data that is read once (not kept in the L1), in program order with stores.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_once(const T* p) {
    Vec<T, V> r;
    if constexpr (Vec<T, V>::BYTES == 32)
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]),
                       "=r"(r.w[6]), "=r"(r.w[7])
                     : "l"(p)
                     : "memory");
    else if constexpr (Vec<T, V>::BYTES == 16)
        asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                     : "l"(p)
                     : "memory");
    else if constexpr (Vec<T, V>::BYTES == 8)
        asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];"
                     : "=r"(r.w[0]), "=r"(r.w[1])
                     : "l"(p)
                     : "memory");
    else if constexpr (Vec<T, V>::BYTES == 4)
        asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(r.w[0]) : "l"(p) : "memory");
    else {
        uint16_t h;
        asm volatile("ld.global.L1::no_allocate.b16 %0, [%1];" : "=h"(h) : "l"(p) : "memory");
        r.w[0] = h;
    }
    return r;
}

// Loads of data that no thread of the kernel writes and others read too (kept in the L1).
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_shared_data(const T* p) {
    Vec<T, V> r;
    if constexpr (Vec<T, V>::BYTES == 32)
        asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
              "=r"(r.w[7])
            : "l"(p));
    else if constexpr (Vec<T, V>::BYTES == 16)
        asm("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];"
            : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
            : "l"(p));
    else if constexpr (Vec<T, V>::BYTES == 8)
        asm("ld.global.nc.v2.b32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    else if constexpr (Vec<T, V>::BYTES == 4)
        asm("ld.global.nc.b32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
    else {
        uint16_t h;
        asm("ld.global.nc.b16 %0, [%1];" : "=h"(h) : "l"(p));
        r.w[0] = h;
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const Vec<T, V>& r) {
    if constexpr (Vec<T, V>::BYTES == 32)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]),
                     "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7])
                     : "memory");
    else if constexpr (Vec<T, V>::BYTES == 16)
        asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                     "r"(r.w[3])
                     : "memory");
    else if constexpr (Vec<T, V>::BYTES == 8)
        asm volatile("st.global.v2.b32 [%0], {%1, %2};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]) : "memory");
    else if constexpr (Vec<T, V>::BYTES == 4)
        asm volatile("st.global.b32 [%0], %1;" ::"l"(p), "r"(r.w[0]) : "memory");
    else
        asm volatile("st.global.b16 [%0], %1;" ::"l"(p), "h"((uint16_t)r.w[0]) : "memory");
}

// The widest vector (elements) in which rows of `channels` elements of every given buffer can move:
// rows split into whole vectors and every base is a multiple of the vector's bytes.
struct Buffer {
    const void* p;
    int type;
};

inline size_t element_size(int type) { return type == HDS_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == HDS_TYPE_F32 || type == HDS_TYPE_BF16 || type == HDS_TYPE_F16; }

inline int widest_vector(int64_t channels, std::initializer_list<Buffer> buffers) {
    for (int v = 8; v > 1; v /= 2) {
        bool fits = channels % v == 0;
        for (const Buffer& b : buffers) fits = fits && ((uintptr_t)b.p & (v * element_size(b.type) - 1)) == 0;
        if (fits) return v;
    }
    return 1;
}

// Calls f(std::integral_constant<int, V>) with V = 8, 4, 2 or 1.
template <typename F>
int with_vector(int v, F&& f) {
    if (v == 8) return f(std::integral_constant<int, 8>{});
    if (v == 4) return f(std::integral_constant<int, 4>{});
    if (v == 2) return f(std::integral_constant<int, 2>{});
    return f(std::integral_constant<int, 1>{});
}

// Exact quotients by a fixed divisor d < 2^16 of numbers a with a * d < 2^32: a * ceil(2^32 / d) >> 32.
struct Divider {
    uint64_t magic;
    uint32_t d;
    __device__ __forceinline__ uint32_t quotient(uint32_t a) const { return (uint32_t)((a * magic) >> 32); }
};

inline Divider divider(uint32_t d) { return Divider{((1ull << 32) + d - 1) / d, d}; }

// Calls f(T{}) with the element type of a HDS_TYPE_* code (checked before).
template <typename F>
int with_type(int type, F&& f) {
    if (type == HDS_TYPE_BF16) return f(bf16{});
    if (type == HDS_TYPE_F16) return f(f16{});
    return f(float{});
}

}  // namespace hds
