// elements.cuh -- the element types of the codebook operators (fp32, bf16, fp16): arithmetic is fp32,
// with one rounding (to nearest) at the store.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

inline size_t element_size(int type) { return type == HDS_TYPE_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == HDS_TYPE_F32 || type == HDS_TYPE_BF16 || type == HDS_TYPE_F16; }

// Calls f(T{}) with the element type of a HDS_TYPE_* code (checked before).
template <typename F>
int with_type(int type, F&& f) {
    if (type == HDS_TYPE_BF16) return f(bf16{});
    if (type == HDS_TYPE_F16) return f(f16{});
    return f(float{});
}

}  // namespace hds
