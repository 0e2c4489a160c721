// Helpers shared by the attention kernels.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "basalt_cuda.h"

namespace bst {

template <typename T>
__device__ __forceinline__ void put(T* p, float v);
template <>
__device__ __forceinline__ void put<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
}

// Calls fn with the value as a constant or type.
template <typename Fn>
cudaError_t by_head_dim(int hd, Fn&& fn) {
    switch (hd) {
        case 32: return fn(std::integral_constant<int, 32>());
        case 64: return fn(std::integral_constant<int, 64>());
        default: return fn(std::integral_constant<int, 128>());
    }
}

template <typename Fn>
cudaError_t by_dtype(int dtype, Fn&& fn) {
    return dtype == BST_DTYPE_BF16 ? fn(__nv_bfloat16()) : fn(float());
}

template <typename Fn>
cudaError_t by_storage(int storage, Fn&& fn) {
    switch (storage) {
        case BST_DTYPE_U4: return fn(std::integral_constant<int, BST_DTYPE_U4>());
        case BST_DTYPE_BF16: return fn(std::integral_constant<int, BST_DTYPE_BF16>());
        default: return fn(std::integral_constant<int, BST_DTYPE_F32>());
    }
}

}  // namespace bst
