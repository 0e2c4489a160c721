// The cache of keys and values: storing a batch's tokens (in float32, bf16 or 4 bits) and reading
// them back.
//
// 4 bits. 32 consecutive channels of one head of one token form a group with its own scale, so a
// token is stored without touching any other. low = minimum rounded down to bf16 and
// step = (maximum - low) / 15 rounded up to bf16, so every value lies inside [low, low + 15 step]
// and no code is clipped: the error is at most step / 2. Both are bf16 because the products that
// read them (code * step, 12 bits) are then exact in float32. 5 bits a value in all.
//
// Both kernels are bound by memory: values in (or out) once, 0.625 bytes of cache per value. Eight
// lanes take one head of one token: lane h holds the channels 4 h .. 4 h + 3 of every group, so its
// loads are 16 bytes (contiguous over the lanes), a group's extremes are three shuffles, and the
// lane's codes of all groups are the consecutive bytes [h][group] of the cache's layout. That
// layout is chosen for the attention kernel, whose lanes read whole words of it.

#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>

#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

constexpr int kThreads = 256;

// x rounded to bf16 towards -infinity / +infinity, as a float. x is not NaN.
__device__ __forceinline__ float bf16_down(float x) {
    const uint32_t u = __float_as_uint(x);
    uint32_t r = u & 0xffff0000u;
    if ((u >> 31) && (u & 0xffffu)) r += 0x10000u;
    return __uint_as_float(r);
}
__device__ __forceinline__ float bf16_up_positive(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float((u & 0xffffu) ? (u & 0xffff0000u) + 0x10000u : u);
}

// step of a group with this low and maximum. The quotient in double, rounded up to bf16. In float
// with directed roundings the two bounds nearly always round to the same bf16; only where they do
// not is the double quotient taken.
__device__ __forceinline__ float group_step(float low, float high) {
    const float up = bf16_up_positive(__fdiv_ru(__fsub_ru(high, low), 15.0f));
    const float down = bf16_up_positive(__fdiv_rd(__fsub_rd(high, low), 15.0f));
    if (up == down) return up;
    const double d = (static_cast<double>(high) - static_cast<double>(low)) / 15.0;
    float f = __double2float_ru(d);
    return bf16_up_positive(f);
}

// rint((x - low) / step) of the double quotient, in 0..15. The float quotient is within
// 15 * 3 * 2^-24 < 3e-6 of it, so only quotients within 1e-5 of a tie need the double.
__device__ __forceinline__ uint32_t code_of(float x, float low, float step, float inverse) {
    float q = __fmul_rn(__fsub_rn(x, low), inverse);
    const float f = q - floorf(q);
    if (!(fabsf(f - 0.5f) > 1e-5f) || !(q < 16.0f)) {
        const double d = (static_cast<double>(x) - static_cast<double>(low)) /
                         static_cast<double>(step);
        q = static_cast<float>(fmin(rint(d), 15.0));
    }
    return static_cast<uint32_t>(fminf(rintf(q), 15.0f));
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, bool vector, float* v);
template <>
__device__ __forceinline__ void load4<float>(const float* p, bool vector, float* v) {
    if (vector) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[i];
    }
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, bool vector, float* v) {
    if (vector) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        v[0] = bf16_bits_to_f(u.x & 0xffffu);
        v[1] = bf16_bits_to_f(u.x >> 16);
        v[2] = bf16_bits_to_f(u.y & 0xffffu);
        v[3] = bf16_bits_to_f(u.y >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __bfloat162float(p[i]);
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vector, const float* v);
template <>
__device__ __forceinline__ void store4<float>(float* p, bool vector, const float* v) {
    if (vector) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = v[i];
    }
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, bool vector, const float* v) {
    if (vector) {
        *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __float2bfloat16_rn(v[i]);
    }
}

// The cache entry of packed token t, or -1.
__device__ __forceinline__ int64_t entry_of(const Cache& c, const Batch& b, int t) {
    int seq, first, n;
    if (!find_sequence(b, t, &seq, &first, &n)) return -1;
    const int row = b.rows ? __ldg(b.rows + seq) : seq;
    const int64_t slot = static_cast<int64_t>(__ldg(b.lengths + seq)) - n + (t - first);
    if (row < 0 || row >= c.rows || slot < 0 || slot >= c.slots) return -2;
    return static_cast<int64_t>(row) * c.kv_heads * c.slots + slot;  // head h adds h * slots
}

// blockIdx.y: 0 keys, 1 values. Eight lanes per (token, head).
template <typename T, int HD, int STORAGE>
__global__ void __launch_bounds__(kThreads)
k_kv_append(Cache c, Batch b, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v,
            int64_t v_stride, bool vector) {
    constexpr int G = HD / 32;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 3;
    const int h8 = threadIdx.x & 7;
    const bool values = blockIdx.y != 0;
    const bool live = unit < static_cast<int64_t>(b.tokens) * c.kv_heads;
    const int t = live ? static_cast<int>(unit / c.kv_heads) : 0;
    const int head = live ? static_cast<int>(unit - static_cast<int64_t>(t) * c.kv_heads) : 0;
    const int64_t entry = live ? entry_of(c, b, t) : -1;
    // Lanes without an entry keep running: the shuffles below take the whole warp.
    float x[G][4];
    const T* src = (values ? v + t * v_stride : k + t * k_stride) + head * HD + 4 * h8;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        if (entry >= 0) {
            load4<T>(src + 32 * g, vector, x[g]);
        } else {
            x[g][0] = x[g][1] = x[g][2] = x[g][3] = 0.0f;
        }
    }
    const int64_t at = entry + static_cast<int64_t>(head) * c.slots;
    if constexpr (STORAGE == BST_DTYPE_U4) {
        uint32_t half[G];
        uint32_t scale = 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float lo = x[g][0], hi = x[g][0], worst = fabsf(x[g][0]);
            bool bad = !(worst <= FLT_MAX);
#pragma unroll
            for (int i = 1; i < 4; ++i) {
                lo = fminf(lo, x[g][i]);
                hi = fmaxf(hi, x[g][i]);
                bad |= !(fabsf(x[g][i]) <= FLT_MAX);
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {
                lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
                bad |= __shfl_xor_sync(kFull, static_cast<int>(bad), o) != 0;
            }
            const float low = bf16_down(lo);
            bad |= isinf(low);
            const float step = bad ? 0.0f : group_step(low, hi);
            uint32_t codes = 0;
            if (step > 0.0f) {
                // A reciprocal of a step below the normal range is no float: code_of then sees a
                // quotient that is not below 16 and takes the double.
                const float inverse = __frcp_rn(step);
#pragma unroll
                for (int i = 0; i < 4; ++i) codes |= code_of(x[g][i], low, step, inverse) << (4 * i);
            }
            half[g] = codes;
            if (h8 == g) {
                scale = bad ? (0x7fc0u << 16)
                            : (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xffff0000u);
            }
        }
        if (entry < 0) return;
        unsigned char* codes = static_cast<unsigned char*>(values ? c.v : c.k) + at * (HD / 2);
        if constexpr (G == 1) {
            reinterpret_cast<uint16_t*>(codes)[h8] = static_cast<uint16_t>(half[0]);
        } else if constexpr (G == 2) {
            reinterpret_cast<uint32_t*>(codes)[h8] = half[0] | (half[1] << 16);
        } else {
            reinterpret_cast<uint2*>(codes)[h8] =
                make_uint2(half[0] | (half[1] << 16), half[2] | (half[3] << 16));
        }
        if (h8 < G) static_cast<uint32_t*>(values ? c.v_scale : c.k_scale)[at * G + h8] = scale;
    } else {
        using S = typename std::conditional<STORAGE == BST_DTYPE_F32, float, __nv_bfloat16>::type;
        if (entry < 0) return;
        S* dst = static_cast<S*>(values ? c.v : c.k) + at * HD + 4 * h8;
#pragma unroll
        for (int g = 0; g < G; ++g) store4<S>(dst + 32 * g, true, x[g]);
    }
}

template <typename T, int HD, int STORAGE>
__global__ void __launch_bounds__(kThreads)
k_kv_read(Cache c, Batch b, T* __restrict__ k, int64_t k_stride, T* __restrict__ v,
          int64_t v_stride, bool vector) {
    constexpr int G = HD / 32;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 3;
    const int h8 = threadIdx.x & 7;
    const bool values = blockIdx.y != 0;
    if (unit >= static_cast<int64_t>(b.tokens) * c.kv_heads) return;
    const int t = static_cast<int>(unit / c.kv_heads);
    const int head = static_cast<int>(unit - static_cast<int64_t>(t) * c.kv_heads);
    const int64_t entry = entry_of(c, b, t);
    if (entry == -1) return;
    T* dst = (values ? v + t * v_stride : k + t * k_stride) + head * HD + 4 * h8;
    const int64_t at = entry + static_cast<int64_t>(head) * c.slots;
    float x[G][4] = {};
    if (entry >= 0) {
        if constexpr (STORAGE == BST_DTYPE_U4) {
            const unsigned char* codes =
                static_cast<const unsigned char*>(values ? c.v : c.k) + at * (HD / 2);
            const uint32_t* scale =
                static_cast<const uint32_t*>(values ? c.v_scale : c.k_scale) + at * G;
            uint32_t half[G];
            if constexpr (G == 1) {
                half[0] = reinterpret_cast<const uint16_t*>(codes)[h8];
            } else if constexpr (G == 2) {
                const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[h8];
                half[0] = w & 0xffffu;
                half[1] = w >> 16;
            } else {
                const uint2 w = reinterpret_cast<const uint2*>(codes)[h8];
                half[0] = w.x & 0xffffu;
                half[1] = w.x >> 16;
                half[2] = w.y & 0xffffu;
                half[3] = w.y >> 16;
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t s = scale[g];
                const float step = bf16_bits_to_f(s & 0xffffu), low = bf16_bits_to_f(s >> 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // code * step is exact, so this rounds once.
                    x[g][i] = fmaf(static_cast<float>((half[g] >> (4 * i)) & 15u), step, low);
                }
            }
        } else {
            using S = typename std::conditional<STORAGE == BST_DTYPE_F32, float, __nv_bfloat16>::type;
            const S* src = static_cast<const S*>(values ? c.v : c.k) + at * HD + 4 * h8;
#pragma unroll
            for (int g = 0; g < G; ++g) load4<S>(src + 32 * g, true, x[g]);
        }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) store4<T>(dst + 32 * g, vector, x[g]);
}

template <typename T, int HD, bool APPEND>
cudaError_t launch_storage(cudaStream_t s, const Cache& c, const Batch& b, void* k, int64_t ks,
                           void* v, int64_t vs) {
    const int64_t units = static_cast<int64_t>(b.tokens) * c.kv_heads;
    const dim3 grid(static_cast<unsigned>((units * 8 + kThreads - 1) / kThreads), 2);
    const size_t four = 4 * sizeof(T);
    const bool vector = reinterpret_cast<uintptr_t>(k) % four == 0 &&
                        reinterpret_cast<uintptr_t>(v) % four == 0 && ks % 4 == 0 && vs % 4 == 0;
    T* kk = static_cast<T*>(k);
    T* vv = static_cast<T*>(v);
#define BST_KV(STORAGE)                                                                     \
    if constexpr (APPEND) {                                                                 \
        k_kv_append<T, HD, STORAGE><<<grid, kThreads, 0, s>>>(c, b, kk, ks, vv, vs, vector); \
    } else {                                                                                \
        k_kv_read<T, HD, STORAGE><<<grid, kThreads, 0, s>>>(c, b, kk, ks, vv, vs, vector);   \
    }
    if (c.storage == BST_DTYPE_U4) {
        BST_KV(BST_DTYPE_U4)
    } else if (c.storage == BST_DTYPE_BF16) {
        BST_KV(BST_DTYPE_BF16)
    } else {
        BST_KV(BST_DTYPE_F32)
    }
#undef BST_KV
    return cudaGetLastError();
}

template <bool APPEND>
cudaError_t launch_kv(cudaStream_t s, const Cache& c, const Batch& b, void* k, int64_t ks, void* v,
                      int64_t vs, int dtype) {
    if (b.tokens < 1 || b.count < 1) return cudaSuccess;
    auto pick = [&](auto tag) {
        using T = decltype(tag);
        switch (c.head_dim) {
            case 32: return launch_storage<T, 32, APPEND>(s, c, b, k, ks, v, vs);
            case 64: return launch_storage<T, 64, APPEND>(s, c, b, k, ks, v, vs);
            default: return launch_storage<T, 128, APPEND>(s, c, b, k, ks, v, vs);
        }
    };
    return dtype == BST_DTYPE_BF16 ? pick(__nv_bfloat16()) : pick(float());
}

}  // namespace

cudaError_t launch_kv_append(cudaStream_t s, const Cache& c, const Batch& b, const void* k,
                             int64_t k_stride, const void* v, int64_t v_stride, int dtype) {
    return launch_kv<true>(s, c, b, const_cast<void*>(k), k_stride, const_cast<void*>(v), v_stride,
                           dtype);
}

cudaError_t launch_kv_read(cudaStream_t s, const Cache& c, const Batch& b, void* k,
                           int64_t k_stride, void* v, int64_t v_stride, int dtype) {
    return launch_kv<false>(s, c, b, k, k_stride, v, v_stride, dtype);
}

}  // namespace bst
