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

// step of a group with this low and maximum: the quotient in double, rounded up to bf16. Products
// with the two floats around 1 / 15 enclose the quotient; nearly always both round up to the same
// bf16, and only where they do not is the double quotient taken.
__device__ __forceinline__ float group_step(float low, float high) {
    const float up = bf16_up_positive(__fmul_ru(__fsub_ru(high, low), __uint_as_float(0x3d888889u)));
    const float down = bf16_up_positive(__fmul_rd(__fsub_rd(high, low), __uint_as_float(0x3d888888u)));
    if (up == down) return up;
    const double d = (static_cast<double>(high) - static_cast<double>(low)) / 15.0;
    return bf16_up_positive(__double2float_ru(d));
}

// rint((x - low) / step) of the double quotient, in 0..15. The float quotient q is within
// 15 * 3 * 2^-24 < 3e-6 of it, so only a q within 1e-5 of a tie needs the double (and one that is no
// number, where step's reciprocal overflows). Adding 1.5 * 2^23 rounds q to nearest even and leaves
// it in the lowest bits.
__device__ __forceinline__ uint32_t code_of(float x, float low, float step, float inverse) {
    const float q = __fmul_rn(__fsub_rn(x, low), inverse);
    const float moved = __fadd_rn(q, 12582912.0f);
    if (!(fabsf(__fsub_rn(q, __fsub_rn(moved, 12582912.0f))) <= 0.49999f)) {
        const double d = (static_cast<double>(x) - static_cast<double>(low)) /
                         static_cast<double>(step);
        return static_cast<uint32_t>(fmin(rint(d), 15.0));
    }
    return __float_as_uint(moved) & 15u;
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

// A CTA's tokens: `per` of them from blockIdx.x * per on, whose entries its first threads look up.
// Eight lanes take a head of a token (a unit); blockIdx.y: 0 keys, 1 values.
constexpr int kMaxTokens = 32;

struct Units {
    int first, count;   // tokens
    int heads;
    __device__ Units(const Cache& c, const Batch& b, int per, int64_t* entries) {
        first = blockIdx.x * per;
        count = min(per, b.tokens - first);
        heads = c.kv_heads;
        if (static_cast<int>(threadIdx.x) < count) {
            entries[threadIdx.x] = entry_of(c, b, first + threadIdx.x);
        }
        __syncthreads();
    }
};

template <typename T, int HD, int STORAGE>
__global__ void __launch_bounds__(kThreads)
k_kv_append(Cache c, Batch b, int per, const T* __restrict__ k, int64_t k_stride,
            const T* __restrict__ v, int64_t v_stride, bool vector) {
    constexpr int G = HD / 32;
    __shared__ int64_t entries[kMaxTokens];
    const int h8 = threadIdx.x & 7;
    const bool values = blockIdx.y != 0;
    const Units units(c, b, per, entries);
    const int most = (units.count * units.heads + kThreads / 8 - 1) / (kThreads / 8);
    for (int turn = 0; turn < most; ++turn) {
        const unsigned unit = turn * (kThreads / 8) + (threadIdx.x >> 3);
        const int at_token = unit / static_cast<unsigned>(units.heads);
        const int head = unit - at_token * units.heads;
        const int64_t t = units.first + at_token;
        const int64_t entry = at_token < units.count ? entries[at_token] : -1;
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
            // Extremes of the groups; then lane g computes the scale of group g for all eight.
            float low_mine = 0.0f, high_mine = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float lo = fminf(fminf(x[g][0], x[g][1]), fminf(x[g][2], x[g][3]));
                float hi = fmaxf(fmaxf(x[g][0], x[g][1]), fmaxf(x[g][2], x[g][3]));
                // fminf and fmaxf pass over a NaN.
                bool bad = !(fabsf(x[g][0]) <= FLT_MAX) || !(fabsf(x[g][1]) <= FLT_MAX) ||
                           !(fabsf(x[g][2]) <= FLT_MAX) || !(fabsf(x[g][3]) <= FLT_MAX);
                if (bad) hi = INFINITY;
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) {
                    lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
                    hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
                }
                if (h8 == g) {
                    low_mine = bf16_down(lo);
                    high_mine = hi;
                }
            }
            const bool bad = !(high_mine <= FLT_MAX) || isinf(low_mine);
            const float step_mine = bad ? 0.0f : group_step(low_mine, high_mine);
            const uint32_t scale = bad ? (0x7fc0u << 16)
                                       : (__float_as_uint(step_mine) >> 16) |
                                             (__float_as_uint(low_mine) & 0xffff0000u);
            uint32_t half[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t pair = __shfl_sync(kFull, scale, (threadIdx.x & 24) | g);
                const float step = bf16_bits_to_f(pair & 0xffffu), low = bf16_bits_to_f(pair >> 16);
                half[g] = 0u;
                if (step > 0.0f) {
                    const float inverse = __frcp_rn(step);
#pragma unroll
                    for (int i = 0; i < 4; ++i) half[g] |= code_of(x[g][i], low, step, inverse) << (4 * i);
                }
            }
            if (entry < 0) continue;
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
            if (entry < 0) continue;
            S* dst = static_cast<S*>(values ? c.v : c.k) + at * HD + 4 * h8;
#pragma unroll
            for (int g = 0; g < G; ++g) store4<S>(dst + 32 * g, true, x[g]);
        }
    }
}

template <typename T, int HD, int STORAGE>
__global__ void __launch_bounds__(kThreads)
k_kv_read(Cache c, Batch b, int per, T* __restrict__ k, int64_t k_stride, T* __restrict__ v,
          int64_t v_stride, bool vector) {
    constexpr int G = HD / 32;
    __shared__ int64_t entries[kMaxTokens];
    const int h8 = threadIdx.x & 7;
    const bool values = blockIdx.y != 0;
    const Units units(c, b, per, entries);
#pragma unroll 2
    for (unsigned unit = threadIdx.x >> 3; unit < static_cast<unsigned>(units.count * units.heads);
         unit += kThreads / 8) {
        const int at_token = unit / static_cast<unsigned>(units.heads);
        const int head = unit - at_token * units.heads;
        const int64_t t = units.first + at_token, entry = entries[at_token];
        if (entry == -1) continue;
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
}

template <typename T, int HD, bool APPEND>
cudaError_t launch_storage(cudaStream_t s, const Cache& c, const Batch& b, void* k, int64_t ks,
                           void* v, int64_t vs) {
    // Tokens a CTA: one while that fills the SMs, then up to 32, at least two units a thread.
    int per = std::max(1, 64 / c.kv_heads);
    per = std::max(1, std::min({per, kMaxTokens, b.tokens / (148 * 4)}));
    const dim3 grid(static_cast<unsigned>((b.tokens + per - 1) / per), 2);
    const size_t four = 4 * sizeof(T);
    const bool vector = reinterpret_cast<uintptr_t>(k) % four == 0 &&
                        reinterpret_cast<uintptr_t>(v) % four == 0 && ks % 4 == 0 && vs % 4 == 0;
    T* kk = static_cast<T*>(k);
    T* vv = static_cast<T*>(v);
#define BST_KV(STORAGE)                                                                     \
    if constexpr (APPEND) {                                                                 \
        k_kv_append<T, HD, STORAGE><<<grid, kThreads, 0, s>>>(c, b, per, kk, ks, vv, vs, vector); \
    } else {                                                                                \
        k_kv_read<T, HD, STORAGE><<<grid, kThreads, 0, s>>>(c, b, per, kk, ks, vv, vs, vector);   \
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
