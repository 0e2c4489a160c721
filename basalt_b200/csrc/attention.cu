// Attention over a cache (float32, bf16 or 4-bit) and over packed sequences, with a sliding window
// and a few first tokens that stay visible.
//
//   out[i] = sum_j p_ij v_j,  p_ij = exp(s_ij - max_j s_ij) / sum_j exp(s_ij - max_j s_ij),
//   s_ij = scale q_i . k_j over the keys j that query i sees; zeros when it sees none.
//
// A running maximum and sum per query let every kernel read each key and value once; a key that a
// query does not see takes no part at all, whatever its slot holds (NaN and infinities included).

#include <cuda_bf16.h>

#include <algorithm>

#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

// Keys and values of one sequence and key head, in any of the layouts.
struct Source {
    const char *k, *v;            // token 0's channels
    const uint32_t *ks, *vs;      // 4-bit: token 0's (step, low) pairs
    int64_t k_stride, v_stride;   // elements between tokens (float32 and bf16)
};

template <int STORAGE, int HD>
__device__ __forceinline__ float channel(const char* base, const uint32_t* scale, int64_t stride,
                                         int64_t j, int c) {
    if constexpr (STORAGE == BST_DTYPE_F32) {
        return __ldg(reinterpret_cast<const float*>(base) + j * stride + c);
    } else if constexpr (STORAGE == BST_DTYPE_BF16) {
        return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[j * stride + c]);
    } else {
        constexpr int G = HD / 32;
        const int g = c >> 5, h = (c & 31) >> 2, i = c & 3;
        const uint32_t half =
            reinterpret_cast<const uint16_t*>(base + j * (HD / 2))[h * G + g];
        const uint32_t s = __ldg(scale + j * G + g);
        return fmaf(static_cast<float>((half >> (4 * i)) & 15u), bf16_bits_to_f(s & 0xffffu),
                    bf16_bits_to_f(s >> 16));
    }
}

__device__ __forceinline__ bool sees(int64_t position, int64_t key, int window, int sinks) {
    return key <= position && (window == 0 || position - key < window || key < sinks);
}

template <typename T>
__device__ __forceinline__ void put(T* p, float v);
template <>
__device__ __forceinline__ void put<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
}

// One query by one warp: lanes over the channels, one key at a time.
template <typename T, int STORAGE, int HD>
__device__ __forceinline__ void attend_query(const T* q, T* out, const Source& src, int64_t position,
                                             int64_t keys, int window, int sinks, float scale,
                                             int lane) {
    constexpr int C = HD / 32;
    float qv[C], acc[C], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        qv[i] = to_f(q[lane + 32 * i]);
        acc[i] = 0.0f;
    }
    const int64_t end = min(position + 1, keys);
    const int64_t first = window ? max(static_cast<int64_t>(0), position - window + 1) : 0;
    const int64_t sunk = min(static_cast<int64_t>(sinks), first);  // keys below this come first
    for (int64_t at = 0; at < sunk + max(static_cast<int64_t>(0), end - first); ++at) {
        const int64_t j = at < sunk ? at : first + (at - sunk);
        if (j >= end) break;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            dot = fmaf(qv[i], channel<STORAGE, HD>(src.k, src.ks, src.k_stride, j, lane + 32 * i),
                       dot);
        }
        const float s = warp_sum(dot) * scale;
        const float top = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.0f : expf(m - top);
        const float p = s == -INFINITY ? 0.0f : expf(s - top);  // NaN scores stay NaN
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const float x = channel<STORAGE, HD>(src.v, src.vs, src.v_stride, j, lane + 32 * i);
            acc[i] = fmaf(p, x, acc[i] * keep);
        }
        m = top;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) put(out + lane + 32 * i, l == 0.0f ? 0.0f : acc[i] / l);
}

template <int STORAGE, int HD>
__device__ __forceinline__ Source cache_source(const Cache& c, int row, int head) {
    const int64_t at = (static_cast<int64_t>(row) * c.kv_heads + head) * c.slots;
    constexpr int64_t bytes = STORAGE == BST_DTYPE_U4 ? HD / 2
                                                      : HD * (STORAGE == BST_DTYPE_F32 ? 4 : 2);
    constexpr int G = HD / 32;
    return Source{static_cast<const char*>(c.k) + at * bytes,
                  static_cast<const char*>(c.v) + at * bytes,
                  static_cast<const uint32_t*>(c.k_scale) + at * G,
                  static_cast<const uint32_t*>(c.v_scale) + at * G, HD, HD};
}

// The plain kernels: one warp per (token, head). Right for every case.
template <typename T, int STORAGE, int HD>
__global__ void __launch_bounds__(128)
k_cached_plain(Cache c, Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride,
               T* __restrict__ out, int64_t out_stride) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (unit >= static_cast<int64_t>(b.tokens) * a.heads) return;
    const int t = static_cast<int>(unit / a.heads), head = static_cast<int>(unit % a.heads);
    int seq, first, n;
    if (!find_sequence(b, t, &seq, &first, &n)) return;
    const int row = b.rows ? __ldg(b.rows + seq) : seq;
    const int64_t length = __ldg(b.lengths + seq);
    int64_t position = length - n + (t - first);
    if (row < 0 || row >= c.rows || position >= c.slots) position = -1;
    const Source src = cache_source<STORAGE, HD>(c, position < 0 ? 0 : row,
                                                 head / (a.heads / a.kv_heads));
    attend_query<T, STORAGE, HD>(q + t * q_stride + head * HD, out + t * out_stride + head * HD, src,
                                 position, c.slots, a.window, a.sinks, a.scale, threadIdx.x & 31);
}

template <typename T, int HD>
__global__ void __launch_bounds__(128)
k_packed_plain(Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride,
               const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v, int64_t v_stride,
               T* __restrict__ out, int64_t out_stride) {
    constexpr int STORAGE = sizeof(T) == 4 ? BST_DTYPE_F32 : BST_DTYPE_BF16;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (unit >= static_cast<int64_t>(b.tokens) * a.heads) return;
    const int t = static_cast<int>(unit / a.heads), head = static_cast<int>(unit % a.heads);
    int seq, first, n;
    if (!find_sequence(b, t, &seq, &first, &n)) return;
    const int kvh = head / (a.heads / a.kv_heads);
    const Source src{reinterpret_cast<const char*>(k + first * k_stride + kvh * HD),
                     reinterpret_cast<const char*>(v + first * v_stride + kvh * HD),
                     nullptr, nullptr, k_stride, v_stride};
    attend_query<T, STORAGE, HD>(q + t * q_stride + head * HD, out + t * out_stride + head * HD, src,
                                 t - first, n, a.window, a.sinks, a.scale, threadIdx.x & 31);
}

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

unsigned plain_grid(const Batch& b, const AttnSpec& a) {
    return static_cast<unsigned>((static_cast<int64_t>(b.tokens) * a.heads + 3) / 4);
}

}  // namespace

size_t attention_cached_workspace(const Cache&, const Batch&, const AttnSpec&) { return 0; }

cudaError_t launch_attention_cached(cudaStream_t s, const Cache& c, const Batch& b,
                                    const AttnSpec& a, const void* q, int64_t q_stride, void* out,
                                    int64_t out_stride, void*) {
    return by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_head_dim(a.head_dim, [&](auto hd) {
            return by_storage(c.storage, [&](auto st) {
                k_cached_plain<T, decltype(st)::value, decltype(hd)::value>
                    <<<plain_grid(b, a), 128, 0, s>>>(c, b, a, static_cast<const T*>(q), q_stride,
                                                      static_cast<T*>(out), out_stride);
                return cudaGetLastError();
            });
        });
    });
}

size_t attention_packed_workspace(const Batch&, const AttnSpec&) { return 0; }

cudaError_t launch_attention_packed(cudaStream_t s, const Batch& b, const AttnSpec& a,
                                    const void* q, int64_t q_stride, const void* k,
                                    int64_t k_stride, const void* v, int64_t v_stride, void* out,
                                    int64_t out_stride, void*) {
    return by_dtype(a.dtype, [&](auto t) {
        using T = decltype(t);
        return by_head_dim(a.head_dim, [&](auto hd) {
            k_packed_plain<T, decltype(hd)::value><<<plain_grid(b, a), 128, 0, s>>>(
                b, a, static_cast<const T*>(q), q_stride, static_cast<const T*>(k), k_stride,
                static_cast<const T*>(v), v_stride, static_cast<T*>(out), out_stride);
            return cudaGetLastError();
        });
    });
}

}  // namespace bst
