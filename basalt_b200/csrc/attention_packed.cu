// Causal attention of packed sequences over their own keys and values, with a sliding window and a
// few first tokens that stay visible.
//
//   out[i] = sum_j p_ij v_j,  p_ij = exp(s_ij - max_j s_ij) / sum_j exp(s_ij - max_j s_ij),
//   s_ij = scale q_i . k_j over the keys j that query i sees; zeros when it sees none.
//
// A running maximum and sum per query let every kernel read each key and value once; a key that a
// query does not see takes no part at all, whatever it holds (NaN and infinities included).

#include <cuda_bf16.h>

#include <algorithm>

#include "attention.cuh"
#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

// One query by one warp: lanes over the channels, one key at a time.
template <typename T, int HD>
__device__ __forceinline__ void attend_query(const T* q, const T* k, int64_t k_stride, const T* v,
                                             int64_t v_stride, T* out, int64_t position, int window,
                                             int sinks, float scale, int lane) {
    constexpr int C = HD / 32;
    float qv[C], acc[C], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        qv[i] = to_f(q[lane + 32 * i]);
        acc[i] = 0.0f;
    }
    const int64_t first = window ? max(static_cast<int64_t>(0), position - window + 1) : 0;
    const int64_t sunk = min(static_cast<int64_t>(sinks), first);  // keys below this come first
    for (int64_t at = 0; at < sunk + position + 1 - first; ++at) {
        const int64_t j = at < sunk ? at : first + (at - sunk);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) dot = fmaf(qv[i], to_f(k[j * k_stride + lane + 32 * i]), dot);
        const float s = warp_sum(dot) * scale;
        const float top = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.0f : expf(m - top);
        const float p = s == -INFINITY ? 0.0f : expf(s - top);  // NaN scores stay NaN
        l = l * keep + p;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            acc[i] = fmaf(p, to_f(v[j * v_stride + lane + 32 * i]), acc[i] * keep);
        }
        m = top;
    }
#pragma unroll
    for (int i = 0; i < C; ++i) put(out + lane + 32 * i, l == 0.0f ? 0.0f : acc[i] / l);
}

// The plain kernel: one warp per (token, head). Right for every case.
template <typename T, int HD>
__global__ void __launch_bounds__(128)
k_packed_plain(Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride,
               const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v, int64_t v_stride,
               T* __restrict__ out, int64_t out_stride) {
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (unit >= static_cast<int64_t>(b.tokens) * a.heads) return;
    const int t = static_cast<int>(unit / a.heads), head = static_cast<int>(unit % a.heads);
    int seq, first, n;
    if (!find_sequence(b, t, &seq, &first, &n)) return;
    const int kvh = head / (a.heads / a.kv_heads);
    attend_query<T, HD>(q + t * q_stride + head * HD, k + first * k_stride + kvh * HD, k_stride,
                        v + first * v_stride + kvh * HD, v_stride,
                        out + t * out_stride + head * HD, t - first, a.window, a.sinks, a.scale,
                        threadIdx.x & 31);
}

unsigned plain_grid(const Batch& b, const AttnSpec& a) {
    return static_cast<unsigned>((static_cast<int64_t>(b.tokens) * a.heads + 3) / 4);
}

}  // namespace

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
