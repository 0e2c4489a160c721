// The cache of keys and values: storing a batch's tokens (in float32, bf16 or 4 bits) and reading
// them back.
//
// 4 bits. 32 consecutive channels of one head of one token form a group with its own scale, so a
// token is stored without touching any other. low = minimum rounded down to bf16 and
// step = (maximum - low) / 15 rounded up to bf16, so every value lies inside [low, low + 15 step]
// and no code is clipped: the error is at most step / 2. Both are bf16 because the products that
// read them (code * step, 12 bits) are then exact in float32. 5 bits a value in all.
//
// Both kernels move values in (or out) once and 0.625 bytes of cache per value. Eight lanes take one
// head of one token: lane h holds the channels 4 h .. 4 h + 3 of every group, so its loads are 16 bytes
// (contiguous over the lanes), the groups' extremes meet in three steps of shuffles, and the lane's
// codes of all groups are the consecutive bytes [h][group] of the cache's layout. That layout is
// chosen for the attention kernel, whose lanes read whole words of it.
// 65 536 tokens of 8 heads of 64 float32 channels (310 MB either way, 47 us at the copy rate): reading
// takes 58 us, bound by the stores; storing 75 us, bound by instruction issue (30 a value at first, 20
// with codes rounded and packed as floats and each lane carrying one group's extremes to the end),
// with a lane's next values on their way while it works on the last. bf16 values take 123 us: they lie
// on the middle between two codes far more often (0.27 % against 0.002 % of normal ones within 1e-5 of
// it), so that every fourth warp meets the double quotient.

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

// The codes rint((x - low) / step), of the double quotient, of four values in 16 bits. A float
// quotient q is within 15 * 4 * 2^-24 < 4e-6 of it (the reciprocal is good to 2^-23), so only a q within
// 1e-5 of a tie needs the double (and one that is no number, for steps below 2^-126). Adding 1.5 * 2^23 rounds q to nearest
// even; the four whole numbers, as digits of base 16, are exact in a float, too.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[4], float low, float step) {
    float c[4], off = 0.0f, inverse;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(step));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = __fmul_rn(__fsub_rn(x[i], low), inverse);
        c[i] = __fsub_rn(__fadd_rn(q, 12582912.0f), 12582912.0f);
        off = max_nan(off, fabsf(__fsub_rn(q, c[i])));
    }
    if (!(off <= 0.49999f)) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
            const float from = i < 2 ? (i ? x[1] : x[0]) : (i == 2 ? x[2] : x[3]);
            const double d = (static_cast<double>(from) - static_cast<double>(low)) /
                             static_cast<double>(step);
            const float code = static_cast<float>(fmin(rint(d), 15.0));
            if (i == 0) c[0] = code;
            if (i == 1) c[1] = code;
            if (i == 2) c[2] = code;
            if (i == 3) c[3] = code;
        }
    }
    const float digits = fmaf(c[3], 4096.0f, fmaf(c[2], 256.0f, fmaf(c[1], 16.0f, c[0])));
    return __float_as_uint(digits + 8388608.0f) & 0xffffu;
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

// A CTA's tokens: `per` of them from blockIdx.x * per on. Its first warp finds their places: the row
// and slot of token first + i in entries[i], -1 where no sequence owns the token and -2 where its
// place lies outside the cache. Eight lanes take a head of a token (a unit) and go on 32 units at a
// time; blockIdx.y: 0 keys, 1 values.
constexpr int kMaxTokens = 32;
constexpr int kUnits = kThreads / 8;

// One warp: the last sequence that starts at or before token t, 32 candidates at a time.
__device__ __forceinline__ int last_start(const Batch& b, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = b.count - 1;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32;
        const int64_t at = lo + (lane + 1ll) * step;
        const int n = __popc(__ballot_sync(kFull, at <= hi && __ldg(b.starts + at) <= t));
        lo += n * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

__device__ __forceinline__ void find_entries(const Cache& c, const Batch& b, int first, int count,
                                             int64_t* entries) {
    if (threadIdx.x >= 32) return;
    const int t = first + static_cast<int>(threadIdx.x);
    int seq = t, from = t, to = t + 1;
    if (b.starts) {
        // The first token's sequence, and from there on each token's own.
        seq = last_start(b, first);
        int hi = b.count - 1;
        if (seq == hi || __ldg(b.starts + seq + 1) > t) hi = seq;
        while (seq < hi) {
            const int mid = (seq + hi + 1) >> 1;
            if (__ldg(b.starts + mid) <= t) {
                seq = mid;
            } else {
                hi = mid - 1;
            }
        }
        from = max(0, __ldg(b.starts + seq));
        to = min(__ldg(b.starts + seq + 1), b.tokens);
    }
    int64_t entry = -1;
    if (static_cast<int>(threadIdx.x) < count && seq < b.count && t >= from && t < to) {
        const int row = b.rows ? __ldg(b.rows + seq) : seq;
        const int64_t slot = static_cast<int64_t>(__ldg(b.lengths + seq)) - (to - t);
        const bool inside = row >= 0 && row < c.rows && slot >= 0 && slot < c.slots;
        // Head h adds h * slots.
        entry = inside ? static_cast<int64_t>(row) * c.kv_heads * c.slots + slot : -2;
    }
    entries[threadIdx.x] = entry;
}

// The units of a lane's octet, one after the other.
struct Unit {
    int token, head;   // in the CTA
    int by_token, by_head, heads;
    __device__ Unit(int heads_) : heads(heads_) {
        const unsigned at = threadIdx.x >> 3, n = static_cast<unsigned>(heads_);
        token = at / n;
        head = at - token * n;
        by_token = kUnits / n;
        by_head = kUnits - by_token * n;
    }
    __device__ void next() {
        token += by_token;
        head += by_head;
        if (head >= heads) {
            head -= heads;
            ++token;
        }
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
    const int first = blockIdx.x * per, count = min(per, b.tokens - first);
    const T* const source = (values ? v : k) + 4 * h8;
    const int64_t stride = values ? v_stride : k_stride;
    Unit unit(c.kv_heads);
    float x[G][4] = {}, ahead[G][4] = {};
    auto load = [&](const Unit& u, float (&to)[G][4]) {
        if (u.token < count) {
            const T* src = source + (first + u.token) * stride + u.head * HD;
#pragma unroll
            for (int g = 0; g < G; ++g) load4<T>(src + 32 * g, vector, to[g]);
        }
    };
    load(unit, ahead);
    find_entries(c, b, first, count, entries);
    __syncthreads();
    // The same number of turns for all: the shuffles below take the whole warp.
    const int turns = (count * c.kv_heads + kUnits - 1) / kUnits;
    for (int turn = 0; turn < turns; ++turn) {
        const int64_t place = unit.token < count ? entries[unit.token] : -1;
        const int64_t at = place + static_cast<int64_t>(unit.head) * c.slots;
#pragma unroll
        for (int g = 0; g < G; ++g) {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[g][i] = ahead[g][i];
        }
        unit.next();
        load(unit, ahead);
        if constexpr (STORAGE == BST_DTYPE_U4) {
            // Extremes of the groups, summed up over the octet so that every lane ends with one
            // group's: lane h has group h / (8 / G).
            float lo[G], hi[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                lo[g] = min_nan(min_nan(x[g][0], x[g][1]), min_nan(x[g][2], x[g][3]));
                hi[g] = max_nan(max_nan(x[g][0], x[g][1]), max_nan(x[g][2], x[g][3]));
            }
#pragma unroll
            for (int n = G, o = 4; o > 0; o >>= 1) {
                if (n > 1) {
                    n /= 2;
                    const bool upper = h8 & o;
#pragma unroll
                    for (int g = 0; g < n; ++g) {
                        const float lo_out = upper ? lo[g] : lo[g + n], hi_out = upper ? hi[g] : hi[g + n];
                        lo[g] = min_nan(upper ? lo[g + n] : lo[g], __shfl_xor_sync(kFull, lo_out, o));
                        hi[g] = max_nan(upper ? hi[g + n] : hi[g], __shfl_xor_sync(kFull, hi_out, o));
                    }
                } else {
                    lo[0] = min_nan(lo[0], __shfl_xor_sync(kFull, lo[0], o));
                    hi[0] = max_nan(hi[0], __shfl_xor_sync(kFull, hi[0], o));
                }
            }
            const float my_low = bf16_down(lo[0]);
            const bool bad = !(hi[0] <= FLT_MAX) || isinf(my_low);
            const uint32_t scale = bad ? (0x7fc0u << 16)
                                       : (__float_as_uint(group_step(my_low, hi[0])) >> 16) |
                                             (__float_as_uint(my_low) & 0xffff0000u);
            uint32_t half[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t pair = __shfl_sync(kFull, scale, (threadIdx.x & 24) | (g * (8 / G)));
                const float step = bf16_bits_to_f(pair & 0xffffu), low = bf16_bits_to_f(pair >> 16);
                half[g] = step > 0.0f ? codes_of(x[g], low, step) : 0u;
            }
            if (place < 0) continue;
            unsigned char* codes = static_cast<unsigned char*>(values ? c.v : c.k) + at * (HD / 2);
            if constexpr (G == 1) {
                reinterpret_cast<uint16_t*>(codes)[h8] = static_cast<uint16_t>(half[0]);
            } else if constexpr (G == 2) {
                reinterpret_cast<uint32_t*>(codes)[h8] = half[0] | (half[1] << 16);
            } else {
                reinterpret_cast<uint2*>(codes)[h8] =
                    make_uint2(half[0] | (half[1] << 16), half[2] | (half[3] << 16));
            }
            if (h8 % (8 / G) == 0) {
                static_cast<uint32_t*>(values ? c.v_scale : c.k_scale)[at * G + h8 / (8 / G)] = scale;
            }
        } else {
            using S = typename std::conditional<STORAGE == BST_DTYPE_F32, float, __nv_bfloat16>::type;
            if (place < 0) continue;
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
    const int first = blockIdx.x * per, count = min(per, b.tokens - first);
    T* const target = (values ? v : k) + 4 * h8;
    const int64_t stride = values ? v_stride : k_stride;
    Unit unit(c.kv_heads);
    find_entries(c, b, first, count, entries);
    __syncthreads();
#pragma unroll 4
    for (; unit.token < count; unit.next()) {
        const int64_t place = entries[unit.token];
        if (place == -1) continue;
        T* dst = target + (first + unit.token) * stride + unit.head * HD;
        const int64_t at = place + static_cast<int64_t>(unit.head) * c.slots;
        float x[G][4] = {};
        if (place >= 0) {
            if constexpr (STORAGE == BST_DTYPE_U4) {
                const unsigned char* codes =
                    static_cast<const unsigned char*>(values ? c.v : c.k) + at * (HD / 2);
                const uint32_t* scales =
                    static_cast<const uint32_t*>(values ? c.v_scale : c.k_scale) + at * G;
                uint32_t half[G], scale[G];
                if constexpr (G == 1) {
                    half[0] = reinterpret_cast<const uint16_t*>(codes)[h8];
                    scale[0] = scales[0];
                } else if constexpr (G == 2) {
                    const uint32_t w = reinterpret_cast<const uint32_t*>(codes)[h8];
                    const uint2 s = *reinterpret_cast<const uint2*>(scales);
                    half[0] = w & 0xffffu;
                    half[1] = w >> 16;
                    scale[0] = s.x;
                    scale[1] = s.y;
                } else {
                    const uint2 w = reinterpret_cast<const uint2*>(codes)[h8];
                    const uint4 s = *reinterpret_cast<const uint4*>(scales);
                    half[0] = w.x & 0xffffu;
                    half[1] = w.x >> 16;
                    half[2] = w.y & 0xffffu;
                    half[3] = w.y >> 16;
                    scale[0] = s.x;
                    scale[1] = s.y;
                    scale[2] = s.z;
                    scale[3] = s.w;
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float step = bf16_bits_to_f(scale[g] & 0xffffu);
                    const float low = bf16_bits_to_f(scale[g] >> 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float code =
                            __uint_as_float(((half[g] >> (4 * i)) & 15u) | 0x4b000000u) - 8388608.0f;
                        // code * step is exact, so this rounds once.
                        x[g][i] = fmaf(code, step, low);
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
    // Tokens a CTA: one while that fills the SMs, then up to 32, about eight units an octet, over which
    // the search for their places is spread (two units instead: 168 -> 188 us for storing and reading).
    int per = std::max(1, 256 / c.kv_heads);
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
