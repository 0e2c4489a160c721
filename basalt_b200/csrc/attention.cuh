// Helpers shared by the attention kernels.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include <algorithm>

#include "device.cuh"
#include "operators.h"

namespace bst {

template <typename T>
__device__ __forceinline__ void put(T* p, float v);
template <>
__device__ __forceinline__ void put<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void put<__nv_bfloat16>(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
}

// An asynchronous copy of N bytes to shared memory of which the first `bytes` are read, the rest zero.
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, int bytes) {
    if constexpr (N == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
                     : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N),
                     "r"(bytes)
                     : "memory");
    }
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {  // lo in the low half
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// One tile of query rows of one key head.
struct Tile {
    int seq, first, n;   // the sequence, its first packed token and its tokens
    int r0;              // the tile's first query row: row r is token r / group, head r % group
};

// Tensor-core tiles over a sequence's own row: query rows a tile; the keys that a tile whose last token stands at
// `position` sees, [0, end); and of `splits` the ones that are worth it, 512 keys or more each.
constexpr int kTcTileRows = 256;
__device__ __forceinline__ int tc_end(int position, int row, const Cache& c) {
    return row >= 0 && row < c.rows ? max(0, min(position + 1, c.slots)) : 0;
}
__device__ __forceinline__ int tc_useful(int end, int splits) { return max(1, min(splits, end / 512)); }

// Tile number `index` of a batch whose sequences have n group rows each, tile_rows to a tile. Without
// starts every sequence has the same number of tiles; with them the tiles before each sequence are
// summed, 32 sequences at a time.
__device__ __forceinline__ bool find_tile(const Batch& b, int group, int tile_rows, int index, Tile* t) {
    if (!b.starts) {
        const int per = (group + tile_rows - 1) / tile_rows;
        t->seq = index / per;
        t->first = t->seq;
        t->n = 1;
        t->r0 = (index - t->seq * per) * tile_rows;
        return t->seq < b.count;
    }
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int s0 = 0; s0 < b.count; s0 += 32) {
        const int s = s0 + lane;
        int from = 0, n = 0;
        if (s < b.count) {
            from = max(0, __ldg(b.starts + s));
            n = max(0, min(__ldg(b.starts + s + 1), b.tokens) - from);
        }
        const int tiles = (n * group + tile_rows - 1) / tile_rows;
        int run = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(kFull, run, o);
            if (lane >= o) run += v;
        }
        const unsigned hit = __ballot_sync(kFull, before + run > index);
        if (hit) {
            const int who = __ffs(hit) - 1;
            t->seq = s0 + who;
            t->first = __shfl_sync(kFull, from, who);
            t->n = __shfl_sync(kFull, n, who);
            t->r0 = (index - before - __shfl_sync(kFull, run - tiles, who)) * tile_rows;
            return true;
        }
        before += __shfl_sync(kFull, run, 31);
    }
    return false;
}

// One query's attention over keys key_of(0) .. key_of(n - 1) (negative: none) by one warp, plainly: what
// rows with values that are not finite are added up by. 32 keys at a time: the lanes hold channels, and
// their partial sums change places, half as many at every step, so that lane i ends with the score of
// key i. Leaves the maximum of the scores (to base 2), the sum of weights, and channels lane + 32 i; each
// key's score goes to write_score, up to the first NaN (behind it every weight is one).
struct NoScores {
    __device__ void operator()(int64_t, float) const {}
};
template <int C, typename T, typename S, typename K, typename W = NoScores>
__device__ __forceinline__ void attend_row(const T* q, const S* k, int64_t k_stride, const S* v,
                                           int64_t v_stride, float scale, int64_t n, K&& key_of,
                                           float (&value)[C], float* top_, float* total_,
                                           W&& write_score = W()) {
    const int lane = threadIdx.x & 31;
    float x[C], top = -INFINITY, total = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        x[i] = to_f(q[lane + 32 * i]);
        value[i] = 0.0f;
    }
    for (int64_t at = 0; at < n; at += 32) {
        const int64_t mine = at + lane < n ? key_of(at + lane) : -1;
        const unsigned seen = __ballot_sync(kFull, mine >= 0);
        // Keys that are not there are read as key 0, and left out below.
        const int64_t from = max(mine, static_cast<int64_t>(0));
        float s[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const S* row = k + __shfl_sync(kFull, from, j) * k_stride + lane;
            s[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < C; ++i) s[j] = fmaf(x[i], to_f(row[32 * i]), s[j]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const bool upper = lane & o;
#pragma unroll
            for (int j = 0; j < o; ++j) {
                const float away = upper ? s[j] : s[j + o];
                s[j] = (upper ? s[j + o] : s[j]) + __shfl_xor_sync(kFull, away, o);
            }
        }
        const float score = mine >= 0 ? s[0] * scale : -INFINITY;
        if (mine >= 0) write_score(mine, score);
        const float most = fmaxf(top, warp_max(score));
        const float keep = top == -INFINITY ? 0.0f : exp2f(top - most);
        const float p = score == -INFINITY ? 0.0f : exp2f(score - most);  // a NaN stays one
        total = fmaf(total, keep, warp_sum(p));
        top = most;
        if (isnan(total)) break;  // and so is every channel
#pragma unroll
        for (int i = 0; i < C; ++i) value[i] *= keep;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const float weight = __shfl_sync(kFull, p, j);
            const S* row = v + __shfl_sync(kFull, from, j) * v_stride + lane;
            if (!((seen >> j) & 1u)) continue;
#pragma unroll
            for (int i = 0; i < C; ++i) value[i] = fmaf(weight, to_f(row[32 * i]), value[i]);
        }
    }
    *top_ = top;
    *total_ = total;
}

// Tiles of `rows` query rows: exact without starts, at most one partial tile a sequence with them.
inline int tile_bound(const Batch& b, const AttnSpec& a, int64_t rows) {
    const int64_t group = a.heads / a.kv_heads;
    if (!b.starts) return static_cast<int>(b.count * ((group + rows - 1) / rows));
    return static_cast<int>(std::min<int64_t>((b.tokens * group) / rows + b.count, b.tokens * group));
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
