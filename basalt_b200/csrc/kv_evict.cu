// Eviction from a cache by the weight that its keys have gathered: each key head of a sequence that has more
// than `keep` keys keeps the first `sinks`, the last `recent`, and of the others those of the largest mass,
// ties by the lowest slot. What stays moves in order to the first slots, so that windows and sinks keep
// their meaning; masses move along.
//
// Two kernels. The first finds a head's border, the mass that the last kept key has, by counting 11, 11 and
// 10 bits of the masses' ordered bits at a time, then writes the kept slots in order. The second moves keys
// and values: bound by memory, every kept byte is read and written once.

#include <algorithm>

#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

// ---- which keys stay ---------------------------------------------------------------------------
constexpr int kChoose = 1024;          // threads of the choosing CTA
constexpr int kBins = 2048;
constexpr int kEach = 4;               // keys a thread takes at a time when they are written out

// Masses in the order of whole numbers: NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (isnan(x)) return 0u;
    const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Where sequence `seq` reads and writes, and how many keys it has and keeps; a row outside its cache, or one
// that an earlier sequence writes, makes it empty. By a whole CTA.
struct Route {
    int from, to, length, kept;
};
template <int THREADS>
__device__ __forceinline__ Route route_of(const Cache& c, const Batch& b, const Eviction& e, int seq) {
    Route r;
    r.from = b.rows ? __ldg(b.rows + seq) : seq;
    const int* const to_rows = e.to_rows;
    r.to = to_rows ? __ldg(to_rows + seq) : seq;
    bool taken = false;
    if (to_rows) {
        for (int s = threadIdx.x; s < seq; s += THREADS) taken |= __ldg(to_rows + s) == r.to;
        taken = __syncthreads_or(taken);
    }
    const bool there = r.from >= 0 && r.from < c.rows && r.to >= 0 && r.to < e.to.rows && !taken;
    r.length = there ? min(max(0, __ldg(b.lengths + seq)), c.slots) : 0;
    r.kept = min(r.length, e.keep);
    if (r.to < 0 || r.to >= e.to.rows || taken) r.to = -1;
    return r;
}

// The sum of `x` over the CTA's earlier threads.
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* sums, uint32_t* all) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t run = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(kFull, run, o);
        if (lane >= o) run += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = run;
    __syncthreads();
    const uint32_t mine = sums[lane];
    uint32_t up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(kFull, up, o);
        if (lane >= o) up += y;
    }
    *all = __shfl_sync(kFull, up, 31);
    return run - x + __shfl_sync(kFull, up - mine, warp);
}

__global__ void __launch_bounds__(kChoose)
k_evict_choose(Cache c, Batch b, Eviction e) {
    __shared__ uint32_t bins[kBins], sums[32], found[2];
    const int head = blockIdx.x % c.kv_heads, seq = blockIdx.x / c.kv_heads;
    const Route route = route_of<kChoose>(c, b, e, seq);
    const int length = route.length, kept = route.kept;
    int* const places = e.kept + (static_cast<int64_t>(seq) * c.kv_heads + head) * e.keep;
    if (head == 0 && threadIdx.x == 0) e.lengths[seq] = kept;
    for (int i = kept + threadIdx.x; i < e.keep; i += kChoose) places[i] = -1;
    if (route.to < 0) return;
    const float* const mass = e.mass + (static_cast<int64_t>(max(route.from, 0)) * c.kv_heads + head) * c.slots;
    float* const to_mass = e.to_mass + (static_cast<int64_t>(route.to) * c.kv_heads + head) * e.to.slots;
    // The keys that compete: [first, last), `need` of them stay.
    const bool all = length <= e.keep;
    const int first = all ? length : e.sinks, last = all ? length : length - e.recent;
    uint32_t need = all ? 0 : e.keep - e.sinks - e.recent;
    uint32_t border = 0xffffffffu;  // ordered masses above it stay, and `need` of those equal to it
    if (need > 0) {
        uint32_t known = 0, mask = 0;
#pragma unroll 1
        for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift - 10) {
            const uint32_t bits = shift == 0 ? 10 : 11;
            for (int i = threadIdx.x; i < kBins; i += kChoose) bins[i] = 0;
            __syncthreads();
            for (int i = first + threadIdx.x; i < last; i += kChoose) {
                const uint32_t u = ordered(mass[i]);
                if ((u & mask) == known) atomicAdd(bins + ((u >> shift) & ((1u << bits) - 1)), 1u);
            }
            __syncthreads();
            // From the highest bin down: thread i has bins 2047 - 2 i and 2046 - 2 i.
            const uint32_t high = bins[kBins - 1 - 2 * threadIdx.x], low = bins[kBins - 2 - 2 * threadIdx.x];
            uint32_t total;
            const uint32_t before = sum_before(high + low, sums, &total);
            if (before < need && before + high >= need) {
                found[0] = kBins - 1 - 2 * threadIdx.x;
                found[1] = before;
            } else if (before + high < need && before + high + low >= need) {
                found[0] = kBins - 2 - 2 * threadIdx.x;
                found[1] = before + high;
            }
            __syncthreads();
            known |= found[0] << shift;
            mask |= ((1u << bits) - 1) << shift;
            need -= found[1];
            __syncthreads();
        }
        border = known;
    }
    // In order: a chunk's masses are read before any of its places is written, and places move to lower slots
    // only, so that masses may move in place.
    uint32_t done = 0, ties = 0;
    for (int at = 0; at < length; at += kChoose * kEach) {
        float m[kEach];
        uint32_t above = 0, equal = 0;  // bit i: key i of this thread's
        const int mine = at + threadIdx.x * kEach;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int key = mine + i;
            if (key >= length) break;
            m[i] = mass[key];
            const uint32_t u = ordered(m[i]);
            const bool free = key < first || key >= last;
            if (free || u > border) {
                above |= 1u << i;
            } else if (u == border) {
                equal |= 1u << i;
            }
        }
        uint32_t total;
        const uint32_t before = sum_before(__popc(above) | (__popc(equal) << 16), sums, &total);
        uint32_t tie = ties + (before >> 16), place = done + (before & 0xffffu) + min(tie, need) - min(ties, need);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            bool stays = (above >> i) & 1u;
            if ((equal >> i) & 1u) stays = tie++ < need;
            if (stays) {
                places[place] = mine + i;
                to_mass[place] = m[i];
                ++place;
            }
        }
        done += (total & 0xffffu) + min(ties + (total >> 16), need) - min(ties, need);
        ties += total >> 16;
    }
    __syncthreads();
    for (int i = kept + threadIdx.x; i < e.to.slots; i += kChoose) to_mass[i] = 0.0f;
}

// ---- what stays moves --------------------------------------------------------------------------
constexpr int kMove = 256;
constexpr int kUnits = 8;   // 16-byte units a thread holds at a time

// Rows [i0, i1) of `to` become rows places[i] of `from`: columns [u0, u0 + units) of U-byte units of rows of
// `pitch` units. The CTA reads a run of rows before it writes it, in order: rows move to lower places only, so
// `to` may be `from`.
template <typename U>
__device__ __forceinline__ void move_rows(const char* from_, char* to_, const int* places, int i0, int i1,
                                          int pitch, int u0, int units, bool in_place) {
    const U* const from = reinterpret_cast<const U*>(from_) + u0;
    U* const to = reinterpret_cast<U*>(to_) + u0;
    const int run = kMove * kUnits / units;  // rows at a time
    for (int i = i0; i < i1; i += run) {
        U x[kUnits];
        const int count = min(run, i1 - i) * units;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int at = threadIdx.x + k * kMove;
            if (at < count) x[k] = from[static_cast<int64_t>(places[i + at / units]) * pitch + at % units];
        }
        if (in_place) __syncthreads();
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int at = threadIdx.x + k * kMove;
            if (at < count) to[static_cast<int64_t>(i + at / units) * pitch + at % units] = x[k];
        }
        if (in_place) __syncthreads();
    }
}

// A CTA's share: `rows` kept keys of a head, or in place (rows 0) a slice of the columns of all of them.
__global__ void __launch_bounds__(kMove)
k_evict_move(Cache c, Batch b, Eviction e, int row_bytes, int scale_bytes, int rows, int shares) {
    const int share = blockIdx.x % shares, head = (blockIdx.x / shares) % c.kv_heads;
    const int seq = blockIdx.x / shares / c.kv_heads;
    const bool of_values = blockIdx.y;
    pdl_wait();
    const int kept = e.lengths[seq];
    const int* const places = e.kept + (static_cast<int64_t>(seq) * c.kv_heads + head) * e.keep;
    const int from_row = b.rows ? __ldg(b.rows + seq) : seq, to_row = e.to_rows ? __ldg(e.to_rows + seq) : seq;
    const int64_t from = (static_cast<int64_t>(from_row) * c.kv_heads + head) * c.slots;
    const int64_t to = (static_cast<int64_t>(to_row) * c.kv_heads + head) * e.to.slots;
    const char* const codes = static_cast<const char*>(of_values ? c.v : c.k) + from * row_bytes;
    char* const to_codes = static_cast<char*>(of_values ? e.to.v : e.to.k) + to * row_bytes;
    const char* const scales = static_cast<const char*>(of_values ? c.v_scale : c.k_scale) + from * scale_bytes;
    char* const to_scales = static_cast<char*>(of_values ? e.to.v_scale : e.to.k_scale) + to * scale_bytes;
    const int units = row_bytes / 16;
    const bool in_place = rows == 0;
    int i0 = share * rows, i1 = min(kept, i0 + rows), u0 = 0, u1 = units;
    if (in_place) {
        // Keys before the first one that went stay where they are.
        int lo = 0, hi = kept;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (places[mid] == mid) {
                lo = mid + 1;
            } else {
                hi = mid;
            }
        }
        i0 = lo;
        i1 = kept;
        u0 = units * share / shares;
        u1 = units * (share + 1) / shares;
    }
    if (i0 >= i1) return;
    move_rows<uint4>(codes, to_codes, places, i0, i1, units, u0, u1 - u0, in_place);
    if (scale_bytes == 0 || (in_place && share > 0)) return;
    move_rows<uint32_t>(scales, to_scales, places, i0, i1, scale_bytes / 4, 0, scale_bytes / 4, in_place);
}

}  // namespace

cudaError_t launch_kv_evict(cudaStream_t s, const Cache& c, const Batch& b, const Eviction& e) {
    if (b.count < 1) return cudaSuccess;
    k_evict_choose<<<c.kv_heads * b.count, kChoose, 0, s>>>(c, b, e);
    if (const cudaError_t err = cudaGetLastError()) return err;
    const int u4 = c.storage == BST_DTYPE_U4;
    const int row_bytes = u4 ? c.head_dim / 2 : c.head_dim * (c.storage == BST_DTYPE_BF16 ? 2 : 4);
    const bool in_place = e.to.k == c.k;
    // 32 KB a CTA; in place, 64 bytes of every row.
    const int rows = in_place ? 0 : std::max(1, (32 << 10) / row_bytes);
    const int shares = in_place ? std::max(1, row_bytes / 64) : (e.keep + rows - 1) / rows;
    const int64_t blocks = static_cast<int64_t>(shares) * c.kv_heads * b.count;
    return launch_pdl(k_evict_move, dim3(static_cast<unsigned>(blocks), 2), dim3(kMove), 0, s, c, b, e, row_bytes,
                      u4 ? c.head_dim / 32 * 4 : 0, rows, shares);
}

}  // namespace bst
