// Drawing tokens from filtered distributions: temperature, top-k, top-p, min-p.
//
// With z = (logit - largest) / temperature the weight of a token is exp(z), held as a 64-bit whole
// number of units of 2^-42 (so 2^20 tokens cannot overflow it). Sums of whole numbers do not depend
// on their order: any number of threads may add in any order, with atomics, and a draw still comes
// out the same. Weights below 2^-40 count as nothing. The exponential is a double one, because a
// draw among 10^5 tokens is decided by differences of 10^-10 of their sum: 2^(k / 32) from a table
// times the Taylor polynomial of 2^r, |r| <= 1/64, of degree five (2^-48): eleven double operations,
// where the library's function for all arguments takes four times as many.
//
// No sort of the row. All filters keep a prefix of the order (logit descending, index ascending), so
// each is a threshold: the smallest logit kept and how many of the tokens with exactly that logit. A
// histogram of 2048 bins over the distance from the largest logit (which spreads the tokens evenly,
// where bits of the float would pile them on a few bins) finds the bin in which the sum of counts or
// weights crosses, and the few tokens in that bin are sorted. (Should it hold more than fit, more
// histograms follow, over the bits of its logits.) A top_k that fits the list itself needs no more:
// its candidates are collected with their indices and one CTA finishes on them. Otherwise the draw is
// a running sum over slices of the row, then inside one slice.
//
// A row is worked on by a cluster of CTAs, each with a slice of the row in its shared memory; sums,
// histograms and lists meet through distributed shared memory. The row is read once; what bounds the
// kernel are its passes over the slices in shared memory, the double operations, and for few rows the
// latency of the steps between them: 32 rows of 4096 with top_k 40 take 10 us (16 with all logits counted
// and the list sorted), 2048 unfiltered rows of 8192 take 53, 64 rows of 131 072 with settings of their
// own 64, the time of those whose top_p needs the histogram of weights.

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>
#include <cstddef>

#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

namespace cg = cooperative_groups;

// Threads a CTA: few, so that more CTAs share an SM and cover one another's steps (512 took 101 us
// instead of 78 for 2048 rows of 8192 at that step, and the same for 64 rows of 131 072).
constexpr int kThreads = 256;
constexpr int kBins = 2048;
constexpr int kCoarse = 64;                  // bins / kCoarse = 32 bins, a lane each
constexpr int kCountBins = 256;              // for counts of a list's candidates
constexpr int kMaxCluster = 8;
constexpr double kCut = -27.725887222397812; // ln 2^-40
using u64 = unsigned long long;

// Not the constant, with which loops are unrolled into spills (53 -> 57 us for 2048 rows of 8192).
__device__ __forceinline__ int threads() { return static_cast<int>(blockDim.x); }
__device__ __forceinline__ int warps() { return static_cast<int>(blockDim.x >> 5); }

// Floats in an order of whole numbers: a < b as floats <=> key(a) < key(b); -0 and 0 are one, NaN
// is -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
    x = isnan(x) ? -INFINITY : x + 0.0f;
    const uint32_t u = __float_as_uint(x);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float float_of(uint32_t key) {
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

constexpr int kList = 2048;   // tokens that a list holds

struct Shared {
    u64 coarse[kCoarse];
    double powers[32];                 // 2^(k / 32)
    unsigned listed;                   // tokens that asked for a place in the list
    u64 exchange[2][2];     // this CTA's value of a reduction over the cluster, two pairs in turn
    u64 warp_a[kThreads / 32], warp_b[kThreads / 32];
    u64 result[4];
    // Rows without filters end here.
    alignas(16) uint32_t low[kBins];  // a histogram's 64-bit sums; both halves are a list otherwise
    uint32_t high[kBins];
};
static_assert(sizeof(Shared) % 16 == 0 && offsetof(Shared, low) % 16 == 0, "slices are 16-byte aligned");
static_assert(kList * 8 == kBins * 8, "a list lies in the histogram's place");

// A histogram's 64-bit sum grows by v: two native 32-bit additions, the carry by hand.
__device__ __forceinline__ void add_to(Shared& sh, int bin, u64 v) {
    const uint32_t lo = static_cast<uint32_t>(v);
    uint32_t hi = static_cast<uint32_t>(v >> 32);
    if (lo && atomicAdd(&sh.low[bin], lo) > 0xffffffffu - lo) ++hi;
    if (hi) atomicAdd(&sh.high[bin], hi);
}

// A list lies in the histogram's place.
__device__ __forceinline__ u64* list_of(Shared* sh) { return reinterpret_cast<u64*>(sh->low); }

// Sorts v[0 .. n) (n a power of two) in descending order, with the whole CTA.
__device__ __forceinline__ void sort_descending(u64* v, int n) {
    for (int size = 2; size <= n; size <<= 1) {
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            __syncthreads();
            for (int x = threadIdx.x; x < n / 2; x += threads()) {
                const int i = 2 * x - (x & (stride - 1)), j = i + stride;
                const u64 p = v[i], q = v[j];
                if ((p < q) == ((i & size) == 0)) {
                    v[i] = q;
                    v[j] = p;
                }
            }
        }
    }
    __syncthreads();
}

__device__ __forceinline__ u64 warp_sum_u(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_max_u(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// A row's state, the same in all threads of the cluster.
template <typename T>
struct Row {
    Shared& sh;
    cg::cluster_group cluster;
    int ranks, rank;
    const T* slice;   // this CTA's logits [0, count), of row indices begin + i
    int begin, count;
    int turn = 0;

    __device__ void sync() {
        if (ranks == 1) {
            __syncthreads();
        } else {
            cluster.sync();
        }
    }

    // Sum (or maximum) over all threads of the cluster of two values at once; the CTAs' own
    // results in rank order are in each CTA's exchange slot until the next but one call.
    template <bool MAX>
    __device__ void reduce(u64& a, u64& b) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const u64 wa = MAX ? warp_max_u(a) : warp_sum_u(a);
        const u64 wb = MAX ? warp_max_u(b) : warp_sum_u(b);
        if (lane == 0) {
            sh.warp_a[warp] = wa;
            sh.warp_b[warp] = wb;
        }
        __syncthreads();
        if (warp == 0) {
            u64 x = lane < warps() ? sh.warp_a[lane] : 0, y = lane < warps() ? sh.warp_b[lane] : 0;
            x = MAX ? warp_max_u(x) : warp_sum_u(x);
            y = MAX ? warp_max_u(y) : warp_sum_u(y);
            if (lane == 0) {
                sh.exchange[turn][0] = x;
                sh.exchange[turn][1] = y;
            }
        }
        sync();
        a = b = 0;
        for (int r = 0; r < ranks; ++r) {
            const u64* e = cluster.map_shared_rank(&sh.exchange[turn][0], r);
            a = MAX ? max(a, e[0]) : a + e[0];
            b = MAX ? max(b, e[1]) : b + e[1];
        }
        turn ^= 1;
        __syncthreads();  // warp_a and warp_b are free again
    }

    __device__ float at(int i) const { return to_f(slice[i]); }
};

// Where a running sum from the largest logit down reaches a target.
struct Threshold {
    uint32_t key;   // the smallest key kept; 0: everything
    u64 above;      // the sum over larger keys
    u64 target;
};

// Clears the histogram.
__device__ __forceinline__ void clear_bins(Shared& sh) {
    for (int i = threadIdx.x; i < kBins; i += threads()) sh.low[i] = sh.high[i] = 0u;
    __syncthreads();
}

// The first bin at which the cluster's histogram, summed from bin 0 on top of `above`, reaches
// `target`; sh.result = bin, the sum before it, its own sum.
template <typename T>
__device__ void find_bin(Row<T>& row, u64 above, u64 target) {
    Shared& sh = row.sh;
    auto bin = [](const Shared* s, int i) { return (static_cast<u64>(s->high[i]) << 32) + s->low[i]; };
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < kCoarse; i += warps()) {
        const u64 v = warp_sum_u(bin(&sh, i * 32 + (threadIdx.x & 31)));
        if ((threadIdx.x & 31) == 0) sh.coarse[i] = v;
    }
    row.sync();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        u64 c0 = 0, c1 = 0;
        for (int r = 0; r < row.ranks; ++r) {
            const u64* c = row.cluster.map_shared_rank(sh.coarse, r);
            c0 += c[2 * lane];
            c1 += c[2 * lane + 1];
        }
        u64 run = c0 + c1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(kFull, run, o);
            if (lane >= o) run += v;
        }
        const unsigned hit = __ballot_sync(kFull, above + run >= target);
        const int who = hit ? __ffs(hit) - 1 : 31;
        u64 before = above + run - c0 - c1;
        int coarse = 2 * lane;
        if (before + c0 < target) {
            before += c0;
            ++coarse;
        }
        before = __shfl_sync(kFull, before, who);
        coarse = __shfl_sync(kFull, coarse, who);
        u64 fine = 0;
        for (int r = 0; r < row.ranks; ++r) {
            fine += bin(row.cluster.map_shared_rank(&sh, r), coarse * 32 + lane);
        }
        run = fine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(kFull, run, o);
            if (lane >= o) run += v;
        }
        const unsigned hit2 = __ballot_sync(kFull, before + run >= target);
        const int who2 = hit2 ? __ffs(hit2) - 1 : 31;
        if (lane == who2) {
            sh.result[0] = coarse * 32 + lane;
            sh.result[1] = before + run - fine;
            sh.result[2] = fine;
        }
    }
    row.sync();  // every CTA has read the others' bins
}

// Bins by the distance from the largest logit, over [least, top].
struct Distance {
    float largest, per;
    bool usable;  // the distance tells tokens apart (not over an infinite span, nor one key)
    __device__ Distance(uint32_t top, uint32_t least) {
        largest = float_of(top);
        const float span = largest - float_of(least);
        usable = span > 0.0f && span < FLT_MAX;
        per = usable ? static_cast<float>(kBins) / span : 0.0f;
    }
    __device__ int bin(float x) const {
        return min(kBins - 1, static_cast<int>((largest - x) * per));
    }
    __device__ int bin(uint32_t key) const { return bin(float_of(key)); }
};

// The key at which the sum of weight(key), over the tokens with key >= least, reaches target, which
// must be at least 1; with SHARE it is target_of(whole sum), where 1 or less ends the search at the
// largest key. extra is a sum that belongs to the key extra_key (tokens that weight() leaves out there).
template <bool SHARE, typename T, typename W, typename U>
__device__ Threshold find_threshold(Row<T>& row, uint32_t top, uint32_t least, u64 target,
                                    uint32_t extra_key, u64 extra, W&& weight, U&& target_of) {
    Shared& sh = row.sh;
    const Distance distance(top, least);
    bool by_distance = distance.usable;
    uint32_t lo = least, hi = top;
    u64 above = 0;
    bool first = SHARE;
    while (true) {
        int shift = 0;
        while (((hi - lo) >> shift) >= kBins) ++shift;
        if (shift == 0) by_distance = false;  // a bin is one key already
        auto bin_of = [&](uint32_t key) {
            return by_distance ? distance.bin(key) : static_cast<int>((hi - key) >> shift);
        };
        clear_bins(sh);
        u64 sum = 0;
        for (int i = threadIdx.x; i < row.count; i += threads()) {
            const uint32_t key = key_of(row.at(i));
            if (key < lo || key > hi) continue;
            const u64 w = weight(key);
            sum += w;
            if (w) add_to(sh, bin_of(key), w);
        }
        if (extra && row.rank == 0 && threadIdx.x == 0 && extra_key >= lo && extra_key <= hi) {
            add_to(sh, bin_of(extra_key), extra);
        }
        if (first) {
            u64 unused = 0;
            row.template reduce<false>(sum, unused);
            target = target_of(sum + extra);
            if (target <= 1) return Threshold{top, 0, target};
            first = false;
        }
        find_bin(row, above, target);
        const int bin = static_cast<int>(sh.result[0]);
        above = sh.result[1];
        if (!by_distance && shift == 0) {
            return Threshold{hi - static_cast<uint32_t>(bin), above, target};
        }
        if (!by_distance) {
            const uint32_t new_hi = hi - (static_cast<uint32_t>(bin) << shift);
            const uint32_t width = (1u << shift) - 1u;
            lo = new_hi - lo > width ? new_hi - width : lo;
            hi = new_hi;
            continue;
        }
        // The bin's tokens, collected by CTA 0 (their keys; weights follow from those).
        __syncthreads();
        if (threadIdx.x == 0) sh.listed = 0;
        row.sync();
        Shared* const home = row.cluster.map_shared_rank(&sh, 0);
        u64 high = 0, low = 0;  // the keys' range; low as its complement, so that both are maxima
        for (int i = threadIdx.x; i < row.count; i += threads()) {
            const uint32_t key = key_of(row.at(i));
            if (key < lo || key > hi || bin_of(key) != bin) continue;
            high = max(high, static_cast<u64>(key));
            low = max(low, static_cast<u64>(~key));
            const unsigned at = atomicAdd(&home->listed, 1u);
            if (at < kList) list_of(home)[at] = key;
        }
        row.template reduce<true>(high, low);  // its barrier completes the list, too
        const int n = static_cast<int>(min(home->listed, 1u + kList));
        hi = static_cast<uint32_t>(high);
        lo = ~static_cast<uint32_t>(low);
        by_distance = false;
        if (n > kList) {
            row.sync();  // the list's place is cleared next
            continue;
        }
        if (row.rank == 0) {
            int size = 2;
            while (size < n) size <<= 1;
            u64* const list = list_of(&sh);
            for (int i = n + threadIdx.x; i < size; i += threads()) list[i] = 0;
            sort_descending(list, size);
            if (threadIdx.x < 32) {
                // Lanes walk the sorted keys, 32 at a time, until the running sum reaches the target.
                u64 run = above;
                for (int i0 = 0; i0 < n; i0 += 32) {
                    const int i = i0 + static_cast<int>(threadIdx.x);
                    const uint32_t key = i < n ? static_cast<uint32_t>(list[i]) : 0u;
                    u64 w = i < n ? weight(key) : 0;
                    // What belongs to the extra key counts at its first token here.
                    if (extra && i < n && key == extra_key && (i == 0 || list[i - 1] != key)) w += extra;
                    u64 upto = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const u64 v = __shfl_up_sync(kFull, upto, o);
                        if (threadIdx.x >= o) upto += v;
                    }
                    const unsigned hit = __ballot_sync(kFull, i < n && run + upto >= target);
                    if (hit) {
                        const uint32_t edge = __shfl_sync(kFull, key, __ffs(hit) - 1);
                        // The sum over larger keys: before the first token with this key.
                        u64 larger = 0;
                        for (int x = static_cast<int>(threadIdx.x); x < n; x += 32) {
                            const uint32_t other = static_cast<uint32_t>(list[x]);
                            if (other > edge) larger += weight(other);
                        }
                        larger = warp_sum_u(larger);
                        if (extra && extra_key > edge && extra_key <= hi) larger += extra;
                        if (threadIdx.x == 0) {
                            sh.result[0] = edge;
                            sh.result[1] = above + larger;
                        }
                        break;
                    }
                    run += __shfl_sync(kFull, upto, 31);
                }
            }
        }
        row.sync();
        const uint32_t edge = static_cast<uint32_t>(home->result[0]);
        const u64 larger = home->result[1];
        row.sync();  // read by all before it is written again
        return Threshold{edge, larger, target};
    }
}

// The smallest key of [lo, hi] that holds(key), which is monotone and true at hi. One warp. The 32
// keys around a guess first, then a search in steps of 32 (a guess near zero may be many keys off).
template <typename P>
__device__ uint32_t smallest_key(uint32_t lo, uint32_t hi, uint32_t guess, P&& holds) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t base = guess > lo + 16 ? min(guess, hi) - 16 : lo;
    const unsigned near = __ballot_sync(kFull, holds(min(hi, base + lane)));
    if (near && (!(near & 1u) || base == lo)) return min(hi, base + __ffs(near) - 1);
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 32 + 1;
        const u64 key = static_cast<u64>(lo) + static_cast<u64>(lane) * step + (step - 1);
        const uint32_t mine = key < hi ? static_cast<uint32_t>(key) : hi;
        const int f = __ffs(__ballot_sync(kFull, holds(mine))) - 1;
        hi = __shfl_sync(kFull, mine, f);
        lo += static_cast<uint32_t>(f) * step;
    }
    return hi;
}

// The draw from a list of n tokens (key, ~index), of which the first top_k in order count: sorted by
// logit for the filters, then by index for the draw. One CTA; warp 0 walks the sums.
template <typename W, typename F, typename U>
__device__ void finish_list(Shared& sh, int n, int top_k, float top_p, bool floored, W&& weight,
                            F&& above_floor, U&& target_of, int* token) {
    u64* const list = list_of(&sh);
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += threads()) list[i] = 0;
    sort_descending(list, size);
    const int lane = threadIdx.x & 31;
    // Running sums of w(i), i < m, 32 at a time: the first i at which they reach `target` (m: none),
    // and with it the sum of all before the walk ended.
    auto walk = [&](int m, u64 target, auto&& w, u64* sum) {
        u64 run = 0;
        for (int i0 = 0; i0 < m; i0 += 32) {
            const int i = i0 + lane;
            u64 upto = i < m ? w(i) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 v = __shfl_up_sync(kFull, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned hit = __ballot_sync(kFull, i < m && run + upto >= target);
            if (hit) return i0 + __ffs(hit) - 1;
            run += __shfl_sync(kFull, upto, 31);
        }
        *sum = run;
        return m;
    };
    auto by_logit = [&](int i) { return weight(static_cast<uint32_t>(list[i] >> 32)); };
    if (threadIdx.x < 32) {
        int m = min(n, top_k);
        u64 sum = 0;
        if (top_p < 1.0f) {
            walk(m, ~0ull, by_logit, &sum);
            const double want = static_cast<double>(top_p) * static_cast<double>(sum);
            const u64 target = want > 0.0 ? min(sum, static_cast<u64>(ceil(want))) : 0;
            m = target <= 1 ? 1 : walk(m, target, by_logit, &sum) + 1;
        }
        if (floored) {
            int kept = 0;
            for (int i0 = 0; i0 < m; i0 += 32) {
                const int i = i0 + lane;
                kept += __popc(__ballot_sync(
                    kFull, i < m && above_floor(static_cast<uint32_t>(list[i] >> 32))));
            }
            m = kept;
        }
        if (lane == 0) sh.result[0] = m;
    }
    __syncthreads();
    const int m = static_cast<int>(sh.result[0]);
    size = 2;
    while (size < m) size <<= 1;
    for (int i = threadIdx.x; i < size; i += threads()) {
        const u64 v = list[i];
        list[i] = i < m ? (v << 32) | (v >> 32) : 0;
    }
    sort_descending(list, size);
    if (threadIdx.x < 32) {
        auto by_index = [&](int i) { return weight(static_cast<uint32_t>(list[i])); };
        u64 sum = 0;
        walk(m, ~0ull, by_index, &sum);
        // The first whose running sum exceeds the target.
        const int i = walk(m, target_of(sum) + 1, by_index, &sum);
        if (lane == 0) *token = static_cast<int>(~static_cast<uint32_t>(list[min(i, m - 1)] >> 32));
    }
}

// The same from a list of at most kRanked: every token finds its rank by comparing, and its running
// sum, in the order of the indices, by adding (tens of cycles a token where the steps of a sort and of
// two walks wait for one another).
constexpr int kRanked = 512;
template <typename W, typename F, typename U>
__device__ void finish_short_list(Shared& sh, int n, int top_k, float top_p, bool floored, W&& weight,
                                  F&& above_floor, U&& target_of, int* token) {
    const u64* const list = list_of(&sh);
    u64* const sorted = list_of(&sh) + kRanked;
    u64* const weights = sorted + kRanked;
    for (int i = threadIdx.x; i < n; i += threads()) {
        const u64 mine = list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += list[j] > mine;
        sorted[rank] = mine;
        weights[rank] = weight(static_cast<uint32_t>(mine >> 32));
    }
    int m = min(n, top_k);
    __syncthreads();
    const int lane = threadIdx.x & 31;
    // A lane's share of the first m, and the sum up to its end.
    auto scan = [&](int each) {
        u64 sum = 0;
        for (int i = lane * each; i < min(m, lane * each + each); ++i) sum += weights[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(kFull, sum, o);
            if (lane >= o) sum += v;
        }
        return sum;
    };
    if (top_p < 1.0f) {
        if (threadIdx.x < 32) {
            const int each = (m + 31) / 32;
            const u64 upto = scan(each), sum = __shfl_sync(kFull, upto, 31);
            const double want = static_cast<double>(top_p) * static_cast<double>(sum);
            const u64 target = want > 0.0 ? min(sum, static_cast<u64>(ceil(want))) : 0;
            // The first token at which the running sum reaches the target.
            const int who = __ffs(__ballot_sync(kFull, upto >= target)) - 1;
            if (lane == who) {
                int i = min(m, lane * each + each) - 1;
                for (u64 run = upto - weights[i]; i > lane * each && run >= target; run -= weights[i]) --i;
                sh.result[0] = target <= 1 ? 1 : i + 1;
            }
        }
        __syncthreads();
        m = static_cast<int>(sh.result[0]);
    }
    if (floored) {
        int kept = 0;
        for (int i0 = 0; i0 < m; i0 += threads()) {
            const int i = i0 + static_cast<int>(threadIdx.x);
            kept += __syncthreads_count(i < m && above_floor(static_cast<uint32_t>(sorted[i] >> 32)));
        }
        m = kept;
    }
    if (threadIdx.x < 32) {
        const u64 whole = scan((m + 31) / 32);
        if (lane == 31) sh.result[1] = target_of(whole);
    }
    __syncthreads();
    const u64 target = sh.result[1];
    for (int i = threadIdx.x; i < m; i += threads()) {
        // The low words are the indices' complements.
        const uint32_t mine = static_cast<uint32_t>(sorted[i]);
        u64 before = 0;
#pragma unroll 4
        for (int j = 0; j < m; ++j) before += static_cast<uint32_t>(sorted[j]) > mine ? weights[j] : 0;
        if (before <= target && target < before + weights[i]) *token = static_cast<int>(~mine);
    }
}

struct Args {
    const void* logits;
    int V, per;            // per: a CTA's slice
    int64_t stride;
    bool staged;           // slices fit in shared memory
    Sampling p;
    const double* uniforms;
    int64_t uniform_stride;
    const int* step;
    int* tokens;
};

// FILTERS false: no row has any, which leaves the histogram's memory to more CTAs an SM and half of the
// code out (2048 rows of 8192: 61.6 -> 53.3 us).
template <typename T, bool FILTERS>
__global__ void __launch_bounds__(kThreads, FILTERS ? 3 : 6)
k_sample_tokens(Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    T* staged = reinterpret_cast<T*>(smem + (FILTERS ? sizeof(Shared) : offsetof(Shared, low)));
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks());
    const int rank = static_cast<int>(cluster.block_rank());
    const int r = blockIdx.x / ranks;
    const int begin = min(a.V, rank * a.per), end = min(a.V, begin + a.per);
    const T* global = static_cast<const T*>(a.logits) + r * a.stride + begin;
    Row<T> row{sh, cluster, ranks, rank, a.staged ? staged : global, begin, end - begin};

    const float temperature = a.p.temperatures ? a.p.temperatures[r] : a.p.temperature;
    const float top_p = !FILTERS ? 1.0f : a.p.top_ps ? a.p.top_ps[r] : a.p.top_p;
    const float min_p = !FILTERS ? 0.0f : a.p.min_ps ? a.p.min_ps[r] : a.p.min_p;
    const int top_k = !FILTERS ? 0 : a.p.top_ks ? a.p.top_ks[r] : a.p.top_k;

    if (threadIdx.x < 32) sh.powers[threadIdx.x] = exp2(threadIdx.x / 32.0);
    // The largest logit (fmaxf passes over NaN).
    float most = -INFINITY;
    constexpr int kWide = 16 / sizeof(T);
    const int wide = reinterpret_cast<uintptr_t>(global) % 16 == 0 ? row.count / kWide : 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < wide; i += threads()) {
        const uint4 chunk = reinterpret_cast<const uint4*>(global)[i];
        if (a.staged) reinterpret_cast<uint4*>(staged)[i] = chunk;
        const T* x = reinterpret_cast<const T*>(&chunk);
#pragma unroll
        for (int j = 0; j < kWide; ++j) most = fmaxf(most, to_f(x[j]));
    }
    for (int i = wide * kWide + threadIdx.x; i < row.count; i += threads()) {
        const T x = global[i];
        if (a.staged) staged[i] = x;
        most = fmaxf(most, to_f(x));
    }
    u64 unused = 0, best = key_of(most);
    row.template reduce<true>(best, unused);
    const uint32_t top = static_cast<uint32_t>(best);
    const float largest = float_of(top);
    if (largest == -INFINITY || !(temperature > 0.0f)) {
        // Nothing to draw, or the first of the largest: the most tokens from it to the row's end.
        u64 rest = 0;
        for (int i = threadIdx.x; i < row.count; i += threads()) {
            if (row.at(i) == largest) rest = max(rest, static_cast<u64>(a.V - (begin + i)));
        }
        row.template reduce<true>(rest, unused);
        if (rank == 0 && threadIdx.x == 0) {
            a.tokens[r] = largest == -INFINITY ? -1 : a.V - static_cast<int>(rest);
        }
        row.sync();  // the exchange slots are read by others until here
        return;
    }

    const double T_ = temperature, top_d = largest, per_two = 1.4426950408889634 / T_;
    // The smallest key with a weight (everything, down to the lowest finite logit, at an infinite
    // temperature; the largest alone when that is infinite).
    if (threadIdx.x < 32) {
        uint32_t least = top;
        if (!isinf(largest)) {
            const float guess = static_cast<float>(fmax(top_d + kCut * T_, -static_cast<double>(FLT_MAX)));
            least = smallest_key(key_of(-FLT_MAX), top, key_of(guess), [&](uint32_t key) {
                return key == top || (static_cast<double>(float_of(key)) - top_d) / T_ >= kCut;
            });
        }
        if (threadIdx.x == 0) sh.result[3] = least;
    }
    __syncthreads();
    const uint32_t least = static_cast<uint32_t>(sh.result[3]);

    // exp((x - largest) / temperature) of a logit from `least` on, in [2^-40, 1]: 2^(k / 32 + r).
    auto real_weight = [&](float x, int* shift) -> double {
        const double y = x == largest ? 0.0 : (static_cast<double>(x) - top_d) * per_two;
        const double moved = y + 211106232532992.0;  // 1.5 * 2^47: y in whole 32nds in the low bits
        const int k = __double2loint(moved);
        const double r = y - (moved - 211106232532992.0);
        double p = fma(r, 0.0013333558146428441, 0.009618129107628477);
        p = fma(r, p, 0.055504108664821576);
        p = fma(r, p, 0.2402265069591007);
        p = fma(r, p, 0.6931471805599453);
        p = fma(r, p, 1.0);
        *shift = -(k >> 5);
        return p * sh.powers[k & 31];
    };
    // In units of 2^-42, to the nearest: adding 2^52 leaves them in the low bits.
    auto weight_of = [&](float x) -> u64 {
        int shift;
        const double w = real_weight(x, &shift);
        const double units = fma(w, __hiloint2double((1023 + 42 - shift) << 20, 0), 4503599627370496.0);
        return static_cast<u64>(__double_as_longlong(units)) & 0xfffffffffffffull;
    };
    auto weight = [&](uint32_t key) -> u64 { return key < least ? 0 : weight_of(float_of(key)); };
    const double floor_w = fmin(static_cast<double>(min_p), 1.0);
    const bool floored = min_p > 0.0f;  // a NaN is no filter
    auto above_floor = [&](uint32_t key) {
        int shift;
        const double w = real_weight(float_of(key), &shift);
        return key == top || w * __hiloint2double((1023 - shift) << 20, 0) >= floor_w;
    };
    double u = a.uniforms[r * a.uniform_stride + (a.step ? *a.step : 0)];
    u = u >= 0.0 ? fmin(u, 1.0) : 0.0;  // NaN too
    auto target_of = [&](u64 whole) {
        return min(static_cast<u64>(u * static_cast<double>(whole)), whole - 1);
    };

    // A top_k whose candidates fit a list: collected and finished by CTA 0. The k-th largest of the
    // threads' own largest logits bounds the k-th largest of all from below, closely as long as k is
    // well below the threads' number, so those alone are counted in bins; with fewer threads than k
    // all logits are.
    const Distance distance(top, least);
    if constexpr (FILTERS) if (top_k > 0 && top_k <= kList / 2 && distance.usable) {
        const float least_f = float_of(least);
        for (int i = threadIdx.x; i < kCountBins; i += threads()) sh.low[i] = 0u;
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        auto count_bin = [&](float x) { return distance.bin(x) / (kBins / kCountBins); };
        if (top_k <= ranks * threads()) {
            if (most >= least_f) atomicAdd(&sh.low[count_bin(most)], 1u);
        } else {
            for (int i = threadIdx.x; i < row.count; i += threads()) {
                const float x = row.at(i);
                if (x >= least_f) atomicAdd(&sh.low[count_bin(x)], 1u);
            }
        }
        row.sync();
        if (threadIdx.x < 32) {
            // A lane sums eight bins; the first bin at which the running sum reaches top_k.
            constexpr int kEach = kCountBins / 32;
            static_assert(kEach == 8, "two 16-byte loads a lane");
            uint32_t bins[kEach] = {};
            for (int q = 0; q < ranks; ++q) {
                const uint4* from = reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.low, q)) +
                                    2 * threadIdx.x;
                const uint4 x = from[0], y = from[1];
                bins[0] += x.x; bins[1] += x.y; bins[2] += x.z; bins[3] += x.w;
                bins[4] += y.x; bins[5] += y.y; bins[6] += y.z; bins[7] += y.w;
            }
            uint32_t upto = 0;
#pragma unroll
            for (int i = 0; i < kEach; ++i) upto += bins[i];
            const uint32_t own = upto;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(kFull, upto, o);
                if (static_cast<int>(threadIdx.x) >= o) upto += v;
            }
            const unsigned hit = __ballot_sync(kFull, upto >= static_cast<uint32_t>(top_k));
            const int who = hit ? __ffs(hit) - 1 : 31;
            if (static_cast<int>(threadIdx.x) == who) {
                int last = 0;  // bins of these before which the sum stays below top_k
                uint32_t run = upto - own;
#pragma unroll
                for (int i = 0; i < kEach - 1; ++i) {
                    run += bins[i];
                    if (run < static_cast<uint32_t>(top_k)) last = i + 1;
                }
                sh.result[0] = who * kEach + last;
            }
        }
        row.sync();  // every CTA has read the others' bins, whose place the list takes
        const int last = static_cast<int>(sh.result[0]);
        Shared* const home = cluster.map_shared_rank(&sh, 0);
        for (int i = threadIdx.x; i < row.count; i += threads()) {
            const float x = row.at(i);
            if (x >= least_f && count_bin(x) <= last) {
                const unsigned at = atomicAdd(&home->listed, 1u);
                if (at < kList) {
                    list_of(home)[at] = (static_cast<u64>(key_of(x)) << 32) |
                                        static_cast<uint32_t>(~(begin + i));
                }
            }
        }
        row.sync();
        const unsigned listed = home->listed;
        row.sync();  // the last access to other CTAs' memory, where the list is finished
        if (listed <= kList) {
            if (rank != 0) return;
            if (listed <= kRanked) {
                finish_short_list(sh, static_cast<int>(listed), top_k, top_p, floored, weight,
                                  above_floor, target_of, a.tokens + r);
            } else {
                finish_list(sh, static_cast<int>(listed), top_k, top_p, floored, weight, above_floor,
                            target_of, a.tokens + r);
            }
            return;
        }
    }

    // Kept: keys above `edge` and the first `ties` tokens, by index, with exactly that key.
    uint32_t edge = 0;
    u64 ties = 0;
    if constexpr (FILTERS) if (top_k > 0 && top_k < a.V) {
        u64 n = 0;
        for (int i = threadIdx.x; i < row.count; i += threads()) n += key_of(row.at(i)) >= least;
        unused = 0;
        row.template reduce<false>(n, unused);
        if (n > static_cast<u64>(top_k)) {
            const Threshold t = find_threshold<false>(row, top, least, static_cast<u64>(top_k), 0u, 0ull,
                                                      [](uint32_t) -> u64 { return 1; },
                                                      [](u64) -> u64 { return 0; });
            edge = t.key;
            ties = static_cast<u64>(top_k) - t.above;
        }
    }
    if constexpr (FILTERS) if (top_p < 1.0f) {
        const uint32_t from = max(least, edge + (edge ? 1u : 0u));
        const u64 tied = edge ? ties * weight(edge) : 0;
        const Threshold t = find_threshold<true>(
            row, top, edge ? edge : least, 0, edge, tied,
            [&](uint32_t key) -> u64 { return key >= from ? weight(key) : 0; },
            [&](u64 sum) -> u64 {
                // The fewest tokens whose sum is at least want: the sum has to reach ceil(want).
                const double want = static_cast<double>(top_p) * static_cast<double>(sum);
                return want > 0.0 ? min(sum, static_cast<u64>(ceil(want))) : 0;
            });
        if (t.target <= 1) {
            edge = top;
            ties = 1;
        } else {
            const u64 w = weight(t.key);
            u64 need = (t.target - t.above + w - 1) / w;
            if (t.key == edge) need = min(need, ties);
            edge = t.key;
            ties = need;
        }
    }
    if constexpr (FILTERS) if (floored) {
        // The smallest key with a weight of at least min_p; all of its tokens are kept.
        if (threadIdx.x < 32) {
            uint32_t low = top;
            if (!isinf(largest) && floor_w < 1.0) {
                const float guess = static_cast<float>(
                    fmax(top_d + log(floor_w) * T_, -static_cast<double>(FLT_MAX)));
                low = smallest_key(least, top, max(least, min(top, key_of(guess))),
                                   [&](uint32_t key) { return above_floor(max(key, least)); });
            }
            if (threadIdx.x == 0) sh.result[3] = low;
        }
        __syncthreads();
        const uint32_t low = static_cast<uint32_t>(sh.result[3]);
        if (low > edge) {
            edge = low;
            ties = ~0ull;
        }
    }
    if (edge == 0) {
        edge = least;
        ties = ~0ull;
    }

    // The draw: sums of slices in index order, then inside the slice that the target falls into.
    const u64 tie_weight = weight(edge);
    auto joined = [&](u64 sum, u64 tied) { return sum + tie_weight * min(tied, ties); };
    const float edge_f = float_of(edge);
    const bool all_ties = ties == ~0ull;  // then tokens at the edge are like the others
    auto count_range = [&](int from, int to, u64* sum, u64* tied) {  // one warp, [from, to)
        u64 s = 0, n = 0;
        if (all_ties) {
#pragma unroll 4
            for (int i = from + (threadIdx.x & 31); i < to; i += 32) {
                const float x = row.at(i);
                if (x >= edge_f) s += weight_of(x);
            }
        } else {
            for (int i = from + (threadIdx.x & 31); i < to; i += 32) {
                const float x = row.at(i);
                if (x > edge_f) s += weight_of(x);
                n += x == edge_f;
            }
        }
        *sum = warp_sum_u(s);
        *tied = warp_sum_u(n);
    };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = (row.count + warps() - 1) / warps();
    const int w0 = min(row.count, warp * part), w1 = min(row.count, w0 + part);
    u64 my_sum, my_ties;
    count_range(w0, w1, &my_sum, &my_ties);
    // Lane 0 alone carries the warp's sums into the reduction.
    u64 sum = lane == 0 ? my_sum : 0, tied = lane == 0 ? my_ties : 0;
    row.template reduce<false>(sum, tied);
    const u64 whole = joined(sum, tied);
    const u64 target = target_of(whole);
    // The CTA that holds the target: sums before it by rank. The slots written by the reduction
    // above are the ones of the other turn.
    u64 before_sum = 0, before_ties = 0;
    bool mine = false;
    for (int q = 0; q <= rank; ++q) {
        const u64* e = cluster.map_shared_rank(&sh.exchange[row.turn ^ 1][0], q);
        const u64 s = e[0], n = e[1];
        if (q == rank) {
            mine = joined(before_sum, before_ties) <= target &&
                   joined(before_sum + s, before_ties + n) > target;
        } else {
            before_sum += s;
            before_ties += n;
        }
    }
    row.sync();  // the last access to other CTAs' memory
    if (!mine) return;
    // Twice: the sums of the warps' parts pick one, and its elements become the next parts.
    int from = 0, to = row.count;
    for (int round = 0; round < 2; ++round) {
        const int step = (to - from + warps() - 1) / warps();
        const int p0 = min(to, from + warp * step), p1 = min(to, p0 + step);
        if (round > 0) count_range(p0, p1, &my_sum, &my_ties);
        __syncthreads();
        if (lane == 0) {
            sh.warp_a[warp] = my_sum;
            sh.warp_b[warp] = my_ties;
        }
        __syncthreads();
        int pick = 0;
        for (; pick < warps() - 1; ++pick) {
            const u64 s = before_sum + sh.warp_a[pick], n = before_ties + sh.warp_b[pick];
            if (joined(s, n) > target) break;
            before_sum = s;
            before_ties = n;
        }
        const int f = min(to, from + pick * step);
        to = min(to, f + step);
        from = f;
    }
    if (warp != 0) return;
    for (int i0 = from; i0 < to; i0 += 32) {
        const int i = i0 + lane;
        const float x = i < to ? row.at(i) : -INFINITY;
        u64 s = x > edge_f || (all_ties && x == edge_f) ? weight_of(x) : 0;
        u64 n = !all_ties && x == edge_f ? 1 : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 vs = __shfl_up_sync(kFull, s, o), vn = __shfl_up_sync(kFull, n, o);
            if (lane >= o) {
                s += vs;
                n += vn;
            }
        }
        const unsigned hit = __ballot_sync(kFull, i < to && joined(before_sum + s, before_ties + n) > target);
        if (hit) {
            if (lane == 0) a.tokens[r] = begin + i0 + __ffs(hit) - 1;
            return;
        }
        before_sum += __shfl_sync(kFull, s, 31);
        before_ties += __shfl_sync(kFull, n, 31);
    }
}

template <typename T, bool FILTERS>
cudaError_t launch_typed(cudaStream_t s, Args a, int rows) {
    // A slice of at most 16 Ki logits a CTA keeps the passes over it short; beyond eight CTAs (the
    // portable cluster) slices grow, and past the shared memory they are read through L2.
    int cluster = 1;
    while (cluster < kMaxCluster && (a.V + cluster - 1) / cluster > (1 << 14)) cluster *= 2;
    a.per = ((a.V + cluster - 1) / cluster + 7) / 8 * 8;  // 16-byte chunks do not straddle slices
    const size_t slice = static_cast<size_t>(a.per) * sizeof(T);
    const size_t fixed = FILTERS ? sizeof(Shared) : offsetof(Shared, low);
    a.staged = fixed + slice <= 200 * 1024;
    const size_t smem = fixed + (a.staged ? slice : 0);
    const auto kernel = k_sample_tokens<T, FILTERS>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (e) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

cudaError_t launch_sample_tokens(cudaStream_t s, const void* logits, int dtype, int rows, int V,
                                 int64_t row_stride, const Sampling& sampling,
                                 const double* uniforms, int64_t uniform_stride, const int* step,
                                 int* tokens) {
    Args a{};
    a.logits = logits;
    a.V = V;
    a.stride = row_stride;
    a.p = sampling;
    a.uniforms = uniforms;
    a.uniform_stride = uniform_stride;
    a.step = step;
    a.tokens = tokens;
    const Sampling& p = a.p;
    const bool filters = p.top_ks || p.top_ps || p.min_ps || p.top_k > 0 || p.top_p < 1.0f || p.min_p > 0.0f;
    if (dtype == BST_DTYPE_BF16) {
        return filters ? launch_typed<__nv_bfloat16, true>(s, a, rows)
                       : launch_typed<__nv_bfloat16, false>(s, a, rows);
    }
    return filters ? launch_typed<float, true>(s, a, rows) : launch_typed<float, false>(s, a, rows);
}

}  // namespace bst
