// Drawing tokens from filtered distributions: temperature, top-k, top-p, min-p.
//
// With z = (logit - largest) / temperature the weight of a token is exp(z), held as a 64-bit whole
// number of units of 2^-42 (so 2^20 tokens cannot overflow it). Sums of whole numbers do not depend
// on their order: any number of threads may add in any order, with atomics, and a draw still comes
// out the same. Weights below 2^-40 count as nothing.
//
// No sort. All filters keep a prefix of the order (logit descending, index ascending), so each is a
// threshold: the smallest logit kept and how many of the tokens with exactly that logit. A threshold
// is found by histograms of 2048 bins: the first over the distance from the largest logit (spreads
// the tokens evenly, where bits of the float would pile them on a few bins), then over the bits of
// the logits inside the bin where the sum crosses, until a bin is one value. The draw itself is a
// running sum over slices of the row, then inside one slice.
//
// A row is worked on by a cluster of CTAs, each with a slice of the row in its shared memory; sums
// and histograms meet through distributed shared memory.

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>

#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kCoarse = 64;                  // bins / kCoarse = 32 bins, a lane each
constexpr int kMaxCluster = 8;
constexpr double kUnit = 4398046511104.0;    // 2^42 units in the largest weight
constexpr double kCut = -27.725887222397812; // ln 2^-40
using u64 = unsigned long long;

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

struct Shared {
    u64 bins[kBins];
    u64 coarse[kCoarse];
    u64 exchange[2][2];     // this CTA's value of a reduction over the cluster, two pairs in turn
    u64 warp_a[kWarps], warp_b[kWarps];
    u64 result[4];
};

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
            u64 x = lane < kWarps ? sh.warp_a[lane] : 0, y = lane < kWarps ? sh.warp_b[lane] : 0;
            x = MAX ? warp_max_u(x) : warp_sum_u(x);
            y = MAX ? warp_max_u(y) : warp_sum_u(y);
            if (lane == 0) {
                sh.exchange[turn][0] = x;
                sh.exchange[turn][1] = y;
            }
        }
        cluster.sync();
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
    uint32_t key;  // the smallest key kept; 0: everything
    u64 above;     // the sum over larger keys
    u64 total;     // the sum over this key's tokens
};

// The key at which the sum of weight(key), over the tokens with key >= least, reaches target (which
// must be between 1 and their whole sum). extra is a sum that belongs to the key extra_key (tokens
// that weight() leaves out there).
template <typename T, typename W>
__device__ Threshold find_threshold(Row<T>& row, uint32_t top, uint32_t least, u64 target,
                                    uint32_t extra_key, u64 extra, W&& weight) {
    Shared& sh = row.sh;
    const float largest = float_of(top);
    const float span = largest - float_of(least);
    // Distance bins first, unless they could not tell anything apart (an infinite span, one key).
    bool by_distance = span > 0.0f && span < FLT_MAX;
    const float per = by_distance ? static_cast<float>(kBins) / span : 0.0f;
    uint32_t lo = least, hi = top;
    u64 above = 0;
    while (true) {
        int shift = 0;
        while (((hi - lo) >> shift) >= kBins) ++shift;
        if (shift == 0) by_distance = false;  // a bin is one key already
        auto bin_of = [&](uint32_t key) {
            return by_distance ? min(kBins - 1, static_cast<int>((largest - float_of(key)) * per))
                               : static_cast<int>((hi - key) >> shift);
        };
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < row.count; i += kThreads) {
            const uint32_t key = key_of(row.at(i));
            if (key < lo || key > hi) continue;
            const u64 w = weight(key);
            if (w) atomicAdd(&sh.bins[bin_of(key)], w);
        }
        if (extra && row.rank == 0 && threadIdx.x == 0 && extra_key >= lo && extra_key <= hi) {
            atomicAdd(&sh.bins[bin_of(extra_key)], extra);
        }
        __syncthreads();
        for (int i = threadIdx.x >> 5; i < kCoarse; i += kWarps) {
            const u64 v = warp_sum_u(sh.bins[i * 32 + (threadIdx.x & 31)]);
            if ((threadIdx.x & 31) == 0) sh.coarse[i] = v;
        }
        row.cluster.sync();
        // The first coarse bin, then the first bin, where the sum from above reaches the target.
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
                fine += row.cluster.map_shared_rank(sh.bins, r)[coarse * 32 + lane];
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
        row.cluster.sync();  // every CTA has read the others' bins
        const int bin = static_cast<int>(sh.result[0]);
        above = sh.result[1];
        const u64 total = sh.result[2];
        if (!by_distance && shift == 0) {
            return Threshold{hi - static_cast<uint32_t>(bin), above, total};
        }
        if (by_distance) {
            // The keys that fell into the bin, as a range.
            u64 high = 0, low = 0;  // low as its complement, so that both are maxima
            for (int i = threadIdx.x; i < row.count; i += kThreads) {
                const uint32_t key = key_of(row.at(i));
                if (key < lo || key > hi || bin_of(key) != bin) continue;
                high = max(high, static_cast<u64>(key));
                low = max(low, static_cast<u64>(~key));
            }
            row.template reduce<true>(high, low);
            hi = static_cast<uint32_t>(high);
            lo = ~static_cast<uint32_t>(low);
            by_distance = false;
        } else {
            const uint32_t new_hi = hi - (static_cast<uint32_t>(bin) << shift);
            const uint32_t width = (1u << shift) - 1u;
            lo = new_hi - lo > width ? new_hi - width : lo;
            hi = new_hi;
        }
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

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample_tokens(Args a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem);
    T* staged = reinterpret_cast<T*>(smem + sizeof(Shared));
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = static_cast<int>(cluster.num_blocks());
    const int rank = static_cast<int>(cluster.block_rank());
    const int r = blockIdx.x / ranks;
    const int begin = min(a.V, rank * a.per), end = min(a.V, begin + a.per);
    const T* global = static_cast<const T*>(a.logits) + r * a.stride + begin;
    Row<T> row{sh, cluster, ranks, rank, a.staged ? staged : global, begin, end - begin};

    const float temperature = a.p.temperatures ? a.p.temperatures[r] : a.p.temperature;
    const float top_p = a.p.top_ps ? a.p.top_ps[r] : a.p.top_p;
    const float min_p = a.p.min_ps ? a.p.min_ps[r] : a.p.min_p;
    const int top_k = a.p.top_ks ? a.p.top_ks[r] : a.p.top_k;

    // The largest logit and its first index: the maximum of (key, V - index).
    u64 best = 0, unused = 0;
    for (int i = threadIdx.x; i < row.count; i += kThreads) {
        const T x = global[i];
        if (a.staged) staged[i] = x;
        const u64 v = (static_cast<u64>(key_of(to_f(x))) << 32) |
                      static_cast<uint32_t>(a.V - (begin + i));
        best = max(best, v);
    }
    row.template reduce<true>(best, unused);
    const uint32_t top = static_cast<uint32_t>(best >> 32);
    const float largest = float_of(top);
    const int first = a.V - static_cast<int>(best & 0xffffffffu);
    if (largest == -INFINITY || !(temperature > 0.0f)) {
        if (rank == 0 && threadIdx.x == 0) a.tokens[r] = largest == -INFINITY ? -1 : first;
        cluster.sync();  // the exchange slots are read by others until here
        return;
    }

    const double T_ = temperature, top_d = largest;
    auto real_weight = [&](uint32_t key) -> double {
        if (key == top) return 1.0;
        const double z = (static_cast<double>(float_of(key)) - top_d) / T_;
        return z >= kCut ? exp(z) : 0.0;
    };
    auto weight = [&](uint32_t key) -> u64 {
        return static_cast<u64>(__double2ll_rn(real_weight(key) * kUnit));
    };
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

    // Kept: keys above `edge` and the first `ties` tokens, by index, with exactly that key.
    uint32_t edge = 0;
    u64 ties = 0;
    if (top_k > 0 && top_k < a.V) {
        u64 n = 0;
        for (int i = threadIdx.x; i < row.count; i += kThreads) n += key_of(row.at(i)) >= least;
        unused = 0;
        row.template reduce<false>(n, unused);
        if (n > static_cast<u64>(top_k)) {
            const Threshold t = find_threshold(row, top, least, static_cast<u64>(top_k), 0u, 0ull,
                                               [](uint32_t) -> u64 { return 1; });
            edge = t.key;
            ties = static_cast<u64>(top_k) - t.above;
        }
    }
    if (top_p < 1.0f) {
        u64 sum = 0;
        unused = 0;
        const uint32_t from = max(least, edge + (edge ? 1u : 0u));
        for (int i = threadIdx.x; i < row.count; i += kThreads) {
            const uint32_t key = key_of(row.at(i));
            if (key >= from) sum += weight(key);
        }
        row.template reduce<false>(sum, unused);
        const u64 tied = edge ? ties * weight(edge) : 0;
        sum += tied;
        const double want = static_cast<double>(top_p) * static_cast<double>(sum);
        // The fewest tokens whose sum is at least want: the sum has to reach ceil(want), at least 1.
        const u64 target = want > 0.0 ? min(sum, static_cast<u64>(ceil(want))) : 0;
        if (target <= 1) {
            edge = top;
            ties = 1;
        } else {
            const Threshold t = find_threshold(row, top, edge ? edge : least, target, edge, tied,
                                               [&](uint32_t key) -> u64 {
                                                   return key >= from ? weight(key) : 0;
                                               });
            const u64 w = weight(t.key);
            u64 need = (target - t.above + w - 1) / w;
            if (t.key == edge) need = min(need, ties);
            edge = t.key;
            ties = need;
        }
    }
    if (!(min_p <= 0.0f) && !isnan(min_p)) {
        // The smallest key with a weight of at least min_p; all of its tokens are kept.
        const double floor_w = fmin(static_cast<double>(min_p), 1.0);
        if (threadIdx.x < 32) {
            uint32_t low = top;
            if (!isinf(largest) && floor_w < 1.0) {
                const float guess = static_cast<float>(
                    fmax(top_d + log(floor_w) * T_, -static_cast<double>(FLT_MAX)));
                low = smallest_key(least, top, max(least, min(top, key_of(guess))),
                                   [&](uint32_t key) { return real_weight(key) >= floor_w; });
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
    auto count_range = [&](int from, int to, u64* sum, u64* tied) {  // one warp, [from, to)
        u64 s = 0, n = 0;
        for (int i = from + (threadIdx.x & 31); i < to; i += 32) {
            const uint32_t key = key_of(row.at(i));
            if (key > edge) {
                s += weight(key);
            } else if (key == edge) {
                ++n;
            }
        }
        *sum = warp_sum_u(s);
        *tied = warp_sum_u(n);
    };
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = (row.count + kWarps - 1) / kWarps;
    const int w0 = min(row.count, warp * part), w1 = min(row.count, w0 + part);
    u64 my_sum, my_ties;
    count_range(w0, w1, &my_sum, &my_ties);
    // Lane 0 alone carries the warp's sums into the reduction.
    u64 sum = lane == 0 ? my_sum : 0, tied = lane == 0 ? my_ties : 0;
    row.template reduce<false>(sum, tied);
    const u64 whole = joined(sum, tied);
    double u = a.uniforms[r * a.uniform_stride + (a.step ? *a.step : 0)];
    u = u >= 0.0 ? u : 0.0;  // NaN too
    u64 target = static_cast<u64>(fmin(u, 1.0) * static_cast<double>(whole));
    target = min(target, whole - 1);
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
    cluster.sync();  // the last access to other CTAs' memory
    if (!mine) return;
    // Twice: the sums of the warps' parts pick one, and its elements become the next parts.
    int from = 0, to = row.count;
    for (int round = 0; round < 2; ++round) {
        const int step = (to - from + kWarps - 1) / kWarps;
        const int p0 = min(to, from + warp * step), p1 = min(to, p0 + step);
        if (round > 0) count_range(p0, p1, &my_sum, &my_ties);
        __syncthreads();
        if (lane == 0) {
            sh.warp_a[warp] = my_sum;
            sh.warp_b[warp] = my_ties;
        }
        __syncthreads();
        int pick = 0;
        for (; pick < kWarps - 1; ++pick) {
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
        const uint32_t key = i < to ? key_of(row.at(i)) : 0u;
        u64 s = i < to && key > edge ? weight(key) : 0, n = i < to && key == edge ? 1 : 0;
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

template <typename T>
cudaError_t launch_typed(cudaStream_t s, Args a, int rows) {
    // A slice of at most 16 Ki logits a CTA keeps the passes over it short; beyond eight CTAs (the
    // portable cluster) slices grow, and past the shared memory they are read through L2.
    int cluster = 1;
    while (cluster < kMaxCluster && (a.V + cluster - 1) / cluster > (1 << 14)) cluster *= 2;
    a.per = (a.V + cluster - 1) / cluster;
    const size_t slice = static_cast<size_t>(a.per) * sizeof(T);
    a.staged = sizeof(Shared) + slice <= 200 * 1024;
    const size_t smem = sizeof(Shared) + (a.staged ? slice : 0);
    cudaError_t e = cudaFuncSetAttribute(k_sample_tokens<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         200 * 1024);
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
    return cudaLaunchKernelEx(&cfg, k_sample_tokens<T>, a);
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
    return dtype == BST_DTYPE_BF16 ? launch_typed<__nv_bfloat16>(s, a, rows)
                                   : launch_typed<float>(s, a, rows);
}

}  // namespace bst
