// Eviction from a cache by the weight that its keys have gathered: each key head of a sequence that has more
// than `keep` keys keeps the first `sinks`, the last `recent`, and of the others those of the largest mass,
// ties by the lowest slot. What stays moves in order to the first slots, so that windows and sinks keep
// their meaning; masses move along.
//
// Two kernels. The first finds a head's border, the mass that the last kept key has, by counting 11, 11 and
// 10 bits of the masses' ordered bits at a time, then writes the kept slots in order. A head is one CTA, or,
// where rows are long and heads few, a cluster of up to eight that add up their counts through one
// another's shared memory. Bound by the latency of its few steps: masses are read once, into shared memory. 32
// sequences of 900 to 8192 keys of eight heads take 18 us, one of 131 000 23 (its 64 CTAs have 64 of the SMs).
// The second moves keys, values and masses: bound by memory, every kept byte is read and written once. 32 x 1024
// bf16 keys of eight heads of 128 take 50 us (5.4 TB/s).

#include <cooperative_groups.h>

#include <algorithm>

#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

namespace cg = cooperative_groups;

// Where sequence `seq` reads and writes, and how many keys it has and keeps; a row outside its cache, or one
// that an earlier sequence writes, makes it empty. By a whole CTA.
struct Route {
    int from, to, length, kept;  // to: -1 where nothing is written
};
template <int THREADS>
__device__ __forceinline__ Route route_of(const Cache& c, const Batch& b, const Eviction& e, int seq) {
    Route r;
    r.from = b.rows ? __ldg(b.rows + seq) : seq;
    r.to = e.to_rows ? __ldg(e.to_rows + seq) : seq;
    bool taken = false;
    if (e.to_rows) {
        for (int s = threadIdx.x; s < seq; s += THREADS) taken |= __ldg(e.to_rows + s) == r.to;
        taken = __syncthreads_or(taken);
    }
    if (r.to < 0 || r.to >= e.to.rows || taken) r.to = -1;
    const bool there = r.to >= 0 && r.from >= 0 && r.from < c.rows;
    r.length = there ? min(max(0, __ldg(b.lengths + seq)), c.slots) : 0;
    r.kept = min(r.length, e.keep);
    return r;
}

// ---- which keys stay ---------------------------------------------------------------------------
// Threads of a choosing CTA, more where a head has long rows and a cluster: 131 000 keys evicted down to 16 384 take
// 52 us with 512 and 49 with 1024, 32 prompts of up to 8192 keys, a CTA a head, 68 and 70.
template <int CTAS>
constexpr int kChooseThreads = CTAS > 1 ? 1024 : 512;
constexpr int kBins = 2048;
constexpr int kHeld = 40960;           // masses that a CTA's shared memory holds

// Masses in the order of whole numbers: NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (isnan(x)) return 0u;
    const uint32_t u = x == 0.0f ? 0u : __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The sum of `x` over the CTA's earlier threads.
template <int THREADS>
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t* sums, uint32_t* all) {
    constexpr int kWarps = THREADS / 32;
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
    const uint32_t mine = lane < kWarps ? sums[lane] : 0u;
    uint32_t up = mine;
#pragma unroll
    for (int o = 1; o < kWarps; o <<= 1) {
        const uint32_t y = __shfl_up_sync(kFull, up, o);
        if (lane >= o) up += y;
    }
    *all = __shfl_sync(kFull, up, kWarps - 1);
    return run - x + __shfl_sync(kFull, up - mine, warp);
}

// CTAS: of a cluster, which has one head.
template <int CTAS>
__global__ void __launch_bounds__(kChooseThreads<CTAS>)
k_evict_choose(Cache c, Batch b, Eviction e, int held) {
    constexpr int kChoose = kChooseThreads<CTAS>;
    __shared__ __align__(16) uint32_t bins[3][kBins];
    __shared__ uint32_t sums[kChoose / 32], found[2], counts[2];
    extern __shared__ float masses[];
    const int rank = CTAS > 1 ? blockIdx.x % CTAS : 0, unit = blockIdx.x / CTAS;
    const int head = unit % c.kv_heads, seq = unit / c.kv_heads;
    auto meet = [] {
        if constexpr (CTAS > 1) {
            cg::this_cluster().sync();
        } else {
            __syncthreads();
        }
    };
    const Route route = route_of<kChoose>(c, b, e, seq);
    const int length = route.length, kept = route.kept;
    int* const places = e.kept + static_cast<int64_t>(unit) * e.keep;
    if (head == 0 && rank == 0 && threadIdx.x == 0) e.lengths[seq] = kept;
    for (int i = kept + rank * kChoose + threadIdx.x; i < e.keep; i += CTAS * kChoose) places[i] = -1;
    if (length <= e.keep) {  // the same for all CTAs of the cluster
        for (int i = rank * kChoose + threadIdx.x; i < length; i += CTAS * kChoose) places[i] = i;
        return;
    }
    // The CTA's keys, [lo, hi), in runs of an odd number a thread (which meets no bank twice).
    const int run = ((length + CTAS * kChoose - 1) / (CTAS * kChoose)) | 1;
    const int lo = min(rank * run * kChoose, length), hi = lo + min(run * kChoose, length - lo);
    const float* mass = e.mass + (static_cast<int64_t>(route.from) * c.kv_heads + head) * c.slots + lo;
    for (int i = threadIdx.x; i < 3 * kBins; i += kChoose) bins[0][i] = 0u;
    __syncthreads();
    // The keys that compete: [first, last), `need` of them stay.
    const int first = e.sinks, last = length - e.recent;
    uint32_t need = e.keep - e.sinks - e.recent;
    uint32_t border = 0xffffffffu;  // ordered masses above it stay, and `need` of those equal to it
    // The upper bits are counted on the way into shared memory, or from where masses lie.
    const bool fits = run * kChoose <= held;
#pragma unroll 8
    for (int i = threadIdx.x; i < hi - lo; i += kChoose) {
        const float m = mass[i];
        if (fits) masses[i] = m;
        if (lo + i >= first && lo + i < last) atomicAdd(bins[0] + (ordered(m) >> 21), 1u);
    }
    if (fits) mass = masses;
    if (need > 0) {
        uint32_t known = 0, mask = 0;
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            constexpr int kShift[3] = {21, 10, 0};
            const int shift = pass == 0 ? kShift[0] : (pass == 1 ? kShift[1] : kShift[2]);
            const uint32_t digit = pass == 2 ? 1023u : 2047u;
            const int end = pass == 0 ? 0 : min(hi, last) - lo;
#pragma unroll 4
            for (int i = max(lo, first) - lo + threadIdx.x; i < end; i += kChoose) {
                const uint32_t u = ordered(mass[i]);
                if ((u & mask) == known) atomicAdd(bins[pass] + ((u >> shift) & digit), 1u);
            }
            meet();
            // Counts of the cluster, from the highest bin down: thread i has bins 2047 - 4 i to 2044 - 4 i, if any.
            uint4 x = {};
#pragma unroll
            for (int r = 0; r < CTAS && threadIdx.x < kBins / 4; ++r) {
                const uint32_t* of = bins[pass];
                if constexpr (CTAS > 1) of = cg::this_cluster().map_shared_rank(bins[pass], (rank + r) % CTAS);
                const uint4 y = reinterpret_cast<const uint4*>(of)[kBins / 4 - 1 - threadIdx.x];
                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            }
            const uint32_t each[4] = {x.w, x.z, x.y, x.x};
            uint32_t total;
            uint32_t before = sum_before<kChoose>(x.x + x.y + x.z + x.w, sums, &total);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < need && before + each[i] >= need) {
                    found[0] = kBins - 1 - 4 * threadIdx.x - i;
                    found[1] = before;
                }
                before += each[i];
            }
            __syncthreads();
            known |= found[0] << shift;
            mask |= digit << shift;
            need -= found[1];
        }
        border = known;
    }
    __syncthreads();
    // This thread's keys above the border (or kept anyway) and at it, then where its places begin.
    const int mine = threadIdx.x * run, n = min(run, hi - lo - mine);
    uint32_t above = 0, equal = 0;
    for (int i = 0; i < n; ++i) {
        const int key = lo + mine + i;
        const uint32_t u = ordered(mass[mine + i]);
        const bool free = key < first || key >= last;
        above += free || u > border;
        equal += !free && u == border;
    }
    uint32_t total;
    uint32_t above_before = sum_before<kChoose>(above, sums, &total);
    if (threadIdx.x == 0) counts[0] = total;
    uint32_t ties = sum_before<kChoose>(equal, sums, &total);
    if (threadIdx.x == 0) counts[1] = total;
    meet();
    if constexpr (CTAS > 1) {
        for (int r = 0; r < rank; ++r) {
            const uint32_t* of = cg::this_cluster().map_shared_rank(counts, r);
            above_before += of[0];
            ties += of[1];
        }
        meet();  // no CTA leaves while another reads its counts
    }
    uint32_t place = above_before + min(ties, need);
    for (int i = 0; i < n; ++i) {
        const int key = lo + mine + i;
        const uint32_t u = ordered(mass[mine + i]);
        bool stays = key < first || key >= last || u > border;
        if (!stays && u == border) stays = ties++ < need;
        if (stays) places[place++] = key;
    }
}

// ---- what stays moves --------------------------------------------------------------------------
constexpr int kMove = 256;
constexpr int kUnits = 8;   // units a thread holds at a time

// Rows [i0, i1) of `to` become rows places[i] of `from`: 1 << units columns from u0 on of rows of 1 << pitch
// units of type U. The CTA reads a run of rows before it writes it, in order: rows move to lower places only,
// so `to` may be `from`.
template <typename U, bool IN_PLACE>
__device__ __forceinline__ void move_rows(const void* from_, void* to_, const int* places, int i0, int i1,
                                          int pitch, int u0, int units) {
    const U* const from = static_cast<const U*>(from_) + u0;
    U* const to = static_cast<U*>(to_) + u0;
    const int run = kMove * kUnits >> units;  // rows at a time
    for (int i = i0; i < i1; i += run) {
        U x[kUnits];
        int place[kUnits];
        const int count = min(run, i1 - i) << units;
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int at = threadIdx.x + k * kMove;
            place[k] = at < count ? places[i + (at >> units)] : 0;
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int at = threadIdx.x + k * kMove;
            if (at < count) x[k] = __ldcs(from + (static_cast<int64_t>(place[k]) << pitch) + (at & ((1 << units) - 1)));
        }
        if (IN_PLACE) __syncthreads();
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int at = threadIdx.x + k * kMove;
            if (at < count) to[(static_cast<int64_t>(i + (at >> units)) << pitch) + (at & ((1 << units) - 1))] = x[k];
        }
        if (IN_PLACE) __syncthreads();
    }
}

// A CTA's share of a head's keys (blockIdx.y 0) or values: `rows` of those that are kept, or, in place, 64 bytes
// of each of them. Rows are 1 << row_units units of 16 bytes, their scales 1 << scale_units of 4 (none: -1).
template <bool IN_PLACE>
__global__ void __launch_bounds__(kMove)
k_evict_move(Cache c, Batch b, Eviction e, int row_units, int scale_units, int rows, int shares) {
    const int share = blockIdx.x % shares, unit = blockIdx.x / shares;
    const int head = unit % c.kv_heads, seq = unit / c.kv_heads;
    const bool of_values = blockIdx.y;
    pdl_wait();
    const int kept = e.lengths[seq];
    const int* const places = e.kept + static_cast<int64_t>(unit) * e.keep;
    const int from_row = b.rows ? b.rows[seq] : seq, to_row = e.to_rows ? e.to_rows[seq] : seq;
    // Without keys the row may be none, or another sequence's.
    if (kept == 0 && route_of<kMove>(c, b, e, seq).to < 0) return;
    const int64_t from = (static_cast<int64_t>(from_row) * c.kv_heads + head) * c.slots;
    const int64_t to = (static_cast<int64_t>(to_row) * c.kv_heads + head) * e.to.slots;
    int i0 = IN_PLACE ? 0 : share * rows, i1 = IN_PLACE ? kept : min(kept, i0 + rows);
    if (IN_PLACE) {
        // Keys before the first one that went stay where they are.
        for (int hi = kept; i0 < hi;) {
            const int mid = i0 + ((hi - i0) >> 1);
            if (places[mid] == mid) {
                i0 = mid + 1;
            } else {
                hi = mid;
            }
        }
    }
    const int units = IN_PLACE ? min(row_units, 2) : row_units, u0 = IN_PLACE ? share << units : 0;
    auto at = [](void* p, int64_t row, int shift) { return static_cast<char*>(p) + (row << shift); };
    move_rows<uint4, IN_PLACE>(at(of_values ? c.v : c.k, from, row_units + 4),
                               at(of_values ? e.to.v : e.to.k, to, row_units + 4), places, i0, i1, row_units, u0,
                               units);
    const bool first = !IN_PLACE || share == 0;
    if (scale_units >= 0 && first) {
        move_rows<uint32_t, IN_PLACE>(at(of_values ? c.v_scale : c.k_scale, from, scale_units + 2),
                                      at(of_values ? e.to.v_scale : e.to.k_scale, to, scale_units + 2), places, i0,
                                      i1, scale_units, 0, scale_units);
    }
    if (of_values || !first) return;
    // In place too masses may go to another array, and then those of the keys that stay as well.
    const int m0 = IN_PLACE && e.to_mass != e.mass ? 0 : i0;
    move_rows<float, IN_PLACE>(e.mass + from, e.to_mass + to, places, m0, i1, 0, 0, 0);
    const int64_t step = IN_PLACE ? kMove : static_cast<int64_t>(shares) * kMove;
    for (int64_t i = kept + (IN_PLACE ? 0 : static_cast<int64_t>(share) * kMove) + threadIdx.x; i < e.to.slots; i += step) {
        e.to_mass[to + i] = 0.0f;
    }
}

template <int CTAS>
cudaError_t choose(cudaStream_t s, const Cache& c, const Batch& b, const Eviction& e) {
    constexpr int kChoose = kChooseThreads<CTAS>;
    const int run = ((c.slots + CTAS * kChoose - 1) / (CTAS * kChoose)) | 1;
    const int held = static_cast<int64_t>(run) * kChoose <= kHeld ? run * kChoose : 0;
    if (held > 4096) {  // beside 24 KB of counts, more than a kernel has by itself
        // The limit is the kernel's, not the call's, so it is the same for all: one thread's call could lower it between
        // another's and its launch.
        const cudaError_t err = cudaFuncSetAttribute(k_evict_choose<CTAS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeld * 4);
        if (err) return err;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(c.kv_heads) * b.count * CTAS));
    cfg.blockDim = dim3(kChoose);
    cfg.dynamicSmemBytes = held * 4;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CTAS > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_evict_choose<CTAS>, c, b, e, held);
}

// CTAs a head, so that long rows get several and many heads leave one another the card (a cluster of eight with 1024
// threads each has an SM a CTA, and twelve such clusters fit). Calls of 1, 64 and 256 heads with one, two, four and eight
// CTAs each (us): 8192 slots 16 15 16 18, 16 16 23 75, 27 44 74 253; 16 384 slots 23 18 19 21, 26 21 29 83, 47 62 96 286;
// 40 000 slots 40 25 22 22, 50 35 45 100, 137 126 156 368; 131 072 slots 207 77 35 29, 270 126 107 164, 691 453 443 610.
int ctas_of(int64_t heads, int slots) {
    if (slots > 40960 && heads <= 12) return 8;
    if (slots > 16384 && heads <= 32) return 4;
    if (slots > 98304) return 4;
    // Fewer heads than a wave, or masses that one CTA could hardly keep in shared memory.
    return (slots > 8192 && heads <= 64) || slots > 32768 ? 2 : 1;
}

int log2_of(int x) {
    int n = 0;
    while (x >>= 1) ++n;
    return n;
}

}  // namespace

cudaError_t launch_kv_evict(cudaStream_t s, const Cache& c, const Batch& b, const Eviction& e) {
    if (b.count < 1) return cudaSuccess;
    const int ctas = ctas_of(static_cast<int64_t>(c.kv_heads) * b.count, c.slots);
    const cudaError_t err = ctas == 1   ? choose<1>(s, c, b, e)
                            : ctas == 2 ? choose<2>(s, c, b, e)
                            : ctas == 4 ? choose<4>(s, c, b, e)
                                        : choose<8>(s, c, b, e);
    if (err) return err;
    const bool u4 = c.storage == BST_DTYPE_U4, in_place = e.to.k == c.k;
    const int row_bytes = u4 ? c.head_dim / 2 : c.head_dim * (c.storage == BST_DTYPE_BF16 ? 2 : 4);
    // 32 KB a CTA; in place, 64 bytes of every row.
    const int rows = (32 << 10) / row_bytes;
    const int shares = in_place ? std::max(1, row_bytes / 64) : (e.keep + rows - 1) / rows;
    const int64_t blocks = static_cast<int64_t>(shares) * c.kv_heads * b.count;
    return launch_pdl(in_place ? k_evict_move<true> : k_evict_move<false>, dim3(static_cast<unsigned>(blocks), 2),
                      dim3(kMove), 0, s, c, b, e, log2_of(row_bytes / 16), u4 ? log2_of(c.head_dim / 32) : -1, rows,
                      shares);
}

}  // namespace bst
