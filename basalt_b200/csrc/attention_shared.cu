// Attention for a batch that shares a long prefix: every query sees the keys of one common row of a cache
// besides those of its own sequence's row.
//
//   out_i = sum_x exp(s_ix - m_i) v_x / sum_x exp(s_ix - m_i),  x over the prefix and the own keys
//
// Sums over disjoint sets of keys join exactly (each set leaves its maximum, its sum of weights and its
// weighted values), so the prefix is a pass of its own: its queries are those of the whole batch, a tile of
// them reads it once, where attention over a copy in every row would read it once a sequence. The own keys
// are the pass of attention_cached, which runs beside the first as far as that leaves room, and one kernel
// joins both passes' splits.

#include "attention_cached.cuh"

namespace bst {
namespace {

struct Plan {
    int rows, tiles, splits;  // query rows a tile, tiles, splits of the keys
};

// On mma.sync, 8 or 16 query rows a tile.
Plan plan_small(const Batch& b, const AttnSpec& a, const Prefix& p) {
    Plan plan{8, 0, 1};
    const int64_t queries = static_cast<int64_t>(b.tokens) * (a.heads / a.kv_heads);
    if (a.dtype == BST_DTYPE_BF16 && queries > 8) plan.rows = 16;
    plan.tiles = static_cast<int>((queries + plan.rows - 1) / plan.rows);
    const int64_t units = static_cast<int64_t>(plan.tiles) * a.kv_heads;
    const int64_t fill = 148 * ctas_per_sm(p.cache) / units;
    plan.splits = static_cast<int>(
        std::max<int64_t>(1, std::min<int64_t>({fill, p.length / 128, static_cast<int64_t>(kMaxSplits)})));
    return plan;
}

// On tcgen05, 256 rows a tile and a CTA an SM: the split with the least waves x (tiles of 64 keys a CTA and
// what a CTA costs besides, in such tiles).
constexpr int kCost = 6, kMostShares = 64;
Plan plan_large(const Batch& b, const AttnSpec& a, const Prefix& p) {
    Plan plan{256, prefix_tc_tiles(b, a), 1};
    const int64_t units = static_cast<int64_t>(plan.tiles) * a.kv_heads, keys = (p.length + 63) / 64;
    int64_t best = 0;
    for (int splits = 1; splits <= std::min<int64_t>(kMostShares, keys); ++splits) {
        const int64_t time = (units * splits + 147) / 148 * ((keys + splits - 1) / splits + kCost);
        if (splits == 1 || time < best) {
            best = time;
            plan.splits = splits;
        }
    }
    return plan;
}

// Rows of a key head from which on tcgen05's tiles of 128 pay, however few of them are filled. Whole calls with own keys
// of 10 to 120, eight key heads, tcgen05 and mma.sync (us).
// bf16 of 128 channels: behind 500 keys 9.8 and 10.6 with 8 rows, 10.2 and 13.1 with 12; behind 4000 14.5 and 17.5, 14.9
// and 20.6; behind 30 000 33.9 and 34.4, 33.9 and 38.5. Of 64 channels: behind 4000 keys 13.7 and 18.6 with 12 rows, behind
// 16 000 21.2 and 21.2; but where every SM has more than 1000 keys, one CTA's chain of tiles takes longer than four small
// CTAs beside one another: behind 30 000 29.6 and 24.0 with 12, 31.3 and 29.1 with 32, 33.1 and 38.9 with 48 (six key heads 28.5 and 30.0 with
// 40; two heads behind 120 000, whose small CTAs leave too many splits to join, 32.1 and 35.2 with 12).
// 4 bits, which take longer to unpack for tcgen05: of 128 channels behind 500 keys 17.9 and 16.9 with 32 rows, 18.6 and 18.4
// with 64, 18.9 and 20.8 with 96; behind 1500 20.5 and 20.1, 20.5 and 21.1 with 40; behind 16 000 40.3 and 38.6, 40.7 and
// 45.0 with 48; behind 30 000 (four heads) 40.0 and 38.2, 40.0 and 42.5. Of 64 behind 1000 16.2 and 12.2, 17.7 and 14.1 with
// 64, 21.0 and 15.4 with 96; behind 30 000 42.7 and 35.5, 42.7 and 49.0 with 48.
constexpr int kLargeRows = 12, kLargeRowsLong = 40, kLongKeys = 148 * 1024;
constexpr int kLargeCodeRows = 40, kLargeCodeRowsShort = 96, kShortKeys = 1280;
bool large(const Batch& b, const AttnSpec& a, const Prefix& p) {
    const int64_t rows = static_cast<int64_t>(b.tokens) * (a.heads / a.kv_heads);
    int least = kLargeRows;
    if (p.cache.storage == BST_DTYPE_U4) {
        least = p.length < kShortKeys ? kLargeCodeRowsShort : kLargeCodeRows;
    } else if (a.head_dim == 64 && a.kv_heads >= 4 && static_cast<int64_t>(p.length) * a.kv_heads >= kLongKeys) {
        least = kLargeRowsLong;
    }
    return prefix_tc_takes(p, a) && rows >= least;
}

// Splits of the own keys: no more than fill the card (spreading 64 rows of 20 to 1000 keys over four waves took
// 64 us where this takes 62, 24 x 4 drafts 93 instead of 88).
int own_splits(const Cache& c, const Batch& b, const AttnSpec& a) {
    return split_count(c, b, a, plain_query(c, b, a) ? plain_per_sm(a) : 0);
}

size_t part_bytes(const Batch& b, const AttnSpec& a, int splits) {
    return static_cast<size_t>(b.tokens) * a.heads * splits * (a.head_dim + 2) * sizeof(float);
}

// A CTA a query; or, for at most 32 splits in all, a warp for 32 channels of one. Bound by the latency of L2 and of
// the hand-over between kernels: 2048 queries of 128 channels and 18 splits take 11 us (1.7 TB/s), 8192 of six 20.
template <typename T, int HD, bool WARP>
__global__ void __launch_bounds__(kThreads)
k_shared_join(Cache c, Batch b, AttnSpec a, int tile_rows, T* __restrict__ out, int64_t out_stride,
              int own_splits, const float* __restrict__ own, int prefix_splits,
              const float* __restrict__ prefix) {
    const uint32_t unit = WARP ? blockIdx.x * kWarps + (threadIdx.x >> 5) : blockIdx.x;
    const uint32_t query = WARP ? unit / (HD / 32) : unit;
    const int token = query / static_cast<uint32_t>(a.heads), head = query - static_cast<uint32_t>(token) * a.heads;
    int seq, first, n;
    if (token >= b.tokens || !find_sequence(b, token, &seq, &first, &n)) {
        pdl_wait();  // every CTA does: this kernel's end is that of all three
        return;
    }
    const int use = used_splits(c, b, a, tile_rows, own_splits, seq, token - first, n, head);
    pdl_wait();
    const float* const mine = own + static_cast<int64_t>(query) * own_splits * (HD + 2);
    const float* const common = prefix + static_cast<int64_t>(query) * prefix_splits * (HD + 2);
    auto at = [&](int s) { return s < use ? mine + s * (HD + 2) : common + (s - use) * (HD + 2); };
    T* const to = out + token * out_stride + head * HD;
    if constexpr (WARP) {
        join_by_warp<T, HD>(use + prefix_splits, at, to, unit % (HD / 32));
    } else {
        join_splits<2 * kMaxSplits, T, HD>(use + prefix_splits, at, to);
    }
}

}  // namespace

size_t attention_shared_workspace(const Cache& c, const Batch& b, const AttnSpec& a, const Prefix& p) {
    if (b.tokens < 1) return 0;
    int splits = p.length > 0 ? plan_small(b, a, p).splits : 0;
    if (p.length > 0 && large(b, a, p)) splits = std::max(splits, plan_large(b, a, p).splits);
    return part_bytes(b, a, own_splits(c, b, a) + splits);
}

cudaError_t launch_attention_shared(cudaStream_t s, const Cache& c, const Batch& b, const AttnSpec& a,
                                    const Prefix& p, const void* q, int64_t q_stride, void* out,
                                    int64_t out_stride, void* workspace) {
    if (b.tokens < 1 || b.count < 1) return cudaSuccess;
    const int own_count = own_splits(c, b, a), rows = rows_of_tile(b, a);
    float* const own = static_cast<float*>(workspace);
    float* const prefix = own + part_bytes(b, a, own_count) / sizeof(float);
    int splits = 0;
    if (p.length > 0) {
        cudaError_t e;
        if (large(b, a, p) && reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride % 8 == 0) {
            const Plan of = plan_large(b, a, p);
            splits = of.splits;
            e = launch_prefix_tc(s, p, b, a, q, q_stride, of.tiles, splits, prefix);
        } else {
            const Plan of = plan_small(b, a, p);
            splits = of.splits;
            Extra extra;
            extra.row = p.row;
            extra.length = p.length;
            e = run_cached<kPrefix>(s, p.cache, b, a, q, q_stride, nullptr, 0, of.tiles, of.rows, splits, prefix,
                                    extra);
        }
        if (e) return e;
    }
    Extra beside;
    beside.early = splits > 0;
    const cudaError_t e = run_cached<kBeside>(s, c, b, a, q, q_stride, nullptr, 0, tile_bound(b, a, rows), rows,
                                              own_count, own, beside);
    if (e) return e;
    return by_dtype(a.dtype, [&](auto type) {
        using T = decltype(type);
        return by_head_dim(a.head_dim, [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            const int64_t queries = static_cast<int64_t>(b.tokens) * a.heads;
            const bool warp = own_count + splits <= 32;
            return launch_pdl(warp ? k_shared_join<T, HD, true> : k_shared_join<T, HD, false>,
                              dim3(static_cast<unsigned>(warp ? (queries * (HD / 32) + kWarps - 1) / kWarps : queries)),
                              dim3(kThreads), 0, s, c, b, a, rows, static_cast<T*>(out), out_stride, own_count,
                              static_cast<const float*>(own), splits, static_cast<const float*>(prefix));
        });
    });
}

}  // namespace bst
