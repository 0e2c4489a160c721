// Attention over a cache that also adds up the weight each key receives:
//
//   mass'_j = decay mass_j + sum over the sequence's queries i and the key head's query heads of p_ij,
//   p_ij = exp(s_ij - max s_i) / sum exp(s_ij - max s_i)
//
// A weight is known only when all of a query's scores are, so the pass over the cache keeps every score
// (4 bytes a query and key, where reading the keys again takes 80 to 512 a key) and a second kernel joins
// the splits and turns scores into weights. Its CTAs own keys: each adds the weights of all queries to a key
// in the order of the queries, so that results do not depend on how CTAs are scheduled.

#include "attention_cached.cuh"

namespace bst {
namespace {

constexpr int kMassKeys = 4 * kThreads;   // keys of a CTA at a time: four next to one another a thread
constexpr int kMassRows = 64;             // query rows whose maxima and sums are held at a time

// Whether the batch's sequence `seq` is the first that names its row, and the next one that names the same.
// (A row that is named twice gets the weights of both.)
__device__ __forceinline__ bool first_of_row(const Batch& b, int seq, int row) {
    if (!b.rows) return true;
    bool before = false;
    for (int s = threadIdx.x; s < seq; s += kThreads) before |= __ldg(b.rows + s) == row;
    return !__syncthreads_or(before);
}
__device__ __forceinline__ int next_of_row(const Batch& b, int seq, int row) {
    if (!b.rows) return b.count;
    __shared__ int next;
    __syncthreads();
    if (threadIdx.x == 0) next = b.count;
    __syncthreads();
    for (int s0 = seq + 1; s0 < b.count; s0 += kThreads) {
        const int s = s0 + threadIdx.x;
        const bool hit = s < b.count && __ldg(b.rows + s) == row;
        if (hit) atomicMin(&next, s);
        if (__syncthreads_or(hit)) break;
    }
    return next;
}

// A split's maximum and sum into those of the splits before. One that saw nothing has nothing to add; one whose
// scores are NaN has.
__device__ __forceinline__ void add_split(float* m, float* total, float top, float sum) {
    const float most = fmaxf(*m, top);
    auto scaled = [&](float x, float at) { return at == -INFINITY ? (x == 0.0f ? 0.0f : x) : x * exp2_fast(at - most); };
    *total = scaled(*total, *m) + scaled(sum, top);
    *m = most;
}

// Maxima and sums of query rows r0 .. r0 + rows - 1 of a sequence and key head, by the CTA: as many lanes a row as
// there are to spare.
template <int HD>
__device__ __forceinline__ void row_sums(const Cache& c, const AttnSpec& a, int tile_rows, int splits,
                                         const float* part, int row, int length, int first, int n, int kvh, int r0,
                                         int rows, float* tops, float* inverse) {
    const int group = a.heads / a.kv_heads, lane = threadIdx.x & 31;
    int lanes = 32;
    while (lanes > 1 && rows * lanes > kThreads) lanes >>= 1;
    const int of_warp = 32 / lanes;  // a warp takes that many rows at a time
    __syncthreads();
    for (int r = threadIdx.x / lanes; r < (rows + of_warp - 1) / of_warp * of_warp; r += kThreads / lanes) {
        float m = -INFINITY, total = 0.0f;
        if (r < rows) {
            const int token = (r0 + r) / group, head = kvh * group + (r0 + r) - token * group;
            const int use = used_splits(c, a, tile_rows, splits, row, length, token, n, head);
            const float* from = part + (static_cast<int64_t>(first + token) * a.heads + head) * splits * (HD + 2) + HD;
#pragma unroll 4
            for (int s = lane % lanes; s < use; s += lanes) {
                const float2 y = *reinterpret_cast<const float2*>(from + s * (HD + 2));
                add_split(&m, &total, y.x, y.y);
            }
        }
        for (int o = lanes / 2; o > 0; o >>= 1) {
            const float other = __shfl_xor_sync(kFull, m, o), others = __shfl_xor_sync(kFull, total, o);
            add_split(&m, &total, other, others);
        }
        if (r < rows && lane % lanes == 0) {
            tops[r] = m == -INFINITY ? 0.0f : m;
            inverse[r] = total == 0.0f ? 0.0f : 1.0f / total;
        }
    }
    __syncthreads();
}

// Joins splits, and turns scores into weights: 64 sequences of 500 to 8192 keys with 32 query heads take 15 us (36 MB
// of scores, 18 of masses: 3.5 TB/s), eight of 1000 to 16 384 with 16 tokens each 31 (127 MB). Bound by how many scores
// are under way: a thread's four rows of four keys, and the four after them.
template <typename T, int HD, bool WARP>
__global__ void __launch_bounds__(kThreads)
k_weights_join(Cache c, Batch b, AttnSpec a, int tile_rows, T* __restrict__ out, int64_t out_stride,
               int splits, const float* __restrict__ part, const float* __restrict__ scores, int64_t pitch,
               const float* previous, float decay, float* mass, int joins, int per) {
    // The last CTAs join: short ones, which fill up what the others leave (first, they took a batch from 210 to 214 us).
    const uint32_t weights = gridDim.x - joins;
    if (blockIdx.x >= weights) {
        const uint32_t block = blockIdx.x - weights;
        const uint32_t unit = WARP ? block * kWarps + (threadIdx.x >> 5) : block;
        const uint32_t query = WARP ? unit / (HD / 32) : unit;
        const int token = query / static_cast<uint32_t>(a.heads), head = query - static_cast<uint32_t>(token) * a.heads;
        int seq, first, n;
        if (token >= b.tokens || !find_sequence(b, token, &seq, &first, &n)) {
            pdl_wait();  // every CTA does: this kernel's end is that of the pass before it
            return;
        }
        const int use = used_splits(c, b, a, tile_rows, splits, seq, token - first, n, head);
        pdl_wait();
        const float* const from = part + static_cast<int64_t>(query) * splits * (HD + 2);
        auto at = [&](int s) { return from + s * (HD + 2); };
        T* const to = out + token * out_stride + head * HD;
        if constexpr (WARP) {
            join_by_warp<T, HD>(use, at, to, unit % (HD / 32));
        } else {
            join_splits<kMaxSplits, T, HD>(use, at, to);
        }
        return;
    }
    __shared__ __align__(16) float tops[kMassRows], inverse[kMassRows];
    // In 32 bits: the quotients of 64 took a third of all instructions. A CTA has `per` chunks of keys.
    const int span = per * kMassKeys;
    const uint32_t shares = 1 + (c.slots - 1) / span, place = blockIdx.x;  // slots and a span may pass 2^31
    const uint32_t of_head = place / shares;
    const int begin = static_cast<int>(place - of_head * shares) * span;
    const int first_seq = of_head / static_cast<uint32_t>(a.kv_heads);
    const int kvh = of_head - static_cast<uint32_t>(first_seq) * a.kv_heads;
    const int row = b.rows ? __ldg(b.rows + first_seq) : first_seq;
    const bool first_one = first_of_row(b, first_seq, row);
    pdl_wait();
    if (row < 0 || row >= c.rows || !first_one) return;
    const int group = a.heads / a.kv_heads;
    constexpr int N = 4, kBatch = 4;  // rows whose scores are under way together
    static_assert(N * kThreads == kMassKeys, "four keys a thread");
    const int64_t base = (static_cast<int64_t>(row) * c.kv_heads + kvh) * c.slots;
    // The usual case, one sequence a row with a token for a few heads: what its rows need is in registers, and a
    // chunk's scores and masses are loaded while the chunk before it is added up (64 rows of up to 8192 keys: 35 us
    // by the general loop below).
    const int only = b.rows ? next_of_row(b, first_seq, row) : b.count;
    if (only == b.count && !b.starts && group <= kBatch) {
        const int length = max(0, __ldg(b.lengths + first_seq)), stop = min(min(length, c.slots), begin + min(span, c.slots - begin));
        if (stop <= begin) return;
        row_sums<HD>(c, a, tile_rows, splits, part, row, length, first_seq, 1, kvh, 0, group, tops, inverse);
        float top[kBatch], by[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            top[k] = tops[min(k, group - 1)];
            by[k] = inverse[min(k, group - 1)];
        }
        const float* const from = scores + (static_cast<int64_t>(first_seq) * a.heads + kvh * group) * pitch;
        const int position = length - 1;
        auto load = [&](int key, float4 (&x)[kBatch], float (&old)[N]) {
            if (key >= stop) return;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (k < group) x[k] = __ldcs(reinterpret_cast<const float4*>(from + k * pitch + key));
            }
#pragma unroll
            for (int i = 0; i < N; ++i) old[i] = decay != 0.0f && key + i < stop ? previous[base + key + i] : 0.0f;
        };
        float4 x[kBatch] = {}, next[kBatch] = {};
        float old[N] = {}, next_old[N] = {};
        int key = begin + N * static_cast<int>(threadIdx.x);
        load(key, x, old);
        for (; key < stop; key += kMassKeys) {
            load(key + kMassKeys, next, next_old);
            float sum[N] = {};
            // A token outside the cache sees nothing.
            if (position < c.slots) {
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    if (k >= group) continue;
                    const float s[N] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float more = fmaf(exp2_fast(s[i] - top[k]), by[k], sum[i]);
                        const bool seen = a.window == 0 || position - (key + i) < a.window || key + i < a.sinks;
                        sum[i] = seen ? more : sum[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (key + i < stop) mass[base + key + i] = decay == 0.0f ? sum[i] : fmaf(decay, old[i], sum[i]);
                old[i] = next_old[i];
            }
#pragma unroll
            for (int k = 0; k < kBatch; ++k) x[k] = next[k];
        }
        return;
    }
    const int64_t to_next = static_cast<int64_t>(a.heads - group) * pitch;  // behind a token's heads to the next's
    int known = -1;  // the sequence whose maxima and sums are held, all of them
    for (int chunk = 0; chunk < per; ++chunk) {
        const int key0 = begin + chunk * kMassKeys;
        if (key0 >= c.slots) break;
        const int my_key = key0 + N * threadIdx.x, offset = min(my_key, static_cast<int>(pitch) - N);
        float sum[N] = {}, old[N] = {};
        if (decay != 0.0f) {  // without decay the old mass is not read: it may be anything
#pragma unroll
            for (int i = 0; i < N; ++i) old[i] = my_key + i < c.slots ? previous[base + my_key + i] : 0.0f;
        }
        int end = 0;
        for (int seq = first_seq; seq < b.count; seq = next_of_row(b, seq, row)) {
            const int length = max(0, __ldg(b.lengths + seq));
            end = max(end, min(length, c.slots));
            if (min(length, c.slots) <= key0) continue;
            int first = seq, n = 1;
            if (b.starts) {
                first = max(0, __ldg(b.starts + seq));
                n = max(0, min(__ldg(b.starts + seq + 1), b.tokens) - first);
            }
            const int all = n * group;
            // Scores of kBatch rows from r on; what lies beside the rows or what they see is read, not used.
            int load_left = all, load_head = 0;
            const float* row_at = scores + (static_cast<int64_t>(first) * a.heads + kvh * group) * pitch + offset;
            auto load = [&](float4 (&x)[kBatch]) {
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (load_left-- > 0) x[k] = __ldcs(reinterpret_cast<const float4*>(row_at));
                    row_at += pitch;
                    if (++load_head == group) {
                        load_head = 0;
                        row_at += to_next;
                    }
                }
            };
            // Whether all tokens see all of the chunk (one outside the cache sees nothing).
            const bool whole = a.window == 0 && key0 + kMassKeys - 1 <= length - n && length <= c.slots;
            float4 x[kBatch];
            load(x);
            for (int r0 = 0; r0 < all; r0 += kMassRows) {
                const int rows = min(kMassRows, all - r0);
                if (known != seq) {
                    row_sums<HD>(c, a, tile_rows, splits, part, row, length, first, n, kvh, r0, rows, tops, inverse);
                    known = all <= kMassRows ? seq : -1;
                }
                for (int r = 0; r < rows; r += kBatch) {  // kMassRows are whole batches
                    float4 next[kBatch];
                    load(next);
                    if (whole && r + kBatch <= rows) {
                        const float4 top4 = *reinterpret_cast<const float4*>(tops + r);
                        const float4 by4 = *reinterpret_cast<const float4*>(inverse + r);
                        const float top[kBatch] = {top4.x, top4.y, top4.z, top4.w};
                        const float by[kBatch] = {by4.x, by4.y, by4.z, by4.w};
#pragma unroll
                        for (int k = 0; k < kBatch; ++k) {
                            const float s[N] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                            for (int i = 0; i < N; ++i) sum[i] = fmaf(exp2_fast(s[i] - top[k]), by[k], sum[i]);
                            x[k] = next[k];
                        }
                        continue;
                    }
                    // The first of the rows' tokens and heads.
                    int at = (r0 + r) / group, head_of = r0 + r - at * group;
#pragma unroll
                    for (int k = 0; k < kBatch; ++k) {
                        if (r + k < rows) {
                            // A token outside the cache sees nothing.
                            const int p = length - n + at;
                            const float top = tops[r + k], by = inverse[r + k];
                            const float s[N] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
                            for (int i = 0; i < N; ++i) {
                                const int key = my_key + i;
                                const bool seen =
                                    key <= p && p < c.slots && (a.window == 0 || p - key < a.window || key < a.sinks);
                                const float more = fmaf(exp2_fast(s[i] - top), by, sum[i]);
                                sum[i] = seen ? more : sum[i];
                            }
                        }
                        if (++head_of == group) {
                            head_of = 0;
                            ++at;
                        }
                        x[k] = next[k];
                    }
                }
            }
        }
        if (end <= key0) break;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (my_key + i < end) mass[base + my_key + i] = decay == 0.0f ? sum[i] : fmaf(decay, old[i], sum[i]);
        }
    }
}

// Several tokens of each sequence on tcgen05, from kLargeRows query rows a sequence and key head and kLargeSlots on (what
// the lengths are is not known here). Whole calls of eight sequences, eight key heads, tcgen05 and mma.sync (us). Of 128
// channels: rows of 700 to 2000 keys 72.6 and 66.5 with 48 query rows, 74.9 and 71.3 with 64, 85.7 and 113 with 96; of 1700 to
// 5000 keys 99 and 76 with 32, 116 and 136 with 64; of 200 to 600 47.9 and 44.6 with 64, 58 and 72 with 96. Of 64 channels,
// whose products leave the unpacking less behind: of 700 to 2000 keys 62.5 and 59.7 with 64, 71.9 and 74.6 with 96; of 1700 to
// 5000 96.5 and 92.0 with 64, 114 and 133 with 96; of 5000 to 16 000 227 and 176 with 48, 208 and 221 with 64. (Four key heads
// of 64: of 700 to 2000 keys 45.4 and 42.2 with 64, 54.0 and 53.8 with 96; of 5000 to 16 000 131 and 134 with 64.)
constexpr int kLargeRows = 64, kLargeSlots = 2048, kLargeRowsOf64 = 96, kLargeSlotsOf64 = 8192;
bool large(const Cache& c, const Batch& b, const AttnSpec& a) {
    if (!own_tc_takes(c, b, a) || c.slots < kLargeSlots) return false;
    const int64_t rows = static_cast<int64_t>(b.tokens) * (a.heads / a.kv_heads);
    const int least = a.head_dim == 64 && c.slots < kLargeSlotsOf64 ? kLargeRowsOf64 : kLargeRows;
    return rows >= static_cast<int64_t>(b.count) * least;
}

// Four waves of CTAs there, since lengths differ and are not known here.
int large_splits(const Cache& c, const Batch& b, const AttnSpec& a) {
    const int64_t units = static_cast<int64_t>(tile_bound(b, a, kTcTileRows)) * a.kv_heads;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({4 * 148 / std::max<int64_t>(1, units), c.slots / 512, 32})));
}

int small_splits(const Cache& c, const Batch& b, const AttnSpec& a) {
    return split_count(c, b, a, plain_query(c, b, a) ? plain_per_sm(a) : 0);
}

int64_t pitch_of(const Cache& c) { return (static_cast<int64_t>(c.slots) + kBlock - 1) / kBlock * kBlock; }

size_t score_bytes(const Cache& c, const Batch& b, const AttnSpec& a) {
    return static_cast<size_t>(b.tokens) * a.heads * pitch_of(c) * sizeof(float);
}

}  // namespace

size_t attention_weights_workspace(const Cache& c, const Batch& b, const AttnSpec& a) {
    const int splits = std::max(small_splits(c, b, a), large(c, b, a) ? large_splits(c, b, a) : 0);
    const size_t query = static_cast<size_t>(splits) * (a.head_dim + 2) * sizeof(float);
    return score_bytes(c, b, a) + static_cast<size_t>(b.tokens) * a.heads * query;
}

cudaError_t launch_attention_weights(cudaStream_t s, const Cache& c, const Batch& b, const AttnSpec& a,
                                     const void* q, int64_t q_stride, void* out, int64_t out_stride,
                                     const float* previous, float decay, float* mass, void* workspace) {
    if (b.count < 1) return cudaSuccess;
    const bool tc = b.tokens > 0 && large(c, b, a) && reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride % 8 == 0;
    const int splits = tc ? large_splits(c, b, a) : small_splits(c, b, a), rows = tc ? kTcTileRows : rows_of_tile(b, a);
    Extra extra;
    extra.scores = static_cast<float*>(workspace);
    extra.pitch = pitch_of(c);
    float* const part = extra.scores + score_bytes(c, b, a) / sizeof(float);
    if (b.tokens > 0) {
        const cudaError_t e = tc ? launch_own_tc(s, c, b, a, q, q_stride, splits, part, extra.scores, extra.pitch)
                                 : run_cached<kScores>(s, c, b, a, q, q_stride, nullptr, 0, tile_bound(b, a, rows),
                                                       rows, splits, part, extra);
        if (e) return e;
    }
    const int64_t queries = static_cast<int64_t>(b.tokens) * a.heads;
    const bool warp = splits <= 32;
    const int64_t joins = warp ? (queries * (a.head_dim / 32) + kWarps - 1) / kWarps : queries;
    // Six CTAs an SM, each of whole chunks (one chunk a CTA: 35 instead of 20 us for 64 rows of up to 8192 keys).
    const int64_t heads = static_cast<int64_t>(b.count) * a.kv_heads, chunks = (c.slots + kMassKeys - 1) / kMassKeys;
    // From 16 query rows a sequence on two chunks at most: eight sequences' 16 tokens of four heads over 16 384 keys take
    // 231 us, with three 240, with one 237; four rows of 64 sequences, without this, 343 with nineteen, 352 with two.
    int64_t per = std::min(chunks, (heads * chunks + 148 * 6 - 1) / (148 * 6));
    if (static_cast<int64_t>(b.tokens) * (a.heads / a.kv_heads) >= 16 * static_cast<int64_t>(b.count)) {
        per = std::min<int64_t>(per, 2);
    }
    const int64_t blocks = joins + heads * ((c.slots + per * kMassKeys - 1) / (per * kMassKeys));
    return by_dtype(a.dtype, [&](auto type) {
        using T = decltype(type);
        return by_head_dim(a.head_dim, [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            const auto kernel = warp ? k_weights_join<T, HD, true> : k_weights_join<T, HD, false>;
            const dim3 grid(static_cast<unsigned>(blocks));
            auto launch = [&](auto... args) {
                if (b.tokens > 0) return launch_pdl(kernel, grid, dim3(kThreads), 0, s, args...);
                // Without a pass before it the kernel stands behind the caller's own, which may write `rows`, read here
                // before the wait.
                kernel<<<grid, kThreads, 0, s>>>(args...);
                return cudaGetLastError();
            };
            return launch(c, b, a, rows, static_cast<T*>(out), out_stride, splits, static_cast<const float*>(part),
                          static_cast<const float*>(extra.scores), extra.pitch, previous, decay, mass,
                          static_cast<int>(joins), static_cast<int>(per));
        });
    });
}

}  // namespace bst
