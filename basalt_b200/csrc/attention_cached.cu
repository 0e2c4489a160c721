// Attention of one or a few new tokens per sequence over a cache, split over the keys.
//
// Bound by memory: every visible key and value is read once (0.625 bytes a value in 4 bits) and
// takes two multiply-adds per query head. With the 4-bit codes the reading is so short that the
// arithmetic has to stay below four lane operations a value, which rules out scaling each value;
// so the codes go to the tensor cores as they are and the scales are applied around the products:
//
//   s_ij    = sum_g step_jg (q_ig . c_jg) + low_jg sum(q_ig)         g: groups of 32 channels
//   out_icg = sum_j (p_ij step_jg) c_jgc + sum_j p_ij low_jg
//
// A nibble becomes an fp16 number without a conversion: its bits in the lowest mantissa bits, c or
// 16 c, are the subnormals c 2^-24 and 16 c 2^-24. The other operand carries the 2^15 or 2^11 that
// bring them near one: queries, normalised by a power of two per row so that nothing overflows, and
// weights p step, normalised by a power of two above the largest of the group so far (which
// moves as the maximum of the scores does, by rescaling). fp16 has 11 bits where bf16 has 8: one
// term is more than bf16 outputs show, and two carry 22 bits for float32. float32 also takes
// 1024 + c, or 1024 + 16 c, to c - 8 with one fp16 operation: sums of low and of step c would
// otherwise cancel one another (over 42 000 keys that left 7e-5 of the output where this leaves 6e-7),
// and the tensor cores add subnormals with fewer bits.
// mma.sync m16n8k16 reads its B operand from registers, which is where unpacked codes are;
// tcgen05 would need them written to shared memory at four times their size first, and a tile
// of at most eight query rows would leave 120 of its 128 rows empty.
//
// The sixteen rows of the A operand hold sixteen queries (tokens x heads of one key head), or eight:
// then rows 8-15 hold what rounding the weights (and float32 q) of rows 0-7 left, so that one product
// carries both terms. The lows, and caches that are not in 4 bits, are multiplied in bf16 the same way,
// float32 ones in three terms. Weights, sums and the running maximum are float32.
//
// A warp works on 16 keys at a time and alone: it copies its keys into its own ring in shared memory
// with cp.async (keys that nobody sees are filled with zeros there, whatever their slots hold), and
// warps meet only at the end. Lane (g, t) = (lane / 4, lane % 4) owns query row g, and its
// fragments' key columns 2 t and 2 t + 1 of either half of the 16. Splits leave their maximum, sum
// and output in the workspace and a second kernel joins them.
//
// What that reaches: a bf16 cache is read at 0.90 of the copy rate (64 sequences of 2052 keys, 8 heads
// of 128: 84 us), a float32 one, whose entries are split in three terms by every warp, at half of it (the
// same in float32: 283 us). With codes a warp's own chain of unpacking, scaling and multiplying is the limit, at
// the two warps a scheduler that registers leave (half of the issue slots are empty): 131 000 keys of 8
// heads of 128 with 32 query heads take 64 us (2.6 TB/s), 24 sequences of 900 to 16 384 keys with 4
// tokens each 183 us (1.5 TB/s, for four times the products; 174 with one normalisation of weight x step
// for all queries of a lane, by the steps alone, which lost what a few large values hid). One query a
// key head has a kernel of its own below.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>

#include "attention.cuh"
#include "device.cuh"
#include "operators.h"

namespace bst {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBlock = 16;   // keys a warp takes at a time
constexpr float kLeastSteps = 0x1p114f;  // the normalisation of steps below 2^-100

template <int STORAGE, int HD>
struct Layout {
    static constexpr int kGroups = HD / 32;
    static constexpr bool kCodes = STORAGE == BST_DTYPE_U4;
    static constexpr int kRowBytes = kCodes ? HD / 2 : (STORAGE == BST_DTYPE_F32 ? 4 : 2) * HD;
    static constexpr int kScaleBytes = kCodes ? kBlock * kGroups * 4 : 0;
    static constexpr int kStage = 2 * (kBlock * kRowBytes + kScaleBytes);
    // Enough in flight to cover the memory's latency from every SM: 20 to 130 KB a CTA.
    static constexpr int kStages = kStage <= 2560 ? 4 : (kStage <= 8192 ? 3 : 2);
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int smem(int rows) {
        return kRing > kWarps * rows * (HD + 2) * 4 ? kRing : kWarps * rows * (HD + 2) * 4;
    }
};

// Where 16-byte chunk `chunk` of key row `row` of a block lies in its row in shared memory, so that
// the reads below meet no bank twice.
template <int STORAGE, int HD>
__device__ __forceinline__ int swizzled(int row, int chunk) {
    if constexpr (STORAGE == BST_DTYPE_U4) {
        return HD == 128 ? chunk ^ (row & 2) : chunk;
    } else if constexpr (STORAGE == BST_DTYPE_BF16) {
        return HD == 32 ? chunk ^ ((row >> 1) & 3) : chunk ^ (((row & 1) << 2) | ((row >> 1) & 3));
    } else {
        return chunk ^ (row & 7);
    }
}

// The key row (0..7) behind column n of a fragment's eight key columns. For 4-bit rows, which are
// shorter than the banks, an order in which neither the key nor the value reads collide.
template <int STORAGE, int HD>
__device__ __forceinline__ int row_of_column(int n) {
    if constexpr (STORAGE == BST_DTYPE_U4) {
        const int t = n >> 1;
        return (n & 1) ? 4 + (t ^ (HD == 128 ? 1 : 2)) : t;
    } else {
        return n;
    }
}

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same from zero.
__device__ __forceinline__ void mma_bf16_start(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_f16_start(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ float low_of(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float high_of(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// (a, b) as bf16 pairs whose sum is (a, b) to 8 bits a term.
template <int TERMS>
__device__ __forceinline__ void terms_of(float a, float b, uint32_t* out) {
    out[0] = pack2(a, b);
#pragma unroll
    for (int i = 1; i < TERMS; ++i) {
        a -= low_of(out[i - 1]);
        b -= high_of(out[i - 1]);
        out[i] = pack2(a, b);
    }
}

// The same as fp16 pairs, 11 bits a term.
template <int TERMS>
__device__ __forceinline__ void half_terms_of(float a, float b, uint32_t* out) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        const __half2 h = __floats2half2_rn(a, b);
        out[i] = *reinterpret_cast<const uint32_t*>(&h);
        if (i + 1 < TERMS) {
            a -= __low2float(h);
            b -= __high2float(h);
        }
    }
}

// Nibbles 0 and 1 of both halves of x as fp16 pairs c - 8.
__device__ __forceinline__ uint32_t centred0(uint32_t x) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"((x & 0x000f000fu) | 0x64006400u), "r"(0x64086408u));
    return r;
}
__device__ __forceinline__ uint32_t centred1(uint32_t x) {  // (1024 + 16 c) / 16 - 72
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;"
        : "=r"(r)
        : "r"((x & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(0xd480d480u));
    return r;
}
// The same as c 2^-24 and 16 c 2^-24, or centred.
template <bool CENTRED>
__device__ __forceinline__ uint32_t nibble0(uint32_t x) {
    return CENTRED ? centred0(x) : x & 0x000f000fu;
}
template <bool CENTRED>
__device__ __forceinline__ uint32_t nibble1(uint32_t x) {
    return CENTRED ? centred1(x) : x & 0x00f000f0u;
}

template <int G>
__device__ __forceinline__ void load_words(uint32_t addr, uint32_t (&w)[G]) {
    if constexpr (G == 1) {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
    } else if constexpr (G == 2) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    } else {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    }
}

// The keys that a tile of queries at positions p0..p1 sees: blocks of 16 that hold the sinks before
// the window, then blocks from the window's first key (rounded down) to the last key.
struct Visible {
    int first, end;       // the window
    int aligned;          // first, rounded down to a block
    int sinks;            // keys below it are visible too
    int sink_blocks, blocks;
    __device__ Visible(int p0, int p1, int slots, int window, int sinks_) {
        end = min(p1 + 1, slots);
        first = window ? max(0, p0 - window + 1) : 0;
        aligned = first & ~(kBlock - 1);
        sinks = sinks_;
        blocks = sink_blocks = 0;
        if (first < end) {
            sink_blocks = (min(sinks, aligned) + kBlock - 1) / kBlock;
            blocks = sink_blocks + (end - aligned + kBlock - 1) / kBlock;
        }
    }
    __device__ int key(int block) const {
        return block < sink_blocks ? block * kBlock : aligned + (block - sink_blocks) * kBlock;
    }
    __device__ bool holds(int key) const { return key < end && (key >= first || key < sinks); }
    // Whether all keys of the block at key0 are held.
    __device__ bool whole(int key0) const {
        return key0 + kBlock <= end && (key0 >= first || key0 + kBlock <= sinks);
    }
};

// Splits that a tile of this many blocks is worth: at least 8 blocks a split, two a warp.
__host__ __device__ __forceinline__ int useful_splits(int blocks, int splits) {
    const int most = blocks / 8;
    return most < 1 ? 1 : (most < splits ? most : splits);
}

// CTAs an SM must hold, which caps the registers: measured, more warps beat the few spills.
template <typename T, int STORAGE, int HD, int ROWS>
constexpr int min_ctas() {
    if (STORAGE == BST_DTYPE_F32) return 1;
    return HD == 128 ? 2 : (HD == 64 ? 4 : 5);
}

// The A fragment's terms times (b0, b1). With one query row a lane, the tile's rows 8-15 carry the
// second term of rows 0-7; with two they are queries of their own and every term is a product.
template <bool HALF, bool START, int R, int N>
__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[R][2][N], uint32_t b0,
                                        uint32_t b1) {
    auto one = [&](bool first, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
        if (START && first) {
            if constexpr (HALF) {
                mma_f16_start(c, a0, a1, a2, a3, b0, b1);
            } else {
                mma_bf16_start(c, a0, a1, a2, a3, b0, b1);
            }
        } else if constexpr (HALF) {
            mma_f16(c, a0, a1, a2, a3, b0, b1);
        } else {
            mma_bf16(c, a0, a1, a2, a3, b0, b1);
        }
    };
    if constexpr (R == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) one(i == 0, a[0][0][i], a[1][0][i], a[0][1][i], a[1][1][i]);
    } else if constexpr (N == 1) {
        one(true, a[0][0][0], 0u, a[0][1][0], 0u);
    } else {
        one(true, a[0][0][0], a[0][0][1], a[0][1][0], a[0][1][1]);
        if constexpr (N == 3) one(false, a[0][0][2], 0u, a[0][1][2], 0u);
    }
}
// One product with the leading term of every query (and the second where it is free).
template <int R, int N>
__device__ __forceinline__ void leading(float (&c)[4], const uint32_t (&a)[R][2][N], uint32_t b0,
                                        uint32_t b1) {
    if constexpr (R == 2) {
        mma_bf16(c, a[0][0][0], a[1][0][0], a[0][1][0], a[1][1][0], b0, b1);
    } else if constexpr (N == 1) {
        mma_bf16(c, a[0][0][0], 0u, a[0][1][0], 0u, b0, b1);
    } else {
        mma_bf16(c, a[0][0][0], a[0][0][1], a[0][1][0], a[0][1][1], b0, b1);
    }
}
// Column e of such a product for this lane's query row r.
template <int R, int N>
__device__ __forceinline__ float entry(const float (&c)[4], int r, int e) {
    if constexpr (R == 2) return c[2 * r + e];
    if constexpr (N == 1) return c[e];
    return c[e] + c[2 + e];
}

// The sums of one query over the keys of blocks [b0, b1) of an unquantised cache, plainly, by one warp:
// [HD outputs, maximum, sum] as k_cached leaves them.
template <typename T, typename S, int HD>
__device__ __noinline__ void attend_plainly(const S* k, const S* v, const T* q, float scale,
                                            const Visible& seen, int b0, int b1, float* to) {
    constexpr int C = HD / 32;
    const int lane = threadIdx.x & 31;
    float value[C], top, total;
    attend_row<C>(q, k, HD, v, HD, scale, static_cast<int64_t>(b1 - b0) * kBlock,
                  [&](int64_t at) {
                      const int key = seen.key(b0 + static_cast<int>(at / kBlock)) + static_cast<int>(at % kBlock);
                      return static_cast<int64_t>(seen.holds(key) ? key : -1);
                  },
                  value, &top, &total);
#pragma unroll
    for (int i = 0; i < C; ++i) to[lane + 32 * i] = value[i];
    if (lane == 0) {
        to[HD] = top;
        to[HD + 1] = total;
    }
}

// Whether the keys and values of blocks [b0, b1), or `rows` queries of one token, hold an infinity or a
// float that bf16 rounds to one. This thread's share of the CTA's.
template <typename T, int STORAGE, int HD>
__device__ __noinline__ bool meets_infinity(const char* k, const char* v, const Visible& seen, int b0, int b1,
                                            const T* q, int rows) {
    auto rounds = [](uint32_t u) { return (u & 0x7fffffffu) - 0x7f7f8000u <= 0x8000u; };
    auto bad = [&](uint32_t u) {
        return STORAGE == BST_DTYPE_F32 ? rounds(u) : ((u & 0x7fffu) == 0x7f80u) | ((u & 0x7fff0000u) == 0x7f800000u);
    };
    using L = Layout<STORAGE, HD>;
    constexpr int kChunks = L::kRowBytes / 16;
    bool found = false;
    for (int block = b0; block < b1; ++block) {
        const int key0 = seen.key(block);
#pragma unroll 4
        for (int x = threadIdx.x; x < kBlock * kChunks; x += kThreads) {
            const int key = key0 + x / kChunks;
            uint4 u = {}, w = {};
            if (seen.holds(key)) {
                const int64_t at = static_cast<int64_t>(key) * kChunks + x % kChunks;
                u = reinterpret_cast<const uint4*>(k)[at];
                w = reinterpret_cast<const uint4*>(v)[at];
            }
            found |= bad(u.x) | bad(u.y) | bad(u.z) | bad(u.w) | bad(w.x) | bad(w.y) | bad(w.z) | bad(w.w);
        }
    }
    for (int x = threadIdx.x; x < rows * HD; x += kThreads) found |= rounds(__float_as_uint(to_f(q[x])));
    return found;
}

// ROWS queries a tile: 8, or 16 for bf16 batches that have more than eight to a key head, so that
// unpacking the codes, which bounds the kernel, is shared by twice as many.
template <typename T, int STORAGE, int HD, int ROWS>
__global__ void __launch_bounds__(kThreads, min_ctas<T, STORAGE, HD, ROWS>())
k_cached(Cache c, Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride,
         T* __restrict__ out, int64_t out_stride, int splits, float* __restrict__ part) {
    using L = Layout<STORAGE, HD>;
    constexpr int G = L::kGroups;
    constexpr int R = ROWS / 8;                  // query rows of a lane: g, and g + 8
    constexpr bool kExact = sizeof(T) == 4;      // float32: 24-bit operands
    constexpr int kTerms = kExact ? 3 : 2;       // of the weights and query sums, in bf16
    constexpr int kHalf = kExact ? 2 : 1;        // of weights x steps, in fp16
    // Of the queries: in fp16 for codes, in bf16 otherwise; a bf16 query is one term of either.
    constexpr int kQ = kExact ? (L::kCodes ? 2 : 3) : 1;
    constexpr int kK = STORAGE == BST_DTYPE_F32 ? (kExact ? 3 : 2) : 1;  // of keys and values
    constexpr int kMma = HD / 16;
    constexpr float kOdd = kExact ? 0x1p15f : 0x1p11f;  // takes the 16 of nibbles 1 and 3 back
    static_assert(!kExact || R == 1, "float32 tiles have eight rows");
    extern __shared__ __align__(16) unsigned char smem[];

    const int group = a.heads / a.kv_heads;
    const int kvh = blockIdx.y;
    const int split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    Tile tile;
    if (!find_tile(b, group, ROWS, blockIdx.x, &tile)) return;
    const int row = b.rows ? __ldg(b.rows + tile.seq) : tile.seq;
    const int length = max(0, __ldg(b.lengths + tile.seq));
    const int rows = min(ROWS, tile.n * group - tile.r0);
    // Positions of the tile's tokens; a row or slot outside the cache sees nothing.
    const bool inside = row >= 0 && row < c.rows;
    // A sequence's only token, or token row / group of several.
    const int first_token = tile.n == 1 ? 0 : tile.r0 / group;
    const int last_token = tile.n == 1 ? 0 : (tile.r0 + rows - 1) / group;
    const int p_first = length - tile.n + first_token, p_last = length - tile.n + last_token;
    const Visible seen(p_first, inside ? p_last : -1, c.slots, a.window, a.sinks);
    const int use = useful_splits(seen.blocks, splits);
    if (split >= use) return;
    const int b0 = static_cast<int>(static_cast<int64_t>(seen.blocks) * split / use);
    const int b1 = static_cast<int>(static_cast<int64_t>(seen.blocks) * (split + 1) / use);

    const int64_t at = (static_cast<int64_t>(inside ? row : 0) * c.kv_heads + kvh) * c.slots;
    const char* kb = static_cast<const char*>(c.k) + at * L::kRowBytes;
    const char* vb = static_cast<const char*>(c.v) + at * L::kRowBytes;
    const char* ksb = static_cast<const char*>(c.k_scale) + at * (G * 4);
    const char* vsb = static_cast<const char*>(c.v_scale) + at * (G * 4);
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) +
                          warp * L::kStages * L::kStage;
    // A block is contiguous in its source: chunk i of this lane lies 512 i bytes after chunk 0.
    const int lane_row = lane / (L::kRowBytes / 16), lane_chunk = lane % (L::kRowBytes / 16);
    constexpr int kKeyBytes = kBlock * L::kRowBytes;      // bytes of a block's keys
    constexpr int kLoads = kKeyBytes / 512 ? kKeyBytes / 512 : 1;  // of each lane, for the keys
    auto lane_to = [&](int i) {
        const int r = lane_row + i * (512 / L::kRowBytes);
        return r * L::kRowBytes + swizzled<STORAGE, HD>(r, lane_chunk) * 16;
    };
    // Rows of 16 bytes: sixteen lanes take the keys, sixteen the values.
    constexpr bool kShared = kKeyBytes < 512;
    const char* const k_lane = (kShared && lane >= 16 ? vb - kKeyBytes : kb) + lane * 16;
    const char* const v_lane = vb + lane * 16;
    const char* const s_lane = (lane >= 16 ? vsb : ksb) + (lane & 15) * (G * 4);
    auto fetch = [&](int block, int stage) {
        if (block < b1) {
            const int key0 = seen.key(block);
            const uint32_t dst = ring + stage * L::kStage;
            const char* const ks = k_lane + static_cast<int64_t>(key0) * L::kRowBytes;
            const char* const vs = v_lane + static_cast<int64_t>(key0) * L::kRowBytes;
            const char* const ss = s_lane + static_cast<int64_t>(key0) * (G * 4);
            const uint32_t scale_to = dst + 2 * kKeyBytes + lane * (G * 4);
            if (seen.whole(key0)) {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) cp_async<16>(dst + lane_to(i), ks + 512 * i, 16);
                if constexpr (!kShared) {
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        cp_async<16>(dst + kKeyBytes + lane_to(i), vs + 512 * i, 16);
                    }
                }
                if constexpr (L::kCodes) cp_async<G * 4>(scale_to, ss, G * 4);
            } else {
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = lane_row + i * (512 / L::kRowBytes);
                    const bool ok = seen.holds(key0 + (kShared ? r & 15 : r));
                    cp_async<16>(dst + lane_to(i), ok ? ks + 512 * i : kb, ok ? 16 : 0);
                    if constexpr (!kShared) {
                        cp_async<16>(dst + kKeyBytes + lane_to(i), ok ? vs + 512 * i : vb, ok ? 16 : 0);
                    }
                }
                if constexpr (L::kCodes) {
                    const bool ok = seen.holds(key0 + (lane & 15));
                    cp_async<G * 4>(scale_to, ok ? ss : ksb, ok ? G * 4 : 0);
                }
            }
        }
        cp_commit();
    };
    int next = b0 + warp;
#pragma unroll
    for (int i = 0; i < L::kStages - 1; ++i) {
        fetch(next, i);
        next += kWarps;
    }

    // This lane's part of the queries as A fragments: product m of group gr takes, for 4-bit
    // keys, channels 8 t + {2 m, 2 m + 4} and {2 m + 1, 2 m + 5} (the order in which nibbles
    // unpack, the second pair 16 times too large), otherwise 8 t + 4 m + {0, 1} and {2, 3}.
    // to_score takes a product to the base-2 logarithm of its weight. With codes, one more product
    // (qs) of the groups' query sums and the keys' lows completes a score.
    uint32_t qa[kMma][R][2][kQ], qs[R][2][kTerms] = {};
    float to_score[R], qsum[G] = {};
    int position[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int my_row = tile.r0 + g + 8 * r;
        const bool live = g + 8 * r < rows;
        const int my_token = tile.n == 1 ? 0 : my_row / group;
        position[r] = length - tile.n + my_token;
        if (!live || !inside || position[r] >= c.slots) position[r] = -1;
        to_score[r] = a.scale * kLog2e;
        const int64_t token = tile.first + my_token;
        const T* src = q + token * q_stride + (kvh * group + my_row - my_token * group) * HD + 8 * t;
        float x[G][8], largest = 0.0f;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[gr][i] = live ? to_f(src[32 * gr + i]) : 0.0f;
                largest = fmaxf(largest, fabsf(x[gr][i]));
            }
        }
        if constexpr (L::kCodes) {
            // Normalised to |q| < 1; products come out 2^-9 too small (2^15 for 2^24), or 2^15 too
            // large.
            largest = fmaxf(largest, __shfl_xor_sync(kFull, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(kFull, largest, 2));
            const int e = max(min(ilogbf(fmaxf(largest, FLT_MIN)), 126) + 1, -100);
            const float shrink = exp2f(static_cast<float>(-e));
            to_score[r] *= exp2f(static_cast<float>(e));
            to_score[r] *= kExact ? 0x1p-15f : 512.0f;
            float mine[2] = {0.0f, 0.0f};  // sums of groups 2 t and 2 t + 1
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += x[gr][i] *= shrink;
                sum += __shfl_xor_sync(kFull, sum, 1);
                sum += __shfl_xor_sync(kFull, sum, 2);
                if (t == gr / 2) mine[gr & 1] = sum * 0.001953125f;
                qsum[gr] = sum * 0x1p15f;
            }
            if constexpr (!kExact) terms_of<kTerms>(mine[0], mine[1], qs[r][0]);
        }
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if constexpr (L::kCodes) {
                    half_terms_of<kQ>(x[gr][2 * m] * 0x1p15f, x[gr][2 * m + 4] * 0x1p15f,
                                      qa[2 * gr + m][r][0]);
                    half_terms_of<kQ>(x[gr][2 * m + 1] * kOdd, x[gr][2 * m + 5] * kOdd,
                                      qa[2 * gr + m][r][1]);
                } else {
                    terms_of<kQ>(x[gr][4 * m], x[gr][4 * m + 1], qa[2 * gr + m][r][0]);
                    terms_of<kQ>(x[gr][4 * m + 2], x[gr][4 * m + 3], qa[2 * gr + m][r][1]);
                }
            }
        }
    }

    // Output columns, and with codes the sums over keys of weight x low (column n: of group n) and the
    // normalisation of weight x step, a power of two for each query and group: 2^14 over the one above
    // the largest step so far, or above 64 times the largest weight x step where that is less (steps of
    // keys that a query does not see, or gives next to no weight, would leave the others no bits). It
    // moves up again by what the maximum of the scores has grown since, in steps of 2^6 or more.
    float o[G * 4][4], lows[4] = {}, middles[G] = {}, top[R], total[R], shrink[R][G], grown[R] = {};
    unsigned poison[R];  // groups in which a key that the query sees holds a NaN
#pragma unroll
    for (int i = 0; i < G * 4; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        top[r] = -INFINITY;
        total[r] = 0.0f;
        poison[r] = 0u;
    }
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
#pragma unroll
        for (int r = 0; r < R; ++r) shrink[r][gr] = kLeastSteps;
    }
    // The key rows of this lane's score columns 2 t and 2 t + 1, and of the key that it loads.
    const int key_row[2] = {row_of_column<STORAGE, HD>(2 * t), row_of_column<STORAGE, HD>(2 * t + 1)};
    const int load_row = row_of_column<STORAGE, HD>(g);
    // Offsets of this lane's reads in a stage, for the first eight keys (the other eight follow at
    // eight rows' distance, which the swizzle does not look at): its keys' codes, the lows of groups
    // 2 t and 2 t + 1, the scales of its score columns, its entries of the values.
    int k_at = 0, lows_at = 0, scale_at[2] = {}, v_at[2] = {};
    if constexpr (L::kCodes) {
        k_at = load_row * L::kRowBytes + swizzled<STORAGE, HD>(load_row, t * 4 * G / 16) * 16 + t * 4 * G % 16;
        lows_at = 2 * kKeyBytes + load_row * (G * 4) + (2 * t < G ? t * 8 : 0);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            scale_at[e] = 2 * kKeyBytes + key_row[e] * (G * 4);
            v_at[e] = kKeyBytes + key_row[e] * L::kRowBytes +
                      swizzled<STORAGE, HD>(key_row[e], g * 2 * G / 16) * 16 + g * 2 * G % 16;
        }
    }

    int stage = 0;
    for (int block = b0 + warp; block < b1; block += kWarps) {
        cp_wait<L::kStages - 2>();
        __syncwarp();
        const uint32_t ks = ring + stage * L::kStage;
        const uint32_t vs = ks + kKeyBytes;
        const uint32_t vss = ks + 2 * kKeyBytes + L::kScaleBytes;
        const int key0 = seen.key(block);

        // Scores of keys key0 + 8 nb + key_row[e].
        float s[R][2][2];
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
            const int lr = 8 * nb + load_row;
            if constexpr (L::kCodes) {
                // Bytes [t * 4 G, ...) of the row: half 2 t of every group, then half 2 t + 1.
                uint32_t w[G], sa[G], sb[G];
                load_words<G>(ks + k_at + nb * 8 * L::kRowBytes, w);
                load_words<G>(ks + scale_at[0] + nb * 8 * (G * 4), sa);  // (step, low) of the two
                load_words<G>(ks + scale_at[1] + nb * 8 * (G * 4), sb);  // keys this lane scores
                if constexpr (kExact) {
                    s[0][nb][0] = s[0][nb][1] = 0.0f;
                } else {
                    uint32_t key_lows;
                    if constexpr (G == 1) {
                        uint32_t w1[1];
                        load_words<1>(ks + lows_at + nb * 8 * (G * 4), w1);
                        key_lows = w1[0] >> 16;
                    } else {
                        uint32_t w2[2];
                        load_words<2>(ks + lows_at + nb * 8 * (G * 4), w2);
                        key_lows = __byte_perm(w2[0], w2[1], 0x7632);
                    }
                    if (2 * t >= G) key_lows = 0u;
                    float low[4];
                    product<false, true>(low, qs, key_lows, 0u);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        s[r][nb][0] = entry<R, kTerms>(low, r, 0);
                        s[r][nb][1] = entry<R, kTerms>(low, r, 1);
                    }
                }
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    uint32_t x;
                    if constexpr (G == 1) {
                        x = w[0];
                    } else {
                        // 16-bit entries gr and G + gr of the lane's 2 G.
                        x = __byte_perm(w[gr / 2], w[G / 2 + gr / 2], gr & 1 ? 0x7632 : 0x5410);
                    }
                    float acc[4];
                    product<true, true>(acc, qa[2 * gr], nibble0<kExact>(x), nibble1<kExact>(x));
                    x >>= 8;
                    product<true, false>(acc, qa[2 * gr + 1], nibble0<kExact>(x), nibble1<kExact>(x));
                    const float step_a = low_of(sa[gr]), step_b = low_of(sb[gr]);
                    if constexpr (kExact) {
                        // The group's middle, low + 8 step, times the sum of the query's channels.
                        s[0][nb][0] = fmaf(fmaf(8.0f, step_a, high_of(sa[gr])), qsum[gr], s[0][nb][0]);
                        s[0][nb][1] = fmaf(fmaf(8.0f, step_b, high_of(sb[gr])), qsum[gr], s[0][nb][1]);
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        s[r][nb][0] = fmaf(step_a, entry<R, kQ>(acc, r, 0), s[r][nb][0]);
                        s[r][nb][1] = fmaf(step_b, entry<R, kQ>(acc, r, 1), s[r][nb][1]);
                    }
                }
            } else {
                float acc[4] = {};
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    uint32_t kw[4][kK];  // channels 8 t .. 8 t + 7 of the group, in pairs
                    if constexpr (STORAGE == BST_DTYPE_BF16) {
                        uint32_t w[4];
                        load_words<4>(ks + lr * L::kRowBytes + swizzled<STORAGE, HD>(lr, 4 * gr + t) * 16, w);
#pragma unroll
                        for (int i = 0; i < 4; ++i) kw[i][0] = w[i];
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t w[4];
                            load_words<4>(ks + lr * L::kRowBytes +
                                              swizzled<STORAGE, HD>(lr, 8 * gr + 2 * t + h) * 16, w);
                            terms_of<kK>(__uint_as_float(w[0]), __uint_as_float(w[1]), kw[2 * h]);
                            terms_of<kK>(__uint_as_float(w[2]), __uint_as_float(w[3]), kw[2 * h + 1]);
                        }
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        // All of the query's terms with the key's first, its leading ones with the
                        // others.
                        product<false, false>(acc, qa[2 * gr + m], kw[2 * m][0], kw[2 * m + 1][0]);
#pragma unroll
                        for (int i = 1; i < kK; ++i) {
                            leading<R, kQ>(acc, qa[2 * gr + m], kw[2 * m][i], kw[2 * m + 1][i]);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    s[r][nb][0] = entry<R, kQ>(acc, r, 0);
                    s[r][nb][1] = entry<R, kQ>(acc, r, 1);
                }
            }
        }
        // Mask, running maximum. Every query of the tile sees all of a block in the middle.
        const bool all = key0 + kBlock - 1 <= p_first && p_last < c.slots &&
                         (a.window == 0 || p_last - key0 < a.window || key0 + kBlock <= a.sinks);
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[r][i / 2][i % 2] *= to_score[r];
        }
        if (!all) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key_at = 8 * (i / 2) + key_row[i % 2], key = key0 + key_at;
                // A NaN that some query does not see is taken out of the products below; the
                // queries that see it remember.
                unsigned bad = 0u;
                if constexpr (L::kCodes && !kExact) {
                    uint32_t w[G];
                    load_words<G>(vss + key_at * (G * 4), w);
#pragma unroll
                    for (int gr = 0; gr < G; ++gr) {
                        bad |= (w[gr] & 0x7f800000u) == 0x7f800000u ? 1u << gr : 0u;
                    }
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (key > position[r] || (a.window != 0 && position[r] - key >= a.window &&
                                              key >= a.sinks)) {
                        s[r][i / 2][i % 2] = -INFINITY;
                    } else {
                        poison[r] |= bad;
                    }
                }
            }
        }
        bool grows = false;
        float keep[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float block_top = fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][1][0], s[r][1][1]));
            block_top = fmaxf(block_top, __shfl_xor_sync(kFull, block_top, 1));
            block_top = fmaxf(block_top, __shfl_xor_sync(kFull, block_top, 2));
            const bool up = block_top > top[r];
            keep[r] = up ? (top[r] == -INFINITY ? 0.0f : exp2_fast(top[r] - block_top)) : 1.0f;
            if constexpr (L::kCodes) grown[r] += up && top[r] != -INFINITY ? block_top - top[r] : 0.0f;
            top[r] = up ? block_top : top[r];
            grows |= up;
        }
        if (__any_sync(kFull, grows)) {
#pragma unroll
            for (int r = 0; r < R; ++r) total[r] *= keep[r];
            // Columns 2 and 3 are row g + 8: of the same query, or of the second.
#pragma unroll
            for (int j = 0; j < 4; ++j) lows[j] *= keep[R == 2 ? j / 2 : 0];
#pragma unroll
            for (int gr = 0; gr < G; ++gr) middles[gr] *= keep[0];
#pragma unroll
            for (int i = 0; i < G * 4; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[i][j] *= keep[R == 2 ? j / 2 : 0];
            }
            if constexpr (L::kCodes) {
                bool far = false;
#pragma unroll
                for (int r = 0; r < R; ++r) far |= grown[r] >= 6.0f;
                if (__any_sync(kFull, far)) {
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        if (grown[r] < 6.0f) continue;
                        const uint32_t by_most = min(static_cast<int>(grown[r]), 126);
                        grown[r] = 0.0f;
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) {
                            const uint32_t room = (__float_as_uint(kLeastSteps) - __float_as_uint(shrink[r][gr])) >> 23;
                            const float by = __uint_as_float((127u + min(by_most, room)) << 23);
                            shrink[r][gr] *= by;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    if (R == 1 || e / 2 == r) o[4 * gr + j][e] *= by;
                                }
                            }
                        }
                    }
                }
            }
        }
        float p[R][2][2];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float base = top[r] == -INFINITY ? 0.0f : top[r];
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    p[r][nb][e] = exp2_fast(s[r][nb][e] - base);
                    total[r] += p[r][nb][e];
                }
            }
        }

        // Weights times values.
        uint32_t pa[R][2][kTerms];
        if constexpr (!(L::kCodes && kExact)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                terms_of<kTerms>(p[r][0][0], p[r][0][1], pa[r][0]);
                terms_of<kTerms>(p[r][1][0], p[r][1][1], pa[r][1]);
            }
        }
        if constexpr (L::kCodes) {
            uint32_t sv[2][2][G];
            uint32_t wv[2][2][(G + 1) / 2];
            uint16_t column[2][2];  // the keys' lows of group g
#pragma unroll
            for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    load_words<G>(ks + scale_at[e] + L::kScaleBytes + nb * 8 * (G * 4), sv[nb][e]);
                    if constexpr (!kExact) {
                        asm volatile("ld.shared.u16 %0, [%1];"
                                     : "=h"(column[nb][e])
                                     : "r"(ks + scale_at[e] + L::kScaleBytes + nb * 8 * (G * 4) +
                                           (g & (G - 1)) * 4 + 2));
                        if (g >= G) column[nb][e] = 0;
                        if (!all && (column[nb][e] & 0x7f80u) == 0x7f80u) column[nb][e] = 0;
                    } else if (!all && s[0][nb][e] == -INFINITY) {
                        // A key that the query does not see (its low may be a NaN).
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) sv[nb][e][gr] = 0u;
                    }
                    // 16-bit entries [g][0 .. G): nibble j is channel 4 g + j of a group.
                    const uint32_t va = ks + v_at[e] + nb * 8 * L::kRowBytes;
                    if constexpr (G == 1) {
                        uint16_t h;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(va));
                        wv[nb][e][0] = h;
                    } else {
                        load_words<G / 2>(va, wv[nb][e]);
                    }
                }
            }
            if constexpr (!kExact) {
                product<false, false>(lows, pa, __byte_perm(column[0][0], column[0][1], 0x5410),
                                      __byte_perm(column[1][0], column[1][1], 0x5410));
            }
            // One test for all groups, so that their products below stand side by side. Steps are the low
            // halves, and order as whole numbers do.
            float largest[G];
            bool above_any = false;
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                const uint32_t most = __vimax3_u16x2(__vmaxu2(sv[0][0][gr], sv[0][1][gr]),
                                                     sv[1][0][gr], sv[1][1][gr]);
                largest[gr] = low_of(most);
#pragma unroll
                for (int r = 0; r < R; ++r) above_any |= largest[gr] * shrink[r][gr] > 0x1p14f;
            }
            if (__any_sync(kFull, above_any)) {
                // A step above its group's power of two: the next one, for a row's lanes (each has seen
                // four of the keys), if the row gives it any weight.
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    float step = fmaxf(largest[gr], __shfl_xor_sync(kFull, largest[gr], 1));
                    step = fmaxf(step, __shfl_xor_sync(kFull, step, 2));
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        float most = 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            most = fmaxf(most, p[r][i / 2][i % 2] * low_of(sv[i / 2][i % 2][gr]));
                        }
                        most = fmaxf(most, __shfl_xor_sync(kFull, most, 1));
                        most = fmaxf(most, __shfl_xor_sync(kFull, most, 2));
                        most = fminf(64.0f * most, step);
                        const uint32_t above = (__float_as_uint(most) & 0x7f800000u) + 0x00800000u;
                        const float next = most * shrink[r][gr] > 0x1p14f
                                               ? __uint_as_float((268u << 23) - above)  // 2^14 / above
                                               : shrink[r][gr];
                        const float by = next / shrink[r][gr];
                        shrink[r][gr] = next;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if (R == 1 || e / 2 == r) o[4 * gr + j][e] *= by;
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                const float steps[2][2] = {{low_of(sv[0][0][gr]), low_of(sv[0][1][gr])},
                                           {low_of(sv[1][0][gr]), low_of(sv[1][1][gr])}};
                uint32_t ps[R][2][kHalf], x[2];
#pragma unroll
                for (int nb = 0; nb < 2; ++nb) {
                    // The weight first: zero times a step that is far above the normalisation is zero.
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        half_terms_of<kHalf>(p[r][nb][0] * shrink[r][gr] * steps[nb][0],
                                             p[r][nb][1] * shrink[r][gr] * steps[nb][1], ps[r][nb]);
                    }
                    x[nb] = __byte_perm(wv[nb][0][gr / 2], wv[nb][1][gr / 2], gr & 1 ? 0x7632 : 0x5410);
                }
                if constexpr (kExact) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        middles[gr] = fmaf(p[0][i / 2][i % 2],
                                           fmaf(8.0f, steps[i / 2][i % 2], high_of(sv[i / 2][i % 2][gr])),
                                           middles[gr]);
                    }
                }
                const uint32_t y0 = x[0] >> 8, y1 = x[1] >> 8;
                product<true, false>(o[4 * gr], ps, nibble0<kExact>(x[0]), nibble0<kExact>(x[1]));
                product<true, false>(o[4 * gr + 1], ps, nibble1<kExact>(x[0]), nibble1<kExact>(x[1]));
                product<true, false>(o[4 * gr + 2], ps, nibble0<kExact>(y0), nibble0<kExact>(y1));
                product<true, false>(o[4 * gr + 3], ps, nibble1<kExact>(y0), nibble1<kExact>(y1));
            }
        } else {
#pragma unroll
            for (int j = 0; j < G * 4; ++j) {  // channels 8 j .. 8 j + 7, column n of them at lane n = g
                uint32_t v0[kK], v1[kK];
                if constexpr (STORAGE == BST_DTYPE_BF16) {
                    // Lanes 0-15 name the rows; the transposed 8x8 pair is this lane's fragment.
                    const int r = lane & 15;
                    const uint32_t addr = vs + r * L::kRowBytes + swizzled<STORAGE, HD>(r, j) * 16;
                    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];"
                                 : "=r"(v0[0]), "=r"(v1[0]) : "r"(addr));
                } else {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 2 * t + (i & 1) + 8 * (i >> 1);
                        const int chunk = 2 * j + (g >> 2);
                        asm volatile("ld.shared.f32 %0, [%1];"
                                     : "=f"(v[i])
                                     : "r"(vs + r * L::kRowBytes + swizzled<STORAGE, HD>(r, chunk) * 16 +
                                           (g & 3) * 4));
                    }
                    terms_of<kK>(v[0], v[1], v0);
                    terms_of<kK>(v[2], v[3], v1);
                }
                product<false, false>(o[j], pa, v0[0], v1[0]);
#pragma unroll
                for (int i = 1; i < kK; ++i) {
                    leading<R, kTerms>(o[j], pa, v0[i], v1[i]);
                }
            }
        }
        __syncwarp();
        fetch(next, (stage + L::kStages - 1) % L::kStages);
        next += kWarps;
        stage = (stage + 1) % L::kStages;
    }
    cp_wait<0>();
    __syncthreads();  // the rings become the merge buffer

    // The warps' results: [warp][row][HD outputs, maximum, sum].
    float* merge = reinterpret_cast<float*>(smem);
    float largest_result = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        total[r] += __shfl_xor_sync(kFull, total[r], 1);
        total[r] += __shfl_xor_sync(kFull, total[r], 2);
        if constexpr (L::kCodes) {
            poison[r] |= __shfl_xor_sync(kFull, poison[r], 1);
            poison[r] |= __shfl_xor_sync(kFull, poison[r], 2);
        }
        float* mine = merge + (warp * ROWS + g + 8 * r) * (HD + 2);
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            float low = 0.0f, by = 1.0f;
            if constexpr (L::kCodes) {
                // The sum of lows of group gr is column gr: entry gr & 1 of lane t = gr / 2.
                if constexpr (kExact) {
                    low = middles[gr] + __shfl_xor_sync(kFull, middles[gr], 1);
                    low += __shfl_xor_sync(kFull, low, 2);
                } else {
                    low = __shfl_sync(kFull, entry<R, kTerms>(lows, r, gr & 1), (lane & ~3) | (gr >> 1));
                    if ((poison[r] >> gr) & 1u) low = NAN;
                }
                by = 1.0f / shrink[r][gr];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // Columns 2 t and 2 t + 1: channels 4 n + j of the group (codes) or 8 j + n.
                const int c0 = L::kCodes ? 32 * gr + 8 * t + j : 32 * gr + 8 * j + 2 * t;
                constexpr int N = L::kCodes ? kHalf : kTerms;
                // Nibbles 0 and 2 count 2^-24, 1 and 3 16 times that.
                const float unit = !L::kCodes || kExact ? 1.0f : (j & 1 ? 0x1p20f : 0x1p24f);
                const float y0 = fmaf(entry<R, N>(o[4 * gr + j], r, 0) * unit, by, low);
                const float y1 = fmaf(entry<R, N>(o[4 * gr + j], r, 1) * unit, by, low);
                mine[c0] = y0;
                mine[c0 + (L::kCodes ? 4 : 1)] = y1;
                largest_result = max_nan(largest_result, max_nan(fabsf(y0), fabsf(y1)));
            }
        }
        if (t == 0) {
            mine[HD] = top[r];
            mine[HD + 1] = total[r];
        }
        largest_result = max_nan(largest_result, total[r]);
    }
    if constexpr (L::kCodes) {
        __syncthreads();
    } else if (__syncthreads_or(!(largest_result <= FLT_MAX)) &&
               __syncthreads_or(meets_infinity<T, STORAGE, HD>(
                   kb, vb, seen, b0, b1, q + tile.first * q_stride + (kvh * group + tile.r0) * HD, rows))) {
        // The terms of an infinity, and of a float that bf16 rounds to one, leave NaN where the formula
        // may have a weight of zero, an infinity or a number (a NaN leaves what it should): the CTA's sums
        // again, a warp a row.
        using S = typename std::conditional<STORAGE == BST_DTYPE_F32, float, __nv_bfloat16>::type;
        for (int r = warp; r < rows; r += kWarps) {
            // A sequence has one token here.
            const T* src = q + tile.first * q_stride + (kvh * group + tile.r0 + r) * HD;
            attend_plainly<T, S, HD>(reinterpret_cast<const S*>(kb), reinterpret_cast<const S*>(vb), src,
                                     a.scale * kLog2e, seen, b0, b1, merge + r * (HD + 2));
            for (int w = 1; w < kWarps && lane == 0; ++w) {
                float* none = merge + (w * ROWS + r) * (HD + 2);
                none[HD] = -INFINITY;
                none[HD + 1] = 0.0f;
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < rows * HD; i += kThreads) {
        const int r = i / HD, ch = i % HD;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, merge[(w * ROWS + r) * (HD + 2) + HD]);
        float sum = 0.0f, value = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* from = merge + (w * ROWS + r) * (HD + 2);
            const float f = from[HD] == -INFINITY ? 0.0f : exp2_fast(from[HD] - m);
            // A warp that saw no key has nothing to add, not even zero times its output.
            if (from[HD] != -INFINITY || from[HD + 1] != 0.0f) {
                sum = fmaf(from[HD + 1], f, sum);
                value = fmaf(from[ch], f, value);
            }
        }
        const int query = tile.r0 + r, my_token = tile.n == 1 ? 0 : query / group;
        const int64_t token = tile.first + my_token;
        const int head = kvh * group + query - my_token * group;
        if (splits == 1) {
            put(out + token * out_stride + head * HD + ch, sum == 0.0f ? 0.0f : value / sum);
        } else {
            float* to = part + ((token * a.heads + head) * splits + split) * (HD + 2);
            to[ch] = value;
            if (ch == 0) {
                to[HD] = m;
                to[HD + 1] = sum;
            }
        }
    }
}

// ---- one query a key head ------------------------------------------------------------------------
// Where a key head has one query the tensor cores' other rows would be empty, so this kernel multiplies
// on the ordinary units, two operations a value: a nibble masked out of its word is, as a float, the
// subnormal c 2^(4 i - 149), and the other factor of the fused multiply-add (the query's channel, or
// weight x step) carries the power of two that is missing. Both are normalised so that neither they
// nor the products leave float32's range: queries by a power of two of the row, steps by the largest
// so far. Sums start 8 times the other factors lower, as if the codes were c - 8 (the middle,
// low + 8 step, makes up for it): without that they cancel what the lows bring, and 256 rows of 385 keys
// came out with an error of 1.3e-6 (of their norm) instead of 4e-7.
// HD / 8 lanes take a key, a word of eight codes each, and the warp 256 / HD keys a pass. After eight
// passes the partial sums change places, half as many at every step, so that a lane ends with the
// whole sums of one key, its own: it loads that key's scales, finishes and masks the score, and hands
// weight x step back by shuffles. Words go to registers, the values' before the scores and the next
// keys' behind them.
// A query sees all keys of two ranges, sinks and window, so nothing inside them is masked; lanes behind
// the end take the last key with a weight of zero.
// 256 sequences of 257 to 512 keys of eight heads of 64 take 32 us where the kernel above took 45 (64 MB,
// 2.0 TB/s), in 1.4 waves of CTAs of unequal length, five warp instructions a value at 53-55 % of the issue
// slots; 64 sequences of 4000 keys of 16 heads 110 (153); 60 000 keys of
// 32 heads 51 (82). bf16, which is cheaper above, gains as well: 31 (45), 110 (134), 51 (72). Scaling in
// the lanes that hold the words, every scale loaded by eight of them, took 36 us for the first.
constexpr int kOneWarps = 2, kOneCtas = 20 / kOneWarps;  // warps a CTA, CTAs an SM

// Whether a call is for this kernel.
bool one_query(const Cache& c, const Batch& b, const AttnSpec& a) {
    return c.storage == BST_DTYPE_U4 && a.heads == a.kv_heads && !b.starts;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kOneWarps * 32, kOneCtas)
k_cached_one(Cache c, Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride,
             T* __restrict__ out, int64_t out_stride, int splits, float* __restrict__ part) {
    constexpr int G = HD / 32;
    constexpr int kLanes = HD / 8, kAtOnce = 32 / kLanes, kPasses = 8, kKeys = kAtOnce * kPasses;
    constexpr int kMine = kLanes < 8 ? 8 / kLanes : 1;  // keys of a lane
    constexpr int kSums = G == 1 ? 1 : 2;               // groups of a lane's word
    // Lanes with the same groups: all, or every other one.
    constexpr int kNext = G == 4 ? 2 : 1;
    __shared__ float merge[kOneWarps][HD + 2];
    const int seq = blockIdx.x, head = blockIdx.y, split = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int word = lane % kLanes, sub = lane / kLanes;
    const int row = b.rows ? __ldg(b.rows + seq) : seq;
    const int position = max(0, __ldg(b.lengths + seq)) - 1;
    const bool inside = row >= 0 && row < c.rows;
    const Visible seen(position, inside ? position : -1, c.slots, a.window, a.sinks);
    const int use = useful_splits(seen.blocks, splits);
    if (split >= use) return;
    // Places 0 .. sunk are the sinks before the window, the others the window's keys.
    const bool sees = inside && position >= 0 && position < c.slots;
    const int sunk = sees ? min(a.sinks, seen.first) : 0, skipped = seen.first - sunk;
    const int64_t places = sees ? static_cast<int64_t>(sunk) + seen.end - seen.first : 0;
    const int x0 = static_cast<int>(places * split / use), x1 = static_cast<int>(places * (split + 1) / use);

    const int64_t at = (static_cast<int64_t>(inside ? row : 0) * c.kv_heads + head) * c.slots;
    const char* const kb = static_cast<const char*>(c.k) + at * (HD / 2) + word * 4;
    const char* const vb = static_cast<const char*>(c.v) + at * (HD / 2) + word * 4;
    const int scale_offset = G == 4 ? (word & 1) * 8 : 0;
    const char* const ksb = static_cast<const char*>(c.k_scale) + at * (G * 4) + scale_offset;
    const char* const vsb = static_cast<const char*>(c.v_scale) + at * (G * 4) + scale_offset;
    const int my_pass = word * 8 / kLanes;  // and the one behind it with two keys a lane
    auto key_at = [&](int place) {
        place = min(place, x1 - 1);
        return static_cast<int64_t>(place + (place >= sunk ? skipped : 0));
    };
    // The words of the keys at places x + i kAtOnce + sub, and the scales of the lane's own.
    auto load = [&](int x, const char* codes, const char* scales, uint32_t (&w)[kPasses],
                    uint32_t (&sc)[kMine][kSums]) {
        if (x >= x1) return;
        if (x + kKeys <= x1 && (x >= sunk || x + kKeys <= sunk)) {
            const char* const from = codes + key_at(x + sub) * (HD / 2);
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                w[i] = __ldg(reinterpret_cast<const uint32_t*>(from + i * kAtOnce * (HD / 2)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPasses; ++i) {
                w[i] = __ldg(reinterpret_cast<const uint32_t*>(
                    codes + key_at(x + i * kAtOnce + sub) * (HD / 2)));
            }
        }
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
            const char* const from = scales + key_at(x + (my_pass + m) * kAtOnce + sub) * (G * 4);
            if constexpr (kSums == 1) {
                sc[m][0] = __ldg(reinterpret_cast<const uint32_t*>(from));
            } else {
                const uint2 both = __ldg(reinterpret_cast<const uint2*>(from));
                sc[m][0] = both.x;
                sc[m][1] = both.y;
            }
        }
    };
    uint32_t kw[kPasses] = {}, ks[kMine][kSums] = {};
    int x = x0 + warp * kKeys;
    load(x, kb, ksb, kw, ks);

    // The query's channels of this lane's eight nibbles: of group 0 (HD 32), or nibbles 0-3 of one
    // group and 4-7 of the next.
    auto channel = [&](int n) {
        if constexpr (G == 1) return 8 * word + n;
        if constexpr (G == 2) return 32 * (n >> 2) + 4 * word + (n & 3);
        return 32 * (2 * (word & 1) + (n >> 2)) + 4 * (word >> 1) + (n & 3);
    };
    float qv[8], qsum[2] = {0.0f, 0.0f}, below[2] = {0.0f, 0.0f}, largest = 0.0f;
    const T* const src = q + seq * q_stride + head * HD;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        qv[n] = to_f(src[channel(n)]);
        largest = fmaxf(largest, fabsf(qv[n]));
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(kFull, largest, o));
    // |q| < 1 then (2 at the upper end); products come out 2^-49 too small.
    const int e = max(min(static_cast<int>(__float_as_uint(largest) >> 23) - 126, 126), -100);
    const float to_one = __uint_as_float((127 - e) << 23);
    const float to_score = a.scale * kLog2e * __uint_as_float((127 + e) << 23);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        qv[n] *= to_one;
        qsum[kSums == 1 ? 0 : n >> 2] += qv[n];
        below[n >> 2] = fmaf(-8.0f * 0x1p-49f, qv[n], below[n >> 2]);
        qv[n] *= __uint_as_float((127u + 100u - 4u * (n & 3)) << 23);
    }
#pragma unroll
    for (int g = 0; g < kSums; ++g) {
#pragma unroll
        for (int o = kLanes / 2; o >= kNext; o >>= 1) qsum[g] += __shfl_xor_sync(kFull, qsum[g], o);
        qsum[g] *= 0x1p-49f;
    }

    float acc[8] = {}, middles[kSums] = {}, top = -INFINITY, total = 0.0f;
    float shrink = 0x1p127f;  // 2^110 over the power of two above the largest step so far, from 2^-17 on
    auto nibble = [](uint32_t w, int n) {  // of a word's half: c 2^(4 n - 149)
        return __uint_as_float(w & (15u << (4 * n)));
    };
    for (; x < x1; x += kOneWarps * kKeys) {
        uint32_t vw[kPasses] = {}, vs[kMine][kSums] = {};
        load(x, vb, vsb, vw, vs);
        float s[kSums][kPasses];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            float sum[2] = {below[0], below[1]};
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                sum[0] = fmaf(nibble(kw[i], n), qv[n], sum[0]);
                sum[1] = fmaf(nibble(kw[i] >> 16, n), qv[4 + n], sum[1]);
            }
            if constexpr (kSums == 1) {
                s[0][i] = sum[0] + sum[1];
            } else {
                s[0][i] = sum[0];
                s[1][i] = sum[1];
            }
        }
#pragma unroll
        for (int g = 0; g < kSums; ++g) {
#pragma unroll
            for (int n = kPasses, o = kLanes / 2; o >= kNext; o >>= 1) {
                n /= 2;
                const bool upper = lane & o;
#pragma unroll
                for (int i = 0; i < n; ++i) {
                    const float away = upper ? s[g][i] : s[g][i + n];
                    s[g][i] = (upper ? s[g][i + n] : s[g][i]) + __shfl_xor_sync(kFull, away, o);
                }
            }
        }
        float score[kMine], most = -INFINITY;
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
            score[m] = 0.0f;
#pragma unroll
            for (int g = 0; g < kSums; ++g) {
                const float step = low_of(ks[m][g]);
                score[m] += fmaf(step, s[g][m], fmaf(8.0f, step, high_of(ks[m][g])) * qsum[g]);
            }
            if constexpr (G == 4) score[m] += __shfl_xor_sync(kFull, score[m], 1);
            score[m] = score[m] * 0x1p49f * to_score;
            if (x + (my_pass + m) * kAtOnce + sub >= x1) score[m] = -INFINITY;
            most = fmaxf(most, score[m]);
        }
        load(x + kOneWarps * kKeys, kb, ksb, kw, ks);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(kFull, most, o));
        if (most > top) {
            const float keep = top == -INFINITY ? 0.0f : exp2_fast(top - most);
            top = most;
            total *= keep;
#pragma unroll
            for (int g = 0; g < kSums; ++g) middles[g] *= keep;
#pragma unroll
            for (int n = 0; n < 8; ++n) acc[n] *= keep;
        }
        const float base = top == -INFINITY ? 0.0f : top;
        float step = 0.0f;
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
#pragma unroll
            for (int g = 0; g < kSums; ++g) step = fmaxf(step, low_of(vs[m][g]));
        }
        if (__any_sync(kFull, step * shrink > 0x1p110f)) {
            step = warp_max(step);
            const uint32_t above = (__float_as_uint(step) & 0x7f800000u) + 0x00800000u;
            const float next = __uint_as_float(((127u + 110u + 127u) << 23) - above);  // 2^110 / above
            const float by = next / shrink;
            shrink = next;
#pragma unroll
            for (int n = 0; n < 8; ++n) acc[n] *= by;
        }
        float weight[kMine][kSums];  // x step
#pragma unroll
        for (int m = 0; m < kMine; ++m) {
            const float p = exp2_fast(score[m] - base);
            total += p;
#pragma unroll
            for (int g = 0; g < kSums; ++g) {
                const float step = low_of(vs[m][g]);
                weight[m][g] = p * shrink * step;
                middles[g] = fmaf(p, fmaf(8.0f, step, high_of(vs[m][g])), middles[g]);
            }
        }
        float w[kPasses][kSums], whole[kSums] = {};
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int owner = sub * kLanes + i * kLanes / 8 + (G == 4 ? word & 1 : 0);
#pragma unroll
            for (int g = 0; g < kSums; ++g) {
                w[i][g] = __shfl_sync(kFull, weight[i % kMine][g], owner);
                whole[g] += w[i][g];
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) acc[n] = fmaf(-nibble(0x8888u, n & 3), whole[n / 4 % kSums], acc[n]);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                acc[n] = fmaf(nibble(vw[i], n), w[i][0], acc[n]);
                acc[4 + n] = fmaf(nibble(vw[i] >> 16, n), w[i][kSums - 1], acc[4 + n]);
            }
        }
    }

    // The lanes' sums, then the warps'. With four groups two lanes count every weight.
    total = warp_sum(total) * (G == 4 ? 0.5f : 1.0f);
#pragma unroll
    for (int g = 0; g < kSums; ++g) {
#pragma unroll
        for (int o = 16; o >= kNext; o >>= 1) middles[g] += __shfl_xor_sync(kFull, middles[g], o);
    }
    const float by = 1.0f / shrink;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
#pragma unroll
        for (int o = kLanes; o < 32; o <<= 1) acc[n] += __shfl_xor_sync(kFull, acc[n], o);
    }
    if (lane < kLanes) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            // acc has 2^(4 i - 149) and the normalisation in it.
            merge[warp][channel(n)] =
                acc[n] * 0x1p90f * by * __uint_as_float((127u + 59u - 4u * (n & 3)) << 23) +
                middles[kSums == 1 ? 0 : n >> 2];
        }
    }
    if (lane == 0) {
        merge[warp][HD] = top;
        merge[warp][HD + 1] = total;
    }
    __syncthreads();
    for (int ch = threadIdx.x; ch < HD; ch += kOneWarps * 32) {
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kOneWarps; ++w) m = fmaxf(m, merge[w][HD]);
        float sum = 0.0f, value = 0.0f;
#pragma unroll
        for (int w = 0; w < kOneWarps; ++w) {
            const float f = merge[w][HD] == -INFINITY ? 0.0f : exp2_fast(merge[w][HD] - m);
            // A warp that saw no key has nothing to add, and one whose scores are all NaN has that.
            if (merge[w][HD] != -INFINITY || merge[w][HD + 1] != 0.0f) {
                sum = fmaf(merge[w][HD + 1], f, sum);
                value = fmaf(merge[w][ch], f, value);
            }
        }
        if (splits == 1) {
            put(out + seq * out_stride + head * HD + ch, sum == 0.0f ? 0.0f : value / sum);
        } else {
            float* to = part + ((static_cast<int64_t>(seq) * a.heads + head) * splits + split) * (HD + 2);
            to[ch] = value;
            if (ch == 0) {
                to[HD] = m;
                to[HD + 1] = sum;
            }
        }
    }
}

// Joins the splits of a query, one CTA each: the splits' factors first, then every warp sums its
// share of the splits with all loads independent of one another.
constexpr int kMaxSplits = 512;

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads)
k_cached_join(Cache c, Batch b, AttnSpec a, int tile_rows, T* __restrict__ out,
              int64_t out_stride, int splits, const float* __restrict__ part) {
    constexpr int C = HD / 32;
    __shared__ float factor[kMaxSplits], tops[kWarps], sums[kWarps], values[kWarps][HD];
    const int token = blockIdx.x, head = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int seq, first, n;
    if (!find_sequence(b, token, &seq, &first, &n)) return;
    // How many splits the query's tile used, as k_cached found it.
    const int group = a.heads / a.kv_heads;
    const int row = b.rows ? __ldg(b.rows + seq) : seq;
    const int length = max(0, __ldg(b.lengths + seq));
    const int r0 = ((token - first) * group + head % group) / tile_rows * tile_rows;
    const int rows = min(tile_rows, n * group - r0);
    const int p_last = row >= 0 && row < c.rows ? length - n + (r0 + rows - 1) / group : -1;
    const Visible seen(length - n + r0 / group, p_last, c.slots, a.window, a.sinks);
    const int use = useful_splits(seen.blocks, splits);
    pdl_wait();
    const float* from =
        part + (static_cast<int64_t>(token) * a.heads + head) * splits * (HD + 2);
    float m = -INFINITY;
    for (int s = threadIdx.x; s < use; s += kThreads) m = fmaxf(m, from[s * (HD + 2) + HD]);
    m = warp_max(m);
    if (lane == 0) tops[warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    float sum = 0.0f;
    for (int s = threadIdx.x; s < use; s += kThreads) {
        const float top = from[s * (HD + 2) + HD], total = from[s * (HD + 2) + HD + 1];
        // A split that saw nothing has nothing to add; one whose scores are NaN has.
        const float f = top == -INFINITY ? (total == 0.0f ? 0.0f : total) : exp2_fast(top - m);
        factor[s] = f;
        sum = fmaf(total, f, sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    float value[C] = {};
#pragma unroll 8
    for (int s = warp; s < use; s += kWarps) {
        const float f = factor[s];
        const float* x = from + s * (HD + 2);
#pragma unroll
        for (int i = 0; i < C; ++i) value[i] = fmaf(x[lane + 32 * i], f, value[i]);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) values[warp][lane + 32 * i] = value[i];
    __syncthreads();
    T* to = out + token * out_stride + head * HD;
    if (threadIdx.x < HD) {
        const int ch = threadIdx.x;
        const float v = values[0][ch] + values[1][ch] + values[2][ch] + values[3][ch];
        put(to + ch, sum == 0.0f ? 0.0f : v / sum);
    }
}

// Query rows a tile: 16 where bf16 sequences have more than eight to a key head on average. For
// four tokens of four heads that took a step over 24 caches of up to 16 384 keys from 330 to 219 us.
int rows_of_tile(const Batch& b, const AttnSpec& a) {
    const int64_t group = a.heads / a.kv_heads;
    return a.dtype == BST_DTYPE_BF16 && b.tokens * group > 8ll * b.count ? 16 : 8;
}

// CTAs that an SM holds, by registers and shared memory.
int ctas_per_sm(const Cache& c, const Batch& b, const AttnSpec& a) {
    if (one_query(c, b, a)) return kOneCtas;
    const int size = c.head_dim == 128 ? 0 : (c.head_dim == 64 ? 1 : 2);
    return c.storage == BST_DTYPE_F32 ? 1 << size : (size == 0 ? 2 : (size == 1 ? 4 : 5));
}

// One full wave of CTAs where the tiles alone are fewer (131 000 keys of eight heads: two waves took
// 80 us, one 68 at that step), and among several sequences splits of at most 4096 keys, so that long ones
// spread over the SMs beside short ones; never less than 128 keys a split. The lengths are on the device,
// so the bound is what the cache and the window allow; tiles with fewer keys use fewer splits
// (useful_splits). Splits of 4096 keys end where a sequence's own tiles and their splits fill the card,
// and where their workspace would pass kSplitBytes: two prompts' chunks of 4096 tokens over 131 072 slots
// (32 heads of 128 over 8) took 4.4 GB, of which no SM had any use, and now take none.
constexpr int64_t kSplitBytes = 128 << 20;  // about what L2 holds
int split_count(const Cache& c, const Batch& b, const AttnSpec& a) {
    int64_t keys = c.slots;
    if (a.window) keys = std::min<int64_t>(keys, static_cast<int64_t>(a.window) + a.sinks + 2 * kBlock);
    const int64_t units = static_cast<int64_t>(tile_bound(b, a, rows_of_tile(b, a))) * a.kv_heads;
    const int64_t card = 148 * ctas_per_sm(c, b, a);
    const int64_t fill = card / std::max<int64_t>(units, 1);
    int64_t even = 1;
    if (b.count > 1) {
        const int64_t own = std::max<int64_t>(1, units / b.count);
        const int64_t split = static_cast<int64_t>(b.tokens) * a.heads * (a.head_dim + 2) * sizeof(float);
        even = std::min<int64_t>({(keys + 4095) / 4096, (card + own - 1) / own,
                                  std::max<int64_t>(1, kSplitBytes / std::max<int64_t>(split, 1))});
    }
    const int64_t most = std::max<int64_t>(1, keys / 128);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({std::max(fill, even), most, kMaxSplits})));
}

}  // namespace

size_t attention_cached_workspace(const Cache& c, const Batch& b, const AttnSpec& a) {
    const int splits = split_count(c, b, a);
    if (splits == 1) return 0;
    return static_cast<size_t>(b.tokens) * a.heads * splits * (a.head_dim + 2) * sizeof(float);
}

cudaError_t launch_attention_cached(cudaStream_t s, const Cache& c, const Batch& b,
                                    const AttnSpec& a, const void* q, int64_t q_stride, void* out,
                                    int64_t out_stride, void* workspace) {
    if (b.tokens < 1 || b.count < 1) return cudaSuccess;
    return by_dtype(a.dtype, [&](auto type) {
        using T = decltype(type);
        return by_head_dim(a.head_dim, [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            return by_storage(c.storage, [&](auto st) {
                constexpr int STORAGE = decltype(st)::value;
                using L = Layout<STORAGE, HD>;
                const int splits = split_count(c, b, a), rows = rows_of_tile(b, a);
                const dim3 grid(tile_bound(b, a, rows_of_tile(b, a)), a.kv_heads, splits);
                auto run = [&](auto tile_rows) {
                    constexpr int ROWS = decltype(tile_rows)::value;
                    const auto kernel = k_cached<T, STORAGE, HD, ROWS>;
                    const cudaError_t err = cudaFuncSetAttribute(
                        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(ROWS));
                    if (err) return err;
                    kernel<<<grid, kThreads, L::smem(ROWS), s>>>(
                        c, b, a, static_cast<const T*>(q), q_stride, static_cast<T*>(out), out_stride,
                        splits, static_cast<float*>(workspace));
                    return cudaGetLastError();
                };
                cudaError_t e;
                if (STORAGE == BST_DTYPE_U4 && one_query(c, b, a)) {
                    k_cached_one<T, HD><<<dim3(b.count, a.heads, splits), kOneWarps * 32, 0, s>>>(
                        c, b, a, static_cast<const T*>(q), q_stride, static_cast<T*>(out), out_stride,
                        splits, static_cast<float*>(workspace));
                    e = cudaGetLastError();
                } else if constexpr (sizeof(T) == 2) {
                    e = rows == 16 ? run(std::integral_constant<int, 16>())
                                   : run(std::integral_constant<int, 8>());
                } else {
                    e = run(std::integral_constant<int, 8>());
                }
                if (e || splits == 1) return e;
                return launch_pdl(k_cached_join<T, HD>, dim3(b.tokens, a.heads), dim3(kThreads), 0, s, c, b, a, rows, static_cast<T*>(out), out_stride,
                                  splits, static_cast<const float*>(workspace));
            });
        });
    });
}

}  // namespace bst
