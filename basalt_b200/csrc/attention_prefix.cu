// Attention of a whole batch's queries over one prefix, on tcgen05: the sums of attention_shared's first pass.
//
//   S = Q K^T,  P = exp2(S f - m),  O = P V  over a share of the prefix's keys; m the running maximum
//
// A CTA takes 256 query rows of one key head (tokens x heads of its group: every row sees every key, so nothing
// but the end of the prefix is masked) and a share of the keys, in tiles of 64: two M = 128 tiles of queries,
// whose scores, weights and outputs live in TMEM and take turns, as in attention over packed prompts. It leaves
// outputs, maximum and sum of weights of every row in float32; the shares are joined with the sequences' own
// keys' sums. Weights are bf16 (8 bits) in the product with bf16 values (a product's operands are of one type),
// whose rounding is of the size of bf16 outputs' own; maxima and sums are float32.
//
// A 4-bit prefix is unpacked on its way into shared memory by four warps in the copy's place, so that every key
// is unpacked once for 256 rows. Scores are good to float32: a key's channel is (c - 8) step + middle, of which
// the first, a code of 4 bits times a step of 8, is an fp16 number as it is; the middles, low + 8 step, are one more
// step of the product, sixteen deep: of every group the query's sum and the middle, both in two fp16 terms, whose
// smallest product is left out. Values and weights become fp16, 11 bits, values by one fused multiply-add for two
// of them, rounded once (with bf16 ones the error was 1.6 times the outputs' own rounding instead of 1.0). Powers
// of two keep all of it in fp16's range: one for each query row and each tile of keys, which the scores' factor f
// takes back; and one for the values of each group of 32 channels, that of the largest so far with two bits to spare,
// by which O is rescaled when a tile passes it. Entries far below those keep fewer bits: keys 2^-12 of the tile's largest
// are off by up to 2^-30 of that, values 2^-20 of the group's so far by 2^-38 of that. Where that could move a score by 2^-12
// or an output by 2^-11 of itself (sizes that no trained model has) the CTA's rows are added up again, plainly, which
// takes 200 times as long: 21 ms for 96 tokens of 32 heads behind 16 384 keys. Each of the four warps unpacks whole tiles by itself, so that they wait for one another nowhere.
//
// The same kernel takes several tokens of each sequence over its own 4-bit row (OWN): then rows see the keys up to
// their position, and every score may be kept.
//
// 256 tokens of 32 heads behind 32 768 bf16 keys of eight heads of 128 take 130 us (1060 TFLOP/s), 96 tokens behind
// 16 384 4-bit ones 59 (430), eight sequences' own 16 tokens over 1000 to 16 384 with scores 200 (their 127 MB
// included). Bound by a softmax thread's chain of dependent instructions, three warps a scheduler, with the tensor
// pipe busy for half, a quarter and a seventh of the time.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>

#include "attention_tc.cuh"
#include "operators.h"

namespace bst {
namespace {

constexpr int kRows = kTcTileRows;
// Warps 0-3 and 4-7: a tile's rows, a thread each; 8: products; 9 on: copies, or four warps that unpack.
constexpr int kSoft = 256, kUnpack = 128;
template <bool CODES>
constexpr int kThreadsOf = kSoft + 32 + (CODES ? kUnpack : 32);

template <int HD, bool CODES>
struct PrefixLayout {
    static constexpr int kQuery = 128 * HD * 2;       // a tile of query rows
    static constexpr int kTile = kTcKeys * HD * 2;    // a tile of keys or values
    static constexpr int kSlots = CODES ? 6 : 8;
    static constexpr int kBars = 2 * kQuery + kSlots * kTile;
    static constexpr int kFactors = kBars + 256;      // of rows, eight tiles of keys, eight tiles of values by groups
    // Middles: the queries' sums, [half][128 rows], and four tiles of keys, 32 bytes a row in the 32-byte swizzle.
    static constexpr int kSums = kFactors + (kRows + 64) * 4, kMiddles = kSums + (CODES ? 2 * 128 * 32 : 0);
    static constexpr int kRaw = kMiddles + (CODES ? 4 * kTcKeys * 32 : 0);
    // Codes and scales as the unpacking lanes copy them: [warp][stage][16-byte pieces][lane].
    static constexpr int kStages = 2, kPieces = HD / 16 + 4;
    static constexpr int kEnd = kRaw + (CODES ? kUnpack * kStages * kPieces * 16 : 0);
    // More than half of an SM's shared memory: one CTA an SM, which owns all of TMEM.
    static constexpr int kSmem = (kEnd > 120 * 1024 ? kEnd : 120 * 1024) + 1024;  // the base is aligned to 1024 bytes
    static_assert(kSums % 256 == 0, "swizzled tiles start at whole atoms");
    static_assert(kBars >= kRows * HD * 4, "outputs are staged where queries and the ring are");
};

// The channels of one head of one key of a 4-bit cache, for rows that are added up plainly.
__device__ __forceinline__ float code_value(const unsigned char* codes, const __nv_bfloat16* scales, int groups,
                                            int channel) {
    const int g = channel >> 5, h = (channel >> 2) & 7, j = channel & 3;
    const int byte = codes[(h * groups + g) * 2 + (j >> 1)];
    return fmaf(static_cast<float>(j & 1 ? byte >> 4 : byte & 15), __bfloat162float(scales[2 * g]),
                __bfloat162float(scales[2 * g + 1]));
}

// Two floats a register pair, and operations on both at once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void of_pair(uint64_t x, float* a, float* b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t sub_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t fma_f16x2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
// 2^e for e in [-126, 127], and the e for which |x| < 2^e, within [-100, 126].
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ __forceinline__ int exponent_above(uint32_t bits) {
    return max(min(static_cast<int>(bits >> 23) - 126, 126), -100);
}

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// One word of codes (nibble j of the low half: channel j of one group; of the high half: of the next) as 16 bytes of
// fp16, c step + low, or, of keys, (c - 8) step. The two groups' channels stay next to one another, so tiles hold
// channels in an order of their own: 16-byte place 4 y + x of a pair of groups has channels 8 x + 4 y .. + 3 of both,
// in turn. Queries are laid out alike, and outputs are put in order when they are written.
template <bool KEYS>
__device__ __forceinline__ uint4 unpack(uint32_t w, uint32_t step, uint32_t low) {
    constexpr uint32_t base = 0x64006400u;      // 1024; in an odd place a code counts 16 times
    constexpr uint32_t sixteenth = 0x2c002c00u, zero0 = KEYS ? 0x64086408u : base, zero1 = KEYS ? 0xd480d480u : 0xd400d400u;
    const uint32_t z = w >> 8;
    uint32_t x[4] = {(w & 0x000f000fu) | base, (w & 0x00f000f0u) | base, (z & 0x000f000fu) | base, (z & 0x00f000f0u) | base};
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // c or c - 8, exactly
        x[j] = j & 1 ? fma_f16x2(x[j], sixteenth, zero1) : sub_f16x2(x[j], zero0);
        x[j] = KEYS ? mul_f16x2(x[j], step) : fma_f16x2(x[j], step, low);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}

// Tiles of 32-byte rows in the 32-byte swizzle: atoms of eight rows, 256 bytes apart.
constexpr uint32_t kDesc32High = (256u >> 4) | (1u << 14) | (6u << 29);
__device__ __forceinline__ int middle_at(int row, int chunk) { return row * 32 + ((chunk ^ ((row >> 2) & 1)) << 4); }
// x in two fp16 terms, the first in the low half.
__device__ __forceinline__ uint32_t two_halves(float x) {
    const __half high = __float2half_rn(x);
    return half2_of(__half2float(high), x - __half2float(high));
}

template <int HD, bool CODES, bool OWN>
__global__ void __launch_bounds__(kThreadsOf<CODES>, 1)
k_prefix_tc(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, Prefix prefix,
            Batch b, AttnSpec a, const __nv_bfloat16* __restrict__ q, int64_t q_stride, int tiles, int splits,
            float* __restrict__ part, float* __restrict__ scores, int64_t pitch) {
    static_assert(CODES || !OWN, "own rows are in 4 bits");
    using L = PrefixLayout<HD, CODES>;
    constexpr int kBlocks = HD / 64;     // 128-byte columns of a tile
    extern __shared__ unsigned char raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads;
    // The tiles of a share of a head's keys stand next to one another, so that they read it together.
    const int kvh = blockIdx.x / tiles % a.kv_heads, split = blockIdx.x / tiles / a.kv_heads;
    int first, n, end;             // the tokens, and the keys that some row sees: those below `end`
    int64_t r0;
    int cache_row = prefix.row, position0 = 0;  // of OWN: the first token's position
    if constexpr (OWN) {
        Tile tile;
        if (!find_tile(b, group, kRows, blockIdx.x % tiles, &tile)) return;
        first = tile.first;
        n = tile.n;
        r0 = tile.r0;
        cache_row = b.rows ? __ldg(b.rows + tile.seq) : tile.seq;
        position0 = max(0, __ldg(b.lengths + tile.seq)) - n;
        end = 0;
    } else {
        pdl_trigger();  // the own keys' pass may fill what this one leaves free
        if (!owned_tokens(b, &first, &n)) return;
        r0 = static_cast<int64_t>(blockIdx.x % tiles) * kRows;
        if (r0 >= static_cast<int64_t>(n) * group) return;
        end = prefix.length;
    }
    const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), static_cast<int64_t>(n) * group - r0));
    if constexpr (OWN) end = tc_end(position0 + static_cast<int>((r0 + rows - 1) / group), cache_row, prefix.cache);
    const int all = (end + kTcKeys - 1) / kTcKeys, use = OWN ? tc_useful(end, splits) : splits;
    if (split >= use) return;
    const int t0 = static_cast<int>(static_cast<int64_t>(all) * split / use);
    const int key_tiles = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / use) - t0;
    const int sees_all = OWN ? position0 + static_cast<int>(r0 / group) : end - 1;  // keys up to it: every row
    const int halves = rows > 128 ? 2 : 1;

    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* const smem = raw + (base - smem_u32(raw));
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
    uint64_t* const full = bars;                 // [kSlots] a tile has arrived
    uint64_t* const empty = full + L::kSlots;    // [kSlots] its readers are done
    uint64_t* const s_full = empty + L::kSlots;  // [half][buffer] scores are done
    uint64_t* const p_full = s_full + 4;         // [half][buffer] weights are written
    uint64_t* const o_done = p_full + 4;         // [half] a product into O is done
    // [half] the last one is. (Its phase of o_done can be over, and the parity of the one before it be that of
    // the next, when a warp that was held up comes to wait for that.)
    uint64_t* const o_last = o_done + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(o_last + 2);
    int* const status = reinterpret_cast<int*>(tmem_slot + 1);  // [0] error code, [1] abort, [2] redo, [3] small values
    float* const row_factor = reinterpret_cast<float*>(smem + L::kFactors);   // what a row was divided by,
    float* const key_factor = row_factor + kRows;                             // a tile of keys, [8],
    float* const value_factor = key_factor + 8;                               // and of values and weights, [8][groups]

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kSlots; ++i) {
            mbar_init(full + i, CODES ? 32 : 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, kSoft / 2);
        }
        for (int i = 0; i < 4; ++i) mbar_init(o_done + i, 1);
        status[0] = status[1] = status[2] = status[3] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Token and head of the CTA's query row `at`: the quotient of two small numbers, in float.
    const int token0 = static_cast<int>(r0 / group), r_first = static_cast<int>(r0 - static_cast<int64_t>(token0) * group);
    const float by_group = 1.0f / static_cast<float>(group);
    auto place = [&](int at, int64_t* token, int* head) {
        const int x = static_cast<int>((static_cast<float>(r_first + at) + 0.5f) * by_group);
        *token = static_cast<int64_t>(first) + token0 + x;
        *head = kvh * group + r_first + at - x * group;
    };
    if (OWN && key_tiles == 0) {  // nobody sees a key
        for (int x = threadIdx.x; x < rows * (HD + 2); x += kThreadsOf<CODES>) {
            int64_t token;
            int head;
            place(x / (HD + 2), &token, &head);
            const int ch = x % (HD + 2);
            part[((token * a.heads + head) * splits + split) * (HD + 2) + ch] = ch == HD ? -INFINITY : 0.0f;
        }
        return;
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    __syncthreads();  // the barriers are there: copies may start
    // The tiles in the order in which they are used: K0 K1 V0 K2 V1 K3 ... V(n-1).
    const int copies = 2 * key_tiles;
    auto k_copy = [&](int i) { return i == 0 ? 0 : 2 * i - 1; };
    auto v_copy = [&](int i) { return i == key_tiles - 1 ? 2 * i + 1 : 2 * i + 2; };
    auto copy_of_keys = [&](int i) { return i == 0 || ((i & 1) && i != copies - 1); };
    auto copy_tile = [&](int i) {
        return i == 0 ? 0 : (copy_of_keys(i) ? (i + 1) / 2 : (i == copies - 1 ? key_tiles - 1 : i / 2 - 1));
    };
    auto copy = [&](int i) {
        const int slot = i % L::kSlots;
        mbar_expect_tx(full + slot, L::kTile);
        for (int x = 0; x < kBlocks; ++x) {
            tma_load_3d(copy_of_keys(i) ? &k_map : &v_map, full + slot,
                        smem + 2 * L::kQuery + slot * L::kTile + x * (kTcKeys * 128), 64 * x,
                        (t0 + copy_tile(i)) * kTcKeys, kvh);
        }
    };
    volatile int* const abort = status + 1;
    auto await = [&](int i, int code) {
        return mbar_wait(full + i % L::kSlots, (i / L::kSlots) & 1, status, code, abort);
    };
    if (!CODES && threadIdx.x == 9 * 32) {
        for (int i = 0; i < min(copies, L::kSlots); ++i) copy(i);
    }
    // Queries, 16-byte chunks into the swizzle, all loads of a thread at once. A negative scale moves
    // into them.
    if (threadIdx.x < kSoft) {
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        constexpr int kLoads = kRows * (HD / 8) / kSoft;
        uint4 x[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = (threadIdx.x + i * kSoft) / (HD / 8), c = threadIdx.x % (HD / 8);
            int64_t token;
            int head;
            place(at, &token, &head);
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (at < rows) x[i] = *reinterpret_cast<const uint4*>(q + token * q_stride + head * HD + 8 * c);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = (threadIdx.x + i * kSoft) / (HD / 8), c = threadIdx.x % (HD / 8), r = at & 127;
            uint32_t w[4] = {x[i].x ^ flip, x[i].y ^ flip, x[i].z ^ flip, x[i].w ^ flip};
            if constexpr (CODES) {
                // The row to fp16 below 2^8, by the exponent of its largest.
                uint32_t most = 0u;
#pragma unroll
                for (int y = 0; y < 4; ++y) most = max(most, max((w[y] << 16) & 0x7fff0000u, w[y] & 0x7fff0000u));
#pragma unroll
                for (int o = HD / 16; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(kFull, most, o));
                const int e = exponent_above(most);
                const float by = power_of_two(-e);
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    w[y] = half2_of(__uint_as_float(w[y] << 16) * by * 256.0f,
                                    __uint_as_float(w[y] & 0xffff0000u) * by * 256.0f);
                }
                // A query that is not finite makes every score NaN.
                if (c == 0) row_factor[at] = most >= 0x7f800000u ? NAN : power_of_two(e) * 0x1p-8f;
                // The sums of its groups: high terms, low ones, high ones again, zeros (four groups' places each).
                float sum = 0.0f;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const __half2 h = *reinterpret_cast<const __half2*>(&w[y]);
                    sum += __low2float(h) + __high2float(h);
                }
                sum += __shfl_xor_sync(kFull, sum, 1);
                sum += __shfl_xor_sync(kFull, sum, 2);
                if ((c & 3) == 0) {
                    constexpr int kSpare = 4 / (HD / 32);  // places a group fills, the others with zeros
                    const uint32_t terms = two_halves(sum);
                    unsigned char* const to = smem + L::kSums + (at >> 7) * (128 * 32);
#pragma unroll
                    for (int y = 0; y < kSpare; ++y) {
                        const int g = (c >> 2) + y * (HD / 32);
                        *reinterpret_cast<uint16_t*>(to + middle_at(r, 0) + 2 * g) = y == 0 ? terms & 0xffffu : 0u;
                        *reinterpret_cast<uint16_t*>(to + middle_at(r, 0) + 8 + 2 * g) = y == 0 ? terms >> 16 : 0u;
                        *reinterpret_cast<uint16_t*>(to + middle_at(r, 1) + 2 * g) = y == 0 ? terms & 0xffffu : 0u;
                        *reinterpret_cast<uint16_t*>(to + middle_at(r, 1) + 8 + 2 * g) = 0u;
                    }
                }
                // Places of keys: this thread's four channels and those of its neighbour's group, in turn.
                const bool odd = c & 4;
                const uint32_t other0 = __shfl_xor_sync(kFull, odd ? w[0] : w[2], 4);
                const uint32_t other1 = __shfl_xor_sync(kFull, odd ? w[1] : w[3], 4);
                const uint32_t a0 = odd ? other0 : w[0], a1 = odd ? other1 : w[1];
                const uint32_t b0 = odd ? w[2] : other0, b1 = odd ? w[3] : other1;
                w[0] = __byte_perm(a0, b0, 0x5410);
                w[1] = __byte_perm(a0, b0, 0x7632);
                w[2] = __byte_perm(a1, b1, 0x5410);
                w[3] = __byte_perm(a1, b1, 0x7632);
            }
            *reinterpret_cast<uint4*>(smem + (at >> 7) * L::kQuery + r * 128 + (c >> 3) * 16384 +
                                      (((c & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    if (warp >= 9) {
        if constexpr (!CODES) {
            if (lane == 0) {
                for (int i = L::kSlots; i < copies; ++i) {
                    if (!mbar_wait(empty + i % L::kSlots, ((i / L::kSlots) - 1) & 1, status, 1, abort)) break;
                    copy(i);
                }
            }
        } else {
            // Two warps take the keys' even and odd tiles, two the values'; a lane has two keys of a tile.
            constexpr int G = HD / 32, kChunks = HD / 32;  // chunks of 16 code bytes of a key
            const int u = warp - 9;
            const bool keys = u < 2;
            const char* const codes_at = static_cast<const char*>(keys ? prefix.cache.k : prefix.cache.v);
            const char* const scales_at = static_cast<const char*>(keys ? prefix.cache.k_scale : prefix.cache.v_scale);
            const int64_t at = (static_cast<int64_t>(cache_row) * a.kv_heads + kvh) * prefix.cache.slots;
            auto piece = [&](int stage, int x) {
                return base + L::kRaw + (((u * L::kStages + stage) * L::kPieces + x) * 32 + lane) * 16;
            };
            auto load = [&](int tile, int stage) {
                if (tile < key_tiles) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int key = (t0 + tile) * kTcKeys + 32 * half + lane;
                        const bool there = key < end;  // zeros behind it
                        const int64_t from = at + (there ? key : 0);
#pragma unroll
                        for (int x = 0; x < kChunks; ++x) {
                            cp_async<16>(piece(stage, half * kChunks + x), codes_at + from * (HD / 2) + 16 * x, there ? 16 : 0);
                        }
                        cp_async<G * 4>(piece(stage, 2 * kChunks + half), scales_at + from * (G * 4), there ? G * 4 : 0);
                        // The scales of the tile before, which the other warp unpacks.
                        if (!keys && tile > 0) {
                            cp_async<G * 4>(piece(stage, 2 * kChunks + 2 + half), scales_at + (at + key - kTcKeys) * (G * 4), G * 4);
                        }
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            auto scale_words = [&](int stage, int x, uint32_t (&w)[G]) {
                if constexpr (G == 4) {
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(piece(stage, x)));
                } else {
                    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(piece(stage, x)));
                }
            };
            // What a group's entries are at most: |low| + 15 step.
            auto top_of = [](uint32_t w) {
                return fmaf(15.0f, __uint_as_float(w << 16), fabsf(__uint_as_float(w & 0xffff0000u)));
            };
            // The exponents above the groups' largest entries in a tile (not of a NaN).
            auto exponents_of = [&](int stage, int x, int (&e)[G]) {
                uint32_t most[G] = {};
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t w[G];
                    scale_words(stage, x + half, w);
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float top = top_of(w[g]);
                        most[g] = max(most[g], top <= FLT_MAX ? __float_as_uint(top) : (isnan(top) ? 0u : 0x7f000000u));
                    }
                }
#pragma unroll
                for (int g = 0; g < G; ++g) e[g] = exponent_above(__reduce_max_sync(kFull, most[g]));
            };
            int below[G];  // values of the groups are below 2^this; what they are divided by goes with it
#pragma unroll
            for (int g = 0; g < G; ++g) below[g] = -1000;
            load(u & 1, 0);
            for (int tile = u & 1, stage = 0; tile < key_tiles; tile += 2, stage ^= 1) {
                load(tile + 2, stage ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
                __syncwarp();
                const int i = keys ? k_copy(tile) : v_copy(tile);
                float by[G];
                int e[G];
                if (!keys && tile > 0) {
                    exponents_of(stage, 2 * kChunks + 2, e);
#pragma unroll
                    for (int g = 0; g < G; ++g) below[g] = e[g] > below[g] ? e[g] + 2 : below[g];
                }
                exponents_of(stage, 2 * kChunks, e);
                if (keys) {
#pragma unroll
                    for (int g = 1; g < G; ++g) e[0] = max(e[0], e[g]);
                }
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    if (!keys) below[g] = e[g] > below[g] ? e[g] + 2 : below[g];
                    by[g] = power_of_two(keys ? 8 - e[0] : 15 - below[g]);
                }
                if (i >= L::kSlots && !mbar_wait(empty + i % L::kSlots, ((i / L::kSlots) - 1) & 1, status, 1, abort)) break;
                if (lane == 0) {
                    if (keys) {
                        key_factor[tile & 7] = power_of_two(e[0] - 8);
                    } else {
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            value_factor[(tile & 7) * 4 + g] = power_of_two(below[g] - 22);  // weights are 2^7 too large
                        }
                    }
                }
                bool small = false;  // whether an entry of the lane's keys has fewer bits
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    const int key = 32 * half + lane;
                    unsigned char* const to = smem + 2 * L::kQuery + (i % L::kSlots) * L::kTile + key * 128;
                    uint32_t scale[G], step[G / 2], low[G / 2];
                    scale_words(stage, 2 * kChunks + half, scale);
                    float key_top = 0.0f;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const float top = top_of(scale[g]);
                        key_top = fmaxf(key_top, top);
                        small |= !keys && top > 0.0f && top * by[g] < 0x1p-7f;
                    }
                    small |= keys && key_top > 0.0f && key_top * by[0] < 0x1p-4f;
                    if (OWN && !keys && (t0 + tile) * kTcKeys + key > sees_all) {
                        // Zero times a NaN is one: rows that do not see it must not get it, the others have to.
                        bool bad = false;
#pragma unroll
                        for (int g = 0; g < G; ++g) bad |= (scale[g] & 0x7f80u) == 0x7f80u || (scale[g] & 0x7f800000u) == 0x7f800000u;
                        if (bad) {
                            status[2] = 1;
#pragma unroll
                            for (int g = 0; g < G; ++g) scale[g] = 0u;
                        }
                    }
#pragma unroll
                    for (int g = 0; g < G; g += 2) {
                        step[g / 2] = half2_of(__uint_as_float(scale[g] << 16) * by[g], __uint_as_float(scale[g + 1] << 16) * by[g + 1]);
                        low[g / 2] = half2_of(__uint_as_float(scale[g] & 0xffff0000u) * by[g],
                                              __uint_as_float(scale[g + 1] & 0xffff0000u) * by[g + 1]);
                    }
                    if (keys) {
                        // Middles beside the queries' sums: high terms twice, low ones, zeros.
                        uint32_t terms[4] = {};
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            terms[g] = two_halves(fmaf(8.0f, __uint_as_float(scale[g] << 16), __uint_as_float(scale[g] & 0xffff0000u)) * by[0]);
                        }
                        unsigned char* const middle = smem + L::kMiddles + (tile & 3) * (kTcKeys * 32);
                        const uint32_t h0 = __byte_perm(terms[0], terms[1], 0x5410), h1 = __byte_perm(terms[2], terms[3], 0x5410);
                        *reinterpret_cast<uint4*>(middle + middle_at(key, 0)) = make_uint4(h0, h1, h0, h1);
                        *reinterpret_cast<uint4*>(middle + middle_at(key, 1)) =
                            make_uint4(__byte_perm(terms[0], terms[1], 0x7632), __byte_perm(terms[2], terms[3], 0x7632), 0u, 0u);
                    }
                    // A loop that is not unrolled: all warps together run at the rate at which instructions arrive.
                    auto unpack_all = [&](auto of_keys) {
                        constexpr bool KEYS = decltype(of_keys)::value;
#pragma unroll 1
                        for (int x = 0; x < kChunks; ++x) {
                            // Words of a chunk: two halves of eight channels by pairs of groups (128 channels), or
                            // four halves.
                            uint32_t w[4];
                            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                         : "r"(piece(stage, half * kChunks + x)));
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int g = G == 4 ? y : 0;               // pair of groups
                                const int eighth = G == 4 ? x : 2 * x + y;  // which eight of a group's 32 channels
                                unsigned char* const block = to + g * (kTcKeys * 128);
                                *reinterpret_cast<uint4*>(block + ((eighth ^ (key & 7)) << 4)) =
                                    unpack<KEYS>(w[G == 4 ? y : 2 * y], step[g], low[g]);
                                *reinterpret_cast<uint4*>(block + (((4 + eighth) ^ (key & 7)) << 4)) =
                                    unpack<KEYS>(w[G == 4 ? 2 + y : 2 * y + 1], step[g], low[g]);
                            }
                        }
                    };
                    if (keys) {
                        unpack_all(std::true_type());
                    } else {
                        unpack_all(std::false_type());
                    }
                }
                // The softmax's threads know what that means for their rows.
                if (__any_sync(kFull, small) && lane == 0) {
                    if (keys) {
                        key_factor[tile & 7] = -key_factor[tile & 7];
                    } else {
                        status[3] = 1;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(full + i % L::kSlots);
                __syncwarp();  // the stage has been read before it is loaded again
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
    } else if (warp == 8) {
        // The whole warp keeps time; one lane issues. Tiles are multiplied whole (what lies behind
        // their keys is masked), and all of TMEM starts at address 0, so that operands are constants but for
        // the slot.
        const int n_tiles = __shfl_sync(kFull, key_tiles, 0), n_halves = __shfl_sync(kFull, halves, 0);
        constexpr uint32_t s_idesc = tc_idesc(kTcKeys, false, CODES), o_idesc = tc_idesc(HD, true, CODES);
        const uint32_t q_desc = desc_k(base), kv_at = base + 2 * L::kQuery;
        auto slot = [&](int i) { return kv_at + (i % L::kSlots) * L::kTile; };
        auto scores = [&](int half, int i) {  // S = Q K^T
            const uint32_t d = half * 256 + (i & 1) * 64;
            const uint32_t qa = q_desc + half * (L::kQuery >> 4), ka = desc_k(slot(k_copy(i)));
#pragma unroll
            for (int k = 0; k < HD / 16; ++k) {
                tc_mma_ss(d, qa + (k >> 2) * (16384 >> 4) + (k & 3) * 2,
                          ka + (k >> 2) * (kTcKeys * 128 >> 4) + (k & 3) * 2, kDescHigh, s_idesc, k > 0);
            }
            if constexpr (CODES) {  // the middles
                tc_mma_ss(d, desc_k(base + L::kSums + half * (128 * 32)), desc_k(base + L::kMiddles + (i & 3) * (kTcKeys * 32)),
                          kDesc32High, s_idesc, true);
            }
            mma_commit(s_full + 2 * half + (i & 1));
        };
        bool ok = true;
        for (int i = 0; ok && i < min(2, n_tiles); ++i) {
            ok = await(k_copy(i), 2);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (elect_one()) {
                scores(0, i);
                if (n_halves > 1) scores(1, i);
                mma_commit(empty + k_copy(i) % L::kSlots);
            }
            __syncwarp();
        }
#pragma unroll 2
        for (int i = 0; ok && i < n_tiles; ++i) {
            const bool more = i + 2 < n_tiles;
            ok = await(v_copy(i), 3) && (!more || await(k_copy(i + 2), 4));
            const uint32_t va = desc_mn(slot(v_copy(i)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= n_halves || !ok) break;
                ok = mbar_wait(p_full + 2 * h + (i & 1), (i >> 1) & 1, status, 5, abort);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) {
                    const uint32_t p = h * 256 + (i & 1) * 64;
#pragma unroll
                    for (int k = 0; k < kTcKeys / 16; ++k) {  // O += P V
                        tc_mma_ts(h * 256 + 128, p + 8 * k, va + k * (2048 >> 4), kDescHigh, o_idesc,
                                  i > 0 || k > 0);
                    }
                    mma_commit(i + 1 < n_tiles ? o_done + h : o_last + h);
                    // Into the buffer that the product above has just read.
                    if (more) scores(h, i + 2);
                }
                __syncwarp();
            }
            if (ok && elect_one()) {
                mma_commit(empty + v_copy(i) % L::kSlots);
                if (more) mma_commit(empty + k_copy(i + 2) % L::kSlots);
            }
            __syncwarp();
        }
    } else {
        const int half = warp >> 2, in_tile = threadIdx.x & 127, at = 128 * half + in_tile;
        constexpr int kUnroll = CODES ? 1 : 2;
        const uint32_t s_at = tmem + half * 256 + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        const uint32_t o_at = s_at + 128;
        // A score's factor to base 2. It stays above zero: the mask's -infinity is multiplied by it.
        float scale = fabsf(a.scale) * kLog2e * (CODES ? row_factor[at] : 1.0f);
        constexpr int G = HD / 32;
        float top = -INFINITY, total = 0.0f, values_by[G];
#pragma unroll
        for (int g = 0; g < G; ++g) values_by[g] = 1.0f;
        // Keys that the row sees, and where its scores go.
        int sees = end;
        float* kept = nullptr;
        if constexpr (OWN) {
            int64_t token;
            int head;
            place(at, &token, &head);
            const int position = position0 + static_cast<int>(token - first);
            sees = at < rows && position < prefix.cache.slots ? position + 1 : 0;
            if (sees <= 0) scale = 0.0f;  // nothing of a query that sees nothing counts, its NaN neither
            if (at < rows) kept = scores + (token * a.heads + head) * pitch;
        }
        // A wait that runs out ends no loop here: the tile's threads meet at a barrier behind it, and
        // what they write then is computed again.
        bool ok = true;
        for (int i = 0; half < halves && i < key_tiles; ++i) {
            const uint32_t buffer = s_at + (i & 1) * 64;
            ok = ok && mbar_wait(s_full + 2 * half + (i & 1), (i >> 1) & 1, status, 7, abort);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            float by = CODES ? scale * key_factor[i & 7] : scale;
            if constexpr (CODES) {
                // Negative: some of the tile's keys have channels that are off by 2^-22, beside queries below 2^8.
                if (by < 0.0f) {
                    by = -by;
                    if (by * (HD * 0x1p-14f) > 0x1p-12f) status[2] = 1;
                }
            }
            by = by < FLT_MIN ? FLT_MIN : by;
            const int left = sees - (t0 + i) * kTcKeys;  // keys of the tile, or more
            // Scores are read twice, 32 at a time: 64 held, the registers that thirteen warps leave were spilled.
            auto columns = [&](int c, uint32_t (&s)[32]) {
                tmem_ld32(buffer + 32 * c, s);
                tmem_ld_wait();
                if (left < 32 * c + 32) {
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        if (32 * c + x >= left) s[x] = 0xff800000u;
                    }
                }
            };
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll kUnroll
            for (int c = 0; c < 2; ++c) {
                uint32_t s[32];
                columns(c, s);
                if constexpr (OWN) {
                    float* const to = kept + (t0 + i) * kTcKeys + 32 * c;
                    const int64_t room = pitch - static_cast<int64_t>(t0 + i) * kTcKeys - 32 * c;  // whole blocks of 16
#pragma unroll
                    for (int x = 0; x < 32; x += 4) {
                        if (kept && x < room) {
                            *reinterpret_cast<float4*>(to + x) = make_float4(__uint_as_float(s[x]) * by, __uint_as_float(s[x + 1]) * by,
                                                                             __uint_as_float(s[x + 2]) * by, __uint_as_float(s[x + 3]) * by);
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                    m[(x >> 1) & 3] = max3(m[(x >> 1) & 3], __uint_as_float(s[x]), __uint_as_float(s[x + 1]));
                }
            }
            const float most = fmaxf(max3(m[0], m[1], m[2]), m[3]) * by;
            // The maximum that weights are taken against moves only when a row's grows by more than 2^8 (a published
            // step of attention kernels for this architecture).
            const bool move = most > top + 8.0f || (top == -INFINITY && most > top);
            auto rescale = [&](const float (&keep)[G]) {
                ok = ok && mbar_wait(o_done + half, (i - 1) & 1, status, 8, abort);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t o[32];
                    tmem_ld32(o_at + 32 * c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int x = 0; x < 32; ++x) {  // columns of two groups in turn
                        o[x] = __float_as_uint(__uint_as_float(o[x]) * keep[c / 2 * 2 + (x & 1)]);
                    }
                    tmem_st16(o_at + 32 * c, o);
                    tmem_st16(o_at + 32 * c + 16, o + 16);
                }
                tmem_st_wait();  // a tile may rescale twice: the second time reads what the first has written
            };
            if (__any_sync(kFull, move)) {
                float keep[G];
                keep[0] = move ? (top == -INFINITY ? 0.0f : exp2_fast(top - most)) : 1.0f;
#pragma unroll
                for (int g = 1; g < G; ++g) keep[g] = keep[0];
                if (move) top = most;
                total *= keep[0];
                if (i > 0) rescale(keep);
            }
            // Weights for fp16 are 2^7 too large, and so is their sum.
            const float from = (CODES ? 7.0f : 0.0f) - (top == -INFINITY ? 0.0f : top);
            const uint64_t by2 = pair_of(by, by), from2 = pair_of(from, from);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll kUnroll
            for (int c = 0; c < 2; ++c) {
                uint32_t s[32], p[16];
                columns(c, s);
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const uint64_t y = fma2(pair_of(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1])), by2, from2);
                    float e0, e1;
                    of_pair(y, &e0, &e1);
                    e0 = exp2_fast(e0);
                    e1 = exp2_fast(e1);
                    sum[x & 1] = add2(sum[x & 1], pair_of(e0, e1));
                    p[x] = CODES ? half2_of(e0, e1) : pack2(e0, e1);
                }
                tmem_st16(buffer + 16 * c, p);
            }
            float sum0, sum1;
            of_pair(add2(sum[0], sum[1]), &sum0, &sum1);
            total += sum0 + sum1;
            if constexpr (CODES) {
                // Values of this tile that are divided by more than those before: what was summed has to be, too.
                // (The tile is there until these weights have been multiplied with it.)
                ok = ok && await(v_copy(i), 6);
                float keep[G];
                bool changed = false;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const float now = value_factor[(i & 7) * 4 + g];
                    keep[g] = values_by[g] / now;
                    changed |= now != values_by[g];
                    values_by[g] = now;
                }
                if (i > 0 && changed) rescale(keep);
            }
            tmem_st_wait();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(p_full + 2 * half + (i & 1));
        }
        if (half < halves) {
            // Products are done in order.
            ok = ok && mbar_wait(o_last + half, 0, status, 9, abort);
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // Both halves' products are done, so queries and ring may give way to the rows, which are then written whole.
        asm volatile("bar.sync 1, %0;" ::"n"(kSoft) : "memory");
        unsigned char* const rows_at = smem;
        if (half < halves) {
            float largest[G] = {};  // of the groups' outputs
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(o_at + 32 * c, o);
                tmem_ld_wait();
                if constexpr (CODES) {
                    if (status[3] != 0) {
#pragma unroll
                        for (int x = 0; x < 32; ++x) {
                            largest[c / 2 * 2 + (x & 1)] = fmaxf(largest[c / 2 * 2 + (x & 1)], fabsf(__uint_as_float(o[x])));
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * values_by[c / 2 * 2 + (x & 1)]);
                }
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    // Columns 32 c + 8 (x / 2) .. + 7, the even ones or the odd ones: four channels of a group.
                    const uint32_t* const y = o + 8 * (x >> 1);
                    int chunk = 8 * c + x;
                    uint4 z = make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
                    if constexpr (CODES) {
                        // Place 4 c' + x / 2 of pair c / 2: channels 64 (c / 2) + 32 (x & 1) + 8 (x / 2) + 4 c'.
                        chunk = 16 * (c >> 1) + 8 * (x & 1) + 2 * (x >> 1) + (c & 1);
                        z = x & 1 ? make_uint4(y[1], y[3], y[5], y[7]) : make_uint4(y[0], y[2], y[4], y[6]);
                    }
                    *reinterpret_cast<uint4*>(rows_at + at * (HD * 4) + ((chunk ^ (in_tile & 7)) << 4)) = z;
                }
            }
            if (CODES && status[3] != 0) {
                // Values as they were multiplied are off by up to 2^-25, and the sum of weights times that is the output's.
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    if (at < rows && largest[g] < total * 0x1p-14f) status[2] = 1;
                }
            }
            if (at < rows) {
                int64_t token;
                int head;
                place(at, &token, &head);
                float* const to = part + ((token * a.heads + head) * splits + split) * (HD + 2) + HD;
                *reinterpret_cast<float2*>(to) = make_float2(top, CODES ? total * 0x1p-7f : total);
            }
        }
        __syncwarp();
        // A warp writes the rows that its own threads staged.
        for (int r = 0; half < halves && r < 32; ++r) {
            const int row = 32 * warp + r;
            if (row >= rows) break;
            int64_t token;
            int head;
            place(row, &token, &head);
            float* const to = part + ((token * a.heads + head) * splits + split) * (HD + 2);
#pragma unroll
            for (int x = 0; x < HD / 64; ++x) {
                const int c = 2 * lane + 64 * x;  // channels c and c + 1
                *reinterpret_cast<float2*>(to + c) = *reinterpret_cast<const float2*>(
                    rows_at + row * (HD * 4) + (((c >> 2) ^ (row & 7)) << 4) + (c & 3) * 4);
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    const bool again = status[0] != 0 || status[2] != 0;
    if (status[0] != 0 && threadIdx.x == 0) {
        // A wait ran out: let the copies that were issued land before the memory goes away.
        const uint64_t start = global_ns();
        while (global_ns() - start < 2000000ull) {
        }
    }
    __syncthreads();
    if (warp == 8) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
    if (!again) return;
    // Its rows once more, plainly, a warp a row and a key at a time: slow, but right whatever the entries are.
    constexpr int C = HD / 32;
    const int64_t keys_at = (static_cast<int64_t>(cache_row) * a.kv_heads + kvh) * prefix.cache.slots;
    for (int r = warp; r < rows; r += kThreadsOf<CODES> / 32) {
        int64_t token;
        int head;
        place(r, &token, &head);
        float value[C] = {}, x[C], top = -INFINITY, total = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) x[i] = __bfloat162float(q[token * q_stride + head * HD + lane + 32 * i]);
        int stop = min(end, (t0 + key_tiles) * kTcKeys);
        if constexpr (OWN) {
            const int position = position0 + static_cast<int>(token - first);
            stop = position < prefix.cache.slots ? min(stop, position + 1) : 0;
        }
        for (int key = t0 * kTcKeys; key < stop; ++key) {
            auto read = [&](const void* values, const void* scales, int channel) {
                if constexpr (CODES) {
                    return code_value(static_cast<const unsigned char*>(values) + (keys_at + key) * (HD / 2),
                                      static_cast<const __nv_bfloat16*>(scales) + (keys_at + key) * (HD / 16), C, channel);
                } else {
                    return __bfloat162float(static_cast<const __nv_bfloat16*>(values)[(keys_at + key) * HD + channel]);
                }
            };
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < C; ++i) s = fmaf(x[i], read(prefix.cache.k, prefix.cache.k_scale, lane + 32 * i), s);
            s = warp_sum(s) * a.scale * kLog2e;
            if (OWN && lane == 0) scores[(token * a.heads + head) * pitch + key] = s;
            const float up = fmaxf(top, s), keep = top == -INFINITY ? 0.0f : exp2f(top - up);
            const float p = s == -INFINITY ? 0.0f : exp2f(s - up);
            top = up;
            total = fmaf(total, keep, p);
#pragma unroll
            for (int i = 0; i < C; ++i) {
                value[i] *= keep;
                if (p != 0.0f || isnan(p)) value[i] = fmaf(p, read(prefix.cache.v, prefix.cache.v_scale, lane + 32 * i), value[i]);
            }
        }
        float* const to = part + ((token * a.heads + head) * splits + split) * (HD + 2);
#pragma unroll
        for (int i = 0; i < C; ++i) to[lane + 32 * i] = value[i];
        if (lane == 0) {
            to[HD] = top;
            to[HD + 1] = total;
        }
    }
}

template <int HD, bool CODES, bool OWN>
cudaError_t run(cudaStream_t s, const Prefix& p, const Batch& b, const AttnSpec& a, const __nv_bfloat16* q,
                int64_t q_stride, int tiles, int splits, float* part, float* scores, int64_t pitch) {
    using L = PrefixLayout<HD, CODES>;
    CUtensorMap k_map{}, v_map{};
    if constexpr (!CODES) {
        const int64_t head = static_cast<int64_t>(p.cache.slots) * HD * 2, row = head * a.kv_heads * p.row;
        // Keys behind the prefix lie outside the maps and read as zeros, whatever their slots hold.
        cudaError_t e = make_head_map(&k_map, static_cast<const char*>(p.cache.k) + row, a.kv_heads, p.length, HD,
                                      head, kTcKeys);
        if (!e) {
            e = make_head_map(&v_map, static_cast<const char*>(p.cache.v) + row, a.kv_heads, p.length, HD, head,
                              kTcKeys);
        }
        if (e) return e;
    }
    const auto kernel = k_prefix_tc<HD, CODES, OWN>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
    if (e) return e;
    kernel<<<tiles * a.kv_heads * splits, kThreadsOf<CODES>, L::kSmem, s>>>(k_map, v_map, p, b, a, q, q_stride, tiles,
                                                                          splits, part, scores, pitch);
    return cudaGetLastError();
}

}  // namespace

int prefix_tc_tiles(const Batch& b, const AttnSpec& a) {
    const int64_t queries = static_cast<int64_t>(b.tokens) * (a.heads / a.kv_heads);
    return static_cast<int>((queries + kRows - 1) / kRows);
}

bool prefix_tc_takes(const Prefix& p, const AttnSpec& a) {
    return a.dtype == BST_DTYPE_BF16 && a.head_dim >= 64 && p.cache.storage != BST_DTYPE_F32 && a.scale != 0.0f;
}

cudaError_t launch_prefix_tc(cudaStream_t s, const Prefix& p, const Batch& b, const AttnSpec& a, const void* q_,
                             int64_t q_stride, int tiles, int splits, float* part) {
    const __nv_bfloat16* const q = static_cast<const __nv_bfloat16*>(q_);
    const bool codes = p.cache.storage == BST_DTYPE_U4;
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        return codes ? run<HD, true, false>(s, p, b, a, q, q_stride, tiles, splits, part, nullptr, 0)
                     : run<HD, false, false>(s, p, b, a, q, q_stride, tiles, splits, part, nullptr, 0);
    };
    return a.head_dim == 128 ? go(std::integral_constant<int, 128>()) : go(std::integral_constant<int, 64>());
}

bool own_tc_takes(const Cache& c, const Batch& b, const AttnSpec& a) {
    return c.storage == BST_DTYPE_U4 && a.dtype == BST_DTYPE_BF16 && a.head_dim >= 64 && a.scale != 0.0f &&
           a.window == 0 && b.starts;
}

cudaError_t launch_own_tc(cudaStream_t s, const Cache& c, const Batch& b, const AttnSpec& a, const void* q_,
                          int64_t q_stride, int splits, float* part, float* scores, int64_t pitch) {
    const __nv_bfloat16* const q = static_cast<const __nv_bfloat16*>(q_);
    Prefix p;
    p.cache = c;
    const int tiles = tile_bound(b, a, kRows);
    return a.head_dim == 128 ? run<128, true, true>(s, p, b, a, q, q_stride, tiles, splits, part, scores, pitch)
                             : run<64, true, true>(s, p, b, a, q, q_stride, tiles, splits, part, scores, pitch);
}

}  // namespace bst
