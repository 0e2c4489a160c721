// Causal attention of packed sequences over their own keys and values, with a sliding window and a
// few first tokens that stay visible.
//
//   out[i] = sum_j p_ij v_j,  p_ij = exp(s_ij - max_j s_ij) / sum_j exp(s_ij - max_j s_ij),
//   s_ij = scale q_i . k_j over the keys j that query i sees; zeros when it sees none.
//
// A running maximum and sum per query let every kernel read each key and value once; a key that a
// query does not see takes no part at all, whatever it holds (NaN and infinities included), and those
// that it sees count as in float32 arithmetic.

#include <cuda_bf16.h>

#include <algorithm>
#include <cfloat>

#include "attention.cuh"
#include "attention_tc.cuh"
#include "device.cuh"
#include "operators.h"
#include "sm100.cuh"

namespace bst {
namespace {

// The key tiles of a CTA: the sinks before its window, then the window; a tile is up to KEYS keys
// from key(i), cols(i) of them (a multiple of STEP) multiplied.
template <int KEYS, int STEP>
struct KeyTiles {
    int first, end;      // the window's keys
    int sink_end;        // sinks before it
    int sink_tiles, tiles;
    __device__ KeyTiles(int p0, int p1, int window, int sinks) {
        end = p1 + 1;
        first = window ? max(0, p0 - window + 1) : 0;
        sink_end = min(sinks, first);
        sink_tiles = (sink_end + KEYS - 1) / KEYS;
        tiles = sink_tiles + (end - first + KEYS - 1) / KEYS;
    }
    __device__ int key(int i) const {
        return i < sink_tiles ? i * KEYS : first + (i - sink_tiles) * KEYS;
    }
    __device__ int stop(int i) const { return i < sink_tiles ? sink_end : end; }
    __device__ int cols(int i) const { return min(KEYS, (stop(i) - key(i) + STEP - 1) / STEP * STEP); }
    // Whether queries at positions p0..p1 see all of the tile's columns.
    __device__ bool whole(int i, int p0, int p1, int window) const {
        const int at = key(i), n = cols(i);
        return at + n - 1 <= p0 && (i < sink_tiles ? at + n <= sink_end
                                                   : window == 0 || p1 - at < window);
    }
};

// ---- bf16 on the tensor cores ----------------------------------------------------------------
// A CTA takes 256 query rows of one key head: tokens x heads of its group, so that heads sharing keys
// share their tiles, and a tile of few tokens wastes little of a window. They are two M = 128 tiles;
// four warps a tile turn scores into weights. Keys and values come in tiles of 64 by TMA through a
// ring of 128-byte-swizzled buffers.
//   TMEM, per tile: two buffers of scores S (64 columns each, float32), whose place the weights P
//   take as bf16 and from where the second product reads them as its A operand, and the output O
//   (head_dim columns). The next tile's scores are computed while a tile's weights are, so that the
//   softmax, which is the longer part, never waits for a product it has just fed.
//   O = P V reads V as it lies in memory (its B operand is MN-major).
// The maximum that weights are taken against moves only when a row's grows by more than 2^8: the
// softmax then waits for the last product into O and rescales O itself.
// What bounds it: per 128 keys the exponentials (32 768 at 16 a cycle, 2048 cycles) beside the
// products (4 x 128 x 128 x 128 multiply-adds, 2048 cycles at the nominal rate; the scores' half
// takes half as long again, because 64 columns a product read Q from shared memory twice as often).
// 8192 tokens of 16 heads over 4 of 128, window 1024: 115 us, 0.34 of the measured bf16 rate, in four
// waves of 18 tiles a CTA, a third of whose time is its beginning and end. (CTAs of 128 rows, two an SM
// with half of TMEM each, took 121: the rings then hold half as many tiles.)
//
// Weights of keys that a row does not see are zero, but zero times a NaN or infinity is NaN. Tiles
// that are partly hidden are searched for such values first; a CTA that meets one, or whose waits
// run out, raises its flag, and the plain kernel behind this one computes its rows again.

constexpr int kTcRows = 256;
// Warps 0-3 and 4-7: a tile's rows, a thread each; 8: products; 9: copies. (Two threads a row were
// slower: their meeting in every step kept both tiles' softmaxes in step with one another.)
constexpr int kTcSoft = 256, kTcThreads = kTcSoft + 64;

template <int HD>
struct TcLayout {
    static constexpr int kQuery = 128 * HD * 2;       // a tile of query rows
    static constexpr int kTile = kTcKeys * HD * 2;    // a tile of keys or values
    static constexpr int kSlots = 8;
    static constexpr int kBars = 2 * kQuery + kSlots * kTile;
    // More than half of an SM's shared memory: one CTA an SM, which owns all of TMEM.
    static constexpr int kEnd = kBars + 256;
    static constexpr int kBytes = kEnd > 120 * 1024 ? kEnd : 120 * 1024;
    static constexpr int kSmem = kBytes + 1024;       // the base is aligned to 1024 bytes
};

// The lowest n of 32 bits, for any n.
__device__ __forceinline__ uint32_t first_bits(int n) {
    return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
}

__device__ __forceinline__ bool not_finite(uint32_t pair) {  // of two bf16
    return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u;
}

template <int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
k_packed_tc(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
            Batch b, AttnSpec a, const __nv_bfloat16* __restrict__ q, int64_t q_stride,
            __nv_bfloat16* __restrict__ out, int64_t out_stride, int* __restrict__ flags) {
    using L = TcLayout<HD>;
    constexpr int kBlocks = HD / 64;     // 128-byte columns of a tile
    extern __shared__ unsigned char raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = a.heads / a.kv_heads, tiles = gridDim.x / a.kv_heads;
    // The last tiles of all heads first: a sequence's first ones see the fewest keys and fill the end
    // (4096 tokens of eight heads, no window: 534 -> 474 us in float32, 279 -> 274 for 8192 in bf16).
    const int place_of = blockIdx.x / a.kv_heads, kvh = blockIdx.x - place_of * a.kv_heads;
    const int index = tiles - 1 - place_of;
    int* const flag = flags + kvh * tiles + index;
    Tile tile;
    if (!find_tile(b, group, kTcRows, index, &tile)) {
        if (threadIdx.x == 0) *flag = 0;
        return;
    }
    const int rows = min(kTcRows, tile.n * group - tile.r0);
    const int p0 = tile.r0 / group, p1 = (tile.r0 + rows - 1) / group;
    const KeyTiles<kTcKeys, kTcKeys> keys(p0, p1, a.window, a.sinks);
    // The second tile of a short CTA has no rows: then all is done for the first alone.
    const int halves = rows > 128 ? 2 : 1;

    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char* const smem = raw + (base - smem_u32(raw));
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
    uint64_t* const full = bars;                 // [kSlots] a copy has arrived
    uint64_t* const empty = full + L::kSlots;    // [kSlots] its readers are done
    uint64_t* const s_full = empty + L::kSlots;  // [tile][buffer] scores are done
    uint64_t* const p_full = s_full + 4;         // [tile][buffer] weights are written
    uint64_t* const o_done = p_full + 4;         // [tile] a product into O is done
    // [tile] the last one is. (Its phase of o_done can be over, and the parity of the one before it be that of
    // the next, when a warp that was held up comes to wait for that.)
    uint64_t* const o_last = o_done + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(o_last + 2);
    int* const status = reinterpret_cast<int*>(tmem_slot + 1);  // [0] error code, [1] abort, [2] redo

    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kSlots; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, kTcSoft / 2);
        }
        for (int i = 0; i < 4; ++i) mbar_init(o_done + i, 1);
        status[0] = status[1] = status[2] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // Token and head of the CTA's query row `at`: the quotient of two small numbers, in float.
    const int r_first = tile.r0 - p0 * group;
    const float by_group = 1.0f / static_cast<float>(group);
    auto place = [&](int at, int* token, int* head) {
        const int n = static_cast<int>((static_cast<float>(r_first + at) + 0.5f) * by_group);
        *token = p0 + n;
        *head = kvh * group + r_first + at - n * group;
    };
    __syncthreads();  // the barriers are there: copies may start
    auto slot_at = [&](int i) { return base + 2 * L::kQuery + (i % L::kSlots) * L::kTile; };
    // The copies in the order in which they are used: K0 K1 V0 K2 V1 K3 ... V(n-1).
    const int copies = 2 * keys.tiles;
    auto k_copy = [&](int i) { return i == 0 ? 0 : 2 * i - 1; };
    auto v_copy = [&](int i) { return i == keys.tiles - 1 ? 2 * i + 1 : 2 * i + 2; };
    auto copy = [&](int i) {
        const bool of_keys = i == 0 || ((i & 1) && i != copies - 1);
        const int at = i == 0 ? 0 : (of_keys ? (i + 1) / 2 : (i == copies - 1 ? keys.tiles - 1 : i / 2 - 1));
        const int slot = i % L::kSlots;
        mbar_expect_tx(full + slot, L::kTile);
        for (int x = 0; x < kBlocks; ++x) {
            tma_load_2d(of_keys ? &k_map : &v_map, full + slot,
                        smem + 2 * L::kQuery + slot * L::kTile + x * (kTcKeys * 128),
                        kvh * HD + 64 * x, tile.first + keys.key(at));
        }
    };
    auto await = [&](int i, int code, volatile int* abort) {
        return mbar_wait(full + i % L::kSlots, (i / L::kSlots) & 1, status, code, abort);
    };
    if (threadIdx.x == 9 * 32) {
        for (int i = 0; i < min(copies, L::kSlots); ++i) copy(i);
    }
    // Queries, 16-byte chunks into the swizzle, all loads of a thread at once. A negative scale moves
    // into them.
    if (threadIdx.x < kTcSoft) {
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        constexpr int kLoads = kTcRows * (HD / 8) / kTcSoft;
        uint4 x[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = (threadIdx.x + i * kTcSoft) / (HD / 8), c = threadIdx.x % (HD / 8);
            int token, head;
            place(at, &token, &head);
            x[i] = make_uint4(0u, 0u, 0u, 0u);
            if (at < rows) {
                x[i] = *reinterpret_cast<const uint4*>(
                    q + (tile.first + static_cast<int64_t>(token)) * q_stride + head * HD + 8 * c);
            }
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = (threadIdx.x + i * kTcSoft) / (HD / 8), c = threadIdx.x % (HD / 8), r = at & 127;
            x[i].x ^= flip; x[i].y ^= flip; x[i].z ^= flip; x[i].w ^= flip;
            *reinterpret_cast<uint4*>(smem + (at >> 7) * L::kQuery + r * 128 + (c >> 3) * 16384 +
                                      (((c & 7) ^ (r & 7)) << 4)) = x[i];
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    volatile int* const abort = status + 1;
    if (warp == 9) {
        if (lane == 0) {
            for (int i = L::kSlots; i < copies; ++i) {
                if (!mbar_wait(empty + i % L::kSlots, ((i / L::kSlots) - 1) & 1, status, 1, abort)) break;
                copy(i);
            }
        }
    } else if (warp == 8) {
        // The whole warp keeps time; one lane issues. Tiles are multiplied whole (what lies behind
        // their keys is masked, or has weights of zero), and all of TMEM starts at address 0, so that
        // operands are constants but for the slot.
        const int n_tiles = __shfl_sync(kFull, keys.tiles, 0), n_halves = __shfl_sync(kFull, halves, 0);
        constexpr uint32_t s_idesc = tc_idesc(kTcKeys, false), o_idesc = tc_idesc(HD, true);
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
            mma_commit(s_full + 2 * half + (i & 1));
        };
        bool ok = true;
        for (int i = 0; ok && i < min(2, n_tiles); ++i) {
            ok = await(k_copy(i), 2, abort);
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
            ok = await(v_copy(i), 3, abort) && (!more || await(k_copy(i + 2), 4, abort));
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
        int my_token, my_head;
        place(at, &my_token, &my_head);
        const uint32_t s_at = tmem + half * 256 + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
        const uint32_t o_at = s_at + 128;
        const float scale = fabsf(a.scale) * kLog2e;
        // Rows behind the last query see nothing.
        const int position = at < rows ? my_token : -1;
        const int low = a.window ? position - a.window + 1 : 0;  // the window's first key
        const float slack = 8.0f / scale;                        // infinite for the smallest scales: never moved
        float top = -INFINITY, from = 0.0f, total = 0.0f;
        // A wait that runs out ends no loop here: the tile's threads meet at a barrier behind it, and
        // what they write then is computed again.
        bool ok = true;
        int key0 = keys.key(0);
        for (int i = 0; half < halves && i < keys.tiles; ++i) {
            const uint32_t buffer = s_at + (i & 1) * 64;
            // Most tiles lie inside every row's window and have all of their columns.
            const bool inside = i >= keys.sink_tiles && key0 + kTcKeys - 1 <= p0 &&
                                (a.window == 0 || p1 - key0 < a.window);
            uint32_t s[2][32];
            if (inside) {
                ok = ok && mbar_wait(s_full + 2 * half + (i & 1), (i >> 1) & 1, status, 7, abort);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tmem_ld32(buffer, s[0]);
                tmem_ld32(buffer + 32, s[1]);
                tmem_ld_wait();
            } else {
                // The CTA's softmax threads search the values for what is not finite.
                ok = ok && await(v_copy(i), 6, abort);
                const uint4* v = reinterpret_cast<const uint4*>(smem + 2 * L::kQuery +
                                                                (v_copy(i) % L::kSlots) * L::kTile);
                bool bad = false;
                for (int x = threadIdx.x; x < L::kTile / 16; x += kTcSoft / 2 * halves) {
                    const uint4 u = v[x];
                    bad |= not_finite(u.x) || not_finite(u.y) || not_finite(u.z) || not_finite(u.w);
                }
                if (bad) status[2] = 1;
                ok = ok && mbar_wait(s_full + 2 * half + (i & 1), (i >> 1) & 1, status, 7, abort);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tmem_ld32(buffer, s[0]);
                tmem_ld32(buffer + 32, s[1]);
                tmem_ld_wait();
                // The columns' visibility as bits: below `last`, and from `low` on or below the sinks.
                const int last = i < keys.sink_tiles ? min(position, keys.sink_end - 1) : position;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int first = key0 + 32 * c;
                    const uint32_t see = first_bits(last + 1 - first) &
                                         (~first_bits(low - first) | first_bits(a.sinks - first));
#pragma unroll
                    for (int x = 0; x < 32; ++x) {
                        if (!((see >> x) & 1u)) s[c][x] = 0xff800000u;
                    }
                }
            }
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int x = 0; x < 64; ++x) m[x & 3] = fmaxf(m[x & 3], __uint_as_float(s[x >> 5][x & 31]));
            const float most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            const bool move = most > top + slack || (top == -INFINITY && most > top);
            if (__any_sync(kFull, move)) {
                const float keep = move ? (top == -INFINITY ? 0.0f : exp2_fast((top - most) * scale)) : 1.0f;
                if (move) {
                    top = most;
                    from = top * scale;
                }
                total *= keep;
                if (i > 0) {
                    ok = ok && mbar_wait(o_done + half, (i - 1) & 1, status, 8, abort);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(o_at + 32 * c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * keep);
                        tmem_st16(o_at + 32 * c, o);
                        tmem_st16(o_at + 32 * c + 16, o + 16);
                    }
                }
            }
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int x = 0; x < 16; ++x) {
                    const float e0 = exp2_fast(fmaf(__uint_as_float(s[c][2 * x]), scale, -from));
                    const float e1 = exp2_fast(fmaf(__uint_as_float(s[c][2 * x + 1]), scale, -from));
                    sum[(2 * x) & 3] += e0;
                    sum[(2 * x + 1) & 3] += e1;
                    p[x] = pack2(e0, e1);
                }
                tmem_st16(buffer + 16 * c, p);
            }
            total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_st_wait();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            mbar_arrive(p_full + 2 * half + (i & 1));
            key0 = i + 1 == keys.sink_tiles ? keys.first : key0 + kTcKeys;
        }
        if (half < halves) {
            // Products are done in order.
            ok = ok && mbar_wait(o_last + half, 0, status, 9, abort);
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float by = total == 0.0f ? 0.0f : 1.0f / total;
            // Through the queries' place in shared memory, so that rows are written whole.
            unsigned char* const rows_at = smem + half * L::kQuery;
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(o_at + 32 * c, o);
                tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    uint32_t w[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        w[y] = pack2(__uint_as_float(o[8 * x + 2 * y]) * by,
                                     __uint_as_float(o[8 * x + 2 * y + 1]) * by);
                    }
                    *reinterpret_cast<uint4*>(rows_at + in_tile * (HD * 2) +
                                              (((4 * c + x) ^ (in_tile & 7)) << 4)) =
                        make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + half), "n"(kTcSoft / 2) : "memory");
#pragma unroll 4
            for (int i = 0; i < 128 * (HD / 8) / (kTcSoft / 2); ++i) {
                const int x = in_tile + i * (kTcSoft / 2);
                const int r = x / (HD / 8), c = x % (HD / 8);
                if (128 * half + r < rows) {
                    int token, head;
                    place(128 * half + r, &token, &head);
                    *reinterpret_cast<uint4*>(out + (tile.first + static_cast<int64_t>(token)) * out_stride +
                                              head * HD + 8 * c) =
                        *reinterpret_cast<const uint4*>(rows_at + r * (HD * 2) + ((c ^ (r & 7)) << 4));
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (status[0] != 0 && threadIdx.x == 0) {
        // A wait ran out: let the copies that were issued land before the memory goes away.
        const uint64_t start = global_ns();
        while (global_ns() - start < 2000000ull) {
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) *flag = status[0] != 0 || status[2] != 0;
    if (warp == 8) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ---- float32, and bf16 that the kernel above does not take --------------------------------------
// The same scheme on mma.sync m16n8k8 (tf32): a CTA takes 64 query rows, a warp 16 of them, keys and
// values pass through shared memory in tiles, double-buffered with cp.async. float32 operands are
// split in two tf32 parts, x = h + l with h the upper 10 mantissa bits, and multiplied as
// h h + h l + l h (2^-21 of a product is left out); bf16 ones are tf32 numbers as they are, their
// weights rounded to tf32. A CTA that meets infinities and whose outputs are not all finite has them
// computed again (4096 causal tokens of 8 heads of 64, an infinity in the first value: 0.55 -> 9 ms). The tensor
// cores cut sums where float32 additions round: sums of a whole row came out 3e-6 low, so products are
// summed 32 channels, or a tile of keys, at a time (the small ones apart) and added up in float32.
// Splitting happens in registers after the load, so the tiles stay float32.
// Rows of keys are padded to HD + 8 floats and of values to HD + 4, which keeps the fragments' reads
// (pairs of channels of eight keys; one channel of four keys two apart) free of bank conflicts.
// Bound by the latency between a warp's own instructions at 12 warps an SM (24 float32 sequences of up to
// 700 tokens, 8 heads of 64, window 256: 140 us, tensor cores 42 % busy, issue 53 %). Keys and values
// split once a tile in shared memory instead of by every warp are 15 % fewer instructions and no faster.

template <typename T, int HD>
struct MmaLayout {
    static constexpr int kRows = 64, kThreads = 128;
    static constexpr int kKeys = 32;    // three CTAs an SM
    static constexpr int kKPitch = HD + 8, kVPitch = HD + 4;
    static constexpr int kStage = kKeys * (kKPitch + kVPitch);  // floats
    static constexpr int kQPitch = HD + 8;
    static constexpr int kSmem = (2 * kStage + kRows * kQPitch) * 4;
};

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = high + low, both rounded to tf32's mantissa, which the product itself only cuts (with parts that
// it cuts, every score came out low by the same 5e-7 of itself): high to the nearest by adding half a
// step to its bits, low by adding 0.72 of half a step of its exponent for each one of its mantissa,
// which makes up for the cut on average and leaves at most 1.44 half steps of low, 2^-21 of x. A NaN
// has to come through: adding to its bits may carry into the sign and leave a zero (0x7fffffff, what
// arithmetic makes here), but low is made by arithmetic alone and stays one.
__device__ __forceinline__ void tf32_parts(float x, uint32_t* high, uint32_t* low) {
    *high = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    const float rest = x - __uint_as_float(*high);
    *low = __float_as_uint(fmaf(rest, 0.72f * 0x1p-11f, rest));
}

template <typename T, int HD>
__global__ void __launch_bounds__(128, HD == 128 ? 2 : 3)
k_packed_mma(Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride, const T* __restrict__ k,
             int64_t k_stride, const T* __restrict__ v, int64_t v_stride, T* __restrict__ out,
             int64_t out_stride, bool vector, int* __restrict__ flags) {
    using L = MmaLayout<T, HD>;
    constexpr bool kSplit = sizeof(T) == 4;
    extern __shared__ __align__(16) float shared[];
    __shared__ int redo;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.heads / a.kv_heads, tiles = gridDim.x / a.kv_heads;
    const int place_of = blockIdx.x / a.kv_heads, kvh = blockIdx.x - place_of * a.kv_heads;
    const int index = tiles - 1 - place_of;  // as above
    int* const flag = flags + kvh * tiles + index;
    Tile tile;
    if (!find_tile(b, group, L::kRows, index, &tile)) {
        if (threadIdx.x == 0) *flag = 0;
        return;
    }
    const int rows = min(L::kRows, tile.n * group - tile.r0);
    const int p0 = tile.r0 / group, p1 = (tile.r0 + rows - 1) / group;
    const KeyTiles<L::kKeys, 8> keys(p0, p1, a.window, a.sinks);
    if (threadIdx.x == 0) redo = 0;

    const T* const kb = k + tile.first * k_stride + kvh * HD;
    const T* const vb = v + tile.first * v_stride + kvh * HD;
    float* const queries = shared + 2 * L::kStage;
    // Keys and values of tile i into stage i & 1; keys behind the sequence read as zeros.
    auto fetch = [&](int i) {
        if (i < keys.tiles) {
            float* const ks = shared + (i & 1) * L::kStage;
            float* const vs = ks + L::kKeys * L::kKPitch;
            const int key0 = keys.key(i);
            for (int x = threadIdx.x; x < L::kKeys * (HD / 4); x += L::kThreads) {
                const int r = x / (HD / 4), c = x % (HD / 4) * 4;
                const bool ok = key0 + r < tile.n;
                const T* from_k = kb + (ok ? (key0 + r) * k_stride + c : 0);
                const T* from_v = vb + (ok ? (key0 + r) * v_stride + c : 0);
                float* to_k = ks + r * L::kKPitch + c;
                float* to_v = vs + r * L::kVPitch + c;
                if constexpr (kSplit) {
                    const int bytes = ok ? 16 : 0;
                    if (vector) {
                        cp_async<16>(smem_u32(to_k), from_k, bytes);
                        cp_async<16>(smem_u32(to_v), from_v, bytes);
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            cp_async<4>(smem_u32(to_k + y), from_k + (ok ? y : 0), bytes / 4);
                            cp_async<4>(smem_u32(to_v + y), from_v + (ok ? y : 0), bytes / 4);
                        }
                    }
                } else {
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        to_k[y] = ok ? to_f(from_k[y]) : 0.0f;
                        to_v[y] = ok ? to_f(from_v[y]) : 0.0f;
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(0);
    const float to_log2 = a.scale * kLog2e;
    // Queries, a warp a row, many loads at once (rows behind the last are copies that become zeros).
#pragma unroll 8
    for (int r = warp; r < L::kRows; r += L::kThreads / 32) {
        const int row = tile.r0 + min(r, rows - 1), token = row / group;
        const T* const from = q + (tile.first + static_cast<int64_t>(token)) * q_stride +
                              (kvh * group + row - token * group) * HD + lane;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
            const float value = to_f(from[32 * c]);
            queries[r * L::kQPitch + 32 * c + lane] = r < rows ? value : 0.0f;
        }
    }
    int position[2], low[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = 16 * warp + g + 8 * r;
        position[r] = row < rows ? (tile.r0 + row) / group : -1;
        low[r] = a.window ? position[r] - a.window + 1 : 0;
    }
    float o[HD / 8][4], top[2] = {-INFINITY, -INFINITY}, total[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

    for (int i = 0; i < keys.tiles; ++i) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // tile i is there, and everyone has left tile i - 1
        fetch(i + 1);
        const float* const ks = shared + (i & 1) * L::kStage;
        const float* const vs = ks + L::kKeys * L::kKPitch;
        const int key0 = keys.key(i), blocks = keys.cols(i) / 8;
        const bool all = keys.whole(i, p0, p1, a.window);
        if (!all) {
            bool bad = false;
            for (int x = threadIdx.x; x < L::kKeys * (HD / 4); x += L::kThreads) {
                const float4 y = *reinterpret_cast<const float4*>(vs + x / (HD / 4) * L::kVPitch +
                                                                  x % (HD / 4) * 4);
                bad |= !(fabsf(y.x) <= FLT_MAX) || !(fabsf(y.y) <= FLT_MAX) ||
                       !(fabsf(y.z) <= FLT_MAX) || !(fabsf(y.w) <= FLT_MAX);
            }
            if (bad) redo = 1;
        }
        constexpr int kBlocks = L::kKeys / 8;
        float s[kBlocks][4];
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
        // 32 channels at a time in sums of their own, the small products apart from the large ones.
#pragma unroll
        for (int c0 = 0; c0 < HD / 8; c0 += 4) {
            float large[kBlocks][4], small[kBlocks][4];
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) large[n][e] = small[n][e] = 0.0f;
            }
#pragma unroll
            for (int c = c0; c < c0 + 4; ++c) {  // channels 8 c + {2 t, 2 t + 1} are k = t and t + 4
                uint32_t qh[4], ql[4];
                const float* from = queries + (16 * warp + g) * L::kQPitch + 8 * c + 2 * t;
                const float2 q0 = *reinterpret_cast<const float2*>(from);
                const float2 q1 = *reinterpret_cast<const float2*>(from + 8 * L::kQPitch);
                tf32_parts(q0.x, &qh[0], &ql[0]);
                tf32_parts(q1.x, &qh[1], &ql[1]);
                tf32_parts(q0.y, &qh[2], &ql[2]);
                tf32_parts(q1.y, &qh[3], &ql[3]);
                // Blocks behind `blocks` are multiplied too (their keys are zeros) and masked below.
                uint32_t h[kBlocks][2], l[kBlocks][2];
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    const float2 x = *reinterpret_cast<const float2*>(ks + (8 * n + g) * L::kKPitch +
                                                                      8 * c + 2 * t);
                    tf32_parts(x.x, &h[n][0], &l[n][0]);
                    tf32_parts(x.y, &h[n][1], &l[n][1]);
                }
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) mma_tf32(large[n], qh, h[n][0], h[n][1]);
                if constexpr (kSplit) {
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) mma_tf32(small[n], qh, l[n][0], l[n][1]);
#pragma unroll
                    for (int n = 0; n < kBlocks; ++n) mma_tf32(small[n], ql, h[n][0], h[n][1]);
                }
            }
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] += kSplit ? large[n][e] + small[n][e] : large[n][e];
            }
        }
        float most[2] = {-INFINITY, -INFINITY};
        const int stop = keys.stop(i);
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
            if (n < blocks) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = e >> 1, key = key0 + 8 * n + 2 * t + (e & 1);
                    s[n][e] *= to_log2;
                    if (!all && !(key <= position[r] && key < stop && (key >= low[r] || key < a.sinks))) {
                        s[n][e] = -INFINITY;
                    }
                    most[r] = fmaxf(most[r], s[n][e]);
                }
            }
        }
        float from[2], keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            most[r] = fmaxf(most[r], __shfl_xor_sync(kFull, most[r], 1));
            most[r] = fmaxf(most[r], __shfl_xor_sync(kFull, most[r], 2));
            const bool up = most[r] > top[r];
            keep[r] = up ? (top[r] == -INFINITY ? 0.0f : exp2_fast(top[r] - most[r])) : 1.0f;
            if (up) top[r] = most[r];
            from[r] = top[r] == -INFINITY ? 0.0f : top[r];
            total[r] *= keep[r];
        }
        uint32_t ph[kBlocks][4], pl[kBlocks][4];
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = n < blocks ? exp2_fast(s[n][e] - from[e >> 1]) : 0.0f;
                total[e >> 1] += p;
                // Column 2 t is k = t, column 2 t + 1 is k = t + 4; rows g and g + 8.
                const int at = (e >> 1) + 2 * (e & 1);
                tf32_parts(p, &ph[n][at], &pl[n][at]);
            }
        }
        // Four columns of channels at a time: independent products follow one another.
#pragma unroll
        for (int c0 = 0; c0 < HD / 8; c0 += 4) {
            float large[4][4] = {}, small[4][4] = {};
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) {
                if (n < blocks) {
                    uint32_t h[4][2], l[4][2];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float* x = vs + (8 * n + 2 * t) * L::kVPitch + 8 * (c0 + c) + g;
                        tf32_parts(x[0], &h[c][0], &l[c][0]);
                        tf32_parts(x[L::kVPitch], &h[c][1], &l[c][1]);
                    }
#pragma unroll
                    for (int c = 0; c < 4; ++c) mma_tf32(large[c], ph[n], h[c][0], h[c][1]);
                    if constexpr (kSplit) {
#pragma unroll
                        for (int c = 0; c < 4; ++c) mma_tf32(small[c], ph[n], l[c][0], l[c][1]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) mma_tf32(small[c], pl[n], h[c][0], h[c][1]);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[c0 + c][e] = fmaf(o[c0 + c][e], keep[e >> 1],
                                        kSplit ? large[c][e] + small[c][e] : large[c][e]);
                }
            }
        }
    }
    bool whole = true;  // all outputs are finite
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        total[r] += __shfl_xor_sync(kFull, total[r], 1);
        total[r] += __shfl_xor_sync(kFull, total[r], 2);
        const float by = total[r] == 0.0f ? 0.0f : 1.0f / total[r];
        const int row = 16 * warp + g + 8 * r;
        if (row < rows) {
            const int token = position[r], head = kvh * group + tile.r0 + row - token * group;
            T* to = out + (tile.first + static_cast<int64_t>(token)) * out_stride + head * HD + 2 * t;
            float most = fabsf(total[r]);
#pragma unroll
            for (int c = 0; c < HD / 8; ++c) {
                const float x = o[c][2 * r] * by, y = o[c][2 * r + 1] * by;
                put(to + 8 * c, x);
                put(to + 8 * c + 1, y);
                most = max_nan(most, max_nan(fabsf(x), fabsf(y)));
            }
            whole &= most <= FLT_MAX;
        }
    }
    // The parts of an infinity, and of a float that rounds to one, leave NaN where the formula may have a
    // weight of zero, an infinity or a number. A NaN leaves what it should: rows that are not finite are
    // computed again only if the CTA has met one of the former.
    if constexpr (kSplit) {
        if (__syncthreads_or(!whole)) {
            auto splits = [](float x) {
                const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
                return u - 0x7f7ff000u <= 0x1000u;
            };
            bool found = false;
            for (int i = 0; i < keys.tiles; ++i) {
                const int key0 = keys.key(i), stop = min(keys.stop(i), key0 + L::kKeys);
#pragma unroll 4
                for (int x = threadIdx.x; x < (stop - key0) * HD; x += L::kThreads) {
                    const int64_t key = key0 + x / HD;
                    found |= splits(to_f(kb[key * k_stride + x % HD])) | splits(to_f(vb[key * v_stride + x % HD]));
                }
            }
            for (int x = threadIdx.x; x < rows * HD; x += L::kThreads) {
                found |= splits(queries[x / HD * L::kQPitch + x % HD]);
            }
            if (found) redo = 1;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) *flag = redo;
}

// The rows of CTAs that raised their flag, computed plainly.
template <typename T, int HD>
__global__ void __launch_bounds__(256, 2)
k_packed_again(Batch b, AttnSpec a, const T* __restrict__ q, int64_t q_stride,
               const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v, int64_t v_stride,
               T* __restrict__ out, int64_t out_stride, const int* __restrict__ flags, int tiles,
               int tile_rows) {
    constexpr int C = HD / 32;
    const int lane = threadIdx.x & 31;
    pdl_wait();
    for (int i = blockIdx.x; i < tiles * a.kv_heads; i += gridDim.x) {
        if (flags[i] == 0) continue;
        const int kvh = i / tiles, group = a.heads / a.kv_heads;
        Tile tile;
        if (!find_tile(b, group, tile_rows, i % tiles, &tile)) continue;
        const int rows = min(tile_rows, tile.n * group - tile.r0);
        for (int r = threadIdx.x >> 5; r < rows; r += 8) {
            const int row = tile.r0 + r;
            const int64_t position = row / group, head = kvh * group + row % group;
            const int64_t first = a.window ? max(static_cast<int64_t>(0), position - a.window + 1) : 0;
            const int64_t sunk = min(static_cast<int64_t>(a.sinks), first);  // keys below this come first
            float value[C], top, total;
            attend_row<C>(q + (tile.first + position) * q_stride + head * HD,
                          k + tile.first * k_stride + kvh * HD, k_stride,
                          v + tile.first * v_stride + kvh * HD, v_stride, a.scale * kLog2e,
                          sunk + position + 1 - first,
                          [&](int64_t at) { return at < sunk ? at : first + (at - sunk); }, value, &top,
                          &total);
            T* to = out + (tile.first + position) * out_stride + head * HD + lane;
#pragma unroll
            for (int c = 0; c < C; ++c) put(to + 32 * c, total == 0.0f ? 0.0f : value[c] / total);
        }
    }
}

// Whether TMA and 16-byte accesses can address these bf16 tensors, and the scale is not zero: the kernel
// multiplies by it behind the mask, whose -inf it would turn into NaN.
bool tc_takes(float scale, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
              const void* v, int64_t v_stride, const void* out, int64_t out_stride) {
    auto aligned = [](const void* p, int64_t stride) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0;
    };
    return scale != 0.0f && aligned(q, q_stride) && aligned(k, k_stride) && aligned(v, v_stride) &&
           aligned(out, out_stride);
}

}  // namespace

// A flag for every CTA, of the kernel with the smaller tiles.
size_t attention_packed_workspace(const Batch& b, const AttnSpec& a) {
    return static_cast<size_t>(tile_bound(b, a, 64)) * a.kv_heads * sizeof(int);
}

cudaError_t launch_attention_packed(cudaStream_t s, const Batch& b, const AttnSpec& a,
                                    const void* q_, int64_t q_stride, const void* k_,
                                    int64_t k_stride, const void* v_, int64_t v_stride, void* out_,
                                    int64_t out_stride, void* workspace) {
    if (b.tokens < 1 || b.count < 1) return cudaSuccess;
    int* const flags = static_cast<int*>(workspace);
    return by_dtype(a.dtype, [&](auto type) {
        using T = decltype(type);
        return by_head_dim(a.head_dim, [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            const T *q = static_cast<const T*>(q_), *k = static_cast<const T*>(k_),
                    *v = static_cast<const T*>(v_);
            T* const out = static_cast<T*>(out_);
            int tile_rows = 0, tiles = 0;
            cudaError_t e = cudaSuccess;
            if constexpr (sizeof(T) == 2 && HD >= 64) {
                if (tc_takes(a.scale, q, q_stride, k, k_stride, v, v_stride, out, out_stride)) {
                    tile_rows = kTcRows;
                    tiles = tile_bound(b, a, tile_rows);
                    CUtensorMap k_map, v_map;
                    const int width = a.kv_heads * HD;
                    e = make_tile_map(&k_map, k, b.tokens, width, k_stride * 2, true, kTcKeys);
                    if (!e) e = make_tile_map(&v_map, v, b.tokens, width, v_stride * 2, true, kTcKeys);
                    if (!e) {
                        e = cudaFuncSetAttribute(k_packed_tc<HD>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 TcLayout<HD>::kSmem);
                    }
                    if (e) return e;
                    k_packed_tc<HD><<<tiles * a.kv_heads, kTcThreads, TcLayout<HD>::kSmem, s>>>(
                        k_map, v_map, b, a, q, q_stride, out, out_stride, flags);
                }
            }
            if (tile_rows == 0) {
                using L = MmaLayout<T, HD>;
                tile_rows = L::kRows;
                tiles = tile_bound(b, a, tile_rows);
                const bool vector = (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0 &&
                                    k_stride % 4 == 0 && v_stride % 4 == 0;
                e = cudaFuncSetAttribute(k_packed_mma<T, HD>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem);
                if (e) return e;
                k_packed_mma<T, HD><<<tiles * a.kv_heads, L::kThreads, L::kSmem, s>>>(
                    b, a, q, q_stride, k, k_stride, v, v_stride, out, out_stride, vector, flags);
            }
            if ((e = cudaGetLastError())) return e;
            return launch_pdl(k_packed_again<T, HD>, dim3(std::min(2 * 148, tiles * a.kv_heads)), dim3(256),
                              0, s, b, a, q, q_stride, k, k_stride, v, v_stride, out, out_stride,
                              static_cast<const int*>(flags), tiles, tile_rows);
        });
    });
}

}  // namespace bst
