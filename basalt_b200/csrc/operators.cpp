// The C ABI of the serving operators: argument checks on the host, then one launcher each.

#include "operators.h"

#include <cuda_runtime.h>

#include <cmath>
#include <exception>
#include <new>
#include <string>

#include "kernels.h"

namespace bst {

int check_batch(const bst_sequences* s, bool lengths_needed, Batch* out, std::string* why) {
    if (!s) {
        *why = "sequences must not be null";
        return BST_INVALID;
    }
    if (s->count < 0 || s->tokens < 0) {
        *why = "sequences: count and tokens must not be negative";
        return BST_SHAPE;
    }
    if (lengths_needed && s->count > 0 && !s->lengths) {
        *why = "sequences: lengths must not be null";
        return BST_INVALID;
    }
    if (!s->starts && s->tokens != s->count) {
        *why = "sequences: without starts every sequence has one token, but there are " +
               std::to_string(s->tokens) + " tokens and " + std::to_string(s->count) + " sequences";
        return BST_SHAPE;
    }
    for (const void* p : {s->rows, s->starts, s->lengths}) {
        if (reinterpret_cast<uintptr_t>(p) % 4) {
            *why = "sequences: rows, starts and lengths must be aligned to 4 bytes";
            return BST_INVALID;
        }
    }
    out->count = s->count;
    out->tokens = s->tokens;
    out->rows = s->rows;
    out->starts = s->starts;
    out->lengths = s->lengths;
    return BST_OK;
}

namespace {

int check_head_dim(int hd, std::string* why) {
    if (hd == 32 || hd == 64 || hd == 128) return BST_OK;
    *why = "head dimension " + std::to_string(hd) + " is not one of 32, 64, 128";
    return BST_UNSUPPORTED;
}

int check_dtype(int dtype, std::string* why) {
    if (dtype == BST_DTYPE_F32 || dtype == BST_DTYPE_BF16) return BST_OK;
    *why = "dtype must be BST_DTYPE_F32 or BST_DTYPE_BF16";
    return BST_INVALID;
}

size_t size_of(int dtype) { return dtype == BST_DTYPE_BF16 ? 2 : 4; }

// A packed tensor [tokens][heads][head_dim] with this token stride.
int check_tensor(const char* name, const void* p, int64_t stride, int64_t heads, int head_dim,
                 int dtype, std::string* why) {
    if (!p) {
        *why = std::string(name) + " must not be null";
        return BST_INVALID;
    }
    if (stride < heads * head_dim) {
        *why = std::string(name) + ": tokens are " + std::to_string(stride) +
               " elements apart, less than their " + std::to_string(heads * head_dim) + " elements";
        return BST_SHAPE;
    }
    if (reinterpret_cast<uintptr_t>(p) % size_of(dtype)) {
        *why = std::string(name) + " is not aligned to its elements";
        return BST_INVALID;
    }
    return BST_OK;
}

// A packed tensor's place in memory: `tokens` runs of `run` bytes, `stride` bytes apart.
struct Span {
    uint64_t at, stride, run;
    int64_t tokens;
    uint64_t end() const { return at + (tokens - 1) * stride + run; }
};

// Whether two of them share a byte. Runs at the same stride may lie between one another (slices of
// one tensor); at different ones no byte between the first and the last may be shared.
bool overlap(const Span& x, const Span& y) {
    if (x.end() <= y.at || y.end() <= x.at) return false;
    if (x.stride != y.stride || x.tokens == 1) return true;
    const uint64_t ahead = y.at >= x.at ? (y.at - x.at) % x.stride
                                        : (x.stride - (x.at - y.at) % x.stride) % x.stride;
    return ahead < x.run || x.stride - ahead < y.run;
}

Span span_of(const void* p, int64_t stride, int64_t heads, const AttnSpec& a, int tokens) {
    const uint64_t size = size_of(a.dtype);
    return Span{reinterpret_cast<uint64_t>(p), static_cast<uint64_t>(stride) * size,
                static_cast<uint64_t>(heads) * a.head_dim * size, tokens};
}

}  // namespace

int check_cache(const bst_kv_cache* c, Cache* out, std::string* why) {
    if (!c) {
        *why = "cache must not be null";
        return BST_INVALID;
    }
    if (c->storage != BST_DTYPE_F32 && c->storage != BST_DTYPE_BF16 && c->storage != BST_DTYPE_U4) {
        *why = "cache storage must be BST_DTYPE_F32, BST_DTYPE_BF16 or BST_DTYPE_U4";
        return BST_INVALID;
    }
    for (int r : c->reserved) {
        if (r != 0) {
            *why = "reserved cache fields must be zero";
            return BST_INVALID;
        }
    }
    if (const int st = check_head_dim(c->head_dim, why)) return st;
    if (c->rows < 1 || c->kv_heads < 1 || c->slots < 1 || c->kv_heads > 65535) {
        *why = "cache rows, heads and slots must be positive (and at most 65535 heads)";
        return BST_SHAPE;
    }
    if (c->slots > 0x7fffffff - 65536) {  // slots are counted in 32 bits, in blocks
        *why = "cache slots must stay below 2^31 - 65536";
        return BST_SHAPE;
    }
    const bool scaled = c->storage == BST_DTYPE_U4;
    if (!c->k || !c->v || (scaled && (!c->k_scale || !c->v_scale))) {
        *why = "cache buffers must not be null";
        return BST_INVALID;
    }
    for (const void* p : {c->k, c->v, c->k_scale, c->v_scale}) {
        if (reinterpret_cast<uintptr_t>(p) % 16) {
            *why = "cache buffers must be 16-byte aligned";
            return BST_INVALID;
        }
    }
    out->storage = c->storage;
    out->rows = c->rows;
    out->kv_heads = c->kv_heads;
    out->slots = c->slots;
    out->head_dim = c->head_dim;
    out->k = c->k;
    out->v = c->v;
    out->k_scale = c->k_scale;
    out->v_scale = c->v_scale;
    return BST_OK;
}

namespace {

int check_spec(const bst_attention_spec* a, AttnSpec* out, std::string* why) {
    if (!a) {
        *why = "spec must not be null";
        return BST_INVALID;
    }
    if (a->reserved != 0) {
        *why = "reserved spec fields must be zero";
        return BST_INVALID;
    }
    if (const int st = check_dtype(a->dtype, why)) return st;
    if (const int st = check_head_dim(a->head_dim, why)) return st;
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65535) {
        *why = "heads must be a positive multiple of kv_heads, got " + std::to_string(a->heads) +
               " and " + std::to_string(a->kv_heads);
        return BST_SHAPE;
    }
    if (a->window < 0 || a->sinks < 0) {
        *why = "window and sinks must not be negative";
        return BST_INVALID;
    }
    if (!std::isfinite(a->scale)) {
        *why = "scale must be finite";
        return BST_INVALID;
    }
    out->heads = a->heads;
    out->kv_heads = a->kv_heads;
    out->head_dim = a->head_dim;
    out->dtype = a->dtype;
    out->window = a->window;
    out->sinks = a->sinks;
    out->scale = a->scale;
    return BST_OK;
}

// Positions and keys stay below `keys`: a window that wide hides nothing.
void limit_window(int keys, AttnSpec* a) {
    if (a->window >= keys || a->sinks >= keys) a->window = 0;
    if (a->window == 0) a->sinks = 0;
}

// Query rows are counted in 32 bits.
int check_rows(const Batch& b, const AttnSpec& a, std::string* why) {
    if (static_cast<int64_t>(b.tokens) * a.heads <= 0x7fffffff - 65536) return BST_OK;
    *why = "tokens x heads must stay below 2^31";
    return BST_SHAPE;
}

int check_cached(const bst_kv_cache* cache, const bst_sequences* sequences,
                 const bst_attention_spec* spec, Cache* c, Batch* b, AttnSpec* a,
                 std::string* why) {
    int st = check_cache(cache, c, why);
    if (!st) st = check_batch(sequences, true, b, why);
    if (!st) st = check_spec(spec, a, why);
    if (st) return st;
    if (a->kv_heads != c->kv_heads || a->head_dim != c->head_dim) {
        *why = "spec and cache disagree on kv_heads or head_dim";
        return BST_SHAPE;
    }
    if ((st = check_rows(*b, *a, why))) return st;
    limit_window(c->slots, a);
    if (b->starts && c->storage != BST_DTYPE_U4) {
        *why = "a float32 or bf16 cache takes one token per sequence (starts must be null)";
        return BST_UNSUPPORTED;
    }
    return BST_OK;
}

int check_packed(const bst_sequences* sequences, const bst_attention_spec* spec, Batch* b,
                 AttnSpec* a, std::string* why) {
    int st = check_batch(sequences, false, b, why);
    if (!st) st = check_spec(spec, a, why);
    if (st) return st;
    if (b->count > 0 && !b->starts) {
        *why = "packed attention needs the sequences' starts";
        return BST_INVALID;
    }
    if (b->rows || b->lengths) {
        *why = "packed attention takes no rows and no lengths";
        return BST_INVALID;
    }
    if ((st = check_rows(*b, *a, why))) return st;
    limit_window(b->tokens, a);
    return BST_OK;
}

int check_shared(const bst_kv_cache* cache, const bst_sequences* sequences, const bst_attention_spec* spec,
                 const bst_kv_cache* prefix, int32_t row, int32_t length, Cache* c, Batch* b, AttnSpec* a,
                 Prefix* p, std::string* why) {
    int st = check_cached(cache, sequences, spec, c, b, a, why);
    if (st) return st;
    if (spec->window != 0 || spec->sinks != 0) {
        *why = "attention behind a prefix takes no window and no sinks";
        return BST_UNSUPPORTED;
    }
    if ((st = check_cache(prefix, &p->cache, why))) {
        *why = "prefix: " + *why;
        return st;
    }
    if (p->cache.kv_heads != c->kv_heads || p->cache.head_dim != c->head_dim) {
        *why = "prefix and cache disagree on kv_heads or head_dim";
        return BST_SHAPE;
    }
    if (row < 0 || row >= p->cache.rows || length < 0 || length > p->cache.slots) {
        *why = "the prefix is " + std::to_string(length) + " keys of row " + std::to_string(row) +
               ", its cache has " + std::to_string(p->cache.rows) + " rows of " +
               std::to_string(p->cache.slots);
        return BST_SHAPE;
    }
    p->row = row;
    p->length = length;
    return BST_OK;
}

// A call's CTAs are counted in 31 bits.
int check_blocks(int64_t blocks, std::string* why) {
    if (blocks <= 0x7fffffff) return BST_OK;
    *why = "too many sequences, heads and slots for one call";
    return BST_SHAPE;
}

// Bytes of a whole array, and whether two such share one.
struct Range {
    uint64_t at, bytes;
};
bool overlap(const Range& x, const Range& y) {
    return x.bytes && y.bytes && x.at < y.at + y.bytes && y.at < x.at + x.bytes;
}
Range range_of(const void* p, uint64_t bytes) { return Range{reinterpret_cast<uint64_t>(p), bytes}; }
Range mass_range(const void* mass, const Cache& c) {
    return range_of(mass, 4ull * c.rows * c.kv_heads * c.slots);
}
Range span_range(const Span& x) { return Range{x.at, x.end() - x.at}; }
// A cache's four buffers.
struct Buffers {
    Range each[4];
    explicit Buffers(const Cache& c) {
        const uint64_t values = static_cast<uint64_t>(c.rows) * c.kv_heads * c.slots * c.head_dim;
        const bool u4 = c.storage == BST_DTYPE_U4;
        const uint64_t bytes = u4 ? values / 2 : values * size_of(c.storage), scale = u4 ? values / 8 : 0;
        each[0] = range_of(c.k, bytes);
        each[1] = range_of(c.v, bytes);
        each[2] = range_of(c.k_scale, scale);
        each[3] = range_of(c.v_scale, scale);
    }
    bool meets(const Range& x) const {
        return overlap(each[0], x) || overlap(each[1], x) || overlap(each[2], x) || overlap(each[3], x);
    }
    bool meets(const Buffers& x) const {
        return meets(x.each[0]) || meets(x.each[1]) || meets(x.each[2]) || meets(x.each[3]);
    }
};

int check_eviction(const bst_kv_cache* cache, const bst_sequences* sequences, const float* mass, int32_t keep,
                   int32_t recent, int32_t sinks, const bst_kv_cache* to, const int32_t* to_rows, float* to_mass,
                   int32_t* lengths, int32_t* kept, Cache* c, Batch* b, Eviction* e, std::string* why) {
    int st = check_cache(cache, c, why);
    if (!st) st = check_batch(sequences, true, b, why);
    if (st) return st;
    if (b->starts) {
        *why = "an eviction takes no tokens (starts must be null)";
        return BST_INVALID;
    }
    if (keep < 1 || recent < 0 || sinks < 0 || static_cast<int64_t>(recent) + sinks > keep) {
        *why = "keep must be positive, recent and sinks not negative and together at most keep, got " +
               std::to_string(keep) + ", " + std::to_string(recent) + " and " + std::to_string(sinks);
        return BST_SHAPE;
    }
    if (to) {
        if ((st = check_cache(to, &e->to, why))) {
            *why = "to: " + *why;
            return st;
        }
        if (e->to.storage != c->storage || e->to.kv_heads != c->kv_heads || e->to.head_dim != c->head_dim) {
            *why = "to must have the cache's storage, kv_heads and head_dim";
            return BST_SHAPE;
        }
    } else {
        if (to_rows) {
            *why = "in place keys stay in their rows (to_rows must be null)";
            return BST_INVALID;
        }
        e->to = *c;
    }
    if (keep > e->to.slots) {
        *why = "keep is " + std::to_string(keep) + ", the cache that is written has " +
               std::to_string(e->to.slots) + " slots";
        return BST_SHAPE;
    }
    if ((st = check_blocks(static_cast<int64_t>(b->count) * c->kv_heads * (8 + keep / 64), why))) return st;
    if (b->count > 0) {
        if (!mass || !to_mass || !lengths || !kept) {
            *why = "masses, new lengths and kept slots must not be null";
            return BST_INVALID;
        }
        for (const void* p : {static_cast<const void*>(mass), static_cast<const void*>(to_mass),
                              static_cast<const void*>(lengths), static_cast<const void*>(kept),
                              static_cast<const void*>(to_rows)}) {
            if (reinterpret_cast<uintptr_t>(p) % 4) {
                *why = "masses, rows, lengths and kept slots must be aligned to 4 bytes";
                return BST_INVALID;
            }
        }
        const Buffers read(*c), written(e->to);
        const Range masses = mass_range(mass, *c), to_masses = mass_range(to_mass, e->to);
        const Range slots = range_of(kept, 4ull * b->count * c->kv_heads * keep);
        const Range counts = range_of(lengths, 4ull * b->count);
        const Range indices[3] = {range_of(b->lengths, 4ull * b->count),
                                  range_of(b->rows, b->rows ? 4ull * b->count : 0),
                                  range_of(to_rows, to_rows ? 4ull * b->count : 0)};
        bool bad = to && read.meets(written);
        bad |= !(!to && to_mass == mass) && overlap(masses, to_masses);
        bad |= overlap(slots, counts);
        for (const Range& x : {to_masses, slots, counts}) {
            bad |= read.meets(x) || written.meets(x);
            for (const Range& y : indices) bad |= overlap(x, y);
        }
        bad |= overlap(slots, masses) || overlap(slots, to_masses) || overlap(counts, masses) ||
               overlap(counts, to_masses);
        if (bad) {
            *why = "what is written must not overlap anything else (masses may stay in place when keys do)";
            return BST_INVALID;
        }
    }
    e->keep = keep;
    e->recent = recent;
    e->sinks = sinks;
    e->mass = mass;
    e->to_rows = to ? to_rows : b->rows;
    e->to_mass = to_mass;
    e->lengths = lengths;
    e->kept = kept;
    return BST_OK;
}

int check_workspace(size_t needed, const void* workspace, int64_t bytes, std::string* why) {
    if (needed == 0) return BST_OK;
    if (!workspace || bytes < 0 || static_cast<size_t>(bytes) < needed) {
        *why = "workspace: " + std::to_string(needed) + " bytes are needed, " +
               std::to_string(workspace ? bytes : 0) + " given";
        return BST_SHAPE;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16) {
        *why = "workspace must be 16-byte aligned";
        return BST_INVALID;
    }
    return BST_OK;
}

int32_t refuse(const char* what, int status, const std::string& why) {
    set_thread_error(std::string(what) + ": " + why);
    return status;
}

// Runs fn (a launcher) with `device` current.
template <typename Fn>
int32_t queue(int32_t device, const char* what, Fn&& fn) {
    DeviceScope scope(device);
    if (scope.error()) {
        return refuse(what, BST_UNSUPPORTED, "device " + std::to_string(device) + ": " +
                                                 cudaGetErrorString(scope.error()));
    }
    const cudaError_t e = fn();
    if (e) {
        cudaGetLastError();
        return refuse(what, e == cudaErrorMemoryAllocation ? BST_OOM : BST_PANIC,
                      std::string(cudaGetErrorName(e)) + ": " + cudaGetErrorString(e));
    }
    return BST_OK;
}

}  // namespace
}  // namespace bst

// No C++ exception leaves an entry point.
#define BST_OPERATOR_GUARDED(name, ...)                                            \
    try {                                                                          \
        __VA_ARGS__                                                                \
    } catch (const std::bad_alloc&) {                                              \
        bst::set_thread_error(name ": host allocation failed");                    \
        return BST_OOM;                                                            \
    } catch (const std::exception& ex) {                                           \
        bst::set_thread_error(std::string(name ": internal error: ") + ex.what()); \
        return BST_PANIC;                                                          \
    }

extern "C" {

static int32_t kv_transfer(bool append, int32_t device, void* stream, const bst_kv_cache* cache,
                           const bst_sequences* sequences, const void* k, int64_t k_stride,
                           const void* v, int64_t v_stride, int32_t dtype) {
    using namespace bst;
    const char* what = append ? "kv_append" : "kv_read";
    Cache c;
    Batch b;
    std::string why;
    int st = check_cache(cache, &c, &why);
    if (!st) st = check_batch(sequences, true, &b, &why);
    if (!st) st = check_dtype(dtype, &why);
    if (!st && b.tokens > 0) st = check_tensor("k", k, k_stride, c.kv_heads, c.head_dim, dtype, &why);
    if (!st && b.tokens > 0) st = check_tensor("v", v, v_stride, c.kv_heads, c.head_dim, dtype, &why);
    if (st) return refuse(what, st, why);
    return queue(device, what, [&] {
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        return append ? launch_kv_append(s, c, b, k, k_stride, v, v_stride, dtype)
                      : launch_kv_read(s, c, b, const_cast<void*>(k), k_stride,
                                       const_cast<void*>(v), v_stride, dtype);
    });
}

int32_t bst_kv_append(int32_t device, void* stream, const bst_kv_cache* cache,
                      const bst_sequences* sequences, const void* k, int64_t k_stride,
                      const void* v, int64_t v_stride, int32_t dtype) {
    BST_OPERATOR_GUARDED("kv_append", {
        return kv_transfer(true, device, stream, cache, sequences, k, k_stride, v, v_stride, dtype);
    })
}

int32_t bst_kv_read(int32_t device, void* stream, const bst_kv_cache* cache,
                    const bst_sequences* sequences, void* k, int64_t k_stride, void* v,
                    int64_t v_stride, int32_t dtype) {
    BST_OPERATOR_GUARDED("kv_read", {
        return kv_transfer(false, device, stream, cache, sequences, k, k_stride, v, v_stride,
                           dtype);
    })
}

int32_t bst_attention_cached_workspace(const bst_kv_cache* cache, const bst_sequences* sequences,
                                       const bst_attention_spec* spec, int64_t* bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_cached", {
        Cache c;
        Batch b;
        AttnSpec a;
        std::string why;
        const int st = check_cached(cache, sequences, spec, &c, &b, &a, &why);
        if (st) return refuse("attention_cached", st, why);
        if (!bytes) return refuse("attention_cached", BST_INVALID, "bytes must not be null");
        *bytes = static_cast<int64_t>(attention_cached_workspace(c, b, a));
        return BST_OK;
    })
}

int32_t bst_attention_cached(int32_t device, void* stream, const bst_kv_cache* cache,
                             const bst_sequences* sequences, const bst_attention_spec* spec,
                             const void* q, int64_t q_stride, void* out, int64_t out_stride,
                             void* workspace, int64_t workspace_bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_cached", {
        Cache c;
        Batch b;
        AttnSpec a;
        std::string why;
        int st = check_cached(cache, sequences, spec, &c, &b, &a, &why);
        if (st) return refuse("attention_cached", st, why);
        if (b.tokens == 0 || b.count == 0) return BST_OK;
        st = check_tensor("q", q, q_stride, a.heads, a.head_dim, a.dtype, &why);
        if (!st) st = check_tensor("out", out, out_stride, a.heads, a.head_dim, a.dtype, &why);
        // Every CTA has read its queries when it writes their outputs: those may take their place.
        if (!st && !(out == q && out_stride == q_stride) &&
            overlap(span_of(q, q_stride, a.heads, a, b.tokens),
                    span_of(out, out_stride, a.heads, a, b.tokens))) {
            st = BST_INVALID;
            why = "out overlaps q (it may only be q itself)";
        }
        if (!st) {
            st = check_workspace(attention_cached_workspace(c, b, a), workspace, workspace_bytes,
                                 &why);
        }
        if (st) return refuse("attention_cached", st, why);
        return queue(device, "attention_cached", [&] {
            return launch_attention_cached(static_cast<cudaStream_t>(stream), c, b, a, q, q_stride,
                                           out, out_stride, workspace);
        });
    })
}

int32_t bst_attention_shared_workspace(const bst_kv_cache* cache, const bst_sequences* sequences,
                                       const bst_attention_spec* spec, const bst_kv_cache* prefix,
                                       int32_t prefix_row, int32_t prefix_length, int64_t* bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_shared", {
        Cache c;
        Batch b;
        AttnSpec a;
        Prefix p;
        std::string why;
        const int st =
            check_shared(cache, sequences, spec, prefix, prefix_row, prefix_length, &c, &b, &a, &p, &why);
        if (st) return refuse("attention_shared", st, why);
        if (!bytes) return refuse("attention_shared", BST_INVALID, "bytes must not be null");
        *bytes = static_cast<int64_t>(attention_shared_workspace(c, b, a, p));
        return BST_OK;
    })
}

int32_t bst_attention_shared(int32_t device, void* stream, const bst_kv_cache* cache,
                             const bst_sequences* sequences, const bst_attention_spec* spec,
                             const bst_kv_cache* prefix, int32_t prefix_row, int32_t prefix_length,
                             const void* q, int64_t q_stride, void* out, int64_t out_stride,
                             void* workspace, int64_t workspace_bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_shared", {
        Cache c;
        Batch b;
        AttnSpec a;
        Prefix p;
        std::string why;
        int st = check_shared(cache, sequences, spec, prefix, prefix_row, prefix_length, &c, &b, &a, &p, &why);
        if (st) return refuse("attention_shared", st, why);
        if (b.tokens == 0 || b.count == 0) return BST_OK;
        st = check_tensor("q", q, q_stride, a.heads, a.head_dim, a.dtype, &why);
        if (!st) st = check_tensor("out", out, out_stride, a.heads, a.head_dim, a.dtype, &why);
        // Outputs are written by the kernel that joins, behind all that read queries.
        if (!st && !(out == q && out_stride == q_stride) &&
            overlap(span_of(q, q_stride, a.heads, a, b.tokens),
                    span_of(out, out_stride, a.heads, a, b.tokens))) {
            st = BST_INVALID;
            why = "out overlaps q (it may only be q itself)";
        }
        if (!st) {
            st = check_workspace(attention_shared_workspace(c, b, a, p), workspace, workspace_bytes, &why);
        }
        if (st) return refuse("attention_shared", st, why);
        return queue(device, "attention_shared", [&] {
            return launch_attention_shared(static_cast<cudaStream_t>(stream), c, b, a, p, q, q_stride, out,
                                           out_stride, workspace);
        });
    })
}

int32_t bst_attention_weights_workspace(const bst_kv_cache* cache, const bst_sequences* sequences,
                                        const bst_attention_spec* spec, int64_t* bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_weights", {
        Cache c;
        Batch b;
        AttnSpec a;
        std::string why;
        const int st = check_cached(cache, sequences, spec, &c, &b, &a, &why);
        if (st) return refuse("attention_weights", st, why);
        if (!bytes) return refuse("attention_weights", BST_INVALID, "bytes must not be null");
        *bytes = static_cast<int64_t>(attention_weights_workspace(c, b, a));
        return BST_OK;
    })
}

int32_t bst_attention_weights(int32_t device, void* stream, const bst_kv_cache* cache,
                              const bst_sequences* sequences, const bst_attention_spec* spec, const void* q,
                              int64_t q_stride, void* out, int64_t out_stride, const float* previous,
                              float decay, float* mass, void* workspace, int64_t workspace_bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_weights", {
        Cache c;
        Batch b;
        AttnSpec a;
        std::string why;
        int st = check_cached(cache, sequences, spec, &c, &b, &a, &why);
        if (!st && !(std::isfinite(decay) && decay >= 0.0f)) {
            st = BST_INVALID;
            why = "decay must be finite and not negative";
        }
        if (st) return refuse("attention_weights", st, why);
        if (b.count == 0) return BST_OK;
        if (b.tokens > 0) {
            st = check_tensor("q", q, q_stride, a.heads, a.head_dim, a.dtype, &why);
            if (!st) st = check_tensor("out", out, out_stride, a.heads, a.head_dim, a.dtype, &why);
        }
        if (!st && (!mass || (!previous && decay != 0.0f))) {
            st = BST_INVALID;
            why = "mass must not be null, nor previous unless decay is 0";
        }
        if (!st && (reinterpret_cast<uintptr_t>(mass) % 4 || reinterpret_cast<uintptr_t>(previous) % 4)) {
            st = BST_INVALID;
            why = "masses must be aligned to 4 bytes";
        }
        if (!st) {
            const Range to = mass_range(mass, c);
            const Range from = decay == 0.0f ? Range{0, 0} : mass_range(previous, c);
            bool bad = Buffers(c).meets(to) || (previous != mass && overlap(to, from));
            if (b.tokens > 0) {
                const Span query = span_of(q, q_stride, a.heads, a, b.tokens);
                const Span result = span_of(out, out_stride, a.heads, a, b.tokens);
                bad |= overlap(to, span_range(query)) || overlap(to, span_range(result)) ||
                       overlap(from, span_range(result)) ||
                       (!(out == q && out_stride == q_stride) && overlap(query, result));
            }
            if (bad) {
                st = BST_INVALID;
                why = "mass and out must not overlap what is read (mass may be previous, out may be q)";
            }
        }
        if (!st) {
            const int64_t chunks = (static_cast<int64_t>(c.slots) + 511) / 512;
            st = check_blocks(static_cast<int64_t>(b.tokens) * a.heads + chunks * a.kv_heads * b.count, &why);
        }
        if (!st) {
            st = check_workspace(attention_weights_workspace(c, b, a), workspace, workspace_bytes, &why);
        }
        if (st) return refuse("attention_weights", st, why);
        return queue(device, "attention_weights", [&] {
            return launch_attention_weights(static_cast<cudaStream_t>(stream), c, b, a, q, q_stride, out,
                                            out_stride, previous, decay, mass, workspace);
        });
    })
}

int32_t bst_kv_evict(int32_t device, void* stream, const bst_kv_cache* cache, const bst_sequences* sequences,
                     const float* mass, int32_t keep, int32_t recent, int32_t sinks, const bst_kv_cache* to,
                     const int32_t* to_rows, float* to_mass, int32_t* lengths, int32_t* kept) {
    using namespace bst;
    BST_OPERATOR_GUARDED("kv_evict", {
        Cache c;
        Batch b;
        Eviction e;
        std::string why;
        const int st = check_eviction(cache, sequences, mass, keep, recent, sinks, to, to_rows, to_mass, lengths,
                                      kept, &c, &b, &e, &why);
        if (st) return refuse("kv_evict", st, why);
        if (b.count == 0) return BST_OK;
        return queue(device, "kv_evict",
                     [&] { return launch_kv_evict(static_cast<cudaStream_t>(stream), c, b, e); });
    })
}

int32_t bst_attention_packed_workspace(const bst_sequences* sequences,
                                       const bst_attention_spec* spec, int64_t* bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_packed", {
        Batch b;
        AttnSpec a;
        std::string why;
        const int st = check_packed(sequences, spec, &b, &a, &why);
        if (st) return refuse("attention_packed", st, why);
        if (!bytes) return refuse("attention_packed", BST_INVALID, "bytes must not be null");
        *bytes = static_cast<int64_t>(attention_packed_workspace(b, a));
        return BST_OK;
    })
}

int32_t bst_attention_packed(int32_t device, void* stream, const bst_sequences* sequences,
                             const bst_attention_spec* spec, const void* q, int64_t q_stride,
                             const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                             void* out, int64_t out_stride, void* workspace,
                             int64_t workspace_bytes) {
    using namespace bst;
    BST_OPERATOR_GUARDED("attention_packed", {
        Batch b;
        AttnSpec a;
        std::string why;
        int st = check_packed(sequences, spec, &b, &a, &why);
        if (st) return refuse("attention_packed", st, why);
        if (b.tokens == 0 || b.count == 0) return BST_OK;
        st = check_tensor("q", q, q_stride, a.heads, a.head_dim, a.dtype, &why);
        if (!st) st = check_tensor("k", k, k_stride, a.kv_heads, a.head_dim, a.dtype, &why);
        if (!st) st = check_tensor("v", v, v_stride, a.kv_heads, a.head_dim, a.dtype, &why);
        if (!st) st = check_tensor("out", out, out_stride, a.heads, a.head_dim, a.dtype, &why);
        // Keys and values are read by many CTAs, and queries again where rows are computed again.
        if (!st) {
            const Span to = span_of(out, out_stride, a.heads, a, b.tokens);
            if (overlap(to, span_of(q, q_stride, a.heads, a, b.tokens)) ||
                overlap(to, span_of(k, k_stride, a.kv_heads, a, b.tokens)) ||
                overlap(to, span_of(v, v_stride, a.kv_heads, a, b.tokens))) {
                st = BST_INVALID;
                why = "out must not overlap q, k or v";
            }
        }
        if (!st) {
            st = check_workspace(attention_packed_workspace(b, a), workspace, workspace_bytes, &why);
        }
        if (st) return refuse("attention_packed", st, why);
        return queue(device, "attention_packed", [&] {
            return launch_attention_packed(static_cast<cudaStream_t>(stream), b, a, q, q_stride, k,
                                           k_stride, v, v_stride, out, out_stride, workspace);
        });
    })
}

int32_t bst_sample_tokens(int32_t device, void* stream, const void* logits, int32_t dtype,
                          int32_t rows, int32_t vocabulary, int64_t row_stride,
                          const bst_sampling* sampling, const double* uniforms, int32_t* tokens) {
    using namespace bst;
    BST_OPERATOR_GUARDED("sample_tokens", {
        std::string why;
        int st = check_dtype(dtype, &why);
        if (!st && (rows < 0 || rows > (1 << 27))) {
            st = BST_SHAPE;
            why = "rows must be in [0, 2^27]";
        }
        if (!st && (vocabulary < 1 || vocabulary > (1 << 20))) {
            st = BST_SHAPE;
            why = "vocabulary must be in [1, 2^20], got " + std::to_string(vocabulary);
        }
        if (!st && row_stride < vocabulary) {
            st = BST_SHAPE;
            why = "rows are " + std::to_string(row_stride) + " logits apart, less than the vocabulary";
        }
        if (!st && !sampling) {
            st = BST_INVALID;
            why = "sampling must not be null";
        }
        if (!st && rows > 0 && (!logits || !uniforms || !tokens)) {
            st = BST_INVALID;
            why = "logits, uniforms and tokens must not be null";
        }
        if (!st && (reinterpret_cast<uintptr_t>(logits) % size_of(dtype) ||
                    reinterpret_cast<uintptr_t>(uniforms) % 8 ||
                    reinterpret_cast<uintptr_t>(tokens) % 4)) {
            st = BST_INVALID;
            why = "logits, uniforms and tokens must be aligned to their elements";
        }
        if (!st) {
            for (const void* p : {static_cast<const void*>(sampling->temperatures),
                                  static_cast<const void*>(sampling->top_ps),
                                  static_cast<const void*>(sampling->min_ps),
                                  static_cast<const void*>(sampling->top_ks)}) {
                if (reinterpret_cast<uintptr_t>(p) % 4) {
                    st = BST_INVALID;
                    why = "per-row settings must be aligned to 4 bytes";
                }
            }
        }
        if (st) return refuse("sample_tokens", st, why);
        if (rows == 0) return BST_OK;
        Sampling p;
        p.temperature = sampling->temperature;
        p.top_p = sampling->top_p;
        p.min_p = sampling->min_p;
        p.top_k = sampling->top_k;
        p.temperatures = sampling->temperatures;
        p.top_ps = sampling->top_ps;
        p.min_ps = sampling->min_ps;
        p.top_ks = sampling->top_ks;
        return queue(device, "sample_tokens", [&] {
            return launch_sample_tokens(static_cast<cudaStream_t>(stream), logits, dtype, rows,
                                        vocabulary, row_stride, p, uniforms, 1, nullptr, tokens);
        });
    })
}

}  // extern "C"
