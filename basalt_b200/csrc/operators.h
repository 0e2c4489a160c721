// Internal interface of the serving operators (kv_cache.cu, attention_cached.cu,
// attention_packed.cu, sample.cu): device views
// of the ABI structs and the launchers shared with the engine. Launchers queue on the given stream
// of the current device and return the launch's error.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "basalt_cuda.h"

namespace bst {

// A batch of sequences over packed tokens (bst_sequences).
struct Batch {
    int count = 0, tokens = 0;
    const int* rows = nullptr;
    const int* starts = nullptr;
    const int* lengths = nullptr;
};

// A cache of keys and values (bst_kv_cache).
struct Cache {
    int storage = 0, rows = 0, kv_heads = 0, slots = 0, head_dim = 0;
    void *k = nullptr, *v = nullptr, *k_scale = nullptr, *v_scale = nullptr;
};

struct AttnSpec {
    int heads = 0, kv_heads = 0, head_dim = 0, dtype = 0, window = 0, sinks = 0;
    float scale = 0.0f;
};

cudaError_t launch_kv_append(cudaStream_t s, const Cache& c, const Batch& b, const void* k,
                             int64_t k_stride, const void* v, int64_t v_stride, int dtype);
cudaError_t launch_kv_read(cudaStream_t s, const Cache& c, const Batch& b, void* k,
                           int64_t k_stride, void* v, int64_t v_stride, int dtype);

size_t attention_cached_workspace(const Cache& c, const Batch& b, const AttnSpec& a);
cudaError_t launch_attention_cached(cudaStream_t s, const Cache& c, const Batch& b,
                                    const AttnSpec& a, const void* q, int64_t q_stride, void* out,
                                    int64_t out_stride, void* workspace);
size_t attention_packed_workspace(const Batch& b, const AttnSpec& a);
cudaError_t launch_attention_packed(cudaStream_t s, const Batch& b, const AttnSpec& a,
                                    const void* q, int64_t q_stride, const void* k,
                                    int64_t k_stride, const void* v, int64_t v_stride, void* out,
                                    int64_t out_stride, void* workspace);

struct Sampling {
    float temperature = 1.0f, top_p = 1.0f, min_p = 0.0f;
    int top_k = 0;
    const float *temperatures = nullptr, *top_ps = nullptr, *min_ps = nullptr;
    const int* top_ks = nullptr;
};
// uniforms of row r: uniforms[r * uniform_stride + (step ? *step : 0)].
cudaError_t launch_sample_tokens(cudaStream_t s, const void* logits, int dtype, int rows, int V,
                                 int64_t row_stride, const Sampling& sampling,
                                 const double* uniforms, int64_t uniform_stride, const int* step,
                                 int* tokens);

// Makes `device` current for the scope and restores the caller's on the way out.
class DeviceScope {
   public:
    explicit DeviceScope(int device) {
        error_ = cudaGetDevice(&before_);
        if (!error_ && before_ != device) {
            error_ = cudaSetDevice(device);
            changed_ = !error_;
        }
        if (error_) cudaGetLastError();
    }
    ~DeviceScope() {
        if (changed_) cudaSetDevice(before_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    cudaError_t error() const { return error_; }

   private:
    int before_ = 0;
    bool changed_ = false;
    cudaError_t error_ = cudaSuccess;
};

// Argument checks: BST_OK, or the status with *why set.
int check_batch(const bst_sequences* s, bool lengths_needed, Batch* out, std::string* why);
int check_cache(const bst_kv_cache* c, Cache* out, std::string* why);

#ifdef __CUDACC__
// The sequence that owns packed token t and the token's place in it; false when none does.
__device__ __forceinline__ bool find_sequence(const Batch& b, int t, int* seq, int* first, int* n) {
    if (!b.starts) {
        *seq = t;
        *first = t;
        *n = 1;
        return t < b.count;
    }
    if (b.count < 1) return false;
    // The last sequence that starts at or before t: empty sequences before it share its start.
    int lo = 0, hi = b.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (__ldg(b.starts + mid) <= t) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    const int from = max(0, __ldg(b.starts + lo)), to = min(__ldg(b.starts + lo + 1), b.tokens);
    *seq = lo;
    *first = from;
    *n = to - from;
    return t >= from && t < to;
}
#endif

}  // namespace bst
