// Attention of one or a few new tokens per sequence over a cache: the launches (attention_cached.cuh has
// the kernels).

#include "attention_cached.cuh"

namespace bst {

size_t attention_cached_workspace(const Cache& c, const Batch& b, const AttnSpec& a) {
    const int splits = split_count(c, b, a);
    if (splits == 1) return 0;
    return static_cast<size_t>(b.tokens) * a.heads * splits * (a.head_dim + 2) * sizeof(float);
}

cudaError_t launch_attention_cached(cudaStream_t s, const Cache& c, const Batch& b,
                                    const AttnSpec& a, const void* q, int64_t q_stride, void* out,
                                    int64_t out_stride, void* workspace) {
    if (b.tokens < 1 || b.count < 1) return cudaSuccess;
    const int splits = split_count(c, b, a), rows = rows_of_tile(b, a);
    float* const part = splits > 1 ? static_cast<float*>(workspace) : nullptr;
    const cudaError_t e = run_cached<kOwn>(s, c, b, a, q, q_stride, out, out_stride, tile_bound(b, a, rows),
                                           rows, splits, part, Extra());
    if (e || !part) return e;
    return by_dtype(a.dtype, [&](auto type) {
        using T = decltype(type);
        return by_head_dim(a.head_dim, [&](auto hd) {
            constexpr int HD = decltype(hd)::value;
            return launch_pdl(k_cached_join<T, HD>, dim3(b.tokens, a.heads), dim3(kThreads), 0, s, c, b, a,
                              rows, static_cast<T*>(out), out_stride, splits,
                              static_cast<const float*>(part));
        });
    });
}

}  // namespace bst
