/*
 * basalt_cuda.h — C ABI of libbasalt_cuda.so, the B200 (sm_100a) decode engine behind
 * basalt.infer.TextEngine.
 *
 * The reference runs TextEngine's loop in Java and reaches its Rust kernels one op at a time
 * through JNI (src/main/java/basalt/nativebridge/NativeBindings.java:13-89, implemented by
 * native/src/api.rs:118-709). This library replaces that per-op traffic with one call per
 * TextEngine method: the whole decode loop — embedding, LayerNorm, projections, attention over an
 * HBM KV cache, LM head, argmax or seeded sampling — runs on the GPU. A JNI shim maps each
 * TextEngine method onto the entry point named in its comment.
 *
 * Conventions (native/src/error.rs:9-17, src/main/java/basalt/BasaltExceptionCode.java:7-15):
 * every entry returns 0 on success or a negative status; the message of the last failure is
 * available from bst_last_error. No C++ exception crosses this boundary.
 *
 * Handles are opaque 64-bit ids, never reused (native/src/tensor.rs:150-176 keeps the same rule
 * for tensors); destroying an engine twice returns BST_UNKNOWN_HANDLE. Calls on one engine are
 * serialised by the engine; engines on different devices are independent.
 */
#ifndef BASALT_CUDA_H
#define BASALT_CUDA_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define BST_ABI_VERSION 1

/* Status codes: native/src/error.rs:9-17. */
#define BST_OK 0
#define BST_INVALID (-1)          /* BasaltParameterException */
#define BST_SHAPE (-2)            /* BasaltShapeException */
#define BST_UNKNOWN_HANDLE (-3)   /* stale or unknown handle */
#define BST_CONTEXT (-4)          /* closed engine / mismatched saved model */
#define BST_GRAPH (-5)
#define BST_PANIC (-6)            /* CUDA fault or internal error */
#define BST_OOM (-7)              /* device or host allocation failed */
#define BST_UNSUPPORTED (-8)

/* Model families the engine runs. */
#define BST_FAMILY_PADDED_DECODER 1 /* pre-norm causal decoder (TransformerBlock.java:37-43) whose
                                       mask also hides leading PAD ids (PAD = vocabulary);
                                       positions count from the first non-PAD id */
#define BST_FAMILY_DECODER 2        /* the same blocks with the stock causal mask only: every step
                                       recomputes the full window, as the reference does */
#define BST_FAMILY_CHAR_LM 3        /* Zoo.charLm windowed MLP (zoo/Zoo.java:135-168) */
#define BST_FAMILY_LAST_TOKEN 4     /* TextEngineTest.LastTokenModel (TextEngineTest.java:210-243) */

#define BST_DTYPE_F32 0
#define BST_DTYPE_BF16 1
#define BST_DTYPE_U4 2 /* caches only: 4-bit codes, a bf16 step and low per 32 channels */

typedef uint64_t bst_engine;

typedef struct bst_model_spec {
    int32_t family;
    int32_t vocabulary;   /* V: tokens the head scores (TextEngine.vocabulary()) */
    int32_t window;       /* W: context length (TextEngine.window()) */
    int32_t dimension;    /* d */
    int32_t layers;       /* L (decoders) */
    int32_t heads;        /* H (decoders); d % H == 0 */
    int32_t hidden;       /* FFN width (decoders) or bottleneck width (charLm) */
    int32_t weight_dtype; /* BST_DTYPE_*: storage of matrices and embedding tables */
    int32_t kv_dtype;     /* BST_DTYPE_*: storage of the attention cache */
    int32_t max_rows;     /* rows decoded together per wave; 0 = sized from free memory */
    /* Decoders: a token attends to the last attention_window tokens (0: all of the context) and,
     * with a window, to the first attention_sinks. No counterpart in the reference. */
    int32_t attention_window;
    int32_t attention_sinks;
    int32_t reserved[4];  /* must be zero */
} bst_model_spec;

/* Per-token callback (java.util.function.IntConsumer of TextEngine.stream / streamSampled,
 * TextEngine.java:181-221). Called once per produced token, in step order within each row.
 * Returning non-zero stops the call, which then returns BST_INVALID. */
typedef int32_t (*bst_token_sink)(void* user, int32_t row, int32_t step, int32_t token);

int32_t bst_abi_version(void);
int32_t bst_device_count(int32_t* count);

/* Engine lifecycle. Replaces TextEngine.of (TextEngine.java:61-74) together with the module it
 * binds: the spec names the architecture, parameters are then set by name. */
int32_t bst_engine_create(const bst_model_spec* spec, int32_t device, bst_engine* out);
int32_t bst_engine_destroy(bst_engine engine);

/* Recognition of a module by its namedParameters (torch/Module.java:27-34), the test TextEngine's
 * dispatch makes before it hands a module to this engine. `count` parameters: names[i] with
 * ranks[i] dimensions, all dimensions concatenated in `dims`, in the reference's layout (Linear
 * weight [in, out], bias [1, out]; LayerNorm gamma/beta [d]; Embedding [rows, d]). vocabulary and
 * window are TextEngine.of's arguments (TextEngine.java:61-74); heads is the decoder's head count
 * (MultiheadAttention's parameter shapes do not carry it; ignored otherwise). Recognised: the
 * padded decoder (embedding rows V + 1) and the stock decoder (V rows), Zoo.charLm
 * (zoo/Zoo.java:135-168) and the one-hot last-token head (TextEngineTest.java:210-243). Fills
 * `spec` (f32 storage, max_rows 0) or returns BST_UNSUPPORTED / BST_SHAPE with the reason. */
int32_t bst_recognize_model(const char* const* names, const int32_t* ranks, const int64_t* dims,
                            int32_t count, int32_t vocabulary, int32_t window, int32_t heads,
                            bst_model_spec* spec);
/* TextEngine.of(module, vocabulary, window) for a recognised module: creates the engine on
 * `device` with the given storage dtypes and copies every parameter by name
 * (Module.loadStateDict, torch/Module.java:68-76). values[i] holds parameter i's floats. */
int32_t bst_engine_create_from_parameters(const char* const* names, const int32_t* ranks,
                                          const int64_t* dims, const float* const* values,
                                          int32_t count, int32_t vocabulary, int32_t window,
                                          int32_t heads, int32_t weight_dtype, int32_t kv_dtype,
                                          int32_t device, bst_engine* out);

/* Parameters by name, in Module.namedParameters order (torch/Module.java:27-34). */
int32_t bst_parameter_count(bst_engine engine, int32_t* count);
int32_t bst_parameter_info(bst_engine engine, int32_t index, char* name, int32_t capacity,
                           int64_t* size);
/* Module.loadStateDict entry (torch/Module.java:68-76) / Tensor.setData. */
int32_t bst_set_parameter(bst_engine engine, const char* name, const float* values,
                          int64_t count);
/* Tensor.data of a parameter (float32 values as last set). */
int32_t bst_get_parameter(bst_engine engine, const char* name, float* values, int64_t count);
/* TextEngine.save / load (TextEngine.java:298-350): big-endian vocabulary, window, count, then
 * per parameter a modified-UTF-8 name, an element count and float32 values. */
int32_t bst_save(bst_engine engine, const char* path);
int32_t bst_load(bst_engine engine, const char* path);

/* TextEngine.scoresBatch / scores (TextEngine.java:96-148). contexts: [rows, length] row-major,
 * length >= window; only each row's tail is used. scores: [rows, vocabulary]. */
int32_t bst_scores(bst_engine engine, const int32_t* contexts, int32_t rows, int32_t length,
                   double* scores);

/* TextEngine.generate / stream / generateBatch (TextEngine.java:158-193, 232-254): greedy
 * decoding, first maximum wins. tokens: [rows, steps]. sink may be NULL. */
int32_t bst_generate(bst_engine engine, const int32_t* contexts, int32_t rows, int32_t length,
                     int32_t steps, int32_t* tokens, bst_token_sink sink, void* user);

/* TextEngine.sample / streamSampled (TextEngine.java:201-227, 267-285) with the engine's
 * java.util.Random. Rows are decoded together but draw exactly what `rows` successive calls on
 * one engine would: row r starts from the generator advanced by 2*steps*r, and the engine's
 * generator ends advanced by 2*steps*rows. */
int32_t bst_sample(bst_engine engine, const int32_t* contexts, int32_t rows, int32_t length,
                   int32_t steps, float temperature, int32_t top_k, int32_t* tokens,
                   bst_token_sink sink, void* user);

/* Sampling with bst_sampling's filters (below; its per-row arrays must be NULL) from the caller's
 * random numbers: step g of row r draws with uniforms[r * steps + g] (host memory, [rows, steps]).
 * A row whose logits leave nothing to draw (NaN only) takes token 0. The engine's java.util.Random is
 * not touched. No counterpart in the reference. */
struct bst_sampling;
int32_t bst_sample_filtered(bst_engine engine, const int32_t* contexts, int32_t rows, int32_t length,
                            int32_t steps, const struct bst_sampling* sampling,
                            const double* uniforms, int32_t* tokens, bst_token_sink sink,
                            void* user);
/* The same, also returning the logits each step was decided on ([rows, steps, vocabulary]). */
int32_t bst_sample_filtered_logits(bst_engine engine, const int32_t* contexts, int32_t rows,
                                   int32_t length, int32_t steps,
                                   const struct bst_sampling* sampling, const double* uniforms,
                                   int32_t* tokens, float* logits);

/* bst_generate / bst_sample that also return the logits each step was decided on:
 * logits [rows, steps, vocabulary] float32 (the scores TextEngine.scores would have returned for
 * that step's window, as the decode path computed them). */
int32_t bst_generate_logits(bst_engine engine, const int32_t* contexts, int32_t rows,
                            int32_t length, int32_t steps, int32_t* tokens, float* logits);
int32_t bst_sample_logits(bst_engine engine, const int32_t* contexts, int32_t rows,
                          int32_t length, int32_t steps, float temperature, int32_t top_k,
                          int32_t* tokens, float* logits);

/* bst_generate_logits / bst_sample_logits that keep the logits of `watch_count` chosen rows only:
 * logits [watch_count, steps, vocabulary], entry i for row watch_rows[i]. Lets a caller follow a
 * few sequences of a batch too large for every row's logits (TextEngine.scores of those rows'
 * windows at each step). Rows must be distinct and inside [0, rows). */
int32_t bst_generate_logits_rows(bst_engine engine, const int32_t* contexts, int32_t rows,
                                 int32_t length, int32_t steps, int32_t* tokens,
                                 int32_t watch_count, const int32_t* watch_rows, float* logits);
int32_t bst_sample_logits_rows(bst_engine engine, const int32_t* contexts, int32_t rows,
                               int32_t length, int32_t steps, float temperature, int32_t top_k,
                               int32_t* tokens, int32_t watch_count, const int32_t* watch_rows,
                               float* logits);

/* The same two calls for callers whose contexts and token buffers already live on the engine's
 * device (device pointers; no sink). */
int32_t bst_generate_device(bst_engine engine, const int32_t* contexts, int32_t rows,
                            int32_t length, int32_t steps, int32_t* tokens);
int32_t bst_sample_device(bst_engine engine, const int32_t* contexts, int32_t rows,
                          int32_t length, int32_t steps, float temperature, int32_t top_k,
                          int32_t* tokens);

/* TextEngine.seed (TextEngine.java:288-290) and raw access to the 48-bit generator state. */
int32_t bst_seed(bst_engine engine, int64_t seed);
int32_t bst_get_rng_state(bst_engine engine, int64_t* state);
int32_t bst_set_rng_state(bst_engine engine, int64_t state);

/* NativeContext.beginScope / endScope / scopeDepth (nativebridge/NativeContext.java:229-247,
 * native/src/context.rs:186-221): device buffers the engine allocates while a scope is open are
 * released when it ends. Weights are never scope-owned. */
int32_t bst_begin_scope(bst_engine engine);
int32_t bst_end_scope(bst_engine engine, int32_t* released);
int32_t bst_scope_depth(bst_engine engine, int32_t* depth);

/* NativeContext.stats (nativebridge/NativeContext.java:256-262, context.rs:404-414):
 * out[0] live device buffers, out[1] live device bytes, out[2] graph nodes (always 0: the engine
 * records no autograd graph), out[3] kernels launched so far. */
int32_t bst_engine_stats(bst_engine engine, int64_t out[4]);

/* The CUDA stream (cudaStream_t) all of the engine's work is queued on. */
int32_t bst_engine_stream(bst_engine engine, void** stream);

/* Per-kernel timing, the device-side counterpart of BasaltMetrics.recordOperator
 * (BasaltMetrics.java:203-281). While enabled, each launch is bracketed by CUDA events and the
 * engine accumulates launches, device milliseconds and algorithmic bytes per kernel class. */
#define BST_KERNEL_CLASSES 15
int32_t bst_profile_enable(bst_engine engine, int32_t enabled);
int32_t bst_profile_reset(bst_engine engine);
int32_t bst_profile_read(bst_engine engine, int32_t kernel_class, char* name, int32_t capacity,
                         int64_t* launches, double* milliseconds, double* bytes, double* flops);

/* Tensor.matMul (torch/Tensor.java:214-227) -> gemm::matmul (native/src/gemm.rs:42-74) on device
 * buffers: C[m, n] = A[m, k] * B[k, n], row-major float32, C overwritten. Runs on `device`, queued
 * on `stream` (a cudaStream_t; NULL is the legacy default stream) and returns once C is complete.
 * m <= 8 uses the GEMV kernel, larger m the tcgen05 GEMM (3xTF32). Temporaries (B transposed and
 * the split operand planes) come from the stream-ordered allocator. Errors: bst_last_error(0). */
int32_t bst_matmul(int32_t device, void* stream, const float* a, const float* b, float* c,
                   int64_t m, int64_t k, int64_t n);

/* bst_matmul that allocates no device memory, for callers that may not call cudaMalloc while
 * they run. No counterpart in the reference. Temporaries come from a 16 MiB scratch array built
 * into the library (held on every GPU that loads it until exit); problems whose scratch does not
 * fit are rejected with BST_SHAPE. The first call on a device looks up that array's device address
 * and should come before any stream capture. Calls share the array: work from calls that overlaps
 * on the GPU races, so such calls must be serialised by the caller. */
int32_t bst_matmul_static(int32_t device, void* stream, const float* a, const float* b, float* c,
                          int64_t m, int64_t k, int64_t n);

/* ---- Device tensors and the op queue (NativeContext on Device.cuda(i)) ----
 * A context is bound to one CUDA device. Its tensors live on that device (device tag 1000 + i,
 * Device.java:22,46-59) or on the host (tag 0). Tensor handles are monotonic per context and never
 * reused (native/src/tensor.rs:150-176). Ops run from the reference's packed queue of 128-byte
 * commands (CommandQueueBuilder.java:12-73): u8 op code, u8 flags, 6 pad, u64 inputs A..E, u64
 * output, i32 attrs[16], 8 reserved. Codes run on the GPU: MatMul 1, Add 2, ReLU 3, Sub 4, Mul 5,
 * Sigmoid 6, Tanh 7, Gelu 11, Exp 23, Log 24, Sqrt 25, Abs 26, Neg 27, Div 28 (binary ops broadcast
 * trailing axes as ops.rs:136-164); other codes return BST_UNSUPPORTED. Each executed op is
 * recorded as one graph node, as the reference's Graph::push does; no backward is offered. */
typedef uint64_t bst_context;
typedef uint64_t bst_tensor;
#define BST_DEVICE_TAG_CPU 0
#define BST_DEVICE_TAG_CUDA 1000
#define BST_COMMAND_BYTES 128

/* NativeContext.create for Device.cuda(i): device_tag = 1000 + i. Tag 0 (cpu) returns
 * BST_UNSUPPORTED: host contexts stay on the CPU engine. */
int32_t bst_context_create(int32_t device_tag, bst_context* out);
int32_t bst_context_destroy(bst_context context);
/* NativeContext.of / zeros (values NULL: zeros) on the device named by device_tag (0 or this
 * context's 1000 + i). */
int32_t bst_tensor_create(bst_context context, int32_t device_tag, const int64_t* shape,
                          int32_t rank, const float* values, bst_tensor* out);
/* NativeContext.transferTensor (native/src/context.rs:125-133): a copy on the target device, as
 * a new handle; host <-> device transfers are cudaMemcpy on the context's stream. */
int32_t bst_tensor_transfer(bst_context context, bst_tensor source, int32_t device_tag,
                            bst_tensor* out);
/* NativeTensorHandle.data / setData: count must equal the tensor's element count. */
int32_t bst_tensor_read(bst_context context, bst_tensor tensor, float* values, int64_t count);
int32_t bst_tensor_write(bst_context context, bst_tensor tensor, const float* values,
                         int64_t count);
/* Device tag, rank and up to `capacity` dimensions of a tensor. */
int32_t bst_tensor_info(bst_context context, bst_tensor tensor, int32_t* device_tag,
                        int32_t* rank, int64_t* shape, int32_t capacity);
/* NativeTensorHandle.close: releasing twice is harmless (*released 0 the second time); a handle
 * the context never issued returns BST_UNKNOWN_HANDLE. */
int32_t bst_tensor_release(bst_context context, bst_tensor tensor, int32_t* released);
/* NativeBindings.executeQueue (native/src/engine.rs:118-154): runs `count` commands in order and
 * returns once they have finished; the first failing command stops the queue with its status. */
int32_t bst_execute_queue(bst_context context, const void* commands, int32_t count);
/* out[0] live tensors, out[1] live device bytes, out[2] graph nodes (NativeContext.graphSize),
 * out[3] kernels launched. */
int32_t bst_context_stats(bst_context context, int64_t out[4]);
int32_t bst_context_clear_graph(bst_context context);

/* ---- Serving operators on caller-owned device buffers ----
 * The parts of a decode step that a host program schedules itself: a cache of keys and values (in
 * 4 bits, bf16 or float32), attention over it, attention over packed prompts, and drawing tokens.
 * No counterpart in the reference. All pointers inside the structs and arguments are device
 * pointers on `device`; the structs themselves are host memory, read before the call returns.
 *
 * Every call queues its kernels on `stream` (a cudaStream_t; NULL is the legacy default stream) and
 * returns without waiting for them: it allocates nothing, never synchronises, leaves the calling
 * thread's current device as it was, and may be captured into a CUDA graph (call it once on the
 * device before the first capture: that loads its kernels). Calls may run at the same time on
 * several streams as long as they do not share a workspace or write the same memory. Errors are
 * found from the host's arguments alone, before anything is queued; bst_last_error(0) has the
 * message.
 *
 * A batch is a list of sequences. Sequence s owns cache row rows[s] (distinct rows; s itself when
 * rows is NULL) and the packed tokens [starts[s], starts[s + 1]) of this call (token s alone when
 * starts is NULL, and then tokens == count). lengths[s] counts the row's cached tokens with this
 * call's tokens included: with n tokens, token i of the sequence has position (and cache slot)
 * lengths[s] - n + i. starts must not decrease; what of a sequence lies outside [0, tokens) does
 * not belong to it. The arrays are read on the device: tokens that no
 * sequence owns are left alone (their outputs stay as they were), and tokens whose row or slot lies
 * outside the cache are not stored, see no keys and read as zeros. */
typedef struct bst_sequences {
    int32_t count;
    int32_t tokens;         /* packed tokens: the first dimension of k, v, q and out */
    const int32_t* rows;    /* [count] or NULL */
    const int32_t* starts;  /* [count + 1] or NULL */
    const int32_t* lengths; /* [count] */
} bst_sequences;

/* k and v are [rows][kv_heads][slots][head_dim], head_dim 32, 64 or 128, 16-byte aligned. With
 * BST_DTYPE_U4 a head's channels of one token take head_dim / 2 bytes and k_scale and v_scale are
 * [rows][kv_heads][slots][head_dim / 32][2] bf16: (step, low) of every 32 channels. A code c stands
 * for low + c * step. low is the 32 channels' minimum rounded down to bf16, step is
 * (maximum - low) / 15 rounded up to bf16, and codes are (x - low) / step rounded to nearest even;
 * 32 channels that hold a NaN, an infinity or a value below bf16's lowest read back as NaN. The codes
 * of a token's head are [8][head_dim / 32][4] nibbles, low nibble first: channel 32 g + 4 h + j is
 * nibble j of the 16 bits at [h][g]. */
typedef struct bst_kv_cache {
    int32_t storage; /* BST_DTYPE_F32, BST_DTYPE_BF16 or BST_DTYPE_U4 */
    int32_t rows, kv_heads, slots, head_dim;
    int32_t reserved[3]; /* must be zero */
    void *k, *v;
    void *k_scale, *v_scale; /* BST_DTYPE_U4 only */
} bst_kv_cache;

/* Stores the batch's keys and values in their slots. k and v: [tokens][kv_heads][head_dim] of
 * `dtype`, tokens k_stride and v_stride elements apart (their heads contiguous). */
int32_t bst_kv_append(int32_t device, void* stream, const bst_kv_cache* cache,
                      const bst_sequences* sequences, const void* k, int64_t k_stride,
                      const void* v, int64_t v_stride, int32_t dtype);
/* The values that the batch's slots stand for, in the same layout. */
int32_t bst_kv_read(int32_t device, void* stream, const bst_kv_cache* cache,
                    const bst_sequences* sequences, void* k, int64_t k_stride, void* v,
                    int64_t v_stride, int32_t dtype);

/* heads must be a multiple of kv_heads: query head h reads key head h * kv_heads / heads. A query
 * at position i sees key j when j <= i and (window == 0, or i - j < window, or j < sinks): the
 * last `window` tokens and the first `sinks`. A query that sees nothing, or whose scores are all
 * -infinity, gives zeros. dtype is the type of q and out (and of packed k and v). Scores, their
 * maximum, the sums of weights and the outputs' sums are float32, and so are the weights that are
 * summed. In the products with values, weights keep 21 bits or more in float32 calls; in bf16 calls
 * 16 over a float32 or bf16 cache, 11 over a 4-bit one (as weight times step), and 8 in prompts (11
 * with 32 channels, or where the tensors are not aligned to 16 bytes). NaN and infinities that a
 * query sees count as in float32 arithmetic (but a query that holds an infinity gives NaN over a
 * 4-bit cache), others not at all. */
typedef struct bst_attention_spec {
    int32_t heads, kv_heads, head_dim, dtype;
    int32_t window, sinks;
    float scale; /* of the scores, e.g. 1 / sqrt(head_dim) */
    int32_t reserved; /* must be zero */
} bst_attention_spec;

/* out[t] = attention of the batch's queries over their rows of the cache, this call's own tokens
 * included (append them first). q and out: [tokens][heads][head_dim], tokens q_stride and
 * out_stride elements apart; out may be q itself, and overlaps it in no other way. A cache of
 * float32 or bf16 takes one token per sequence (starts NULL); a 4-bit cache takes any number.
 * workspace: at least the bytes that bst_attention_cached_workspace gives for the same arguments
 * (16-byte aligned, may be NULL when that is 0), not shared with calls that run at the same time. */
int32_t bst_attention_cached_workspace(const bst_kv_cache* cache, const bst_sequences* sequences,
                                       const bst_attention_spec* spec, int64_t* bytes);
int32_t bst_attention_cached(int32_t device, void* stream, const bst_kv_cache* cache,
                             const bst_sequences* sequences, const bst_attention_spec* spec,
                             const void* q, int64_t q_stride, void* out, int64_t out_stride,
                             void* workspace, int64_t workspace_bytes);

/* Causal attention of packed sequences over their own keys and values (prompts that need no cache
 * yet): sequences->starts is required, rows and lengths must be NULL, positions count from 0.
 * q and out [tokens][heads][head_dim], k and v [tokens][kv_heads][head_dim]. out shares no byte with
 * q, k or v (at the same distance between tokens it may lie between theirs). Should a wait inside
 * the bf16 kernel run out (2 s), its rows are computed again by another kernel: the call is slow,
 * its outputs are right. */
int32_t bst_attention_packed_workspace(const bst_sequences* sequences,
                                       const bst_attention_spec* spec, int64_t* bytes);
int32_t bst_attention_packed(int32_t device, void* stream, const bst_sequences* sequences,
                             const bst_attention_spec* spec, const void* q, int64_t q_stride,
                             const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                             void* out, int64_t out_stride, void* workspace,
                             int64_t workspace_bytes);

/* How tokens are drawn; a per-row array, where given, replaces the scalar. In order:
 *   temperature  weights w = exp((logit - largest logit) / temperature); at 0, below, or NaN the
 *                row takes the first of its largest logits instead.
 *                Weights below 2^-40 are never drawn.
 *   top_k        keeps the k largest (<= 0: all), ties lowest index first.
 *   top_p        keeps the fewest of the largest whose weights reach top_p of what is left (at
 *                least one; >= 1 or NaN: all), ties lowest index first.
 *   min_p        keeps weights of at least min_p times the largest (<= 0 or NaN: all).
 * The token is the first, by index, at which the running sum of the kept weights exceeds
 * uniform * their sum. NaN logits count as -infinity; rows with no logit above it give -1. */
typedef struct bst_sampling {
    float temperature, top_p, min_p;
    int32_t top_k;
    const float *temperatures, *top_ps, *min_ps; /* [rows] or NULL */
    const int32_t* top_ks;                       /* [rows] or NULL */
} bst_sampling;

/* tokens[r] drawn from logits [rows][vocabulary] (`dtype`, rows row_stride elements apart) with
 * uniforms[r] in [0, 1) (values outside are clamped). vocabulary <= 2^20. The draw is decided in
 * 64-bit integers, so it does not depend on how rows are scheduled. */
int32_t bst_sample_tokens(int32_t device, void* stream, const void* logits, int32_t dtype,
                          int32_t rows, int32_t vocabulary, int64_t row_stride,
                          const bst_sampling* sampling, const double* uniforms, int32_t* tokens);

/* Message of the last failure on this engine (engine 0: on this thread). */
int32_t bst_last_error(bst_engine engine, char* buffer, int32_t capacity);

/* Synthetic inputs for tests and benchmarks: a TextEngine weight file whose parameters are
 * N(0, stddev) from java.util.Random(seed).nextGaussian (LayerNorm gamma 1, beta 0), and prompts
 * of java.util.Random(seed).nextInt(bound) ids, row after row. */
int32_t bst_write_synthetic_weights(const bst_model_spec* spec, const char* path, int64_t seed,
                                    double stddev);
int32_t bst_synthetic_prompts(int64_t seed, int32_t rows, int32_t length, int32_t bound,
                              int32_t* out);

#ifdef __cplusplus
}
#endif
#endif
