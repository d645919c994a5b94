#ifndef CTORCH_DECODER_C_API_H
#define CTORCH_DECODER_C_API_H
/*
 * Decoder C17 surface: every entry of the reference's include/dl/decoder_c_api.h:13-41 (same names and
 * arguments; bodies in ctorch_amd/csrc/api/decoder_api.cpp), plus additive extensions marked below.
 * The cache handle belongs to one inference request, holds one K/V store per layer and is released
 * independently of the model.
 */
#include "dl/c_api.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct dl_decoder_cache dl_decoder_cache;

/* decoder_c_api.h:15-20 */
DL_API dl_status dl_tensordot(const dl_tensor* a, const dl_tensor* b,
    dl_shape axes_a, dl_shape axes_b, dl_tensor** output);
DL_API dl_status dl_rotary_embedding(const dl_tensor* input, const dl_tensor* cosine,
    const dl_tensor* sine, dl_tensor** output);
DL_API dl_status dl_grouped_query_attention(const dl_tensor* query, const dl_tensor* key,
    const dl_tensor* value, const dl_tensor* keep_mask, dl_tensor** output);

/* No counterpart in the reference: dl_grouped_query_attention for callers that cannot allocate device memory
 * (code under HIP graph capture, serving loops that forbid allocation).  The caller passes device pointers:
 * query [B, L, H, D] f32 (position-major rows, head h at columns h*D), key and value [B, KV, S, D] contiguous in
 * `kv_dtype` (DL_F32 or DL_BF16), output [B, L, H, D] f32.  The result is dl_grouped_query_attention's with no
 * keep mask (every query row sees all S keys) and its kernels; key-split partials live in a fixed 8 MiB device
 * array per GPU instead of allocated memory, and a shape whose partials would not fit (B*H*L * splits * (D + 2)
 * floats) is rejected with DL_ERROR before anything runs.  Work is queued on the library's stream for `device`.
 * The first call on a device sets up its context and the array's address; later calls allocate nothing.  Calls
 * that overlap on one GPU share the array and race: issue them in order on that stream. */
DL_API dl_status dl_grouped_query_attention_noalloc(const float* query, const void* key, const void* value,
    dl_dtype kv_dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t length, int64_t source,
    int64_t head_dim, float* output, int32_t device);

/* decoder_c_api.h:22-35 */
DL_API dl_status dl_swiglu_create(int64_t dimensions, int64_t hidden, int32_t bias,
    dl_tensor_options options, dl_module** output);
DL_API dl_status dl_lora_linear_create(const dl_module* base, int64_t rank, double alpha, dl_module** output);
DL_API dl_status dl_lora_linear_merge(const dl_module* adapter, dl_module** output);
DL_API dl_status dl_rotary_embedding_create(int64_t dimensions, int64_t capacity, double base,
    dl_tensor_options options, dl_module** output);
DL_API dl_status dl_rotary_embedding_forward(dl_module* rotary, const dl_tensor* input,
    int64_t offset, dl_tensor** output);
DL_API dl_status dl_grouped_query_attention_create(int64_t dimensions, int64_t heads, int64_t kv_heads,
    int64_t context, dl_tensor_options options, dl_module** output);
DL_API dl_status dl_transformer_decoder_create(int64_t layers, int64_t dimensions, int64_t heads,
    int64_t kv_heads, int64_t hidden, int64_t context, dl_tensor_options options, dl_module** output);

/* decoder_c_api.h:37-42 */
DL_API dl_status dl_decoder_cache_create(const dl_module* decoder, dl_decoder_cache** output);
DL_API void dl_decoder_cache_release(dl_decoder_cache* cache);
DL_API dl_status dl_decoder_cache_clear(dl_decoder_cache* cache);
DL_API dl_status dl_decoder_cache_truncate(dl_decoder_cache* cache, int64_t length);
DL_API dl_status dl_decoder_cache_length(const dl_decoder_cache* cache, int64_t* length);
DL_API dl_status dl_transformer_decoder_decode(dl_module* decoder, const dl_tensor* input,
    dl_decoder_cache* cache, dl_tensor** output);

/* Extension (no reference counterpart): the same constructor with the RoPE base the reference hard-codes
 * to 10000 (src/nn/decoder.cpp:70), needed by base-500000 models. */
DL_API dl_status dl_transformer_decoder_create_with_base(int64_t layers, int64_t dimensions, int64_t heads,
    int64_t kv_heads, int64_t hidden, int64_t context, double rope_base, dl_tensor_options options,
    dl_module** output);
/* Extension (no reference counterpart): attaches unmerged rank-`rank` LoRA adapters (scale alpha/rank,
 * `up` zero-initialised) to the query and/or value projection of every layer; they appear in the state as
 * layer{i}.attention.{query,value}_adapter.{down,up}.weight. */
DL_API dl_status dl_transformer_decoder_attach_lora(dl_module* decoder, int64_t rank, double alpha,
    int32_t query, int32_t value);
/* Extension (no reference counterpart): the dtype of the K/V storage every layer's decode reserves.  DL_F32, the
 * default, is the reference's: its KVCache takes the dtype of the appended keys (src/nn/kv_cache.cpp:16-21),
 * which is linear's f32 output (src/ops/matmul.cpp:35-67).  DL_BF16 is an opt-in that halves the cache bytes of
 * long-context decode and rounds every stored key and value to bf16.  Set it before the first decode into a
 * cache: a cache already holding storage of the other dtype is refused on the next decode. */
DL_API dl_status dl_transformer_decoder_set_cache_dtype(dl_module* decoder, dl_dtype dtype);
DL_API dl_status dl_transformer_decoder_cache_dtype(const dl_module* decoder, dl_dtype* dtype);
/* The ONNX decoder's cache wire format (reference extensions/onnx/src/decoder.cpp:64-69, docs/onnx.md:68-113):
 * per layer i, past_key_i / past_value_i as f32 [batch, kv_heads, length, head_dim].  cache_state writes the
 * cache under those names (ready to feed an ONNX Runtime session as its next past_* inputs).  cache_load_state
 * replaces the cache's contents with such a state; each layer may be named past_* or present_* (an ONNX
 * session's outputs), all layers must share batch and length, and the values are stored in the decoder's cache
 * dtype.  Nothing changes when the state does not fit (chunk-atomic). */
DL_API dl_status dl_decoder_cache_state(const dl_decoder_cache* cache, dl_state** output);
DL_API dl_status dl_decoder_cache_load_state(const dl_module* decoder, dl_decoder_cache* cache, const dl_state* state);
/* Extension: writes the K and V of one layer's cache directly (keys already rotated), the reference's
 * KVCache::append route (include/dl/decoder.h:52) for seeding a prefix.  key/value are [B, KV, n, D]. */
DL_API dl_status dl_decoder_cache_append(dl_decoder_cache* cache, int64_t layer, const dl_tensor* key,
    const dl_tensor* value);

/* ---- Extensions (no reference counterpart): rows at given positions, and a paged cache for requests of different
 * lengths.  The rules stand at the C++ entries they call, dl/ops.h and dl/paged.h. ---- */
typedef enum dl_rotary_layout { DL_ROTARY_INTERLEAVED = 0, DL_ROTARY_HALF = 1 } dl_rotary_layout;
typedef enum dl_rotary_scaling_kind {
    DL_ROTARY_UNSCALED = 0, DL_ROTARY_LINEAR = 1, DL_ROTARY_BASE = 2, DL_ROTARY_PARTS = 3
} dl_rotary_scaling_kind;
typedef struct dl_rotary_scaling {
    dl_rotary_scaling_kind kind;
    double factor;
    int64_t trained;
    double slow_turns, fast_turns, magnitude;
} dl_rotary_scaling;
/* Cosine and sine tables [capacity, dimensions / 2], f32, on `device`; scaling may be NULL (none, magnitude 1). */
DL_API dl_status dl_rotary_tables(int64_t dimensions, int64_t capacity, double base, const dl_rotary_scaling* scaling,
    dl_device device, dl_tensor** cosine, dl_tensor** sine);
/* input [T, H, D] f32 or bf16, positions [T] i64, tables [capacity, R/2]: the first R entries of each head rotated by
 * its row's position, the others copied; f32 [T, H, D]. */
DL_API dl_status dl_rotary_positions(const dl_tensor* input, const dl_tensor* positions, const dl_tensor* cosine,
    const dl_tensor* sine, dl_rotary_layout layout, dl_tensor** output);

typedef struct dl_paged_cache dl_paged_cache;
typedef struct dl_paged_batch dl_paged_batch;
/* options.dtype (f32 or bf16) is the pages' type; options.device a GPU. */
DL_API dl_status dl_paged_cache_create(int64_t layers, int64_t pages, int64_t page_size, int64_t kv_heads,
    int64_t head_dim, dl_tensor_options options, dl_paged_cache** output);
DL_API void dl_paged_cache_release(dl_paged_cache* cache);
/* Views of a layer's live storage [pages, kv_heads, page_size, head_dim]; either slot may be NULL. */
DL_API dl_status dl_paged_cache_tensors(const dl_paged_cache* cache, int64_t layer, dl_tensor** key, dl_tensor** value);
/* A step: sequence b holds lengths[b] positions and gets counts[b] new ones; its position p lies in page
 * tables[b * width + p / page_size].  `shared` leading positions (whole pages, 0: none) lie in the same pages for all.
 * The arrays are host memory, read during the call.  Sequences with a count of 0 are not looked at.  The call waits for the
 * library's stream. */
DL_API dl_status dl_paged_batch_create(const dl_paged_cache* cache, int64_t heads, int64_t sequences,
    const int64_t* lengths, const int64_t* counts, const int64_t* tables, int64_t width, int64_t shared,
    dl_paged_batch** output);
DL_API void dl_paged_batch_release(dl_paged_batch* batch);
/* The step's keys, rotated, and values, [tokens, kv_heads, head_dim], into their pages of `layer`.  query [tokens, heads,
 * head_dim] and rotated are both NULL, or rotated receives the queries rotated likewise, f32. */
DL_API dl_status dl_paged_cache_append(dl_paged_cache* cache, int64_t layer, const dl_paged_batch* batch,
    const dl_tensor* query, const dl_tensor* key, const dl_tensor* value, const dl_tensor* cosine, const dl_tensor* sine,
    dl_rotary_layout layout, dl_tensor** rotated);
/* The step's queries [tokens, heads, head_dim] over the pages of `layer`, each row over the positions up to its own;
 * f32 [tokens, heads, head_dim]. */
DL_API dl_status dl_paged_attention(const dl_paged_cache* cache, int64_t layer, const dl_paged_batch* batch,
    const dl_tensor* query, dl_tensor** output);

/* ---- Extensions (no reference counterpart): who holds which page, forks and compaction; the gated delta rule over states of
 * fixed size; a layer of experts.  The rules stand at the C++ entries they call, dl/paged.h, dl/delta.h and dl/ops.h.  Arrays
 * of ids are host memory, read (or written) during the call; a refused call changes nothing. ---- */
typedef struct dl_page_pool dl_page_pool;
DL_API dl_status dl_page_pool_create(int64_t pages, dl_page_pool** output);
DL_API void dl_page_pool_release(dl_page_pool* pool);
DL_API dl_status dl_page_pool_available(const dl_page_pool* pool, int64_t* available);
DL_API dl_status dl_page_pool_references(const dl_page_pool* pool, int64_t page, int64_t* references);
/* `count` free pages, the lowest ones, to `pages`. */
DL_API dl_status dl_page_pool_take(dl_page_pool* pool, int64_t count, int64_t* pages);
/* One more holder (claim: of free pages too; share: of held ones), or one fewer, of each page; ids below zero are passed over. */
DL_API dl_status dl_page_pool_claim(dl_page_pool* pool, int64_t count, const int64_t* pages);
DL_API dl_status dl_page_pool_share(dl_page_pool* pool, int64_t count, const int64_t* pages);
DL_API dl_status dl_page_pool_give_back(dl_page_pool* pool, int64_t count, const int64_t* pages);
/* Page sources[i] to page targets[i] in every layer, the first rows[i] positions of it (rows NULL: all). */
DL_API dl_status dl_paged_cache_copy(dl_paged_cache* cache, int64_t count, const int64_t* sources, const int64_t* targets,
    const int64_t* rows);
/* New requests that go on from request parents[i] at its length: tables [sequences, width], forked [children, width]. */
DL_API dl_status dl_paged_cache_fork(dl_paged_cache* cache, dl_page_pool* pool, int64_t sequences, const int64_t* tables,
    int64_t width, const int64_t* lengths, int64_t children, const int64_t* parents, int64_t* forked);
/* Moves the held pages to the front of the pool and renames them in tables (`count` ids, all that hold pages); *moved (may be
 * NULL) receives how many. */
DL_API dl_status dl_paged_cache_compact(dl_paged_cache* cache, dl_page_pool* pool, int64_t count, int64_t* tables,
    int64_t* moved);

typedef struct dl_delta_states dl_delta_states;
typedef struct dl_delta_batch dl_delta_batch;
/* States [slots, heads, key_dim, value_dim], f32, of each layer, zero at first. */
DL_API dl_status dl_delta_states_create(int64_t layers, int64_t slots, int64_t heads, int64_t key_dim, int64_t value_dim,
    dl_device device, dl_delta_states** output);
DL_API void dl_delta_states_release(dl_delta_states* states);
/* A view of a layer's live storage. */
DL_API dl_status dl_delta_states_tensor(const dl_delta_states* states, int64_t layer, dl_tensor** output);
DL_API dl_status dl_delta_states_copy(dl_delta_states* states, int64_t count, const int64_t* sources, const int64_t* targets);
/* A step: request b goes on from slot sources[b] (-1: from zero) by counts[b] tokens and leaves its state in targets[b].  The
 * call waits for the library's stream. */
DL_API dl_status dl_delta_batch_create(const dl_delta_states* states, int64_t key_heads, int64_t requests,
    const int64_t* sources, const int64_t* targets, const int64_t* counts, dl_delta_batch** output);
DL_API void dl_delta_batch_release(dl_delta_batch* batch);
/* query and key [tokens, key_heads, key_dim], value [tokens, heads, value_dim], decay and rate [tokens, heads]; scale may be
 * NULL (1 / sqrt(key_dim)); f32 [tokens, heads, value_dim]. */
DL_API dl_status dl_gated_delta(dl_delta_states* states, int64_t layer, const dl_delta_batch* batch, const dl_tensor* query,
    const dl_tensor* key, const dl_tensor* value, const dl_tensor* decay, const dl_tensor* rate, const double* scale,
    dl_tensor** output);

/* input [..., d], router [E, d], gate and up [E, F, d], down [E, d, F]: output [..., d] f32, chosen [..., top] i64 and weights
 * [..., top] f32; the last two slots may be NULL. */
DL_API dl_status dl_expert_mixture(const dl_tensor* input, const dl_tensor* router, const dl_tensor* gate,
    const dl_tensor* up, const dl_tensor* down, int64_t top, int32_t normalise, dl_tensor** output, dl_tensor** chosen,
    dl_tensor** weights);
/* The module: dl_module_forward gives its output. */
DL_API dl_status dl_expert_mixture_create(int64_t dimensions, int64_t hidden, int64_t experts, int64_t top,
    int32_t normalise, dl_tensor_options options, dl_module** output);

#ifdef __cplusplus
}
#endif

#endif
