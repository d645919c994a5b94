// Launch entries of the hand-written CDNA4 kernels (gfx950).  Plain C structs of device pointers, sizes and a
// stream; each entry returns 0 or a HIP error code.  The host C++ layers fill these from tensors.
#pragma once

#include "backends/hip_backend.h"

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element codes follow dl_dtype */
enum { DLK_F32 = 0, DLK_F64 = 1, DLK_I64 = 2, DLK_BOOL = 3, DLK_BF16 = 5 };

/* ------------------------------------------------------------------------------------------------------
 * Projection GEMV over bf16 (or f32) weights, f32 activations and f32 accumulation:
 *   y[m, n] = epilogue( s_m * sum_k x[m, k] * g[k] * W[n, k] )
 * with g = the RMSNorm weight and s_m = 1/sqrt(mean_k x[m,k]^2 + eps) when apply_norm (the preceding RMSNorm
 * fused into this launch), else g = 1, s_m = 1.
 * Replaces the reference's cast_pair upcast + cuBLAS GEMM of every decoder Linear
 * (src/ops/matmul.cpp:14-67, src/kernels/cuda/matmul.cpp:9-93) and the RMSNorm/RoPE/KV-append/SiLU/residual
 * passes around them (src/kernels/cuda/normalization.cu:12-42, pointwise.cu:38-44,147-153,267-281).
 * ---------------------------------------------------------------------------------------------------- */
enum {
    DLK_EPI_STORE = 0,    /* y = acc (+ bias); optionally advances *bump_position by bump_count */
    DLK_EPI_RESIDUAL = 1, /* y = residual + acc; optionally advances *bump_position by bump_count */
    DLK_EPI_QKV = 2,      /* segments q|k|v: (+LoRA) RoPE on q,k; q -> y, k,v -> cache at position + l */
    DLK_EPI_SWIGLU = 3,   /* segments gate|up: y = silu(gate) * up */
    DLK_EPI_LOGITS = 4    /* y = acc; per-block best (value, index) for greedy / Gumbel-max sampling */
};

typedef struct dlk_sample_partial {
    double score;
    int64_t index;
} dlk_sample_partial;

typedef struct dlk_gemv_params {
    const float* x;         /* [M, ldx] f32 */
    int64_t ldx;
    int M, K;
    int nseg;               /* 1..3 weight segments stacked along n (STORE: their outputs side by side in y) */
    const void* w[3];       /* [seg_rows[i], K] row-major */
    const void* w_tiles[3]; /* optional, bf16: segment i repacked by dlk_pack_tiles, which the batched matrix-core
                               path reads instead of w (1 KB contiguous per load instruction) */
    int seg_rows[3];
    int w_bf16;
    int apply_norm;         /* fuse the preceding RMSNorm: scale row m by 1/sqrt(mean(x^2)+eps), weight g */
    const void* norm_weight; /* RMSNorm weight [K] (f32, or bf16 when norm_bf16); NULL means g = 1 */
    int norm_bf16;
    float epsilon;
    float acc_scale;        /* multiplies the accumulated dot products (1 for a plain projection) */
    int epilogue;
    float* y;               /* output rows [M, ldy] (QKV: the q rows) */
    int64_t ldy;
    const float* residual;  /* RESIDUAL: [M, ldres] f32 (may alias y) */
    int64_t ldres;
    const void* bias;       /* STORE: optional [N] */
    int bias_bf16;
    int64_t m_base;         /* global row of x row 0 (QKV position mapping, sample partial rows) */
    /* QKV */
    int head_dim, kv_heads, length; /* global row m -> batch m / length, position *position + m % length */
    const float* cosine;    /* [capacity, head_dim/2] f32 */
    const float* sine;
    const int64_t* position;
    void* k_cache;          /* [B, kv_heads, capacity, head_dim] */
    void* v_cache;
    int cache_bf16;
    int64_t cache_capacity;
    const float* lora_hidden[3]; /* per segment: [M_total, rank] f32 hidden = down(norm(x)) or NULL */
    int64_t lora_ld;             /* row stride of the lora_hidden rows (0: lora_rank) */
    const void* lora_up[3];      /* per segment: [seg_rows, rank] */
    const void* lora_down[3];    /* per segment: [rank, K] bf16 down rows that the launch applies itself (its
                                    lora_hidden NULL), when dlk_gemv_folds_lora says it can; else NULL */
    int lora_rank;
    float lora_scale;
    /* STORE / RESIDUAL: device cache length advanced by one thread after the launch's reads of it */
    int64_t* bump_position;
    int64_t bump_count;
    /* LOGITS */
    int sample_mode;        /* 0: none, 1: greedy, 2: Gumbel-max */
    double temperature;
    uint64_t key_seed, key_stream;
    const int64_t* key_label; /* if set, the key is fold_in(key, *key_label) */
    dlk_sample_partial* partial; /* [M_total, blocks] */
    int partial_blocks;
    /* Workspace for key-split launches of the matrix-core path (NULL: never split): partial dot products and
     * per-row sums of squares of each key slice, reduced in fixed order by a second launch. */
    float* split_partial;
    int64_t split_capacity; /* floats */
    /* Workspace of the staged (prompt and prefill) path: a preparation launch writes the activation rows (times the norm
     * weight) split into bf16 hi + lo rows and the per-row norm factors.  NULL: many-row launches take the
     * batched matrix-core path (64 rows per launch) instead. */
    void* stage;
    int64_t stage_bytes;
    int stage_ready;        /* the workspace already holds this launch's split rows (same x, norm weight, M, K) */
    int row_parts;          /* set by dlk_gemv for a launch it splits over activation rows (callers leave 0) */
    int defer_reduce;       /* QKV on the key-split matrix-core path: leave the partials for the one-position
                               attention to finish (no reduce launch); see dlk_attention_params.qkv_partial */
    void* stage_out;        /* SWIGLU on the tiled path: write silu(gate) * up, split into bf16 hi + lo, in the
                               staging layout of a following tiled launch over these rows (K = seg_rows[0]) instead
                               of y; that launch then takes it as its stage with stage_ready set */
} dlk_gemv_params;

/* Repacks bf16 weights for the batched matrix-core path: for each 16-row tile and 32-wide k step a 1 KB block
   whose 16 bytes at 16 l hold tile row l % 16, columns 32 s + 8 (l / 16) .. +8 (the MFMA operand of lane l).
   swiglu = 0: rows of w0 [rows, K], tile t = rows 16 t .. +16.  swiglu = 1: w0 = gate, w1 = up, each [rows, K];
   tile t interleaves gate and up rows 8 t .. +8 (tile row 2 j: gate 8 t + j, 2 j + 1: up 8 t + j).  out holds
   rows * K (swiglu: 2 * rows * K) bf16. */
int dlk_pack_tiles(const void* w0, const void* w1, int swiglu, int64_t rows, int64_t K, void* out, dlh_stream stream);
/* The kernel that dlk_gemv launches for these parameters: "gemv", "rows" (gemm_rows or gemm_wide), "narrow", "mid" or
   "tiles" (the staged ones), or "f32 " and its work-group shape. */
const char* dlk_gemv_kernel(const dlk_gemv_params* p);
/* 1 when dlk_gemv takes a batched matrix-core kernel (gemm_rows or gemm_wide, which read w_tiles) for this
   launch. */
int dlk_gemv_uses_rows(const dlk_gemv_params* p);
/* 1 when this QKV launch, with lora_down set for its adapted segments (and their lora_hidden NULL), computes the
   LoRA down projections itself: a launch over at most 16 rows on the few-row matrix-core kernel, bf16 weights,
   rank 4..16 in steps of 4, acc_scale 1.  dlk_gemv refuses lora_down otherwise. */
int dlk_gemv_folds_lora(const dlk_gemv_params* p);
/* Floats of workspace that lets dlk_gemv split the keys of this launch (0 when it would not split). */
int64_t dlk_gemv_split_floats(const dlk_gemv_params* p);
/* Key slices dlk_gemv will use for this launch as attached (1: no split). */
int dlk_gemv_split_count(const dlk_gemv_params* p);
/* Bytes of staging workspace that lets this launch take the tiled (prefill) path: attach it as stage /
   stage_bytes (0 when the shape does not suit that path). */
int64_t dlk_gemv_stage_bytes(const dlk_gemv_params* p);

/* Work-groups of the persistent launch (the LOGITS partial row length: one sampling candidate per work-group);
   -1 when no kernel fits the parameters.  Depends on the current device's CU count and the kernel's occupancy. */
int dlk_gemv_blocks(const dlk_gemv_params* p);
int dlk_gemv(const dlk_gemv_params* p, dlh_stream stream);

/* ------------------------------------------------------------------------------------------------------
 * Split-K GQA decode attention (flash-decoding).  Q rows m = b*L + l of [B*L, H*hd] f32 (post-RoPE);
 * K/V cache [B, KV, capacity, hd] (bf16 or f32, keys already rotated); first = *position (or first_host);
 * S = first + L keys; causal: row l sees keys <= first + l.  One work-group per (key split, query-row
 * block, b, kv head) stages 64-key K/V tiles in LDS and serves all H/KV query heads of that KV head.
 * Replaces grouped_block + attention_weights (src/ops/attention.cpp:65-95) i.e. two batched cuBLAS GEMMs
 * and attention_softmax_kernel (src/kernels/cuda/reduction.cu:149-169).
 * ---------------------------------------------------------------------------------------------------- */
typedef struct dlk_attention_params {
    const float* q;
    int64_t ldq;
    const void* k;
    const void* v;
    int kv_bf16;
    int64_t capacity;        /* rows per (b, kv head) in the K/V storage */
    const int64_t* position; /* device length before this chunk, or NULL to use first_host */
    int64_t first_host;
    int B, L, H, KV, hd;
    float scale;
    int causal;
    float* out;              /* [B*L, ldo] f32, head h at columns h*hd */
    int64_t ldo;
    int splits;              /* key splits; > 1 needs partial buffers */
    int chunk;               /* keys per split (multiple of the tile) */
    float* partial_o;        /* [B*H*L, splits, hd] */
    float* partial_ml;       /* [B*H*L, splits, 2] */
    int partials_only;       /* splits > 1: leave the merge of the partials to the caller (no combine launch) */
    /* One position on the matrix-core kernel: the QKV projection's key-split partials, left unreduced by it
       (dlk_gemv_params.defer_reduce).  The attention sums them in slice order for its sequence's q, k and v
       columns, applies the RMSNorm factor (row sums of squares after the dots) and RoPE at *position, and writes
       the new K/V row into the cache at *position (and uses the finished row for that key in place of the cache's).  Layout: [qkv_splits][B][qkv_width]
       dot products (q columns, then k, then v), then [qkv_splits][B] sums of squares. */
    const float* qkv_partial;
    int qkv_splits, qkv_width, qkv_K, qkv_norm;
    float qkv_scale, qkv_epsilon;
    const float* rope_cos;   /* [capacity, hd/2] */
    const float* rope_sin;
    void* stage_out;         /* prefill kernel only: write the output rows (row b * L + l, K = H * hd) split into
                                bf16 hi + lo in the staging layout of the tiled projection that reads them, instead
                                of out (see dlk_gemv_params.stage_out) */
    void* kv_split;          /* prefill kernel over an f32 cache: dlk_attention_split_bytes of workspace
                                (kv_split_tiles 64-key tiles per (b, kv head), covering the capacity).  A preparation
                                launch splits the live K/V tiles into bf16 hi + lo planes once, and the attention
                                copies them into LDS as they are instead of splitting each tile it reads */
    int kv_split_tiles;
    /* Explicit keep mask (reference grouped_query_attention, src/ops/attention.cpp:48-50,156-183), or NULL: bool
       bytes, key s of query row (b, h, l) kept when keep_mask[b * mask_stride[0] + h * mask_stride[1] +
       l * mask_stride[2] + s * mask_stride[3]] is nonzero (element strides, 0 on broadcast axes).  A dropped key's
       score is -inf before the softmax, and a row that keeps no key comes out NaN, as the reference's softmax of
       an all -inf row does.  Taken by the general and small-head kernels only (not causal, not the matrix-core or
       prefill kernels). */
    const unsigned char* keep_mask;
    int64_t mask_stride[4];
    /* Matrix-core decode kernel: keys the caller knows the cache holds at this launch (its host length plus the
       new position: the capture-time count for a replayed graph, whose length only grows), or 0.  A wave whose run
       of keys starts below it requests its first K/V tile before it reads the device length.  A hint for speed
       only: any value gives the same result. */
    int64_t early_keys;
    /* General kernel (head dim 16 and up): element strides of the query per sequence, position and head where its rows
       are not [B * L, ldq]; q_row 0: they are. */
    int64_t q_batch, q_row, q_head;
} dlk_attention_params;

/* Keys per split of a short one-position decode over a bf16 cache (few keys in all): 256 or 512, one work-group. */
#define DLK_DECODE_CHUNK_MAX 512
/* One-position decodes over at least this many keys in all (B * KV * keys), or over an f32 cache, split the keys
   into runs of 64..256 keys per wave (~4096 runs in all; a work-group per (sequence, KV head) from 256 pairs). */
#define DLK_STREAM_DECODE_KEYS 32768
/* 1 when the matrix-core one-position kernel serves this head layout (head dim 64 or 128, H/KV <= 16). */
int dlk_attention_matrix_heads(int heads, int kv_heads, int head_dim);


int dlk_attention(const dlk_attention_params* p, dlh_stream stream);
/* The kernel that dlk_attention launches for these parameters: "matrix", "prefill", "small", or "rows" and its row tiles
   per work-group. */
const char* dlk_attention_kernel(const dlk_attention_params* p);
/* 1 when dlk_attention takes the general kernel for these parameters, which reads the query through its strides. */
int dlk_attention_takes_strides(const dlk_attention_params* p);
/* Floats of the device-resident scratch array behind the allocation-free attention entry (8 MiB per GPU). */
#define DLK_ATTENTION_SCRATCH_FLOATS (2 << 20)
/* The address of that array on GPU `device` (looked up once per device with the device current; later calls
   return the kept address). */
int dlk_attention_scratch(int device, float** address);
/* The matrix-core causal prefill kernel (attention_prefill.hip), which dlk_attention takes for causal launches
   over bf16 or f32 K/V, head dim 64 or 128, L >= 16 new positions, one split and H/KV dividing 128. */
int dlk_attention_prefill_eligible(const dlk_attention_params* p);
/* Its part about the heads and the chunk: head dim 64 or 128, L >= 16, H/KV dividing 128. */
int dlk_attention_prefill_heads(int heads, int kv_heads, int head_dim, int length);
/* One position on the matrix cores (attention_matrix.hip): eligibility, and the launch of the attention kernel
   alone (with several splits it writes the partials; dlk_attention adds the merge). */
int dlk_attention_matrix_eligible(const dlk_attention_params* p);
int dlk_attention_matrix_decode(const dlk_attention_params* p, dlh_stream stream);
int dlk_attention_prefill(const dlk_attention_params* p, dlh_stream stream);
/* Bytes of kv_split workspace for these parameters: the capacity's 64-key tiles of every (b, kv head) as bf16
   hi + lo planes of K and V^T (0: no such path, a bf16 cache or not the prefill kernel). */
int64_t dlk_attention_split_bytes(const dlk_attention_params* p);

/* ------------------------------------------------------------------------------------------------------
 * Small kernels of the token loop and the tensor API.
 * ---------------------------------------------------------------------------------------------------- */
/* Strided copy with dtype conversion: dst[idx(dst_strides)] = convert(src[idx(src_strides)]), rank <= 8. */
int dlk_copy(const void* src, int src_dtype, const int64_t* src_strides, void* dst, int dst_dtype,
             const int64_t* dst_strides, const int64_t* shape, int rank, dlh_stream stream);
int dlk_fill(void* dst, int dtype, int64_t count, double value, dlh_stream stream);
/* Embedding rows: out[i, :] = weight[ids[i], :] converted to out_dtype; ids outside [0, V) give a zero row
 * and set *error_flag (if given) to 1. */
int dlk_embedding(const int64_t* ids, int64_t count, const void* weight, int weight_dtype, int64_t vocabulary,
                  int64_t width, void* out, int out_dtype, int32_t* error_flag, dlh_stream stream);
/* y[r, :] = x[r, :] / sqrt(mean(x^2) + eps) * weight (weight f32 or bf16, may be NULL); f32 in and out. */
int dlk_rms_norm(const float* x, int64_t rows, int64_t width, const void* weight, int weight_bf16, float epsilon,
                 float* y, dlh_stream stream);
/* Interleaved RoPE on contiguous x [outer, L, D] f32 with tables [L, D/2]. */
int dlk_rope(const float* x, int64_t outer, int64_t length, int64_t dim, const float* cosine, const float* sine,
             float* y, dlh_stream stream);
/* A launch has fewer than 2^32 threads: so many work-groups of 256. */
#define DLK_MOST_GROUPS ((1 << 24) - 1)

/* ------------------------------------------------------------------------------------------------------
 * Rows at given positions (rotary.hip): the queries, keys and values of `tokens` rows, queries and keys rotated by
 * the table row of the token's position, keys and values written to the pages of a paged cache.
 * ---------------------------------------------------------------------------------------------------- */
typedef struct dlk_row_segment {
    const void* x;           /* [tokens, heads, dim], last axis contiguous; NULL: the segment is absent */
    int bf16;                /* bf16 rows, else f32 */
    int heads;
    int64_t row, head;       /* element strides of a token and of a head */
} dlk_row_segment;

typedef struct dlk_rotary_params {
    dlk_row_segment q, k, v;
    int64_t tokens;
    int dim, part;           /* the first `part` (even) of each head's `dim` entries are rotated, the others copied */
    int half;                /* pairs (i, i + part / 2) instead of (2 i, 2 i + 1) */
    const int64_t* positions; /* [tokens] */
    const float* cosine;     /* [capacity, part / 2] */
    const float* sine;
    int64_t capacity;        /* a query row whose position lies outside [0, capacity) comes out NaN */
    float* out;              /* [tokens, q.heads, dim] */
    void* k_pages;           /* [pages, k.heads, page_size, dim] */
    void* v_pages;
    int pages_bf16;
    int page_shift;          /* log2 of the page size */
    const int64_t* places;   /* [tokens]: page * page_size + row of the token's place */
} dlk_rotary_params;
int dlk_rotary(const dlk_rotary_params* p, dlh_stream stream);

/* ------------------------------------------------------------------------------------------------------
 * Attention over the pages of a paged cache (attention_paged.hip).  The work of a call is a list of items, made once
 * for a step's batch: rows of one run of tokens over a range of its keys.  Row r of a run is token r / G and query
 * head r % G of the KV head's group (G = H / KV).
 * ---------------------------------------------------------------------------------------------------- */
typedef struct dlk_paged_item {
    int32_t token;           /* the run's first token */
    int32_t row_begin, row_end;
    int32_t table;           /* where the run's page ids start in `tables` (the page of key 0) */
    int32_t key_begin, key_end;
    int32_t first;           /* row r sees the keys up to first + r / G */
    int32_t slot;            /* the first row's place among the partials, or -1: the item is all that its rows see, and
                                writes the output */
} dlk_paged_item;

/* Items of one kind of work-group.  rows: the most rows of an item, 16 or 32 (the waves of a work-group split its keys) or
   128 (they split its rows). */
typedef struct dlk_paged_list {
    const dlk_paged_item* items;
    int count, rows;
} dlk_paged_list;

enum { DLK_PAGED_FEW = 0, DLK_PAGED_MANY = 1 };

/* One token whose rows several items share: its first row's place among the partials of its run's first split, how far
   apart the splits are, and how many of them hold keys that it sees; and the first row's place among the prefix's. */
typedef struct dlk_paged_merge {
    int32_t token, slot, stride, count, shared_slot;
} dlk_paged_merge;

typedef struct dlk_paged_params {
    const void* q;
    int q_bf16;
    int64_t q_row, q_head;   /* element strides of a token and of a head; 16-byte aligned rows */
    const void* k;           /* [pages, KV, page_size, hd] */
    const void* v;
    int kv_bf16, page_shift, H, KV, hd;
    float scale;
    const int32_t* tables;
    float* out;              /* [tokens, H, hd] */
    dlk_paged_list lists[2]; /* items of few rows, and of many */
    float* partial_o;        /* [KV, places, hd] */
    float* partial_ml;       /* [KV, places, 2]: base (a power of two) and sum */
    int places;
    int shared_splits, shared_stride; /* splits of the prefix that the whole batch shares (0: none), and how far apart */
    const dlk_paged_merge* merges;
    int merge_count, merge_most; /* merges, and the most partials of one */
} dlk_paged_params;
int dlk_paged_attention(const dlk_paged_params* p, dlh_stream stream);
/* Whether a launch holds `items` of each KV head and `merges`. */
int dlk_paged_fits(int64_t items, int64_t merges, int H, int KV, int hd);

/* ------------------------------------------------------------------------------------------------------
 * Copies of pages within pools of one layout [pages, heads, page, row] (page_copy.hip): the first `rows` rows of each head
 * of page `from` to page `to`, in every pool.  A page below zero is page ~from or ~to of the staging memory, which holds
 * `staged` pages for each pool.  No page of a launch is read and written, nor written twice (the caller sees to it).
 * ---------------------------------------------------------------------------------------------------- */
typedef struct dlk_page_pair {
    int32_t from, to, rows;
} dlk_page_pair;
#define DLK_PAGE_PAIRS 240
#define DLK_PAGE_POOLS 64
typedef struct dlk_page_copy_params { /* (an argument block of a launch: 3424 bytes, below 4 KB) */
    int pool_count, count;
    int heads, page, row_units; /* a row is row_units * 16 bytes */
    int staged;
    void* staging;              /* [pool_count, staged, heads, page, row] or NULL */
    void* pools[DLK_PAGE_POOLS];
    dlk_page_pair pairs[DLK_PAGE_PAIRS];
} dlk_page_copy_params;
int dlk_page_copy(const dlk_page_copy_params* p, dlh_stream stream);

/* ------------------------------------------------------------------------------------------------------
 * The gated delta rule over a step's tokens, one after the other (delta_step.hip) or in chunks of 64 (delta_chunk.hip).  Rows
 * are 16-byte aligned, also between heads and tokens; queries and keys are of one type.
 * ---------------------------------------------------------------------------------------------------- */
typedef struct dlk_delta_item { /* a request's new tokens: `count` from `token` on */
    int32_t source, target;     /* slots of its state before (-1: zero) and after */
    int32_t token, count;
    int32_t chunk, unused;      /* the first of its chunks */
} dlk_delta_item;
typedef struct dlk_delta_chunk { /* up to 64 tokens of a request */
    int32_t token, count;
} dlk_delta_chunk;

typedef struct dlk_delta_params {
    dlk_row_segment q, k, v; /* [tokens, heads / group, key_dim] and [tokens, heads, value_dim] */
    const float* decay;      /* [tokens, heads] */
    const float* rate;       /* [tokens, heads] */
    float* states;           /* [slots, heads, key_dim, value_dim] */
    float* out;              /* [tokens, heads, value_dim] */
    int heads, group, key_dim, value_dim;
    float scale;
    const dlk_delta_item* items;
    const dlk_delta_chunk* chunks;
    int item_count, chunk_count;
    /* set by dlk_delta_chunks: its workspace */
    uint16_t* solution;      /* [chunks, heads, 3 parts, 10 tiles, 16, 16] */
    float* within;           /* [chunks, heads, 10 tiles, 16, 16] */
    float* gates;            /* [chunks, heads, 3, 64] */
    uint16_t* turned_keys;   /* [parts, chunks, key heads, key_dim, 64] */
    uint16_t* key_parts;     /* [parts, chunks, key heads, 64, key_dim], f32 queries or keys only */
    uint16_t* query_parts;
} dlk_delta_params;
/* Bytes of workspace for the chunks of these parameters. */
int64_t dlk_delta_workspace(const dlk_delta_params* p);
int dlk_delta_chunks(const dlk_delta_params* p, void* workspace, dlh_stream stream);
int dlk_delta_step(const dlk_delta_params* p, dlh_stream stream);

/* ------------------------------------------------------------------------------------------------------
 * A layer of experts (experts.hip): for each of `tokens` rows x the `top` experts with the largest router logits, and
 *   y = sum_j weights_j down[e_j] (silu(gate[e_j] x) * (up[e_j] x))
 * ---------------------------------------------------------------------------------------------------- */
#define DLK_EXPERTS_MOST 1024    /* experts */
#define DLK_EXPERTS_TOP_MOST 64  /* chosen ones of a row */
typedef struct dlk_experts_params {
    const void* x;           /* [tokens, dim], x_bf16 or f32 */
    int x_bf16;
    const void* router;      /* [experts, dim] */
    const void* gate;        /* [experts, hidden, dim] */
    const void* up;
    const void* down;        /* [experts, dim, hidden] */
    int router_bf16, weights_bf16;
    int64_t tokens;
    int dim, hidden, experts, top;
    int normalise;           /* the chosen experts' weights are divided by their sum */
    float* y;                /* [tokens, dim] */
    int64_t* chosen;         /* [tokens, top] */
    float* weights;          /* [tokens, top] */
    void* workspace;         /* dlk_experts_workspace bytes, 16-byte aligned */
} dlk_experts_params;
/* The most rows of a launch, and the bytes of workspace that it takes. */
int64_t dlk_experts_rows(const dlk_experts_params* p);
int64_t dlk_experts_workspace(const dlk_experts_params* p);
int dlk_experts(const dlk_experts_params* p, dlh_stream stream);

/* First maximum of each row (NaN first); x [rows, n] f32 contiguous -> out i64 [rows]. */
int dlk_argmax(const float* x, int64_t rows, int64_t n, int64_t* out, dlh_stream stream);
/* Per-block candidates of a [rows, n] logits matrix (greedy or Gumbel-max), for dlk_sample_finalize. */
int dlk_sample_partials(const float* logits, int64_t rows, int64_t n, int mode, double temperature,
                        uint64_t key_seed, uint64_t key_stream, const int64_t* key_label,
                        dlk_sample_partial* partial, int blocks, dlh_stream stream);
int dlk_sample_blocks(int64_t n);
/* Reduces partial [rows, blocks] to ids: out[r] (may be NULL), next_ids[r] (may be NULL), and
 * tokens[r * token_stride + *step] when tokens != NULL; then advances *step by one if step != NULL.
 * With embedding != NULL it also writes the next step's input rows x[r, :] = f32(embedding[id, :]). */
int dlk_sample_finalize(const dlk_sample_partial* partial, int64_t rows, int blocks, int64_t* out,
                        int64_t* next_ids, int64_t* tokens, int64_t token_stride, int64_t* step,
                        const void* embedding, int embedding_dtype, int64_t width, float* x, dlh_stream stream);
/* ------------------------------------------------------------------------------------------------------
 * Verification of drafted tokens (verify.hip): target [batch, drafts + 1, vocabulary], draft [batch, drafts, vocabulary]
 * or NULL, uniforms [batch, drafts + 1], all f32 contiguous; drafted [batch, drafts], a negative id ends a row.
 * inverse = 1 / temperature (at most 1e300), or 0: the largest logit decides.
 * ---------------------------------------------------------------------------------------------------- */
typedef struct dlk_verify_slice { /* a slice of a row of logits: its largest, and the sum of exp((l - largest) / T) */
    double sum;
    float largest;
    int32_t index;           /* of the largest (greedy verification only) */
} dlk_verify_slice;

#define DLK_VERIFY_DRAW 1024
typedef struct dlk_verify_params {
    const int64_t* drafted;
    const float* target;
    const float* draft;
    const float* uniforms;
    int64_t batch, drafts, vocabulary;
    double inverse;
    int slices;              /* of a row, dlk_verify_slices */
    int64_t slice;           /* entries of one: slices * slice >= vocabulary */
    dlk_verify_slice* rows;  /* [batch, 2 drafts + 1, slices]: the target's rows, then the draft's */
    double* drawn;           /* [batch, ceil(vocabulary / DLK_VERIFY_DRAW), 2]: of the row that is drawn from, per so many
                                entries, what the target has over a refused draft, and the target's own */
    double* decisions;       /* [batch, 4]: the largest logit and one over the sum, of the row that is drawn from and of
                                the refused draft's (-1: none was refused) */
    int64_t* tokens;         /* [batch, drafts + 1]: accepted drafts, the drawn token, -1 */
    int64_t* accepted;       /* [batch] */
} dlk_verify_params;
/* Slices of a row, where `rows` rows of logits are read. */
int dlk_verify_slices(int64_t rows, int64_t vocabulary);
int dlk_verify(const dlk_verify_params* p, dlh_stream stream);
/* Keyed Philox: mode 0 uniform [low, high), mode 1 standard normal times scale; output f32 or bf16. */
int dlk_random(uint64_t seed, uint64_t stream_bits, int64_t count, int mode, double low, double high,
               double scale, void* out, int out_dtype, dlh_stream stream);
/* Plain y = x W^T (+ bias) for shapes the GEMV cannot take (K not a multiple of the 16-byte chunk). */
int dlk_linear_generic(const float* x, int64_t rows, int64_t K, const void* w, int w_dtype, int64_t N,
                       const void* bias, int bias_dtype, float* y, dlh_stream stream);
/* Streaming copy of `bytes` (multiple of 16) for the bandwidth probe. */
int dlk_stream_copy(const void* src, void* dst, uint64_t bytes, dlh_stream stream);

#ifdef __cplusplus
}
#endif
