/*
 * locus_sampler.h - C ABI of the MI355X (gfx950) token sampler.
 *
 * The drop-in boundary for the reference's per-step sampling path. The
 * reference has no C ABI for it: its callers use free C++ functions
 * (src/locus/model/sampling.hpp:70-89, llama.hpp:352) on host spans, one
 * row at a time (engine.cpp:423-450, engine.cpp:357-396). This ABI is what a
 * backend-registry entry (registry.hpp:107-131) or any FFI binds: plain
 * pointers and sizes, no exceptions, stream-ordered and asynchronous.
 *
 * All buffer pointers in lcs_batch / lcs_out / lcs_verify_* are DEVICE
 * pointers unless the field says "host". Every call is asynchronous on the
 * given HIP stream (a hipStream_t passed as void*, NULL = default stream);
 * outputs are valid once the stream has been synchronised. One context must
 * not be used by two threads at once; separate contexts are independent.
 */
#ifndef LOCUS_SAMPLER_H
#define LOCUS_SAMPLER_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct lcs_ctx lcs_ctx;

/* A row's raw statistics, as the fused lm-head's epilogue leaves them
 * (lcs_lmhead_out.stats): the log-normaliser of logprobs_from
 * (sampling.cpp:155-163) and the first index of the max (llama.cpp:1237-1245)
 * over the row's raw logits. 16 bytes. */
typedef struct lcs_row_stats {
    double log_z;              /* log sum_i exp(logit_i) */
    float max;                 /* largest raw logit */
    int32_t argmax;            /* its first index */
} lcs_row_stats;

enum lcs_status {
    LCS_OK = 0,
    LCS_ERR_INVALID_ARG = -1, /* bad pointer, size, alignment or dtype */
    LCS_ERR_NO_DEVICE = -2,   /* no usable gfx950 device */
    LCS_ERR_HIP = -3,         /* a HIP runtime call failed (see lcs_last_error) */
    LCS_ERR_CAPACITY = -4     /* request exceeds the context's create-time limits */
};

enum lcs_dtype {
    LCS_F32 = 0,
    LCS_BF16 = 1,
    LCS_E4M3 = 2              /* 8 bits (OCP e4m3, no infinities): lcs_add_rmsnorm, lcs_lmhead_ex, lcs_kv_cache */
};

enum lcs_flags {
    LCS_WANT_LOGPROBS = 1u,   /* write chosen_lp and the n_top alternatives */
    LCS_WRITE_PENALIZED = 2u  /* write penalised logits back in place (f32 only) */
};

/* Per-row sampling parameters: field-for-field the reference's
 * SamplingParams (src/locus/model/sampling.hpp:23-40), 32 bytes. */
typedef struct lcs_params {
    float temperature;        /* <= 0: greedy (argmax) */
    uint32_t top_k;           /* 0: disabled */
    float top_p;              /* 1: disabled */
    float min_p;              /* 0: disabled */
    float repeat_penalty;     /* 1: disabled */
    float frequency_penalty;  /* 0: disabled */
    float presence_penalty;   /* 0: disabled */
    uint32_t repeat_last_n;   /* trailing history entries the penalties see */
} lcs_params;

/* One batch of rows to sample: the batched form of
 * sample(logits, params, history, rng, constraint) (sampling.hpp:70-73)
 * followed, when LCS_WANT_LOGPROBS is set, by
 * logprobs_from(raw logits, chosen, n_top, ...) (sampling.hpp:86-89),
 * per row exactly as Engine::sample_from does (engine.cpp:423-450). */
typedef struct lcs_batch {
    uint32_t rows;
    uint32_t vocab;            /* V, 1 <= V <= 262144 */
    uint32_t dtype;            /* lcs_dtype */
    uint32_t flags;            /* lcs_flags */
    uint64_t row_stride;       /* elements between rows; multiple of 4 (f32) / 8 (bf16) */
    const void* logits;        /* rows x row_stride, 16-byte aligned, raw logits */
    const lcs_params* params;  /* rows */
    const lcs_params* params_host; /* optional HOST copy of params (dispatch hint) or NULL */
    const uint32_t* hist_off;  /* rows + 1 CSR offsets into hist_ids, or NULL */
    const int32_t* hist_ids;   /* token history (the request's generated ids) */
    const double* u;           /* rows: uniform in [0,1) per stochastic row, the
                                  generate_canonical<double,53> draw of the row's
                                  mt19937_64 (libstdc++ random.tcc:3348-3380).
                                  May be NULL only when params_host is given and
                                  no row has temperature > 0; otherwise a NULL u
                                  returns LCS_ERR_INVALID_ARG before any launch */
    const uint32_t* mask;      /* rows x mask_words allow-bits (bit t&31 of word
                                  t>>5, LSB first), or NULL for no constraint */
    const uint8_t* has_mask;   /* rows, nonzero = row constrained; NULL = all rows
                                  constrained when mask != NULL */
    uint32_t mask_words;       /* >= ceil(V/32) when mask != NULL */
    uint32_t n_top;            /* alternatives per row (<= the context's max_top) */
    const int32_t* lp_ids;     /* rows, or NULL: with LCS_WANT_LOGPROBS, chosen_lp
                                  reports the logprob of lp_ids[row] instead of the
                                  sampled id (logprobs_from's `chosen` argument,
                                  sampling.hpp:86-89); ids outside [0, V) give 0 */
    /* Device-resident penalty windows (lcs_windows_reserve). NULL: every row's
     * window comes from hist_off / hist_ids. Otherwise every row must be a
     * min-p window row (temperature > 0, min_p > 0, top_k 0, no mask; checked
     * against params_host, which is then required): */
    const int32_t* win_slot;   /* rows: the row's window slot, or -1 (hist_off / hist_ids) */
    const int32_t* win_push;   /* rows: the id the sequence appended since the slot's last
                                  call (its previous sample, engine.cpp:436), read when
                                  win_len grows by one */
    const uint32_t* win_len;   /* rows: the history length after that append: the slot's
                                  stored length (nothing appended) or one more; the slot's
                                  window, vocabulary and repeat_last_n must match the row,
                                  else the row gets id -1 and LCS_STATUS_WINDOW */
    /* Optional (NULL: computed here): each row's raw statistics over the same
     * logits, from the lcs_lmhead call that wrote them (lcs_lmhead_out.stats).
     * With LCS_WANT_LOGPROBS, greedy, min-p window and sliced top-k rows then
     * take their log-normaliser from it instead of summing the row's
     * exponentials again; the other paths compute their own. */
    const lcs_row_stats* raw_stats;
} lcs_batch;

/* Per-row diagnostics (optional output): the survivor set of the reference's
 * candidate walk (sampling.cpp:70-147). */
typedef struct lcs_row_diag {
    uint32_t n_cand;    /* candidates after the constraint */
    uint32_t keep;      /* survivors after top-k, top-p, min-p (0 for greedy) */
    float maxl;         /* max penalised candidate logit */
    float boundary;     /* logit of the last survivor */
    uint32_t path;      /* implementation path taken (LCS_PATH_*) */
    uint32_t reserved;  /* 1: a window row that the nucleus kernels decided, else 0 */
    double sum;         /* softmax normaliser over the candidate list */
    double kept_sum;    /* mass of the survivors */
} lcs_row_diag;

enum lcs_path {
    LCS_PATH_GREEDY = 1u,     /* sliced argmax */
    LCS_PATH_WINDOW = 2u,     /* sliced min-p window, certified normaliser */
    LCS_PATH_WINDOW_EXACT = 3u, /* window with an exactly recomputed normaliser */
    LCS_PATH_GENERAL = 4u,    /* exact selection over the whole row: one workgroup, or (a wide
                                 min-p window in a call that runs the nucleus kernels) theirs */
    LCS_PATH_TOPK = 5u,       /* sliced exact top-k (k <= 64) */
    LCS_PATH_NUCLEUS = 6u     /* sliced histogram passes, exact decisions (no top-k) */
};

typedef struct lcs_out {
    int32_t* ids;              /* rows: sampled token id */
    float* chosen_lp;          /* rows (LCS_WANT_LOGPROBS) */
    int32_t* top_ids;          /* rows x n_top (LCS_WANT_LOGPROBS) */
    float* top_lp;             /* rows x n_top (LCS_WANT_LOGPROBS) */
    lcs_row_diag* diag;        /* rows, or NULL */
} lcs_out;

/* Speculative-decoding verify (engine.cpp:357-396): row j of sequence s holds
 * the logits that predict draft[s*rows_per_seq + j]. */
typedef struct lcs_verify_batch {
    uint32_t n_seq;
    uint32_t rows_per_seq;     /* 1..64 */
    uint32_t vocab;
    uint32_t dtype;            /* lcs_dtype */
    uint64_t row_stride;       /* elements; multiple of 4 (f32) / 8 (bf16) */
    const void* logits;        /* (n_seq * rows_per_seq) x row_stride */
    const int32_t* draft;      /* n_seq * rows_per_seq draft ids */
} lcs_verify_batch;

typedef struct lcs_verify_out {
    int32_t* argmax_ids;       /* per row: argmax (llama.cpp:1237-1245) */
    float* draft_lp;           /* per row: logprobs_from(row, draft, 0).chosen_lp */
    uint32_t* accept_len;      /* per sequence: leading rows whose argmax == draft */
} lcs_verify_out;

/* Prompt-lookup drafts for a batch of device-resident contexts: per
 * sequence, the reference's ngram_draft (src/locus/model/speculative.cpp:7-28,
 * declared at speculative.hpp:9-19). */
typedef struct lcs_draft_batch {
    uint32_t n_seq;
    uint32_t ngram;            /* 0..64 (0: every draft empty) */
    uint32_t max_draft;        /* 0..256 */
    const uint32_t* ctx_off;   /* n_seq + 1 CSR offsets into ctx_ids */
    const int32_t* ctx_ids;    /* each sequence's context (prompt + generated) */
} lcs_draft_batch;

typedef struct lcs_draft_out {
    int32_t* draft;            /* n_seq x max_draft; entries past the draft are -1 */
    uint32_t* draft_len;       /* n_seq: the draft's length (0..max_draft) */
} lcs_draft_out;

/* The lm-head product with the sampler's first statistics in its epilogue:
 * logits = x w^T for bf16 x (rows x hidden, the normed hidden states) and w
 * (vocab x hidden, the output weight), accumulated in f32 - the reference's
 * matvec(out_w, norm(x)) per token (src/locus/model/llama.cpp:512-513,
 * 754-761). From the epilogue, without re-reading the logits: each row's
 * argmax (llama.cpp:1237-1245) and log-normaliser, the log-probability of a
 * draft token (logprobs_from with chosen = draft, sampling.cpp:150-170) and
 * each sequence's acceptance length (engine.cpp:357-383). */
typedef struct lcs_lmhead_batch {
    uint32_t rows;             /* hidden vectors, <= the context's max_rows */
    uint32_t vocab;            /* <= the context's max_vocab */
    uint32_t hidden;           /* multiple of 64 */
    uint32_t rows_per_seq;     /* 1..64 rows per sequence (accept_len), or 0 */
    const void* x;             /* rows x hidden bf16, 16-byte aligned */
    const void* w;             /* vocab x hidden bf16, 16-byte aligned */
    const int32_t* draft;      /* rows, or NULL: the token whose logprob each row reports */
} lcs_lmhead_batch;

typedef struct lcs_lmhead_out {
    float* logits;             /* rows x ld_logits f32, or NULL: not written */
    uint64_t ld_logits;        /* elements between rows of logits (>= vocab) */
    int32_t* argmax_ids;       /* rows */
    float* log_z;              /* rows: log sum exp of the row, or NULL */
    float* draft_lp;           /* rows (when draft != NULL), 0 for ids outside [0, vocab) */
    uint32_t* accept_len;      /* rows / rows_per_seq, or NULL */
    lcs_row_stats* stats;      /* rows, or NULL: each row's log_z, max and argmax, for
                                  lcs_batch.raw_stats of the lcs_sample call that samples
                                  these logits */
} lcs_lmhead_out;

/* The residual's addition and the root-mean-square norm ahead of the lm-head
 * (norm(x) of matvec(out_w, norm(x)), src/locus/model/llama.cpp:512-513):
 *   h = x + residual, y = h / sqrt(mean(h^2) + eps) * weight
 * per row, sums in f32, y and sum rounded once from f32 values (y from the
 * unrounded h). In e4m3, y holds y / y_scale with y_scale = max|y| / 448 of the
 * row (1 for a row of zeros, else 2^-126 at least): the operand of lcs_lmhead_ex.
 * A row that holds a NaN or an infinity has a NaN wherever the formula has one; in
 * e4m3 its y_scale is 1 if its largest |y| is a NaN. Squares and their sum are f32:
 * past 3e38 a row's y is 0. Rows and strides need the alignment of their elements
 * only. */
typedef struct lcs_norm_batch {
    uint32_t rows;
    uint32_t hidden;           /* 1..32768 */
    uint32_t x_dtype;          /* LCS_F32 or LCS_BF16: x, residual, weight and sum */
    uint32_t y_dtype;          /* LCS_F32, LCS_BF16 or LCS_E4M3 */
    float eps;                 /* > 0 */
    const void* x;             /* rows x x_stride */
    const void* residual;      /* rows x residual_stride, or NULL */
    const void* weight;        /* hidden */
    uint64_t x_stride;         /* elements between rows (>= hidden), of each buffer */
    uint64_t residual_stride;
} lcs_norm_batch;

typedef struct lcs_norm_out {
    void* y;                   /* rows x y_stride */
    float* y_scale;            /* rows (LCS_E4M3), else ignored */
    void* sum;                 /* rows x sum_stride: h, or NULL; needs residual; it may be x or
                                  residual itself (same stride), other overlaps may not be */
    uint64_t y_stride;
    uint64_t sum_stride;
} lcs_norm_out;

/* A pool of low-rank adapters beside the lm-head's weight: adapter i adds
 * scale[i] (x a[i]^T) b[i]^T to the logits of the rows that name it. Only an
 * adapter's first rank[i] ranks count, whatever the others hold. Infinities and
 * NaNs come out where the formula has them, in the rows of their adapter: a b of
 * -inf times a state above zero takes that column out. */
typedef struct lcs_adapters {
    uint32_t n;                /* 1..1024 */
    uint32_t wide;             /* ranks a slot of the pool holds: a multiple of 8, up to 256 */
    const void* a;             /* n x wide x hidden bf16, 16-byte aligned */
    const void* b;             /* n x vocab x wide bf16, 16-byte aligned */
    const int32_t* rank;       /* n (clamped to 0..wide), or NULL: wide */
    const float* scale;        /* n, or NULL: 1 */
} lcs_adapters;

/* lcs_lmhead_batch with the operands' type, their scales and the rows' adapters:
 * logits[i][v] = x_scale[i] w_scale[v] sum_k x[i][k] w[v][k], plus the product of
 * the row's adapter on x_scale[i] x[i]. All sums are f32 sums of exact products. */
typedef struct lcs_lmhead_ex_batch {
    uint32_t rows;             /* hidden vectors, <= the context's max_rows */
    uint32_t vocab;            /* <= the context's max_vocab */
    uint32_t hidden;           /* multiple of 64, up to 65536 */
    uint32_t rows_per_seq;     /* 1..64 rows per sequence (accept_len), or 0 */
    uint32_t dtype;            /* LCS_BF16 or LCS_E4M3: x and w */
    const void* x;             /* rows x hidden, 16-byte aligned */
    const void* w;             /* vocab x hidden, 16-byte aligned */
    const float* x_scale;      /* rows (LCS_E4M3), or NULL: 1 */
    const float* w_scale;      /* vocab (LCS_E4M3), or NULL: 1 */
    const int32_t* draft;      /* rows, or NULL: the token whose logprob each row reports */
    const lcs_adapters* adapters;  /* host struct, or NULL: none */
    const int32_t* slot;       /* rows (with adapters): the row's adapter; any id outside
                                  [0, n): none */
} lcs_lmhead_ex_batch;

/* A paged cache of keys and values for all layers. A sequence is a slot of `table`:
 * token t of sequence s lies in page table[s * max_pages + t / page_tokens], row t %
 * page_tokens. A page holds every layer's and head's rows of its tokens, and
 * refs[page] counts the sequences that hold it (0: free); pages may be shared
 * (lcs_kv_fork) and are then replaced by copies ahead of writes (lcs_kv_grow). The
 * reference's counterpart: its ref-counted copy-on-write cache on the host
 * (src/locus/kv/block_allocator.hpp:25-55, paged_cache.hpp:24-120). All buffers
 * are the caller's; a new cache's table is all -1, its refs all 0. */
typedef struct lcs_kv_cache {
    uint32_t layers, pages;
    uint32_t page_tokens;      /* a power of two, 16..1024 */
    uint32_t kv_heads;
    uint32_t head_dim;         /* a multiple of 16, up to 256 */
    uint32_t dtype;            /* LCS_BF16, or LCS_E4M3 with a scale per row */
    uint32_t seqs, max_pages;  /* slots of the table, pages a slot can hold */
    void* k;                   /* element d of a row: base + layer * layer_stride + page * page_stride + */
    void* v;                   /*   head * head_stride + row * token_stride + d, for both */
    float* k_scale;            /* layers x pages x kv_heads x page_tokens (LCS_E4M3): a row holds */
    float* v_scale;            /*   its values / its scale; else NULL */
    uint64_t layer_stride;     /* elements. Bases and strides are multiples of 16 bytes, rows do */
    uint64_t page_stride;      /*   not overlap (a size of 1 leaves its stride free), and a page's */
    uint64_t head_stride;      /*   rows of one head span less than 2 GiB */
    uint64_t token_stride;
    int32_t* table;            /* seqs x max_pages, -1: none */
    int32_t* refs;             /* pages */
} lcs_kv_cache;

/* Attention of a step's new tokens, R = rows_per_seq for each of n_seq sequences (one
 * token, a chain, or a tree of drafts), over their cached context and over each
 * other:
 *   o[r] = sum_j p_j v_j,  p = softmax_j(scale q[r] . k_j),  lse[r] = log sum_j exp(scale q[r] . k_j)
 * where j runs over the sequence's first length[i] cached tokens and over those of
 * its new tokens that row r's mask names. The new tokens' keys and values come from
 * k and v, not from the cache: what becomes of them is known after lcs_tree_verify
 * only (lcs_kv_append puts the accepted ones there). Query head h reads kv head
 * h / (heads / kv_heads). Scores, statistics and sums are f32; a weight is rounded
 * to bf16 for the product with the values, o once at the end. A row that sees
 * nothing (or scores of -inf only) has o = 0 and lse = -inf; one that meets a NaN or a
 * score of +inf is NaN. Scores past 2e38 in size may count as infinite, and an
 * element's sum, of weights up to 2^8, overflows where the number of tokens times their
 * largest |v| comes near 1e36. What a row does not see is no part of its result,
 * whatever it holds. o may not overlap what is read. */
typedef struct lcs_tree_attn_batch {
    uint32_t n_seq;            /* up to 1024, and n_seq * kv_heads up to 65536 */
    uint32_t rows_per_seq;     /* 1..256 */
    uint32_t heads;            /* a multiple of the cache's kv_heads */
    uint32_t layer;
    float scale;               /* at most 1e30, of either sign */
    uint32_t mask_words;       /* >= ceil(rows_per_seq / 32) when mask != NULL */
    const lcs_kv_cache* cache; /* host struct */
    const void* q;             /* row r = i * rows_per_seq + j, head h: q + r * q_stride + h * head_dim; bf16 */
    const void* k;             /* likewise, kv_heads a row */
    const void* v;
    uint64_t q_stride;         /* elements; bases and strides are multiples of 16 bytes, k's and v's at most 2^25 */
    uint64_t k_stride;
    uint64_t v_stride;
    const int32_t* seq;        /* n_seq: the sequence's slot of the cache, -1: no context; NULL: i */
    const int32_t* length;     /* n_seq: cached tokens (below 0: none) */
    const uint32_t* mask;      /* rows x mask_words, bit j & 31 of word j >> 5: the row sees its sequence's new
                                  token j; NULL: new tokens 0 .. its own */
} lcs_tree_attn_batch;

typedef struct lcs_tree_attn_out {
    void* o;                   /* as q, bf16 */
    uint64_t o_stride;         /* elements, a multiple of 16 bytes */
    float* lse;                /* rows x heads, or NULL */
} lcs_tree_attn_out;

/* The greedy verdict on a tree of drafts: lcs_verify for trees. Node j of sequence i
 * is row i * rows_per_seq + j. Node 0 is the root, the last token that is certain;
 * node j > 0 drafts tokens[j] as a continuation of node parent[j] < j (a node with
 * another parent is never accepted). Row j of the logits predicts what follows node
 * j: from the root on, the lowest child whose token is its parent's argmax is
 * accepted (engine.cpp:357-396 along a chain). */
typedef struct lcs_tree_verify_batch {
    uint32_t n_seq;
    uint32_t rows_per_seq;     /* 1..256 */
    uint32_t vocab;
    uint32_t dtype;            /* LCS_F32 or LCS_BF16 */
    uint64_t row_stride;       /* elements; multiple of 4 (f32) / 8 (bf16) */
    const void* logits;        /* rows x row_stride, 16-byte aligned; NULL: out->argmax_ids holds the rows'
                                  argmax (lcs_lmhead), vocab, dtype and row_stride are not read */
    const int32_t* tokens;     /* rows */
    const int32_t* parent;     /* rows (the root's is not read) */
    const int32_t* length;     /* n_seq: cached tokens, for out->length; or NULL */
} lcs_tree_verify_batch;

typedef struct lcs_tree_verify_out {
    int32_t* argmax_ids;       /* rows: argmax (llama.cpp:1237-1245); read where logits is NULL */
    float* node_lp;            /* rows: log-probability of the node's token under its parent's row (0 for the
                                  root, other parents and ids outside [0, vocab)), or NULL; needs logits */
    int32_t* path;             /* rows: each sequence's accepted nodes, the root first, then -1 */
    int32_t* n_path;           /* n_seq: their number, 1 .. rows_per_seq */
    int32_t* next_id;          /* n_seq: the argmax at the path's end */
    int32_t* length;           /* n_seq: length + n_path, or NULL; needs length; it may be the same buffer */
} lcs_tree_verify_out;

/* New rows of a cache: token j < count[i] of sequence i goes to position pos[i] + j,
 * from row i * rows_per_seq + (index ? index[i * rows_per_seq + j] : j) of each of
 * n_layers layers. Into e4m3 as lcs_add_rmsnorm's y: a scale of max|x| / 448 per row
 * (1 for a row of zeros, or one that holds a NaN; 2^-126 at least), x / scale cut to
 * +-448 and rounded to nearest even, a NaN staying one. */
typedef struct lcs_kv_append_batch {
    uint32_t n_seq;            /* up to 1024 */
    uint32_t rows_per_seq;     /* 1..2^20, and n_seq * n_layers * ceil(rows_per_seq / 4) below 2^32 */
    uint32_t layer, n_layers;  /* the first one, and how many */
    const void* k;             /* layer l (from 0), row r, head h: k + l * layer_stride + r * k_stride + h * head_dim; bf16 */
    const void* v;
    uint64_t layer_stride;     /* elements, of both; bases and strides are multiples of 16 bytes */
    uint64_t k_stride, v_stride;
    const int32_t* seq;        /* n_seq: slots, -1: nothing to do; NULL: i */
    const int32_t* pos;        /* n_seq */
    const int32_t* count;      /* n_seq (clamped to 0..rows_per_seq), or NULL: rows_per_seq */
    const int32_t* index;      /* n_seq x rows_per_seq, or NULL */
} lcs_kv_append_batch;

/* Number of usable gfx950 devices (0 when none). Replaces the runtime probe
 * that sets Backend::available (registry.cpp:148-223, cuda_stub.cpp:29). */
int lcs_probe(int* n_devices);

/* Allocates the per-context workspace on `device` once; no call below
 * allocates device memory. Returns NULL on failure (lcs_last_error(NULL)). */
lcs_ctx* lcs_create(int device, uint32_t max_rows, uint32_t max_vocab,
                    uint32_t max_hist, uint32_t max_top);
void lcs_destroy(lcs_ctx* ctx);

/* Device-resident penalty windows: the counts apply_penalties builds from
 * the history's last repeat_last_n ids (sampling.cpp:22-28) kept per
 * sequence slot on the device and updated in place by each lcs_sample call
 * that names the slot (one id enters the window, at most one leaves), so a
 * serving loop uploads no history. Allocates room for `slots` slots of
 * windows up to `max_window` ids (<= 4096), once (call it before the hot
 * loop; calling again with larger limits reallocates and clears every slot).
 * No counterpart in the reference, which rescans the history per call. */
int lcs_windows_reserve(lcs_ctx* ctx, uint32_t slots, uint32_t max_window);

/* (Re)starts slot `slot` for a sequence whose generated history so far is
 * ids[0..n) (device memory; n may be 0, ids may then be NULL), penalised
 * over its last `window` ids (1..max_window: the rows' repeat_last_n) for
 * a vocabulary of `vocab` ids. Asynchronous on `stream`. */
int lcs_windows_load(lcs_ctx* ctx, uint32_t slot, const int32_t* ids, uint32_t n, uint32_t window,
                     uint32_t vocab, void* stream);

/* Batched sample (+ logprobs): replaces per-row sample()/logprobs_from()
 * (sampling.hpp:70-89) as called from engine.cpp:430-442. */
int lcs_sample(lcs_ctx* ctx, const lcs_batch* batch, const lcs_out* out, void* stream);

/* Batched logprobs_from (sampling.hpp:86-89, sampling.cpp:150-190) with no
 * draw: per row, into out->chosen_lp, the log-probability of chosen[row]
 * under the row's raw logits (0 for an id outside [0, V); chosen NULL: of the
 * row's argmax), and into out->top_ids / top_lp the batch's n_top most likely
 * ids with theirs; out->ids, when given, receives each row's argmax. Reads
 * rows, vocab, dtype, row_stride, logits, n_top and raw_stats of batch and
 * ignores the rest (params, history, u, mask, flags, windows). The backend
 * registry's logprobs_batch op. */
int lcs_logprobs(lcs_ctx* ctx, const lcs_batch* batch, const int32_t* chosen, const lcs_out* out, void* stream);

/* lcs_sample without a context, allocating nothing: for callers that cannot
 * call hipMalloc (code under HIP graph capture, tight serving loops, harnesses
 * that forbid it). No counterpart in the reference. Runs on the current
 * device with the same batch, outputs and results as lcs_sample; its
 * workspace is one static device array per GPU (about 38 MiB, held until the
 * process ends), sized for rows <= 64, any vocabulary up to 262144, n_top <=
 * 20 and penalty windows up to 8192. More rows return LCS_ERR_CAPACITY with
 * nothing launched. Calls share that array: calls that overlap on one GPU
 * (two streams, or two threads) race and must be serialised by the caller.
 * Its status bits are not readable (lcs_get_status needs a context); failures
 * are reported by lcs_last_error(NULL). */
int lcs_sample_noalloc(const lcs_batch* batch, const lcs_out* out, void* stream);

/* Batched greedy verify: replaces the argmax loop of engine.cpp:357-396 and
 * adds the draft logprob (sampling.cpp:150-170 with chosen = draft). */
int lcs_verify(lcs_ctx* ctx, const lcs_verify_batch* batch, const lcs_verify_out* out,
               void* stream);

/* Batched n-gram drafts: replaces the per-sequence host call of
 * engine.cpp:328-329 (speculative.cpp:7-28) when contexts live on the device.
 * Drafts feed lcs_verify. Allocates nothing and uses no context workspace, so
 * n_seq is not bounded by the context's max_rows. */
int lcs_ngram_draft(lcs_ctx* ctx, const lcs_draft_batch* batch, const lcs_draft_out* out, void* stream);

/* The fused lm-head product (see lcs_lmhead_batch); no counterpart call in
 * the reference, which computes the logits with matvec and reads them again
 * in argmax / logprobs_from. Allocates nothing. */
int lcs_lmhead(lcs_ctx* ctx, const lcs_lmhead_batch* batch, const lcs_lmhead_out* out, void* stream);

/* The fused lm-head product in bf16 or e4m3, with the rows' low-rank adapters (see
 * lcs_lmhead_ex_batch); outputs as lcs_lmhead. No counterpart call in the
 * reference. Allocates nothing. */
int lcs_lmhead_ex(lcs_ctx* ctx, const lcs_lmhead_ex_batch* batch, const lcs_lmhead_out* out, void* stream);

/* Residual addition and norm, optionally into 8 bits (see lcs_norm_batch). Allocates
 * nothing and uses no context workspace: rows are not bounded by max_rows. */
int lcs_add_rmsnorm(lcs_ctx* ctx, const lcs_norm_batch* batch, const lcs_norm_out* out, void* stream);

/* The workspace of lcs_kv_grow and lcs_tree_attn: room for `new_pages` pages that one
 * lcs_kv_grow call may allocate, and for the partial results of lcs_tree_attn (34 MB).
 * Allocates once, ahead of the hot loop; a call with a larger limit reallocates, and
 * graphs that were captured ahead of it are then to be captured anew. Nothing in it
 * outlives a call, but calls on one context share it: issue them, and graphs that hold
 * them, on one stream, or order the streams. */
int lcs_kv_reserve(lcs_ctx* ctx, uint32_t new_pages);

/* The bookkeeping of a paged cache, on the device, for n <= 1024 requests per call. Slots
 * are in device memory, so bad ones are refused there: result[i] is 0, or -1 for a
 * request that changed nothing, with LCS_STATUS_PAGES set. A slot of -1 asks for
 * nothing (result 0, but behind a shortage in lcs_kv_grow). A slot outside [0, seqs)
 * is refused, and one that an earlier request of the call has named. No counterpart
 * call in the reference, which does this on the host (paged_cache.hpp:24-120).
 *
 * lcs_kv_grow: slot seq[i] gets a page of its own wherever one is missing or shared at
 * its tokens [start[i], end[i]): a missing one a free page, a shared one a copy (all
 * layers) that takes its place, also if all its holders ask in this call. Free pages
 * go to the requests in order, the lowest first; from the first request that there
 * are not enough for, none is served, whatever it asks for: result -1, for a slot of
 * -1 too. start > end and ends past the table are refused.
 * lcs_kv_fork: slot dst[i], which holds no page, shares slot src[i]'s first tokens[i]
 * tokens. Refused where a page of them is missing, dst holds any, or src is itself
 * some request's dst.
 * lcs_kv_free: slot seq[i] gives up its pages past its first keep[i] tokens (keep NULL
 * or below 0: all). A page that nobody else holds is free again. */
int lcs_kv_grow(lcs_ctx* ctx, const lcs_kv_cache* cache, uint32_t n, const int32_t* seq, const int32_t* start,
                const int32_t* end, int32_t* result, void* stream);
int lcs_kv_fork(lcs_ctx* ctx, const lcs_kv_cache* cache, uint32_t n, const int32_t* src, const int32_t* dst,
                const int32_t* tokens, int32_t* result, void* stream);
int lcs_kv_free(lcs_ctx* ctx, const lcs_kv_cache* cache, uint32_t n, const int32_t* seq, const int32_t* keep,
                int32_t* result, void* stream);

/* Keeps count[i] (clamped to 0..max_keep) of slot seq[i]'s tokens, in all layers: row
 * keep[i * max_keep + j] moves to position j, in place. keep is ascending. Refused
 * (result -1, nothing moved) where it is not, where a page is missing, or where a page
 * that would be written is shared (lcs_kv_grow gives copies). What lies past the
 * last one is left as it was; lcs_kv_free gives its pages back. Slots as above. */
int lcs_kv_compact(lcs_ctx* ctx, const lcs_kv_cache* cache, uint32_t n, uint32_t max_keep, const int32_t* seq,
                   const int32_t* count, const int32_t* keep, int32_t* result, void* stream);

/* New rows of a cache (see lcs_kv_append_batch). A row whose page is missing or shared,
 * or whose index or position is out of range, is not written and sets
 * LCS_STATUS_PAGES. Rows that go to one place (a slot named twice) are a race.
 * Allocates nothing and uses no context workspace. */
int lcs_kv_append(lcs_ctx* ctx, const lcs_kv_cache* cache, const lcs_kv_append_batch* batch, void* stream);

/* Attention over the cache and the new tokens (see lcs_tree_attn_batch), after
 * lcs_kv_reserve. Allocates nothing.
 * A page that is missing below length[i] counts as not seen and sets LCS_STATUS_PAGES, as
 * does a slot outside [-1, seqs) or a length past the table. */
int lcs_tree_attn(lcs_ctx* ctx, const lcs_tree_attn_batch* batch, const lcs_tree_attn_out* out, void* stream);

/* Verdict on a tree of drafts (see lcs_tree_verify_batch). Allocates nothing and uses no
 * context workspace. */
int lcs_tree_verify(lcs_ctx* ctx, const lcs_tree_verify_batch* batch, const lcs_tree_verify_out* out, void* stream);

/* Sticky device-side status bits of ctx (LCS_STATUS_*), set by kernels that
 * met an input they could not serve. Every bit of the sampling calls comes with id
 * -1 on each affected row (also from lcs_sample_noalloc, whose status is not readable),
 * so a caller that sees no -1 id needs no status read. Blocking:
 * reads device memory; call after the work's stream has been synchronised.
 * No counterpart in the reference (its sampler cannot fail). */
int lcs_get_status(lcs_ctx* ctx, uint32_t* status_out, int reset);

enum lcs_status_bits {
    LCS_STATUS_HIST_CAPACITY = 1u,  /* a penalty window exceeded max_hist */
    LCS_STATUS_SELECT = 2u,         /* a selection bin exceeded its capacity */
    LCS_STATUS_WINDOW = 4u,         /* a row's window slot did not match it (win_len, window,
                                       vocabulary) */
    LCS_STATUS_PAGES = 8u           /* a cache request was refused, or a page was missing */
};

/* Message of the last failure on ctx (or, when NULL, of the last lcs_create
 * or lcs_sample_noalloc on this thread). */
const char* lcs_last_error(const lcs_ctx* ctx);

#ifdef __cplusplus
}
#endif
#endif /* LOCUS_SAMPLER_H */
