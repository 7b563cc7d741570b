// What the paged cache's calls, lcs_tree_attn and lcs_tree_verify refuse, before any
// launch (plain host code: the CPU tests compile it by itself).
#pragma once

#include "lcs_check.hpp"

namespace lcs {

struct Why {   // (the status of a refusal, and its message)
    const char** why;
    int no(const char* m) const { *why = m; return LCS_ERR_INVALID_ARG; }
    int over(const char* m) const { *why = m; return LCS_ERR_CAPACITY; }
};

// Whether rows of `row` elements at these four sizes and strides do not overlap: each
// dimension's stride, from the smallest on, is past what the smaller ones span.
inline bool rows_apart(uint64_t row, const uint64_t (&size)[4], const uint64_t (&stride)[4]) {
    bool done[4] = {};
    unsigned __int128 span = row;
    for (int n = 0; n < 4; ++n) {
        int at = -1;
        for (int i = 0; i < 4; ++i)
            if (!done[i] && size[i] > 1 && (at < 0 || stride[i] < stride[at])) at = i;
        if (at < 0) break;
        if ((unsigned __int128)stride[at] < span) return false;
        span += (unsigned __int128)stride[at] * (size[at] - 1u);
        done[at] = true;
    }
    return span < ((unsigned __int128)1 << 62);
}

inline int check_kv_cache(const lcs_kv_cache* c, const char** why) {
    const Why w{why};
    if (!c) return w.no("null cache");
    if (c->dtype != LCS_BF16 && c->dtype != LCS_E4M3) return w.no("cache: dtype must be bf16 or e4m3");
    if (c->layers == 0 || c->layers > 4096) return w.no("cache: layers must be 1..4096");
    if (c->pages == 0 || c->pages > 0x7fffffffu) return w.no("cache: pages must be 1..2^31 - 1");
    if (c->page_tokens < 16 || c->page_tokens > 1024 || (c->page_tokens & (c->page_tokens - 1u))) {
        return w.no("cache: page_tokens must be a power of two, 16..1024");
    }
    if (c->kv_heads == 0 || c->kv_heads > 1024) return w.no("cache: kv_heads must be 1..1024");
    if (c->head_dim == 0 || c->head_dim % 16 != 0 || c->head_dim > 256) return w.no("cache: head_dim must be a multiple of 16 up to 256");
    if (c->seqs == 0 || c->max_pages == 0 || (uint64_t)c->seqs * c->max_pages > 0x7fffffffull) {
        return w.no("cache: the table must have 1..2^31 - 1 entries");
    }
    if (!c->k || !c->v || !c->table || !c->refs) return w.no("cache: null k / v / table / refs");
    if (misaligned(c->k, 16u) || misaligned(c->v, 16u) || misaligned(c->refs, 16u)) {
        return w.no("cache: k, v and refs must be 16-byte aligned");
    }
    if (misaligned(c->table, 4u) || misaligned(c->k_scale, 4u) || misaligned(c->v_scale, 4u)) {
        return w.no("a pointer is not aligned to its elements");
    }
    if (c->dtype == LCS_E4M3 ? !c->k_scale || !c->v_scale : c->k_scale || c->v_scale) {
        return w.no("cache: k_scale and v_scale go with e4m3");
    }
    const uint64_t es = c->dtype == LCS_BF16 ? 2u : 1u;
    const uint64_t size[4] = {c->layers, c->pages, c->kv_heads, c->page_tokens};
    const uint64_t stride[4] = {c->layer_stride, c->page_stride, c->head_stride, c->token_stride};
    for (int i = 0; i < 4; ++i)
        if (size[i] > 1 && stride[i] * es % 16u != 0) return w.no("cache: strides must be multiples of 16 bytes");
    if (!rows_apart(c->head_dim, size, stride)) return w.no("cache: rows must not overlap");
    if (c->token_stride >= 0x80000000ull / (c->page_tokens * es)) return w.no("cache: a page's rows of one head must span less than 2 GiB");
    return LCS_OK;
}

inline int check_kv_requests(const lcs_kv_cache* c, uint32_t n, const int32_t* seq, const int32_t* a, const int32_t* b,
                             const int32_t* result, uint32_t max_req, const char** why) {
    const Why w{why};
    const int rc = check_kv_cache(c, why);
    if (rc != LCS_OK) return rc;
    if (n == 0) return LCS_OK;
    if (n > max_req) return w.over("at most 1024 requests a call");
    if (!seq || !a || !b || !result) return w.no("null request array");
    if (misaligned(seq, 4u) || misaligned(a, 4u) || misaligned(b, 4u) || misaligned(result, 4u)) {
        return w.no("a pointer is not aligned to its elements");
    }
    return LCS_OK;
}

inline int check_kv_compact(const lcs_kv_cache* c, uint32_t n, uint32_t max_keep, const int32_t* seq, const int32_t* count,
                            const int32_t* keep, const int32_t* result, uint32_t max_req, const char** why) {
    const Why w{why};
    const int rc = check_kv_requests(c, n, seq, count, max_keep ? keep : count, result, max_req, why);
    if (rc != LCS_OK) return rc;
    if (max_keep > 0x7fffffffu) return w.no("max_keep must be below 2^31");
    if ((uint64_t)n * c->layers * 2u * c->kv_heads > 0x7fffffffull) return w.over("too many requests, layers and heads for a call");
    return LCS_OK;
}

inline int check_kv_append(const lcs_kv_cache* c, const lcs_kv_append_batch* b, uint32_t max_req, const char** why) {
    const Why w{why};
    if (!b) return w.no("null append argument");
    const int rc = check_kv_cache(c, why);
    if (rc != LCS_OK) return rc;
    if (b->n_seq == 0 || b->n_layers == 0) return LCS_OK;
    if (b->n_seq > max_req) return w.over("at most 1024 sequences a call");
    if (b->rows_per_seq == 0 || b->rows_per_seq > 1u << 20) return w.no("rows_per_seq must be 1..2^20");
    if (b->layer >= c->layers || b->n_layers > c->layers - b->layer) return w.no("layers outside the cache's");
    if (!b->k || !b->v || !b->pos) return w.no("null k / v / pos");
    if (misaligned(b->k, 16u) || misaligned(b->v, 16u)) return w.no("k and v must be 16-byte aligned");
    if (misaligned(b->seq, 4u) || misaligned(b->pos, 4u) || misaligned(b->count, 4u) || misaligned(b->index, 4u)) {
        return w.no("a pointer is not aligned to its elements");
    }
    const uint64_t row = (uint64_t)c->kv_heads * c->head_dim;
    if (b->k_stride < row || b->v_stride < row) return w.no("row strides must be at least kv_heads * head_dim");
    if (b->k_stride % 8u || b->v_stride % 8u || (b->n_layers > 1 && b->layer_stride % 8u)) {
        return w.no("strides must be multiples of 16 bytes");
    }
    // (a workgroup for four tokens of a sequence and layer)
    if ((uint64_t)b->n_seq * ((b->rows_per_seq + 3u) / 4u) * b->n_layers > 0xffffffffull) return w.over("too many rows and layers for a call");
    return LCS_OK;
}

inline int check_tree_attn(const lcs_tree_attn_batch* b, const lcs_tree_attn_out* o, uint32_t max_req, uint32_t max_pairs,
                           const char** why) {
    const Why w{why};
    if (!b || !o) return w.no("null attention argument");
    const lcs_kv_cache* c = b->cache;
    const int rc = check_kv_cache(c, why);
    if (rc != LCS_OK) return rc;
    if (b->n_seq == 0) return LCS_OK;
    if (b->n_seq > max_req) return w.over("at most 1024 sequences a call");
    if (b->rows_per_seq == 0 || b->rows_per_seq > 256) return w.no("rows_per_seq must be 1..256");
    if (b->heads == 0 || b->heads % c->kv_heads != 0 || b->heads > 65536) return w.no("heads must be a multiple of kv_heads, up to 65536");
    if (b->layer >= c->layers) return w.no("layer outside the cache's");
    if (!finite_bits(b->scale) || b->scale > 1e30f || b->scale < -1e30f) return w.no("scale must be a number of at most 1e30");
    if (!b->q || !b->k || !b->v || !b->length || !o->o) return w.no("null q / k / v / length / o");
    if (misaligned(b->q, 16u) || misaligned(b->k, 16u) || misaligned(b->v, 16u) || misaligned(o->o, 16u)) {
        return w.no("q, k, v and o must be 16-byte aligned");
    }
    if (misaligned(b->seq, 4u) || misaligned(b->length, 4u) || misaligned(b->mask, 4u) || misaligned(o->lse, 4u)) {
        return w.no("a pointer is not aligned to its elements");
    }
    if (b->mask && b->mask_words < (b->rows_per_seq + 31u) / 32u) return w.no("mask_words < ceil(rows_per_seq / 32)");
    const uint64_t D = c->head_dim;
    if (b->q_stride < b->heads * D || o->o_stride < b->heads * D || b->k_stride < c->kv_heads * D || b->v_stride < c->kv_heads * D) {
        return w.no("row strides must be at least a row's heads");
    }
    if (b->q_stride % 8u || b->k_stride % 8u || b->v_stride % 8u || o->o_stride % 8u) return w.no("strides must be multiples of 16 bytes");
    if (c->pages > 1 && c->page_stride * (c->dtype == LCS_BF16 ? 2u : 1u) > 0xffffffffull) return w.no("the cache's pages must be less than 4 GiB apart");
    if (b->k_stride > 1u << 25 || b->v_stride > 1u << 25) return w.no("k_stride and v_stride must be at most 2^25");
    if ((uint64_t)b->n_seq * b->rows_per_seq * b->heads > 0x7fffffffull) return w.over("too many rows and heads for a call");
    if ((uint64_t)b->n_seq * c->kv_heads > max_pairs) return w.over("at most 65536 sequences x kv heads a call");
    // (steps of 128 tokens, of every sequence and kv head)
    const uint64_t steps = ((uint64_t)c->max_pages * c->page_tokens + 127u) / 128u + 2u;
    if (steps > 0x40000000ull || steps * b->n_seq * c->kv_heads > 0x40000000ull) return w.over("sequences, table and heads beyond 2^30 steps of 128 tokens");
    return LCS_OK;
}

inline int check_tree_verify(const lcs_tree_verify_batch* b, const lcs_tree_verify_out* o, const char** why) {
    const Why w{why};
    if (!b || !o) return w.no("null verify argument");
    if (b->n_seq == 0) return LCS_OK;
    if (b->rows_per_seq == 0 || b->rows_per_seq > 256) return w.no("rows_per_seq must be 1..256");
    if ((uint64_t)b->n_seq * b->rows_per_seq > 0x7fffffffull) return w.over("too many rows for a call");
    if (!b->tokens || !b->parent || !o->argmax_ids || !o->path || !o->n_path || !o->next_id) {
        return w.no("null tokens / parent / argmax_ids / path / n_path / next_id");
    }
    if (misaligned(b->tokens, 4u) || misaligned(b->parent, 4u) || misaligned(b->length, 4u) || misaligned(o->argmax_ids, 4u) ||
        misaligned(o->node_lp, 4u) || misaligned(o->path, 4u) || misaligned(o->n_path, 4u) || misaligned(o->next_id, 4u) ||
        misaligned(o->length, 4u)) {
        return w.no("a pointer is not aligned to its elements");
    }
    if (o->length && !b->length) return w.no("length out needs length");
    if (!b->logits) return o->node_lp ? w.no("node_lp needs logits") : (int)LCS_OK;
    if (b->dtype != LCS_F32 && b->dtype != LCS_BF16) return w.no("dtype must be f32 or bf16");
    if (b->vocab == 0 || b->vocab > 0x7fffffffu || b->row_stride < b->vocab || b->row_stride % (b->dtype == LCS_BF16 ? 8u : 4u) != 0 || misaligned(b->logits, 16u)) {
        return w.no("logits must be 16-byte aligned with row_stride >= vocab and a multiple of 4 (f32) / 8 (bf16)");
    }
    return LCS_OK;
}

}  // namespace lcs
