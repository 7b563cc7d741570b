// What lcs_add_rmsnorm and lcs_lmhead_ex refuse, before any launch (plain host
// code: the CPU tests compile it by itself). Each returns the status and, where
// it is not LCS_OK, the message.
#pragma once

#include <stdint.h>

#include "locus_sampler.h"

namespace lcs {

inline bool misaligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1u)) != 0u; }

inline int check_add_rmsnorm(const lcs_norm_batch* b, const lcs_norm_out* o, uint32_t max_hidden, const char** why) {
    auto no = [&](const char* m) { *why = m; return (int)LCS_ERR_INVALID_ARG; };
    if (!b || !o) return no("null norm argument");
    if (b->rows == 0) return LCS_OK;
    if (b->x_dtype != LCS_F32 && b->x_dtype != LCS_BF16) return no("x_dtype must be f32 or bf16");
    if (b->y_dtype != LCS_F32 && b->y_dtype != LCS_BF16 && b->y_dtype != LCS_E4M3) return no("y_dtype must be f32, bf16 or e4m3");
    if (b->hidden == 0 || b->hidden > max_hidden) return no("hidden must be 1..32768");
    if (!(b->eps > 0.0f && b->eps <= 3.0e38f)) return no("eps must be positive and finite");
    if (!b->x || !b->weight || !o->y) return no("null x / weight / y");
    if (b->y_dtype == LCS_E4M3 && !o->y_scale) return no("y in e4m3 needs y_scale");
    if (o->sum && !b->residual) return no("sum given without residual");
    const uintptr_t n = b->x_dtype == LCS_F32 ? 4u : 2u, m = b->y_dtype == LCS_F32 ? 4u : b->y_dtype == LCS_BF16 ? 2u : 1u;
    if (misaligned(b->x, n) || misaligned(b->residual, n) || misaligned(b->weight, n) || misaligned(o->sum, n) ||
        misaligned(o->y, m) || misaligned(o->y_scale, 4u)) {
        return no("a pointer is not aligned to its elements");
    }
    if (b->x_stride < b->hidden || (b->residual && b->residual_stride < b->hidden) || o->y_stride < b->hidden ||
        (o->sum && o->sum_stride < b->hidden)) {
        return no("row strides must be at least hidden");
    }
    return LCS_OK;
}

inline int check_lmhead_ex(const lcs_lmhead_ex_batch* b, const lcs_lmhead_out* o, uint32_t max_rows, uint32_t max_vocab,
                           const char** why) {
    auto no = [&](const char* m) { *why = m; return (int)LCS_ERR_INVALID_ARG; };
    auto over = [&](const char* m) { *why = m; return (int)LCS_ERR_CAPACITY; };
    if (!b || !o) return no("null lm-head argument");
    if (b->rows == 0) return LCS_OK;
    if (b->dtype != LCS_BF16 && b->dtype != LCS_E4M3) return no("dtype must be bf16 or e4m3");
    if (!b->x || !b->w || !o->argmax_ids) return no("null x / w / argmax_ids");
    if (misaligned(b->x, 16u) || misaligned(b->w, 16u)) return no("x and w must be 16-byte aligned");
    if (b->hidden == 0 || b->hidden % 64 != 0 || b->hidden > 65536) return no("hidden must be a multiple of 64 up to 65536");
    if (b->vocab == 0) return no("vocab must be positive");
    if (o->logits && o->ld_logits < b->vocab) return no("ld_logits < vocab");
    if (b->rows_per_seq > 64 || (b->rows_per_seq && b->rows % b->rows_per_seq)) {
        return no("rows_per_seq must be 0 or 1..64 and divide rows");
    }
    if (b->draft && !o->draft_lp) return no("draft given without draft_lp");
    if (o->accept_len && (!b->draft || !b->rows_per_seq)) return no("accept_len needs draft and rows_per_seq");
    if (b->dtype == LCS_BF16 && (b->x_scale || b->w_scale)) return no("scales go with e4m3 operands");
    if (misaligned(b->x_scale, 4u) || misaligned(b->w_scale, 4u)) return no("a pointer is not aligned to its elements");
    if (b->rows > max_rows || b->vocab > max_vocab) return over("rows or vocab above the context limits");
    if (const lcs_adapters* d = b->adapters) {
        if (d->n == 0 || d->n > 1024) return no("adapters: 1 to 1024");
        if (d->wide == 0 || d->wide % 8 != 0 || d->wide > 256) return no("adapters: wide must be a multiple of 8 up to 256");
        if (!d->a || !d->b || !b->slot) return no("adapters: null a / b / slot");
        if (misaligned(d->a, 16u) || misaligned(d->b, 16u)) return no("adapters: a and b must be 16-byte aligned");
        if (misaligned(d->rank, 4u) || misaligned(d->scale, 4u) || misaligned(b->slot, 4u)) {
            return no("a pointer is not aligned to its elements");
        }
        if ((uint64_t)b->rows * b->hidden * (b->dtype == LCS_BF16 ? 2u : 1u) > 0xffffffffull) {
            return over("adapters: x must be under 4 GiB");
        }
    } else if (b->slot) {
        return no("slot given without adapters");
    }
    return LCS_OK;
}

}  // namespace lcs
