// Argument checks of the sequence operators: plain host C++, no HIP, so that they are tested without a GPU.
#pragma once
#include "../../include/drlvae.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>

struct SeqError {
    int code = DRL_OK;
    char msg[256] = {0};
    int set(int c, const char* fmt, ...) __attribute__((format(printf, 3, 4))) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(msg, sizeof msg, fmt, ap);
        va_end(ap);
        return code = c;
    }
};

// What the checks know of a layout.
struct SeqRows {
    int64_t q_end = 0, k_end = 0;      // rows of q / k that belong to no series behind the last one are not touched
    int n_seg = 0;
};

// Rows are counted in 32 bits, and a tile or two past the last one.
constexpr int64_t SEQ_MAX_ROWS = 0x7fff0000LL;

inline int seq_check_layout(SeqError& e, const int64_t* qo, const int64_t* ko, int n_seg) {
    if (n_seg < 0 || n_seg > (1 << 24)) return e.set(DRL_ERR_ARG, "drl_seq_layout_create: n_seg %d (0 .. 2^24)", n_seg);
    if (!qo) return e.set(DRL_ERR_ARG, "drl_seq_layout_create: q_offsets is NULL");
    for (int side = 0; side < (ko ? 2 : 1); ++side) {
        const int64_t* o = side ? ko : qo;
        if (o[0] < 0) return e.set(DRL_ERR_ARG, "drl_seq_layout_create: negative offset");
        for (int i = 0; i < n_seg; ++i)
            if (o[i + 1] < o[i]) return e.set(DRL_ERR_ARG, "drl_seq_layout_create: %s_offsets decrease at series %d", side ? "k" : "q", i);
        if (o[n_seg] > SEQ_MAX_ROWS) return e.set(DRL_ERR_UNSUPPORTED, "drl_seq_layout_create: more than 2^31 - 2^16 rows");
    }
    return DRL_OK;
}

inline int seq_check_call(SeqError& e, const char* who, const drl_seq_call* c) {
    if (!c) return e.set(DRL_ERR_ARG, "%s: call is NULL", who);
    if (c->struct_size != (int)sizeof(drl_seq_call) || c->abi_revision != DRL_ABI_REVISION)
        return e.set(DRL_ERR_ARG, "%s: drl_seq_call of another header (size %d, revision %d)", who, c->struct_size, c->abi_revision);
    if (c->dtype < DRL_F32 || c->dtype > DRL_BF16) return e.set(DRL_ERR_ARG, "%s: dtype %d", who, c->dtype);
    if (c->on_stream != 0 && c->on_stream != 1) return e.set(DRL_ERR_ARG, "%s: on_stream %d", who, c->on_stream);
    if (c->workspace_bytes < 0 || ((uintptr_t)c->workspace & 15)) return e.set(DRL_ERR_ARG, "%s: workspace not 16-byte aligned", who);
    return DRL_OK;
}

inline int seq_check_workspace(SeqError& e, const char* who, const drl_seq_call* c, int64_t need) {
    if (need > 0 && (!c->workspace || c->workspace_bytes < need))
        return e.set(DRL_ERR_ARG, "%s: workspace of %lld bytes needed, %lld given", who, (long long)need,
                     c->workspace ? (long long)c->workspace_bytes : 0LL);
    return DRL_OK;
}

// A launch counts its threads along x in 32 bits.
inline bool seq_grid_fits(int64_t workgroups, int threads) { return workgroups <= (((int64_t)1 << 32) - 1) / threads; }
inline int seq_check_grid(SeqError& e, const char* who, int64_t workgroups, int threads) {
    if (!seq_grid_fits(workgroups, threads))
        return e.set(DRL_ERR_UNSUPPORTED, "%s: %lld workgroups of %d threads: too many series, rows or heads for one call", who, (long long)workgroups, threads);
    return DRL_OK;
}

inline bool seq_aligned(int dtype, const void* p, int64_t row, int64_t head) {
    const int64_t unit = dtype == DRL_F32 ? 4 : 8;
    const int64_t most = (int64_t)1 << 40;
    return !((uintptr_t)p & 15) && row >= 0 && head >= 0 && row <= most && head <= most && row % unit == 0 && head % unit == 0;
}

// The kernels count the rows of a tile in 32 bits.
constexpr int64_t SEQ_MAX_ROW = (int64_t)1 << 24;

// Rows and heads of an output may lie either way round, but not on each other.
inline bool seq_apart(int64_t rows, int64_t row, int heads, int64_t head, int width) {
    const bool row_major = head >= width && row >= (heads - 1) * head + width;
    const bool head_major = row >= width && head >= (rows - 1) * row + width;
    return (heads == 1 && (row >= width || rows <= 1)) || (rows <= 1 && head >= width) || row_major || head_major;
}

inline int seq_check_heads(SeqError& e, const char* who, int h, int g) {
    if (h < 1 || g < 1 || h > 65535 || h % g) return e.set(DRL_ERR_ARG, "%s: %d heads over %d kv heads", who, h, g);
    return DRL_OK;
}

inline int seq_check_attention(SeqError& e, const SeqRows* l, const drl_seq_call* c, const drl_attn_args* a) {
    const char* who = "drl_attention_dev";
    if (seq_check_call(e, who, c)) return e.code;
    if (!l || !a) return e.set(DRL_ERR_ARG, "%s: layout or args is NULL", who);
    if (seq_check_heads(e, who, a->n_heads, a->n_kv_heads)) return e.code;
    if (a->dim < 8 || a->dim > 128 || a->dim % 8) return e.set(DRL_ERR_UNSUPPORTED, "%s: dim %d (8 .. 128, a multiple of 8)", who, a->dim);
    if (!(a->scale > 0) || !std::isfinite(a->scale)) return e.set(DRL_ERR_ARG, "%s: scale %g (finite and > 0)", who, (double)a->scale);
    if (a->window < 0) return e.set(DRL_ERR_ARG, "%s: window %d", who, a->window);
    if (l->q_end > 0 && (!a->q || !a->out)) return e.set(DRL_ERR_ARG, "%s: q or out is NULL", who);
    if (l->k_end > 0 && (!a->k || !a->v)) return e.set(DRL_ERR_ARG, "%s: k or v is NULL", who);
    if (!seq_aligned(c->dtype, a->q, a->q_row, a->q_head) || !seq_aligned(c->dtype, a->k, a->k_row, a->k_head) ||
        !seq_aligned(c->dtype, a->v, a->v_row, a->v_head) || !seq_aligned(c->dtype, a->out, a->o_row, a->o_head))
        return e.set(DRL_ERR_ARG, "%s: a pointer or stride is negative or not a multiple of 16 bytes", who);
    if (a->k_row > SEQ_MAX_ROW || a->v_row > SEQ_MAX_ROW) return e.set(DRL_ERR_UNSUPPORTED, "%s: a row stride of k or v above 2^24", who);
    if (((uintptr_t)a->lse & 3) || ((uintptr_t)a->k_len & 3)) return e.set(DRL_ERR_ARG, "%s: lse or k_len not 4-byte aligned", who);
    if (!seq_apart(l->q_end, a->o_row, a->n_heads, a->o_head, a->dim)) return e.set(DRL_ERR_ARG, "%s: rows or heads of out overlap", who);
    return DRL_OK;
}

inline int seq_check_linear(SeqError& e, const char* who, int64_t rows, const drl_seq_call* c, const drl_linear_args* a, bool step) {
    if (seq_check_call(e, who, c)) return e.code;
    if (!a) return e.set(DRL_ERR_ARG, "%s: args is NULL", who);
    if (rows < 0 || rows > SEQ_MAX_ROWS) return e.set(DRL_ERR_ARG, "%s: %lld rows", who, (long long)rows);
    if (seq_check_heads(e, who, a->n_heads, a->n_kv_heads)) return e.code;
    if (a->dim_k < 8 || a->dim_k > 128 || a->dim_k % 8) return e.set(DRL_ERR_UNSUPPORTED, "%s: dim_k %d (8 .. 128, a multiple of 8)", who, a->dim_k);
    if (a->dim_v < 8 || a->dim_v > 256 || a->dim_v % 8) return e.set(DRL_ERR_UNSUPPORTED, "%s: dim_v %d (8 .. 256, a multiple of 8)", who, a->dim_v);
    if (!std::isfinite(a->scale)) return e.set(DRL_ERR_ARG, "%s: scale is not finite", who);
    if (a->reserved) return e.set(DRL_ERR_ARG, "%s: reserved is not 0", who);
    if (!a->log_decay) return e.set(DRL_ERR_ARG, "%s: log_decay is NULL", who);
    if (rows > 0 && (!a->q || !a->k || !a->v || !a->out)) return e.set(DRL_ERR_ARG, "%s: q, k, v or out is NULL", who);
    if (step && rows > 0 && (!a->state_in || !a->state_out)) return e.set(DRL_ERR_ARG, "%s: a step needs state_in and state_out", who);
    if (!seq_aligned(c->dtype, a->q, a->q_row, a->q_head) || !seq_aligned(c->dtype, a->k, a->k_row, a->k_head) ||
        !seq_aligned(c->dtype, a->v, a->v_row, a->v_head) || !seq_aligned(c->dtype, a->out, a->o_row, a->o_head) ||
        ((uintptr_t)a->state_in & 15) || ((uintptr_t)a->state_out & 15) || ((uintptr_t)a->log_decay & 3))
        return e.set(DRL_ERR_ARG, "%s: a pointer or stride is negative or not a multiple of 16 bytes", who);
    if (a->q_row > SEQ_MAX_ROW || a->k_row > SEQ_MAX_ROW || a->v_row > SEQ_MAX_ROW)
        return e.set(DRL_ERR_UNSUPPORTED, "%s: a row stride above 2^24", who);
    if (!seq_apart(rows, a->o_row, a->n_heads, a->o_head, a->dim_v)) return e.set(DRL_ERR_ARG, "%s: rows or heads of out overlap", who);
    return DRL_OK;
}

inline int seq_check_norm(SeqError& e, int64_t rows, const drl_seq_call* c, const drl_norm_args* a) {
    const char* who = "drl_group_norm_dev";
    if (seq_check_call(e, who, c)) return e.code;
    if (!a) return e.set(DRL_ERR_ARG, "%s: args is NULL", who);
    if (rows < 0 || rows > SEQ_MAX_ROWS) return e.set(DRL_ERR_ARG, "%s: %lld rows", who, (long long)rows);
    if (a->channels < 1 || a->channels > 65536) return e.set(DRL_ERR_UNSUPPORTED, "%s: %d channels (1 .. 65536)", who, a->channels);
    if (a->groups < 1 || a->channels % a->groups) return e.set(DRL_ERR_ARG, "%s: %d channels in %d groups", who, a->channels, a->groups);
    if (a->act < DRL_ACT_LINEAR || a->act > DRL_ACT_SILU) return e.set(DRL_ERR_ARG, "%s: activation %d", who, a->act);
    if (!(a->eps > 0) || !std::isfinite(a->eps)) return e.set(DRL_ERR_ARG, "%s: eps %g (finite and > 0)", who, (double)a->eps);
    if (rows > 0 && (!a->x || !a->y)) return e.set(DRL_ERR_ARG, "%s: x or y is NULL", who);
    if (a->x_row < a->channels || a->y_row < a->channels) return e.set(DRL_ERR_ARG, "%s: a row stride is less than the channels", who);
    if (a->x == a->y && a->x_row != a->y_row) return e.set(DRL_ERR_ARG, "%s: y is x with another row stride", who);
    const uintptr_t mask = c->dtype == DRL_F32 ? 3 : 1;
    if (((uintptr_t)a->x & mask) || ((uintptr_t)a->y & mask) || ((uintptr_t)a->gamma & 3) || ((uintptr_t)a->beta & 3))
        return e.set(DRL_ERR_ARG, "%s: a pointer is not aligned to its type", who);
    return DRL_OK;
}
