// Host side of the sequence operators (include/drlvae.h): layouts, argument checks, launches.
#include "ctx_internal.h"
#include "seq_check.h"
#include "seq_attn.hip.h"
#include "seq_linear.hip.h"
#include "seq_norm.hip.h"

#include <algorithm>
#include <new>
#include <numeric>
#include <vector>

struct drl_seq_layout {
    int device = 0;
    SeqRows rows;
    int64_t n_q = 0, n_k = 0;         // rows that belong to a series
    int max_q = 0, max_k = 0;
    seq::SegInfo* segs = nullptr;     // device, n_seg + 1 entries
};

namespace {

using seq::bf16;
using seq::f16;

// The context's GPU is current inside a call; the caller's is again behind it.
struct DeviceGuard {
    int was = -1;
    bool ok = true;
    explicit DeviceGuard(int device) {
        if (hipGetDevice(&was) != hipSuccess) { was = -1; ok = hipSetDevice(device) == hipSuccess; return; }
        if (was == device) was = -1;
        else ok = hipSetDevice(device) == hipSuccess;
    }
    ~DeviceGuard() { if (was >= 0) (void)hipSetDevice(was); }
};

int fail(drl_ctx* c, const SeqError& e) { return drl_ctx_fail(c, e.code, e.msg); }

int hip_fail(drl_ctx* c, const char* who, hipError_t err) {
    SeqError e;
    e.set(DRL_ERR_HIP, "%s: %s", who, hipGetErrorString(err));
    return fail(c, e);
}

hipStream_t stream_of(const DrlCtxView& v, const drl_seq_call* call) {
    return (hipStream_t)(call->on_stream ? call->stream : v.stream);
}

// Runs f with a null pointer of the element type.
template <typename F>
void by_type(int dtype, F f) {
    if (dtype == DRL_F32) f((float*)nullptr);
    else if (dtype == DRL_F16) f((f16*)nullptr);
    else f((bf16*)nullptr);
}

int launched(drl_ctx* c, const char* who) {
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? DRL_OK : hip_fail(c, who, err);
}

int check_layout(SeqError& e, const char* who, const DrlCtxView& v, const drl_seq_layout* l) {
    if (!l) return e.set(DRL_ERR_ARG, "%s: layout is NULL", who);
    if (l->device != v.device) return e.set(DRL_ERR_ARG, "%s: the layout is GPU %d's, the context GPU %d's", who, l->device, v.device);
    return DRL_OK;
}

}  // namespace

extern "C" {

int drl_seq_layout_create(drl_ctx* c, const int64_t* qo, const int64_t* ko, int n_seg, drl_seq_layout** out) {
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (!out) { e.set(DRL_ERR_ARG, "drl_seq_layout_create: out is NULL"); return fail(c, e); }
    *out = nullptr;
    if (seq_check_layout(e, qo, ko, n_seg)) return fail(c, e);
    if (!ko) ko = qo;
    const DrlCtxView v = drl_ctx_view(c);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, "drl_seq_layout_create", hipErrorInvalidDevice);
    drl_seq_layout* l = new (std::nothrow) drl_seq_layout();
    if (!l) return drl_ctx_fail(c, DRL_ERR_STATE, "drl_seq_layout_create: out of host memory");
    try {
        l->device = v.device;
        l->rows.n_seg = n_seg;
        l->rows.q_end = qo[n_seg];
        l->rows.k_end = ko[n_seg];
        l->n_q = qo[n_seg] - qo[0];
        l->n_k = ko[n_seg] - ko[0];
        std::vector<int> order(n_seg);
        std::iota(order.begin(), order.end(), 0);
        std::stable_sort(order.begin(), order.end(), [&](int a, int b) {
            const int64_t qa = qo[a + 1] - qo[a], qb = qo[b + 1] - qo[b];
            return qa != qb ? qa > qb : ko[a + 1] - ko[a] > ko[b + 1] - ko[b];
        });
        std::vector<seq::SegInfo> segs((size_t)n_seg + 1);
        int64_t cum = 0;
        for (int i = 0; i < n_seg; ++i) {
            const int s = order[i];
            segs[i] = {qo[s], ko[s], cum, (int32_t)(qo[s + 1] - qo[s]), (int32_t)(ko[s + 1] - ko[s]), s, 0};
            cum += segs[i].nq;
            l->max_q = std::max(l->max_q, segs[i].nq);
            l->max_k = std::max(l->max_k, segs[i].nk);
        }
        segs[n_seg] = {qo[n_seg], ko[n_seg], cum, 0, 0, n_seg, 0};
        const size_t bytes = segs.size() * sizeof(segs[0]);
        drl_count_alloc();
        hipError_t err = hipMalloc((void**)&l->segs, bytes);
        if (err == hipSuccess) err = hipMemcpy(l->segs, segs.data(), bytes, hipMemcpyHostToDevice);
        if (err != hipSuccess) {
            if (l->segs) (void)hipFree(l->segs);
            delete l;
            return hip_fail(c, "drl_seq_layout_create", err);
        }
    } catch (const std::bad_alloc&) {
        delete l;
        return drl_ctx_fail(c, DRL_ERR_STATE, "drl_seq_layout_create: out of host memory");
    }
    *out = l;
    return DRL_OK;
}

void drl_seq_layout_destroy(drl_seq_layout* l) {
    if (!l) return;
    DeviceGuard guard(l->device);
    if (l->segs) (void)hipFree(l->segs);
    delete l;
}

// ---- attention ----------------------------------------------------------------------------------------------------

static int attn_prepare(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a, SeqError& e) {
    const DrlCtxView v = drl_ctx_view(c);
    if (check_layout(e, "drl_attention_dev", v, l)) return e.code;
    return seq_check_attention(e, &l->rows, call, a);
}

int drl_attention_workspace(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a, int64_t* bytes) {
    if (!c || !bytes) return DRL_ERR_ARG;
    SeqError e;
    if (attn_prepare(c, l, call, a, e)) return fail(c, e);
    *bytes = 0;
    return DRL_OK;
}

int drl_attention_dev(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a) {
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (attn_prepare(c, l, call, a, e)) return fail(c, e);
    if (l->n_q == 0) return DRL_OK;
    const DrlCtxView v = drl_ctx_view(c);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, "drl_attention_dev", hipErrorInvalidDevice);
    seq::AttnArgs k = {};
    k.q = a->q; k.k = a->k; k.v = a->v; k.out = a->out; k.lse = a->lse; k.key_mask = a->key_mask; k.k_len = a->k_len;
    k.q_row = a->q_row; k.q_head = a->q_head; k.k_row = a->k_row; k.k_head = a->k_head;
    k.v_row = a->v_row; k.v_head = a->v_head; k.o_row = a->o_row; k.o_head = a->o_head;
    k.segs = l->segs; k.n_seg = l->rows.n_seg; k.heads = a->n_heads; k.rep = a->n_heads / a->n_kv_heads; k.dim = a->dim;
    k.causal = a->causal != 0; k.window = a->window; k.scale = a->scale;
    k.splits = 1;
    const hipStream_t st = stream_of(v, call);
    by_type(call->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        if constexpr (sizeof(T) == 2) {
            constexpr int BM = 128;
            k.blocks = (k.rep + BM - 1) / BM;
            k.rep_b = (k.rep + k.blocks - 1) / k.blocks;
            k.kv_blocks = a->n_kv_heads * k.blocks;
            k.per = BM / k.rep_b;
            const int64_t tiles = (l->n_q / k.per + l->rows.n_seg) * k.kv_blocks;
            const int dt = (a->dim + 31) / 32;
            const size_t shmem = 4 * 64 * 2 * (dt == 1 ? 32 : dt == 2 ? 64 : 128);
            const dim3 grid((unsigned)tiles);
            if (dt == 1) hipLaunchKernelGGL((seq::attn_tile_kernel<T, 1>), grid, dim3(256), shmem, st, k);
            else if (dt == 2) hipLaunchKernelGGL((seq::attn_tile_kernel<T, 2>), grid, dim3(256), shmem, st, k);
            else if (dt == 3) hipLaunchKernelGGL((seq::attn_tile_kernel<T, 3>), grid, dim3(256), shmem, st, k);
            else hipLaunchKernelGGL((seq::attn_tile_kernel<T, 4>), grid, dim3(256), shmem, st, k);
        } else {
            const dim3 grid((unsigned)(l->n_q / 4 + l->rows.n_seg), a->n_heads);
            hipLaunchKernelGGL((seq::attn_rows_kernel<T>), grid, dim3(256), 0, st, k);
        }
    });
    return launched(c, "drl_attention_dev");
}

// ---- linear attention ---------------------------------------------------------------------------------------------

int drl_linear_attention_workspace(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_linear_args* a, int64_t* bytes) {
    if (!c || !bytes) return DRL_ERR_ARG;
    SeqError e;
    if (check_layout(e, "drl_linear_attention_dev", drl_ctx_view(c), l) ||
        seq_check_linear(e, "drl_linear_attention_dev", l->rows.q_end, call, a, false)) return fail(c, e);
    *bytes = 0;
    return DRL_OK;
}

static seq::LinearArgs linear_args(const drl_linear_args* a, const seq::SegInfo* segs, int n_seg) {
    return {a->q, a->k, a->v, a->out, a->log_decay, a->state_in, a->state_out, a->q_row, a->q_head, a->k_row, a->k_head,
            a->v_row, a->v_head, a->o_row, a->o_head, segs, n_seg, a->n_heads, a->n_heads / a->n_kv_heads, a->dim_k, a->dim_v, a->scale};
}

int drl_linear_attention_dev(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_linear_args* a) {
    const char* who = "drl_linear_attention_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    const DrlCtxView v = drl_ctx_view(c);
    if (check_layout(e, who, v, l) || seq_check_linear(e, who, l->rows.q_end, call, a, false)) return fail(c, e);
    if (l->rows.n_seg == 0) return DRL_OK;
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    const seq::LinearArgs k = linear_args(a, l->segs, l->rows.n_seg);
    by_type(call->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        const dim3 grid(l->rows.n_seg, a->n_heads, (a->dim_v + 63) / 64);
        hipLaunchKernelGGL((seq::linear_rows_kernel<T>), grid, dim3(256), 0, stream_of(v, call), k);
    });
    return launched(c, who);
}

int drl_linear_attention_step_dev(drl_ctx* c, int64_t n, const drl_seq_call* call, const drl_linear_args* a) {
    const char* who = "drl_linear_attention_step_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (seq_check_linear(e, who, n, call, a, true)) return fail(c, e);
    if (n == 0) return DRL_OK;
    const DrlCtxView v = drl_ctx_view(c);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    const seq::LinearArgs k = linear_args(a, nullptr, 0);
    by_type(call->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        const dim3 grid((unsigned)n, a->n_heads, (a->dim_v + 63) / 64);
        hipLaunchKernelGGL((seq::linear_rows_kernel<T>), grid, dim3(256), 0, stream_of(v, call), k);
    });
    return launched(c, who);
}

// ---- group norm ---------------------------------------------------------------------------------------------------

static int norm_prepare(drl_ctx* c, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a, SeqError& e) {
    if (l && check_layout(e, "drl_group_norm_dev", drl_ctx_view(c), l)) return e.code;
    return seq_check_norm(e, l ? l->rows.q_end : rows, call, a);
}

int drl_group_norm_workspace(drl_ctx* c, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a, int64_t* bytes) {
    if (!c || !bytes) return DRL_ERR_ARG;
    SeqError e;
    if (norm_prepare(c, l, rows, call, a, e)) return fail(c, e);
    *bytes = 0;
    return DRL_OK;
}

int drl_group_norm_dev(drl_ctx* c, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a) {
    const char* who = "drl_group_norm_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (norm_prepare(c, l, rows, call, a, e)) return fail(c, e);
    if ((l ? l->n_q : rows) == 0) return DRL_OK;
    const DrlCtxView v = drl_ctx_view(c);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    const seq::NormArgs k = {a->x, a->y, a->gamma, a->beta, a->x_row, a->y_row, l ? l->segs : nullptr, a->channels, a->groups, a->act, a->eps};
    by_type(call->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        const dim3 grid((unsigned)(l ? l->rows.n_seg : rows), a->groups);
        hipLaunchKernelGGL((seq::norm_group_kernel<T>), grid, dim3(256), 0, stream_of(v, call), k);
    });
    return launched(c, who);
}

}  // extern "C"
