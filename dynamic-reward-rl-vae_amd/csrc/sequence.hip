// Host side of the sequence operators (include/drlvae.h): layouts, argument checks, launches.
#include "ctx_internal.h"
#include "seq_check.h"
#include "seq_attn.hip.h"
#include "seq_linear.hip.h"
#include "seq_norm.hip.h"

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <new>
#include <numeric>
#include <vector>

struct drl_seq_layout {
    int device = 0;
    SeqRows rows;
    int64_t n_q = 0, n_k = 0;         // rows that belong to a series
    int64_t q_first = 0;
    int max_q = 0, max_k = 0;
    seq::SegInfo* segs = nullptr;     // device, n_seg + 1 entries
    size_t bytes = 0;
};

namespace {

using seq::bf16;
using seq::f16;

// Device memory of the layouts' tables.  Small ones come out of slabs: a layout is made for every new batch, and asking the
// runtime for memory takes longer than the rest of it.  A table given back may still be read by work under way, on any
// stream: it waits among the retired until the device has been waited for once, which happens when many have gathered.  Slabs are kept
// until the process ends.
class TablePool {
    static constexpr size_t SLAB = 256 << 10, LARGEST = 32 << 10, MOST_RETIRED = 64;
    std::mutex mu;
    std::vector<void*> free_[16], retired[16];       // by size: 256 bytes << k
    char* slab = nullptr;
    size_t left = 0, n_retired = 0;
    static int size_class(size_t bytes) {
        int k = 0;
        while (((size_t)256 << k) < bytes) ++k;
        return k;
    }

public:
    hipError_t get(size_t bytes, void** p) {
        if (bytes > LARGEST) {
            drl_count_alloc();
            return hipMalloc(p, bytes);
        }
        std::lock_guard<std::mutex> lk(mu);
        const int k = size_class(bytes);
        if (free_[k].empty() && n_retired >= MOST_RETIRED && hipDeviceSynchronize() == hipSuccess) {
            for (int i = 0; i < 16; ++i) {
                free_[i].insert(free_[i].end(), retired[i].begin(), retired[i].end());
                retired[i].clear();
            }
            n_retired = 0;
        }
        if (!free_[k].empty()) {
            *p = free_[k].back();
            free_[k].pop_back();
            return hipSuccess;
        }
        const size_t size = (size_t)256 << k;
        if (left < size) {
            void* fresh = nullptr;
            drl_count_alloc();
            const hipError_t err = hipMalloc(&fresh, SLAB);
            if (err != hipSuccess) return err;
            slab = (char*)fresh;
            left = SLAB;
        }
        *p = slab;
        slab += size;
        left -= size;
        return hipSuccess;
    }
    void put(void* p, size_t bytes) noexcept {
        if (bytes > LARGEST) {
            (void)hipFree(p);
            return;
        }
        std::lock_guard<std::mutex> lk(mu);
        try {
            retired[size_class(bytes)].push_back(p);
            ++n_retired;
        } catch (const std::bad_alloc&) {}               // the table is lost, not more
    }
};
TablePool& table_pool(int device) {
    static std::mutex mu;
    static auto* pools = new std::map<int, TablePool>();       // never destroyed: layouts may be, after everything else
    std::lock_guard<std::mutex> lk(mu);
    return (*pools)[device];
}

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
    (void)hipGetLastError();               // reported here: not left for the caller's next question as well
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

// How the launches of this thread's call went.  The runtime's own last error is no measure: it may be someone else's, and asking
// for it takes it from them.
thread_local hipError_t launch_error = hipSuccess;
void keep_error(hipError_t err) {
    if (launch_error == hipSuccess) launch_error = err;
}

// A kernel is a handle here, not a function that host code may call: launched through the runtime, not through the pointer.
template <typename A>
void launch(void (*kernel)(A), dim3 grid, dim3 block, size_t shmem, hipStream_t st, A args) {
    void* p[] = {&args};
    keep_error(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, p, shmem, st));
}
// More LDS than a kernel gets unasked.
template <typename A>
void allow_lds(void (*kernel)(A), size_t shmem) {
    if (shmem > 64 * 1024) keep_error(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)shmem));
}

int launched(drl_ctx* c, const char* who) {
    const hipError_t err = launch_error;
    launch_error = hipSuccess;
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
        l->q_first = qo[0];
        l->n_q = qo[n_seg] - qo[0];
        l->n_k = ko[n_seg] - ko[0];
        std::vector<int> order(n_seg);
        std::iota(order.begin(), order.end(), 0);
        std::stable_sort(order.begin(), order.end(), [&](int a, int b) {
            const int64_t qa = qo[a + 1] - qo[a], qb = qo[b + 1] - qo[b];
            return qa != qb ? qa > qb : ko[a + 1] - ko[a] > ko[b + 1] - ko[b];
        });
        std::vector<seq::SegInfo> segs((size_t)n_seg + 1);
        uint32_t cum = 0;
        for (int i = 0; i < n_seg; ++i) {
            const int s = order[i];
            segs[i] = {qo[s], ko[s], cum, (int32_t)(qo[s + 1] - qo[s]), (int32_t)(ko[s + 1] - ko[s]), s};
            cum += segs[i].nq;
            l->max_q = std::max(l->max_q, segs[i].nq);
            l->max_k = std::max(l->max_k, segs[i].nk);
        }
        segs[n_seg] = {qo[n_seg], ko[n_seg], cum, 0, 0, n_seg};
        const size_t bytes = segs.size() * sizeof(segs[0]);
        l->bytes = bytes;
        hipError_t err = table_pool(l->device).get(bytes, (void**)&l->segs);
        if (err == hipSuccess) err = hipMemcpy(l->segs, segs.data(), bytes, hipMemcpyHostToDevice);
        if (err != hipSuccess) {
            if (l->segs) table_pool(l->device).put(l->segs, bytes);
            delete l;
            return hip_fail(c, "drl_seq_layout_create", err);
        }
    } catch (const std::bad_alloc&) {
        if (l->segs) table_pool(l->device).put(l->segs, l->bytes);
        delete l;
        return drl_ctx_fail(c, DRL_ERR_STATE, "drl_seq_layout_create: out of host memory");
    }
    *out = l;
    return DRL_OK;
}

void drl_seq_layout_destroy(drl_seq_layout* l) {
    if (!l) return;
    DeviceGuard guard(l->device);
    if (l->segs) table_pool(l->device).put(l->segs, l->bytes);      // the pool was made when the table came out of it
    delete l;
}

// ---- attention ----------------------------------------------------------------------------------------------------

static int attn_prepare(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a, SeqError& e) {
    const DrlCtxView v = drl_ctx_view(c);
    if (check_layout(e, "drl_attention_dev", v, l)) return e.code;
    return seq_check_attention(e, &l->rows, call, a);
}

// How a call is cut: rows into tiles, and, where these do not fill the GPU, the keys into runs.
struct AttnPlan {
    bool few;
    int blocks, rep_b, per, splits, chunk, turn;
    int64_t tiles, workspace, longest;        // longest: the most keys that one workgroup goes over
};
static AttnPlan attn_plan(const DrlCtxView& v, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a) {
    AttnPlan p = {};
    const int rep = a->n_heads / a->n_kv_heads, rows = 128;
    p.blocks = (rep + rows - 1) / rows;
    p.rep_b = (rep + p.blocks - 1) / p.blocks;
    p.per = rows / p.rep_b;
    p.few = (int64_t)std::min(l->max_q, p.per) * p.rep_b <= 32;
    p.tiles = (l->n_q / p.per + l->rows.n_seg) * (int64_t)(a->n_kv_heads * p.blocks);
    p.splits = 1;
    // Keys one tile can see, cut into runs where the tiles are fewer than what is resident at once: steps one workgroup per
    // CU (two where their LDS lets them), others two.  More and shorter runs only add the reading of q and the joining (16
    // caches of up to 32,768 rows: 256 us at one run per CU, 275 at two, 265 at eight; one of 30,000: 33, 41, 62; 8,192
    // rows of two heads: 71 us at two, 85 at eight, 169 whole).
    const int64_t most = a->window > 0 && a->causal ? std::min<int64_t>(l->max_k, (int64_t)a->window + p.per) : l->max_k;
    const int64_t room = p.few && (call->dtype == DRL_F32 ? a->dim > 32 : a->dim > 64) ? v.n_cu : 2 * v.n_cu, least = p.few && call->dtype == DRL_F32 ? 128 : 256;
    const int64_t want = p.tiles > 0 ? (room + p.tiles / 2) / p.tiles : 1;
    if (most > 2 * least && want > 1) {
        const int64_t chunk = std::max<int64_t>(least, ((most + want - 1) / want + 63) / 64 * 64);
        p.splits = (int)((most + chunk - 1) / chunk);
        p.chunk = (int)chunk;
    }
    p.longest = p.splits > 1 ? p.chunk : most;
    if (p.splits > 1) p.workspace = (int64_t)p.splits * l->n_q * a->n_heads * (a->dim + 2) * 4;
    // Where all workgroups are resident at once, two per CU, each CU's second is taken from the other end of the order, so
    // that a long tile has a short one beside it (8,192 rows of 8 heads, dim 64: 124 -> 120 us, float32 834 -> 667; two
    // series of 4,096 84 -> 65, four of 2,048 45 -> 38).  Short ones would rather have the longest started first (eight
    // series of 1,024, dim 128: 35 -> 39), and so would what does not fit at once (16 series of 4,096: 646 -> 657).
    const bool pairs = !p.few && p.splits == 1 && p.tiles > v.n_cu && p.tiles <= 2 * v.n_cu + v.n_cu / 4 && most >= 2048;
    p.turn = pairs ? std::max(1, v.n_cu / (a->n_kv_heads * p.blocks)) : 0x7fffffff;
    return p;
}

int drl_attention_workspace(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a, int64_t* bytes) {
    if (!c || !bytes) return DRL_ERR_ARG;
    SeqError e;
    if (attn_prepare(c, l, call, a, e)) return fail(c, e);
    *bytes = attn_plan(drl_ctx_view(c), l, call, a).workspace;
    return DRL_OK;
}

}  // extern "C"

// Runs f with the constant n, 1 .. 4.
template <typename F>
static void by_count(int n, F f) {
    if (n == 1) f(std::integral_constant<int, 1>());
    else if (n == 2) f(std::integral_constant<int, 2>());
    else if (n == 3) f(std::integral_constant<int, 3>());
    else f(std::integral_constant<int, 4>());
}

template <typename T>
static void attn_tiles(const AttnPlan& p, const seq::AttnArgs& k, hipStream_t st) {
    const int dt = (k.dim + 31) / 32;
    const size_t tile = 64 * sizeof(T) * (dt == 1 ? 1 : dt == 2 ? 2 : 4) * 16;    // 32 keys (or values)
    const dim3 grid((unsigned)p.tiles, p.splits);
    auto go = [&](auto kernel, int waves, size_t shmem) {
        allow_lds(kernel, shmem);
        launch(kernel, grid, dim3(waves * 64), shmem, st, k);
    };
    by_count(dt, [&](auto d) {
        constexpr int DT = decltype(d)::value;
        constexpr int NW = sizeof(T) == 4 && DT > 2 ? 2 : 4;
        if (p.few) go(seq::attn_step_kernel<T, DT, NW>, NW, std::max(NW * 4 * tile, (size_t)NW * (DT * 4096 + 256)));
        else if constexpr (sizeof(T) == 4) {
            if (DT <= 2 && p.longest <= 1024) go(seq::attn_tile32_kernel<DT, DT >= 3>, 4, 4 * tile);
            else go(seq::attn_tile32_kernel<DT, true>, 4, 4 * tile);
        }
        else if (k.key_mask) go(seq::attn_tile_kernel<T, DT, true>, 4, 8 * tile);
        else go(seq::attn_tile_kernel<T, DT, false>, 4, 8 * tile);
    });
    if (p.splits > 1) {
        const dim3 jg((unsigned)((k.part_rows * k.heads + 3) / 4));
        launch((seq::attn_join_kernel<T>), jg, dim3(256), 0, st, k);
    }
}

extern "C" {

int drl_attention_dev(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_attn_args* a) {
    const char* who = "drl_attention_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (attn_prepare(c, l, call, a, e)) return fail(c, e);
    if (l->n_q == 0) return DRL_OK;
    const DrlCtxView v = drl_ctx_view(c);
    const AttnPlan p = attn_plan(v, l, call, a);
    if (seq_check_grid(e, who, p.tiles, 256) || (p.splits > 1 && seq_check_grid(e, who, (l->n_q * a->n_heads + 3) / 4, 256))) return fail(c, e);
    if (seq_check_workspace(e, who, call, p.workspace)) return fail(c, e);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    seq::AttnArgs k = {};
    k.q = a->q; k.k = a->k; k.v = a->v; k.out = a->out; k.lse = a->lse; k.key_mask = a->key_mask; k.k_len = a->k_len;
    k.q_row = a->q_row; k.q_head = a->q_head; k.k_row = a->k_row; k.k_head = a->k_head;
    k.v_row = a->v_row; k.v_head = a->v_head; k.o_row = a->o_row; k.o_head = a->o_head;
    k.segs = l->segs; k.n_seg = l->rows.n_seg; k.heads = a->n_heads; k.rep = a->n_heads / a->n_kv_heads; k.dim = a->dim;
    k.causal = a->causal != 0; k.window = a->window; k.scale = a->scale;
    k.kv_blocks = a->n_kv_heads * p.blocks; k.blocks = p.blocks; k.rep_b = p.rep_b; k.per = p.per;
    k.turn = p.turn;
    k.splits = p.splits; k.chunk = p.chunk;
    k.part_rows = l->n_q; k.row0 = l->q_first;
    if (p.splits > 1) {
        k.part_o = (float*)call->workspace;
        k.part_ml = (seq::f32x2*)(k.part_o + (int64_t)p.splits * l->n_q * a->n_heads * a->dim);
    }
    const hipStream_t st = stream_of(v, call);
    by_type(call->dtype, [&](auto* t) { attn_tiles<std::remove_pointer_t<decltype(t)>>(p, k, st); });
    return launched(c, who);
}

// ---- linear attention ---------------------------------------------------------------------------------------------

// How a call is cut: value widths into workgroups, and, where series and heads do not fill the GPU, the rows into pieces.
struct LinearPlan {
    int waves, blocks, piece;
    int64_t units, workspace;
};
static LinearPlan linear_plan(const DrlCtxView& v, const drl_seq_layout* l, const drl_seq_call* call, const drl_linear_args* a) {
    LinearPlan p = {};
    const int tiles = (a->dim_v + 31) / 32;
    p.waves = tiles <= 2 ? 2 : 4;
    p.blocks = (tiles + p.waves - 1) / p.waves;
    p.piece = 0x7fffffff;
    p.units = l->rows.n_seg;
    // Pieces cost a second reading of k and v and the states between them: only where the workgroups are fewer than the CUs
    // (384 of 2,048 rows: 222 us whole, 226 in pieces of 512; 64 of 32,768: 2.9 ms whole, 0.76 in pieces of 4,096).
    // A piece is long enough that two workgroups per CU do it all at once, and that going through its chunks twice takes
    // about as long as going through the pieces' states (1.6 us a chunk, 0.3 a state: pieces of sqrt(3 rows), 8,192 rows
    // of 16 heads in 81 us at 256), in whole chunks, rounded down by up to a quarter of one (375 rows of 4 heads,
    // float32: 18.9 us in pieces of 32, 25.1 of 64; 1,000 rows: 26.4 and 26.3; 4,000 rows of 8 heads: 51 at 96, 43 at 128).
    const int64_t groups = (int64_t)a->n_heads * p.blocks;
    if (groups * l->rows.n_seg < v.n_cu) {
        const int64_t rows = std::max<int64_t>(l->n_q * groups / (2 * v.n_cu), (int64_t)std::sqrt(3.0 * l->max_q));
        const int64_t piece = std::max<int64_t>(32, (rows + 23) / 32 * 32);
        if (piece < l->max_q) {
            // pieces of one length
            const int64_t n = (l->max_q + piece - 1) / piece;
            p.piece = (int)(((l->max_q + n - 1) / n + 31) / 32 * 32);
            p.units = l->n_q / p.piece + l->rows.n_seg;
            p.workspace = p.units * a->n_heads * a->dim_k * a->dim_v * 4;
        }
    }
    return p;
}

int drl_linear_attention_workspace(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_linear_args* a, int64_t* bytes) {
    if (!c || !bytes) return DRL_ERR_ARG;
    SeqError e;
    if (check_layout(e, "drl_linear_attention_dev", drl_ctx_view(c), l) ||
        seq_check_linear(e, "drl_linear_attention_dev", l->rows.q_end, call, a, false)) return fail(c, e);
    *bytes = linear_plan(drl_ctx_view(c), l, call, a).workspace;
    return DRL_OK;
}

static seq::LinearArgs linear_args(const drl_linear_args* a, const seq::SegInfo* segs, int n_seg) {
    seq::LinearArgs k = {};
    k.q = a->q; k.k = a->k; k.v = a->v; k.out = a->out; k.log_decay = a->log_decay; k.state_in = a->state_in; k.state_out = a->state_out;
    k.q_row = a->q_row; k.q_head = a->q_head; k.k_row = a->k_row; k.k_head = a->k_head;
    k.v_row = a->v_row; k.v_head = a->v_head; k.o_row = a->o_row; k.o_head = a->o_head;
    k.segs = segs; k.n_seg = n_seg; k.heads = a->n_heads; k.rep = a->n_heads / a->n_kv_heads; k.dk = a->dim_k; k.dv = a->dim_v;
    k.scale = a->scale;
    return k;
}

}  // extern "C"

template <typename T, int KT, int NW, bool STATE>
static void linear_chunks(const LinearPlan& p, const seq::LinearArgs& k, hipStream_t st) {
    constexpr int DP = KT <= 1 ? 32 : KT <= 2 ? 64 : 128;
    constexpr int stage = 32 * sizeof(T) * ((STATE ? 1 : 2) * DP + 32 * NW), stages = sizeof(T) == 2 ? 3 : 2, table = sizeof(T) == 4 ? 0 : STATE ? 256 : 640 + 4096;
    const dim3 grid((unsigned)(p.units * k.heads * p.blocks));
    auto go = [&](auto kernel) {
        allow_lds(kernel, stages * stage + table);
        launch(kernel, grid, dim3(NW * 64), stages * stage + table, st, k);
    };
    if constexpr (sizeof(T) == 2) go(seq::linear_chunk_kernel<T, KT, NW, STATE>);
    else go(seq::linear_chunk32_kernel<KT, NW, STATE>);
}

template <typename T>
static void linear_series(const LinearPlan& p, const seq::LinearArgs& k, hipStream_t st) {
    auto all = [&](auto state) {
        constexpr bool STATE = decltype(state)::value;
        auto by_waves = [&](auto kt) {
            constexpr int KT = decltype(kt)::value;
            if (p.waves == 2) linear_chunks<T, KT, 2, STATE>(p, k, st);
            else linear_chunks<T, KT, 4, STATE>(p, k, st);
        };
        if (k.dk <= 32) by_waves(std::integral_constant<int, 1>());
        else if (k.dk <= 64) by_waves(std::integral_constant<int, 2>());
        else by_waves(std::integral_constant<int, 4>());
    };
    if (k.states) {
        all(std::true_type());
        const dim3 grid(k.n_seg, k.heads, (k.dk * k.dv / 4 + 255) / 256);
        launch(seq::linear_scan_kernel, grid, dim3(256), 0, st, k);
    }
    all(std::false_type());
}

extern "C" {

int drl_linear_attention_dev(drl_ctx* c, const drl_seq_layout* l, const drl_seq_call* call, const drl_linear_args* a) {
    const char* who = "drl_linear_attention_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    const DrlCtxView v = drl_ctx_view(c);
    if (check_layout(e, who, v, l) || seq_check_linear(e, who, l->rows.q_end, call, a, false)) return fail(c, e);
    if (l->rows.n_seg == 0) return DRL_OK;
    const LinearPlan p = linear_plan(v, l, call, a);
    if (seq_check_grid(e, who, p.units * a->n_heads * p.blocks, p.waves * 64)) return fail(c, e);
    if (seq_check_workspace(e, who, call, p.workspace)) return fail(c, e);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    seq::LinearArgs k = linear_args(a, l->segs, l->rows.n_seg);
    k.piece = p.piece;
    k.blocks = p.blocks;
    if (p.workspace) k.states = (float*)call->workspace;
    const hipStream_t st = stream_of(v, call);
    by_type(call->dtype, [&](auto* t) { linear_series<std::remove_pointer_t<decltype(t)>>(p, k, st); });
    return launched(c, who);
}

int drl_linear_attention_step_dev(drl_ctx* c, int64_t n, const drl_seq_call* call, const drl_linear_args* a) {
    const char* who = "drl_linear_attention_step_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (seq_check_linear(e, who, n, call, a, true)) return fail(c, e);
    if (n == 0) return DRL_OK;
    if (seq_check_grid(e, who, n * a->n_heads, 256)) return fail(c, e);
    const DrlCtxView v = drl_ctx_view(c);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    const seq::LinearArgs k = linear_args(a, nullptr, 0);
    by_type(call->dtype, [&](auto* t) {
        typedef std::remove_pointer_t<decltype(t)> T;
        launch((seq::linear_step_kernel<T>), dim3((unsigned)(n * a->n_heads)), dim3(256), 0, stream_of(v, call), k);
    });
    return launched(c, who);
}

// ---- group norm ---------------------------------------------------------------------------------------------------

static int norm_prepare(drl_ctx* c, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a, SeqError& e) {
    if (l && check_layout(e, "drl_group_norm_dev", drl_ctx_view(c), l)) return e.code;
    return seq_check_norm(e, l ? l->rows.q_end : rows, call, a);
}

// How a call is cut: packs of channels, and rows into units.
struct NormPlan {
    int pack, lanes, count, slice, slices, piece, share, threads;      // share > 0: packs per thread of a short series
    int64_t units, blocks, workspace;
};
static NormPlan norm_plan(const DrlCtxView& v, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a) {
    NormPlan p = {};
    const int size = call->dtype == DRL_F32 ? 4 : 2, cg = a->channels / a->groups;
    // the widest pack that a group is made of and that everything is aligned to
    for (p.pack = 16 / size; p.pack > 1; p.pack /= 2) {
        const int64_t bytes = p.pack * size;
        if (cg % p.pack == 0 && (uintptr_t)a->x % bytes == 0 && (uintptr_t)a->y % bytes == 0 && a->x_row % p.pack == 0 && a->y_row % p.pack == 0) break;
    }
    const int packs = cg / p.pack;
    p.lanes = 1;
    if (!l) {
        // two packs per lane hide more latency than one and still leave a group's lanes side by side in memory
        while (p.lanes < 64 && p.lanes * 2 < packs) p.lanes *= 2;
        p.count = (packs + p.lanes - 1) / p.lanes;
        const int per_wave = 64 / p.lanes;
        const int64_t sets = (a->groups + per_wave - 1) / per_wave;
        // waves: a multiple of the sets and of four; eight workgroups per CU, or one row each where that is fewer
        const int64_t want = std::min<int64_t>(rows * sets, (int64_t)8 * 4 * v.n_cu);
        const int64_t unit = sets % 4 == 0 ? sets : sets % 2 == 0 ? sets * 2 : sets * 4;
        p.blocks = std::max<int64_t>(1, (want + unit - 1) / unit) * unit / 4;
        return p;
    }
    // A group of the longest series in the registers of 256 or 1,024 threads, where all is read at about the same time: 67
    // series of 700 rows of 128 channels, float32, 17 us (two launches 23), 128 of 300 rows 9 (16), but 67 of 1,461 rows of
    // 512 channels, bf16, 100 MB, 94 us (78).
    const int64_t most = (int64_t)l->max_q * packs;
    if (most <= 8 * 1024 && l->n_q * a->channels * size <= (int64_t)64 << 20 && seq_grid_fits((int64_t)(l->rows.n_seg + 7) * a->groups, 1024)) {
        p.threads = most <= 512 ? 256 : 1024;
        p.share = std::max<int>(1, (int)((most + p.threads - 1) / p.threads));
        return p;
    }
    p.slice = std::max(1, std::min(a->groups, 256 / std::min(packs, 256)));
    p.slices = (a->groups + p.slice - 1) / p.slice;
    const int share = std::min(packs, 256), rl = 256 / std::min(p.slice * packs, 256);
    while (p.lanes < 64 && p.lanes < share * rl) p.lanes *= 2;
    // four workgroups per CU, of at least 8 rows per thread, at most 256 units to a series (each of which reads the
    // moments of all)
    const int64_t fill = (l->n_q * p.slices + 4 * v.n_cu - 1) / (4 * v.n_cu);
    p.piece = (int)std::max({fill, (int64_t)8 * rl, (int64_t)(l->max_q + 255) / 256});
    p.units = l->n_q / p.piece + l->rows.n_seg;
    if (l->max_q > p.piece) p.workspace = p.units * a->groups * 2 * 4;
    return p;
}

int drl_group_norm_workspace(drl_ctx* c, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a, int64_t* bytes) {
    if (!c || !bytes) return DRL_ERR_ARG;
    SeqError e;
    if (norm_prepare(c, l, rows, call, a, e)) return fail(c, e);
    *bytes = norm_plan(drl_ctx_view(c), l, rows, call, a).workspace;
    return DRL_OK;
}

}  // extern "C"

template <typename T, int V>
static void norm_launch(const NormPlan& p, const seq::NormArgs& k, hipStream_t st) {
    auto go = [&](auto kernel, dim3 grid) { launch(kernel, grid, dim3(256), 0, st, k); };
    if (p.share) {
        auto by = [&](auto r) {
            constexpr int R = decltype(r)::value;
            const dim3 grid((unsigned)((int64_t)((k.n_seg + 7) / 8) * 8 * k.groups));
            auto run = [&](auto kernel) { launch(kernel, grid, dim3(p.threads), 0, st, k); };
            if (p.threads == 1024) run(seq::norm_short_kernel<T, V, R, 1024>);
            else if constexpr (R <= 2) run(seq::norm_short_kernel<T, V, R, 256>);
        };
        if (p.share <= 1) by(std::integral_constant<int, 1>());
        else if (p.share <= 2) by(std::integral_constant<int, 2>());
        else if (p.share <= 4) by(std::integral_constant<int, 4>());
        else if (p.share <= 6) by(std::integral_constant<int, 6>());
        else by(std::integral_constant<int, 8>());
        return;
    }
    if (k.segs) {
        const dim3 grid((unsigned)p.units, p.slices);
        if (k.part) go(seq::norm_series_kernel<T, V, true>, grid);
        go(seq::norm_series_kernel<T, V, false>, grid);
        return;
    }
    const dim3 grid((unsigned)p.blocks);
    if (p.count <= 1) go(seq::norm_rows_kernel<T, V, 1>, grid);
    else if (p.count <= 2) go(seq::norm_rows_kernel<T, V, 2>, grid);
    else if (p.count <= 4) go(seq::norm_rows_kernel<T, V, 4>, grid);
    else go(seq::norm_rows_kernel<T, V, 0>, grid);
}

template <typename T>
static void norm_packs(const NormPlan& p, const seq::NormArgs& k, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (p.pack == 8) return norm_launch<T, 8>(p, k, st);
    if (p.pack == 4) norm_launch<T, 4>(p, k, st);
    else if (p.pack == 2) norm_launch<T, 2>(p, k, st);
    else norm_launch<T, 1>(p, k, st);
}

extern "C" {

int drl_group_norm_dev(drl_ctx* c, const drl_seq_layout* l, int64_t rows, const drl_seq_call* call, const drl_norm_args* a) {
    const char* who = "drl_group_norm_dev";
    if (!c) return DRL_ERR_ARG;
    SeqError e;
    if (norm_prepare(c, l, rows, call, a, e)) return fail(c, e);
    if ((l ? l->n_q : rows) == 0) return DRL_OK;
    const DrlCtxView v = drl_ctx_view(c);
    const NormPlan p = norm_plan(v, l, rows, call, a);
    if (seq_check_grid(e, who, p.units, 256)) return fail(c, e);
    if (seq_check_workspace(e, who, call, p.workspace)) return fail(c, e);
    DeviceGuard guard(v.device);
    if (!guard.ok) return hip_fail(c, who, hipErrorInvalidDevice);
    seq::NormArgs k = {};
    k.x = a->x; k.y = a->y; k.gamma = a->gamma; k.beta = a->beta; k.x_row = a->x_row; k.y_row = a->y_row; k.rows = rows;
    k.segs = l ? l->segs : nullptr; k.n_seg = l ? l->rows.n_seg : 0;
    k.channels = a->channels; k.groups = a->groups; k.act = a->act; k.eps = a->eps;
    k.lanes = p.lanes; k.piece = p.piece; k.slice = p.slice;
    if (p.workspace) k.part = (float*)call->workspace;
    const hipStream_t st = stream_of(v, call);
    by_type(call->dtype, [&](auto* t) { norm_packs<std::remove_pointer_t<decltype(t)>>(p, k, st); });
    return launched(c, who);
}

}  // extern "C"
