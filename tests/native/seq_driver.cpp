// Native caller of the sequence operators (include/drlvae.h), built as abi_driver.cpp is: layouts of many shapes, workspaces,
// refusals and one small call of each operator on the context's stream, in float32, against plain loops in double.
// Prints "seq_driver OK" and exits 0 on success.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <random>
#include <vector>

#include "drlvae.h"

#define EXPECT(cond)                                                                             \
    do {                                                                                         \
        if (!(cond)) { std::fprintf(stderr, "%s:%d expectation failed: %s (%s)\n", __FILE__, __LINE__, #cond, drl_last_error(ctx)); return 1; } \
    } while (0)

static std::mt19937 rng(11);
struct Dev {
    float* p = nullptr;
    std::vector<float> h;
    explicit Dev(size_t n, float spread = 1.0f) : h(n) {
        std::uniform_real_distribution<float> d(-spread, spread);
        for (auto& x : h) x = d(rng);
        if (hipMalloc((void**)&p, n * 4 + 16) != hipSuccess || hipMemcpy(p, h.data(), n * 4, hipMemcpyHostToDevice) != hipSuccess) std::abort();
    }
    ~Dev() { (void)hipFree(p); }
    std::vector<float> back() const {
        std::vector<float> v(h.size());
        if (hipMemcpy(v.data(), p, v.size() * 4, hipMemcpyDeviceToHost) != hipSuccess) std::abort();
        return v;
    }
};
static bool near(double got, double want, double size) { return std::fabs(got - want) <= 1e-4 * (size + 1e-3); }

int main() {
    drl_ctx* ctx = nullptr;
    if (drl_create(0, &ctx) != 0) { std::fprintf(stderr, "drl_create failed\n"); return 1; }

    // layouts: many, empty, large, refused
    for (int i = 0; i < 300; ++i) {
        const int n = i == 7 ? 70000 : i % 50;
        std::vector<int64_t> off(n + 1, 3);
        for (int s = 0; s < n; ++s) off[s + 1] = off[s] + (s * 7 + i) % 5;
        drl_seq_layout* l = nullptr;
        EXPECT(drl_seq_layout_create(ctx, off.data(), i % 2 ? off.data() : nullptr, n, &l) == 0 && l);
        drl_seq_layout_destroy(l);
    }
    drl_seq_layout_destroy(nullptr);
    drl_seq_layout* none = nullptr;
    const int64_t falling[] = {0, 5, 4};
    EXPECT(drl_seq_layout_create(ctx, falling, nullptr, 2, &none) == DRL_ERR_ARG && !none);
    EXPECT(drl_seq_layout_create(ctx, nullptr, nullptr, 2, &none) == DRL_ERR_ARG && !none);

    const int R = 100, H = 2, D = 16, C = 24, G = 3;
    const int64_t off[] = {0, 40, 40, 97};                     // three rows belong to no series
    drl_seq_layout* l = nullptr;
    EXPECT(drl_seq_layout_create(ctx, off, nullptr, 3, &l) == 0);
    Dev q(R * H * D), k(R * H * D), v(R * H * D), out(R * H * D), lse(R * H), x(R * C), y(R * C), state(3 * H * D * D), ld(H, 0.1f);
    drl_seq_call call = {};
    call.struct_size = sizeof call;
    call.abi_revision = DRL_ABI_REVISION;
    call.dtype = DRL_F32;

    drl_attn_args a = {};
    a.q = q.p; a.k = k.p; a.v = v.p; a.out = out.p; a.lse = lse.p;
    a.q_row = a.k_row = a.v_row = a.o_row = H * D;
    a.q_head = a.k_head = a.v_head = a.o_head = D;
    a.n_heads = a.n_kv_heads = H; a.dim = D; a.causal = 1; a.window = 9; a.scale = 0.25f;
    int64_t bytes = -1;
    EXPECT(drl_attention_workspace(ctx, l, &call, &a, &bytes) == 0 && bytes == 0);
    EXPECT(drl_attention_dev(ctx, l, &call, &a) == 0);
    drl_synchronize(ctx);
    std::vector<float> o = out.back(), ls = lse.back();
    for (int s = 0; s < 3; ++s)
        for (int64_t i = off[s]; i < off[s + 1]; ++i)
            for (int h = 0; h < H; ++h) {
                double sum = 0, acc[16] = {0};
                for (int64_t j = std::max(off[s], i - 8); j <= i; ++j) {
                    double z = 0;
                    for (int d = 0; d < D; ++d) z += (double)q.h[(i * H + h) * D + d] * k.h[(j * H + h) * D + d];
                    const double p = std::exp(0.25 * z);
                    sum += p;
                    for (int d = 0; d < D; ++d) acc[d] += p * v.h[(j * H + h) * D + d];
                }
                EXPECT(near(ls[i * H + h], std::log(sum), 1));
                for (int d = 0; d < D; ++d) EXPECT(near(o[(i * H + h) * D + d], acc[d] / sum, 1));
            }
    for (int e = 97 * H * D; e < R * H * D; ++e) EXPECT(o[e] == out.h[e]);

    drl_attn_args bad = a;
    bad.dim = 12;
    EXPECT(drl_attention_dev(ctx, l, &call, &bad) == DRL_ERR_UNSUPPORTED);
    bad = a;
    bad.k = (char*)a.k + 4;
    EXPECT(drl_attention_dev(ctx, l, &call, &bad) == DRL_ERR_ARG);
    EXPECT(drl_attention_dev(ctx, nullptr, &call, &a) == DRL_ERR_ARG && drl_attention_dev(ctx, l, nullptr, &a) == DRL_ERR_ARG);
    EXPECT(drl_attention_dev(ctx, l, &call, nullptr) == DRL_ERR_ARG && drl_attention_dev(nullptr, l, &call, &a) == DRL_ERR_ARG);

    drl_linear_args b = {};
    b.q = q.p; b.k = k.p; b.v = v.p; b.out = out.p; b.log_decay = ld.p; b.state_out = state.p;
    b.q_row = b.k_row = b.v_row = b.o_row = H * D;
    b.q_head = b.k_head = b.v_head = b.o_head = D;
    b.n_heads = b.n_kv_heads = H; b.dim_k = b.dim_v = D; b.scale = 0.25f;
    EXPECT(drl_linear_attention_workspace(ctx, l, &call, &b, &bytes) == 0 && bytes >= 0);
    Dev ws((size_t)bytes / 4 + 4);
    call.workspace = ws.p;
    call.workspace_bytes = bytes;
    EXPECT(drl_linear_attention_dev(ctx, l, &call, &b) == 0);
    drl_synchronize(ctx);
    o = out.back();
    std::vector<float> st = state.back();
    for (int s = 0; s < 3; ++s)
        for (int h = 0; h < H; ++h) {
            double S[16][16] = {{0}};
            const double lam = std::exp(std::min((double)ld.h[h], 0.0));
            for (int64_t i = off[s]; i < off[s + 1]; ++i)
                for (int e = 0; e < D; ++e) {
                    double want = 0;
                    for (int d = 0; d < D; ++d) {
                        S[d][e] = lam * S[d][e] + (double)k.h[(i * H + h) * D + d] * v.h[(i * H + h) * D + e];
                        want += 0.25 * S[d][e] * q.h[(i * H + h) * D + d];
                    }
                    EXPECT(near(o[(i * H + h) * D + e], want, 10));
                }
            for (int d = 0; d < D; ++d)
                for (int e = 0; e < D; ++e) EXPECT(near(st[((s * H + h) * D + d) * D + e], S[d][e], 10));
        }
    b.state_in = state.p;
    EXPECT(drl_linear_attention_step_dev(ctx, 3, &call, &b) == 0);
    drl_synchronize(ctx);
    const std::vector<float> st2 = state.back();
    for (int n = 0; n < 3; ++n)
        for (int h = 0; h < H; ++h)
            for (int d = 0; d < D; ++d)
                for (int e = 0; e < D; ++e) {
                    const int at = ((n * H + h) * D + d) * D + e;
                    const double want = std::exp(std::min((double)ld.h[h], 0.0)) * st[at] + (double)k.h[(n * H + h) * D + d] * v.h[(n * H + h) * D + e];
                    EXPECT(near(st2[at], want, 10));
                }
    o = out.back();
    for (int n = 0; n < 3; ++n)
        for (int h = 0; h < H; ++h)
            for (int e = 0; e < D; ++e) {
                double want = 0;
                for (int d = 0; d < D; ++d) want += 0.25 * st2[((n * H + h) * D + d) * D + e] * q.h[(n * H + h) * D + d];
                EXPECT(near(o[(n * H + h) * D + e], want, 10));
            }
    b.state_in = nullptr;
    EXPECT(drl_linear_attention_step_dev(ctx, 3, &call, &b) == DRL_ERR_ARG);

    drl_norm_args c = {};
    c.x = x.p; c.y = y.p; c.x_row = c.y_row = C; c.channels = C; c.groups = G; c.act = DRL_ACT_SILU; c.eps = 1e-5f;
    for (int rows = 0; rows < 2; ++rows) {                     // per series, per row
        drl_seq_layout* use = rows ? nullptr : l;
        EXPECT(drl_group_norm_workspace(ctx, use, R, &call, &c, &bytes) == 0 && bytes <= call.workspace_bytes);
        EXPECT(drl_group_norm_dev(ctx, use, R, &call, &c) == 0);
        drl_synchronize(ctx);
        const std::vector<float> n = y.back();
        for (int s = 0; s < (rows ? R : 3); ++s)
            for (int g = 0; g < G; ++g) {
                const int64_t from = rows ? s : off[s], to = rows ? s + 1 : off[s + 1];
                double mean = 0, var = 0;
                const double N = (double)(to - from) * (C / G);
                for (int pass = 0; pass < 2; ++pass)
                    for (int64_t i = from; i < to; ++i)
                        for (int e = g * C / G; e < (g + 1) * C / G; ++e) {
                            if (pass == 0) mean += x.h[i * C + e] / N;
                            else var += (x.h[i * C + e] - mean) * (x.h[i * C + e] - mean) / N;
                        }
                for (int64_t i = from; i < to; ++i)
                    for (int e = g * C / G; e < (g + 1) * C / G; ++e) {
                        const double z = (x.h[i * C + e] - mean) / std::sqrt(var + 1e-5);
                        EXPECT(near(n[i * C + e], z / (1 + std::exp(-z)), 10));
                    }
            }
    }
    c.groups = 5;
    EXPECT(drl_group_norm_dev(ctx, l, R, &call, &c) == DRL_ERR_ARG);

    drl_seq_layout_destroy(l);
    drl_destroy(ctx);
    std::printf("seq_driver OK\n");
    return 0;
}
