// What the library's translation units know of a context beside drlvae.hip, which defines it.
#pragma once
#include "../../include/drlvae.h"

struct DrlCtxView {
    int device;
    int n_cu;
    void* stream;       // hipStream_t the context enqueues on
};
__attribute__((visibility("hidden"))) DrlCtxView drl_ctx_view(const drl_ctx* c);
// Keeps `msg` as the context's last error and returns `code`.
__attribute__((visibility("hidden"))) int drl_ctx_fail(drl_ctx* c, int code, const char* msg);
__attribute__((visibility("hidden"))) void drl_count_alloc();
