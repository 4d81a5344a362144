// Group normalisation with an activation, channels last.
#pragma once
#include "seq_common.hip.h"

namespace seq {

struct NormArgs {
    const void* x;
    void* y;
    const float *gamma, *beta;
    int64_t x_row, y_row;
    const SegInfo* segs;      // NULL: every row by itself
    int channels, groups, act;
    float eps;
};

__device__ __forceinline__ float activate(float x, int act) {
    if (act == 1) return x < 0.0f ? 0.0f : x;                       // a NaN stays one
    if (act == 0) return x;
    const float s = 1.0f / (1.0f + exp2_fast(-LOG2E * x));
    return act == 2 ? s : x * s;
}

template <typename T>
__global__ __launch_bounds__(256) void norm_group_kernel(NormArgs a) {
    __shared__ float red[4];
    const int g = blockIdx.y, cg = a.channels / a.groups, c0 = g * cg;
    int64_t first = blockIdx.x;
    int rows = 1;
    if (a.segs) { first = a.segs[blockIdx.x].q0; rows = a.segs[blockIdx.x].nq; }
    const int64_t n = (int64_t)rows * cg;
    if (n == 0) return;
    const T* x = (const T*)a.x + first * a.x_row + c0;
    T* y = (T*)a.y + first * a.y_row + c0;
    auto total = [&](float v) {
        v = wave_sum(v);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        return red[0] + red[1] + red[2] + red[3];
    };
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 256) s += (float)x[i / cg * a.x_row + i % cg];
    const float mean = total(s) / (float)n;
    float d2 = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 256) { const float d = (float)x[i / cg * a.x_row + i % cg] - mean; d2 = fmaf(d, d, d2); }
    const float rstd = 1.0f / sqrtf(total(d2) / (float)n + a.eps);
    for (int64_t i = threadIdx.x; i < n; i += 256) {
        const int c = (int)(i % cg);
        const float w = ((float)x[i / cg * a.x_row + c] - mean) * rstd;
        y[i / cg * a.y_row + c] = (T)activate(fmaf(w, a.gamma ? a.gamma[c0 + c] : 1.0f, a.beta ? a.beta[c0 + c] : 0.0f), a.act);
    }
}

}  // namespace seq
