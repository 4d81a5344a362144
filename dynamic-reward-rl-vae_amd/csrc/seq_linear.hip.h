// Linear attention with a decaying state.
#pragma once
#include "seq_common.hip.h"

namespace seq {

struct LinearArgs {
    const void *q, *k, *v;
    void* out;
    const float* log_decay;
    const float* state_in;
    float* state_out;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    const SegInfo* segs;
    int n_seg;
    int heads, rep, dk, dv;
    float scale;
};

// d_h of the definition: a NaN stays one.
__device__ __forceinline__ float decay_log(const LinearArgs& a, int h) {
    const float d = a.log_decay[h];
    return d > 0.0f ? 0.0f : d;
}

// Row after row, the state's columns in registers: thread (kk, c) holds S[kk*KP .. , c] of one column c.
template <typename T>
__global__ __launch_bounds__(256) void linear_rows_kernel(LinearArgs a) {
    constexpr int KP = 32;                       // dk <= 128: four threads share a column
    __shared__ float part[4][64];
    SegInfo s = {(int64_t)blockIdx.x, 0, 0, 1, 1, (int)blockIdx.x, 0};       // a step: one row each
    if (a.segs) s = a.segs[blockIdx.x];
    const int h = blockIdx.y, c = blockIdx.z * 64 + (threadIdx.x & 63), kk = threadIdx.x >> 6;
    const bool col = c < a.dv;
    const float lam = exp2_fast(decay_log(a, h) * LOG2E);
    const int64_t sb = ((int64_t)s.seg * a.heads + h) * a.dk * a.dv;
    float S[KP];
#pragma unroll
    for (int r = 0; r < KP; ++r) {
        const int kr = kk * KP + r;
        S[r] = a.state_in && col && kr < a.dk ? a.state_in[sb + (int64_t)kr * a.dv + c] : 0.0f;
    }
    const T* q = (const T*)a.q + (int64_t)h * a.q_head;
    const T* k = (const T*)a.k + (int64_t)(h / a.rep) * a.k_head;
    const T* v = (const T*)a.v + (int64_t)(h / a.rep) * a.v_head;
    T* o = (T*)a.out + (int64_t)h * a.o_head;
    for (int t = 0; t < s.nq; ++t) {
        const int64_t row = s.q0 + t;
        const float vc = col ? (float)v[row * a.v_row + c] : 0.0f;
        float acc = 0.0f;
#pragma unroll
        for (int r = 0; r < KP; ++r) {
            const int kr = kk * KP + r;
            if (kr < a.dk) {
                S[r] = fmaf((float)k[row * a.k_row + kr], vc, lam * S[r]);
                acc = fmaf((float)q[row * a.q_row + kr], S[r], acc);
            }
        }
        part[kk][threadIdx.x & 63] = acc;
        __syncthreads();
        if (kk == 0 && col) o[row * a.o_row + c] = (T)((part[0][threadIdx.x] + part[1][threadIdx.x] + part[2][threadIdx.x] + part[3][threadIdx.x]) * a.scale);
        __syncthreads();
    }
    if (a.state_out)
#pragma unroll
        for (int r = 0; r < KP; ++r) {
            const int kr = kk * KP + r;
            if (col && kr < a.dk) a.state_out[sb + (int64_t)kr * a.dv + c] = S[r];
        }
}

}  // namespace seq
