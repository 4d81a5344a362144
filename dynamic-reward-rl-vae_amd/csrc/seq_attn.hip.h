// Softmax attention over packed series.
#pragma once
#include "seq_common.hip.h"

namespace seq {

struct AttnArgs {
    const void *q, *k, *v;
    void* out;
    float* lse;
    const uint8_t* key_mask;
    const int32_t* k_len;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;
    const SegInfo* segs;
    int n_seg;
    int heads, rep, dim;
    int causal, window;
    float scale;
};

// The keys [lo, hi) that row i of a series may see by position (the key mask apart).
__device__ __forceinline__ void visible(const AttnArgs& a, int i, int nq, int nk, int& lo, int& hi) {
    const int64_t end = (int64_t)i + nk - nq;             // the row's own place among the keys
    hi = a.causal ? (int)max((int64_t)0, min((int64_t)nk, end + 1)) : nk;
    lo = a.window > 0 ? (int)max((int64_t)0, min((int64_t)nk, end + 1 - a.window)) : 0;
}

__device__ __forceinline__ int keys_of(const AttnArgs& a, const SegInfo& s) {
    return a.k_len ? max(0, min(a.k_len[s.seg], s.nk)) : s.nk;
}

// One row and head by one wave, straight from the definition: 64 keys at a time, a lane per key for the scores, lanes
// over the width for the sum.  Touches nothing but the visible keys' rows.
template <typename T>
__device__ void attn_row(const AttnArgs& a, const SegInfo& s, int nk, int i, int h) {
    const int lane = threadIdx.x & 63;
    const int64_t row = s.q0 + i;
    const T* q = (const T*)a.q + row * a.q_row + (int64_t)h * a.q_head;
    const T* kb = (const T*)a.k + s.k0 * a.k_row + (int64_t)(h / a.rep) * a.k_head;
    const T* vb = (const T*)a.v + s.k0 * a.v_row + (int64_t)(h / a.rep) * a.v_head;
    int lo, hi;
    visible(a, i, s.nq, nk, lo, hi);
    float top = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int base = lo; base < hi; base += 64) {
        const int j = base + lane;
        const bool seen = j < hi && (!a.key_mask || a.key_mask[s.k0 + j]);
        float z = -INFINITY;
        if (seen) {
            const T* kr = kb + (int64_t)j * a.k_row;
            float d = 0.0f;
            for (int c = 0; c < a.dim; ++c) d = fmaf((float)q[c], (float)kr[c], d);
            z = d * a.scale;
        }
        const float m = fmaxf(top, wave_max(z));
        const float mm = m == -INFINITY ? 0.0f : m;
        const float p = seen ? exp2_fast((z - mm) * LOG2E) : 0.0f;
        const float c = exp2_fast((top - mm) * LOG2E);
        sum = sum * c + wave_sum(p);
        o0 *= c;
        o1 *= c;
        top = m;
        uint64_t todo = __ballot(seen);
        while (todo) {
            const int b = __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            const float pj = __shfl(p, b);
            const T* vr = vb + (int64_t)(base + b) * a.v_row;
            if (lane < a.dim) o0 = fmaf(pj, (float)vr[lane], o0);
            if (lane + 64 < a.dim) o1 = fmaf(pj, (float)vr[lane + 64], o1);
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;      // a NaN sum stays one
    T* o = (T*)a.out + row * a.o_row + (int64_t)h * a.o_head;
    if (lane < a.dim) o[lane] = (T)(o0 * inv);
    if (lane + 64 < a.dim) o[lane + 64] = (T)(o1 * inv);
    if (a.lse && lane == 0)
        a.lse[row * a.heads + h] = sum == 0.0f ? -INFINITY : (top == -INFINITY ? 0.0f : top) + LN2 * __builtin_amdgcn_logf(sum);
}

template <typename T>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
    const int64_t t = (int64_t)blockIdx.x;
    const int slot = find_seg(a.segs, a.n_seg, t, 4);
    const SegInfo s = a.segs[slot];
    const int i = (int)(t - (s.cum / 4 + slot)) * 4 + (int)(threadIdx.x >> 6);
    if (i >= s.nq) return;
    attn_row<T>(a, s, keys_of(a, s), i, blockIdx.y);
}

}  // namespace seq
