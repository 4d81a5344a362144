// Group normalisation with an activation, channels last:  y = act((x - mean) / sqrt(var + eps) * gamma + beta).
//
// Bound by memory: x is read and y written once, and x once more where a group does not fit into registers.  Means and
// squared deviations are never differences of large sums: rows by themselves are summed in two passes over registers,
// series by running means that are joined pairwise (with the counts n, means m and squared deviations s of two parts,
// m = m1 + (m2 - m1) n2/n, s = s1 + s2 + (m2 - m1)^2 n1 n2/n), always in the same order.
#pragma once
#include "seq_common.hip.h"

namespace seq {

struct NormArgs {
    const void* x;
    void* y;
    const float *gamma, *beta;
    int64_t x_row, y_row, rows;
    const SegInfo* segs;
    int n_seg;
    int channels, groups, act;
    float eps;
    // rows by themselves: lanes per group; series: rows per unit, groups per workgroup
    int lanes, piece, slice;
    float* part;              // [units][groups][2]: mean and squared deviation of a unit's rows (NULL: one unit per series)
};

// In float32 the exponent is taken in two parts, the second times ln 2 as a factor: one product's rounding alone, relative to
// the exponent, would make the result's relative error grow with |x| (4e-6 at -40).  What is rounded to 16 bits does not show it.
template <typename T>
__device__ __forceinline__ float activate(float x, int act) {
    if (act == 1) return x < 0.0f ? 0.0f : x;                       // a NaN stays one
    if (act == 0) return x;
    float e;
    if constexpr (sizeof(T) == 4) {
        constexpr float LOG2E_REST = 1.9259629911e-8f;              // log2(e) - LOG2E
        const float t = -LOG2E * x;
        e = exp2_fast(t);                                           // infinite, or nothing beside 1, from 128 on
        e = fabsf(t) < 128.0f ? fmaf(e * LN2, fmaf(-LOG2E_REST, x, fmaf(-LOG2E, x, -t)), e) : e;
    } else e = exp2_fast(-LOG2E * x);
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    return act == 2 ? s : x * s;
}

template <typename T, int V> struct alignas(V * sizeof(T)) Pack { T e[V]; };

struct Moments {
    float n, mean, dev;
};
__device__ __forceinline__ Moments join(const Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (n == 0.0f) return a;
    const float d = b.mean - a.mean, w = b.n / n;
    return {n, fmaf(d, w, a.mean), a.dev + b.dev + d * d * a.n * w};
}
template <int K>
__device__ __forceinline__ Moments join_other(const Moments& m) {
    const Moments o = {other<K>(m.n), other<K>(m.mean), other<K>(m.dev)};
    // the lower lane first on both sides: the same result in both
    return (threadIdx.x & K) ? join(o, m) : join(m, o);
}
__device__ __forceinline__ Moments join_lanes(Moments m, int lanes) {
    if (lanes > 1) m = join_other<1>(m);
    if (lanes > 2) m = join_other<2>(m);
    if (lanes > 4) m = join_other<4>(m);
    if (lanes > 8) m = join_other<8>(m);
    if (lanes > 16) m = join_other<16>(m);
    if (lanes > 32) m = join_other<32>(m);
    return m;
}

// Rows by themselves.  `lanes` lanes hold a group of a row, NV packs of V channels each (NV = 0: it does not fit, and is
// read twice more from the caches); a wave has 64 / lanes neighbouring groups and goes down the rows with them, so that
// gamma and beta stay in registers.  65,536 rows of 4,096 channels in 32 groups, bfloat16: 241 us, 4.5 TB/s (a copy: 4.7); 4
// rows of 1,024: 7.0 us, a launch.
template <typename T, int V, int NV>
__global__ __launch_bounds__(256) void norm_rows_kernel(NormArgs a) {
    typedef Pack<T, V> P;
    const int lane = threadIdx.x & 63, cg = a.channels / a.groups, nv = cg / V;
    const int per_wave = 64 / a.lanes, sets = (a.groups + per_wave - 1) / per_wave;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), waves = (int64_t)gridDim.x * 4;
    const int set = (int)(id % sets), sub = lane % a.lanes, g = set * per_wave + lane / a.lanes;
    const int64_t step = waves / sets;                 // the grid is a multiple of the sets
    const bool on = g < a.groups;
    const int c0 = (on ? g : 0) * cg;
    const float inv = 1.0f / (float)cg;
    auto sum = [&](float v) { return lanes_sum(v, a.lanes); };
    if constexpr (NV > 0) {
        float ga[NV][V], be[NV][V];
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = c0 + (sub + n * a.lanes) * V + e;
                const bool in = sub + n * a.lanes < nv;
                ga[n][e] = a.gamma && in ? a.gamma[c] : 1.0f;
                be[n][e] = a.beta && in ? a.beta[c] : 0.0f;
            }
        auto load = [&](int64_t row, P (&p)[NV]) {
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                p[n] = P{};
                if (on && sub + n * a.lanes < nv) p[n] = *(const P*)((const T*)a.x + row * a.x_row + c0 + (sub + n * a.lanes) * V);
            }
        };
        P next[NV];
        if (id / sets < a.rows) load(id / sets, next);
        for (int64_t row = id / sets; row < a.rows; row += step) {
            T* y = (T*)a.y + row * a.y_row + c0;
            float f[NV][V], s = 0.0f;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) s += f[n][e] = (float)next[n].e[e];
            if (row + step < a.rows) load(row + step, next);          // on its way while this row is done
            const float mean = sum(s) * inv;
            float d2 = 0.0f;
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    f[n][e] -= mean;
                    if (sub + n * a.lanes < nv) d2 = fmaf(f[n][e], f[n][e], d2);
                }
            const float rstd = 1.0f / sqrtf(fmaf(sum(d2), inv, a.eps));
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                P p;
#pragma unroll
                for (int e = 0; e < V; ++e) p.e[e] = (T)activate<T>(fmaf(f[n][e] * rstd, ga[n][e], be[n][e]), a.act);
                if (on && sub + n * a.lanes < nv) *(P*)(y + (sub + n * a.lanes) * V) = p;
            }
        }
    } else {
        for (int64_t row = id / sets; row < a.rows; row += step) {
            const T* x = (const T*)a.x + row * a.x_row + c0;
            T* y = (T*)a.y + row * a.y_row + c0;
            float s = 0.0f, d2 = 0.0f;
            if (on)
                for (int n = sub; n < nv; n += a.lanes) {
                    const P p = *(const P*)(x + n * V);
#pragma unroll
                    for (int e = 0; e < V; ++e) s += (float)p.e[e];
                }
            const float mean = sum(s) * inv;
            if (on)
                for (int n = sub; n < nv; n += a.lanes) {
                    const P p = *(const P*)(x + n * V);
#pragma unroll
                    for (int e = 0; e < V; ++e) { const float d = (float)p.e[e] - mean; d2 = fmaf(d, d, d2); }
                }
            const float rstd = 1.0f / sqrtf(fmaf(sum(d2), inv, a.eps));
            if (on)
                for (int n = sub; n < nv; n += a.lanes) {
                    P p = *(const P*)(x + n * V);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const int c = c0 + n * V + e;
                        p.e[e] = (T)activate<T>(fmaf(((float)p.e[e] - mean) * rstd, a.gamma ? a.gamma[c] : 1.0f, a.beta ? a.beta[c] : 0.0f), a.act);
                    }
                    *(P*)(y + n * V) = p;
                }
        }
    }
}

// Short series: a workgroup has one group of one series in registers, R packs of V channels per thread, and sums it in two
// passes over them: x is read once, in one launch.  67 series of 1,421 rows of 128 channels in 8 groups, float32: 34 us, where
// reading and writing take 21 at a copy's rate: 536 workgroups for 512 places, and each waits for its own reads.
template <typename T, int V, int R, int THREADS>
__global__ __launch_bounds__(THREADS) void norm_short_kernel(NormArgs a) {
    typedef Pack<T, V> P;
    __shared__ float red[2][THREADS / 64];
    // a series' groups share lines of memory: one XCD (the workgroup's number modulo 8) does all of them, one after the other
    const uint32_t eight = blockIdx.x / 8, slot = eight / a.groups * 8 + blockIdx.x % 8;
    if (slot >= (uint32_t)a.n_seg) return;
    const SegInfo s = a.segs[slot];
    if (s.nq == 0) return;
    const int cg = a.channels / a.groups, per = cg / V, packs = s.nq * per, c0 = (int)(eight % a.groups) * cg;
    const T* x = (const T*)a.x + s.q0 * a.x_row + c0;
    T* y = (T*)a.y + s.q0 * a.y_row + c0;
    auto sum = [&](float v, int k) {
        v = wave_sum(v);
        if ((threadIdx.x & 63) == 0) red[k][threadIdx.x >> 6] = v;
        __syncthreads();
        float all = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) all += red[k][w];
        return all;
    };
    P p[R];
    float f = 0.0f;
    int row[R], pos[R];
#pragma unroll
    for (int n = 0; n < R; ++n) {
        const uint32_t i = n * THREADS + threadIdx.x;
        row[n] = i / (uint32_t)per;
        pos[n] = (i - row[n] * per) * V;
        if (i < (uint32_t)packs) p[n] = *(const P*)(x + (int64_t)row[n] * a.x_row + pos[n]);
    }
#pragma unroll
    for (int n = 0; n < R; ++n)
        if (n * THREADS + (int)threadIdx.x < packs)
#pragma unroll
            for (int e = 0; e < V; ++e) f += (float)p[n].e[e];
    const float inv = 1.0f / (float)(s.nq * cg), mean = sum(f, 0) * inv;
    f = 0.0f;
#pragma unroll
    for (int n = 0; n < R; ++n)
        if (n * THREADS + (int)threadIdx.x < packs)
#pragma unroll
            for (int e = 0; e < V; ++e) { const float d = (float)p[n].e[e] - mean; f = fmaf(d, d, f); }
    const float rstd = 1.0f / sqrtf(fmaf(sum(f, 1), inv, a.eps));
#pragma unroll
    for (int n = 0; n < R; ++n)
        if (n * THREADS + (int)threadIdx.x < packs) {
            P q;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int c = c0 + pos[n] + e;
                q.e[e] = (T)activate<T>(fmaf(((float)p[n].e[e] - mean) * rstd, a.gamma ? a.gamma[c] : 1.0f, a.beta ? a.beta[c] : 0.0f), a.act);
            }
            *(P*)(y + (int64_t)row[n] * a.y_row + pos[n]) = q;
        }
}

// Series.  A workgroup has `piece` rows of one series and `slice` groups of channels; a thread has a pack of V channels
// (of one group; where one group alone has more packs than threads, several of them) and every so many rows.
// STATS writes the unit's moments, the second launch joins a series' units and writes y; a series that is one unit
// (part == NULL: all are) is done at once, its second reading out of the caches.  100 MB of 67 series of 512 channels,
// bfloat16: 78 us, 2.6 TB/s of what is needed, with the second reading 3.9.
template <typename T, int V, bool STATS>
__global__ __launch_bounds__(256) void norm_series_kernel(NormArgs a) {
    typedef Pack<T, V> P;
    __shared__ Moments mom[256];
    __shared__ float stat[256][2];
    const int slot = find_seg(a.segs, a.n_seg, blockIdx.x, a.piece);
    const SegInfo s = a.segs[slot];
    const uint32_t unit0 = s.cum / (uint32_t)a.piece + slot;
    const int k = (int)(blockIdx.x - unit0), units = (int)(((uint32_t)s.nq + a.piece - 1) / (uint32_t)a.piece);
    if (k >= units) return;
    const int first = k * a.piece, rows = min(a.piece, s.nq - first);
    const int cg = a.channels / a.groups, g0 = blockIdx.y * a.slice, ng = min(a.slice, a.groups - g0);
    const int per = cg / V, nvec = ng * per, tc = min(nvec, 256), rl = 256 / tc;
    const int c = threadIdx.x % tc, r0 = threadIdx.x / tc;
    const bool on = r0 < rl;
    const T* x = (const T*)a.x + (s.q0 + first) * a.x_row + g0 * cg;
    T* y = (T*)a.y + (s.q0 + first) * a.y_row + g0 * cg;

    if (STATS || !a.part) {
        Moments m = {0.0f, 0.0f, 0.0f};
        if (on)
            for (int v = c; v < nvec; v += tc) {
                float mean[V], dev[V], n = 0.0f;
#pragma unroll
                for (int e = 0; e < V; ++e) mean[e] = dev[e] = 0.0f;
                int r = r0;
                constexpr int U = 4;                                  // rows in flight
                for (; r + (U - 1) * rl < rows; r += U * rl) {
                    P p[U];
#pragma unroll
                    for (int i = 0; i < U; ++i) p[i] = *(const P*)(x + (int64_t)(r + i * rl) * a.x_row + v * V);
#pragma unroll
                    for (int i = 0; i < U; ++i) {
                        n += 1.0f;
                        const float w = __builtin_amdgcn_rcpf(n);
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            const float f = (float)p[i].e[e], d = f - mean[e];
                            mean[e] = fmaf(d, w, mean[e]);
                            dev[e] = fmaf(d, f - mean[e], dev[e]);
                        }
                    }
                }
                for (; r < rows; r += rl) {
                    const P p = *(const P*)(x + (int64_t)r * a.x_row + v * V);
                    n += 1.0f;
                    const float w = __builtin_amdgcn_rcpf(n);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float f = (float)p.e[e], d = f - mean[e];
                        mean[e] = fmaf(d, w, mean[e]);
                        dev[e] = fmaf(d, f - mean[e], dev[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < V; ++e) m = join(m, {n, mean[e], dev[e]});
            }
        mom[threadIdx.x] = m;
        __syncthreads();
        // a wave joins the threads of 64 / lanes groups at a time
        const int per_wave = 64 / a.lanes, w = threadIdx.x >> 6, sub = threadIdx.x % a.lanes, share = min(per, 256);
        for (int g = w * per_wave + (threadIdx.x & 63) / a.lanes; g < (ng + per_wave - 1) / per_wave * per_wave; g += 4 * per_wave) {
            Moments t = {0.0f, 0.0f, 0.0f};
            if (g < ng)
                for (int i = sub; i < share * rl; i += a.lanes) t = join(t, mom[(i / share) * tc + g * share + i % share]);
            t = join_lanes(t, a.lanes);
            if (g < ng && sub == 0) {
                if (STATS) {
                    float* o = a.part + ((int64_t)blockIdx.x * a.groups + g0 + g) * 2;
                    o[0] = t.mean;
                    o[1] = t.dev;
                } else {
                    stat[g][0] = t.mean;
                    stat[g][1] = 1.0f / sqrtf(t.dev / t.n + a.eps);
                }
            }
        }
        if (STATS) return;
    } else {
        for (int g = threadIdx.x >> 6; g < ng; g += 4) {
            Moments t = {0.0f, 0.0f, 0.0f};
            for (int u = threadIdx.x & 63; u < units; u += 64) {
                const float* o = a.part + ((int64_t)(unit0 + u) * a.groups + g0 + g) * 2;
                t = join(t, {(float)min(a.piece, s.nq - u * a.piece) * (float)cg, o[0], o[1]});
            }
            t = join_lanes(t, 64);
            if ((threadIdx.x & 63) == 0) {
                stat[g][0] = t.mean;
                stat[g][1] = 1.0f / sqrtf(t.dev / t.n + a.eps);
            }
        }
    }
    __syncthreads();
    if (!on) return;
    for (int v = c; v < nvec; v += tc) {
        const int g = v / per;
        const float mean = stat[g][0], rstd = stat[g][1];
        float ga[V], be[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            ga[e] = a.gamma ? a.gamma[g0 * cg + v * V + e] : 1.0f;
            be[e] = a.beta ? a.beta[g0 * cg + v * V + e] : 0.0f;
        }
        auto put = [&](P p, int r) {
#pragma unroll
            for (int e = 0; e < V; ++e) p.e[e] = (T)activate<T>(fmaf(((float)p.e[e] - mean) * rstd, ga[e], be[e]), a.act);
            *(P*)(y + (int64_t)r * a.y_row + v * V) = p;
        };
        int r = r0;
        for (; r + 3 * rl < rows; r += 4 * rl) {
            P p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *(const P*)(x + (int64_t)(r + i * rl) * a.x_row + v * V);
#pragma unroll
            for (int i = 0; i < 4; ++i) put(p[i], r + i * rl);
        }
        for (; r < rows; r += rl) put(*(const P*)(x + (int64_t)r * a.x_row + v * V), r);
    }
}

}  // namespace seq
