// Linear attention with a decaying state:  S <- lam S + k_t v_t^T,  out_t = scale S^T q_t,  lam = exp(d_h).
//
// Whole series go in chunks of C = 32 rows.  With S the state before a chunk, i and j rows of it, n its rows,
//   out_i = scale ( lam^(i+1) S^T q_i  +  sum_{j <= i} lam^(i-j) (q_i.k_j) v_j )
//   S'    = lam^n S + sum_j k_j (lam^(n-1-j) v_j)^T
// four matrix products, with no power of lam above 1.
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
    // a series is cut into pieces of `piece` rows (a multiple of the chunk); unit u is a piece, states[u] the state
    // before it, [heads, dk, dv] (NULL: the series are whole)
    int piece, blocks;            // blocks: workgroups per head, over the values' width
    float* states;
};

// log2 of a head's decay per row: a growth is taken as none, a NaN stays one.
__device__ __forceinline__ float decay_log(const LinearArgs& a, int h) {
    const float d = a.log_decay[h];
    return d > 0.0f ? 0.0f : d;
}
__device__ __forceinline__ float power(float ld2, int n) { return n == 0 ? 1.0f : exp2_fast(ld2 * (float)n); }

// A state over n rows: S + (lam^n - 1) S where lam^n is above 1/2, since lam^n itself, rounded, would drift over many times; where
// it is below, lam^n S, since 1 + (lam^n - 1) would keep an error of the old state's last place: all of a state that dies out.
struct Decay {
    float f;
    bool most;
    __device__ __forceinline__ float operator()(float S) const { return fmaf(S, f, most ? S : 0.0f); }
};
__device__ __forceinline__ Decay decay_of(const LinearArgs& a, int h, int n) {
    const float less = expm1f(decay_log(a, h) * (float)n);
    const bool most = !(less < -0.5f);                         // a NaN stays one
    return {most ? less : power(decay_log(a, h) * LOG2E, n), most};
}
// lam^n in its two roundings, f and the one beside it, by turns: the same over chunk after chunk with one product, which would drift
// with f alone.  `owed` is what the factors so far are short of; a column begins with what its state's bits make of it, from -2^-25
// to 2^-25, so that calls that hand a state on do not all round alike either.  (None of this below 1/2: nothing is left to drift.)
struct Factor {
    float f, rest;                // the same in all lanes
    __device__ __forceinline__ Factor(const LinearArgs& a, int h, int n) {
        const Decay d = decay_of(a, h, n);
        f = uniform(d.most ? 1.0f + d.f : d.f);
        rest = uniform(d.most ? d.f - (f - 1.0f) : 0.0f);
    }
    __device__ __forceinline__ float operator()(float& owed) const {
        owed += rest;
        const float more = owed > 0x1p-25f ? 0x1p-24f : owed < -0x1p-25f ? -0x1p-24f : 0.0f;      // a last place of [1/2, 1)
        owed -= more;
        return f + more;
    }
};
template <int KT>
__device__ __forceinline__ float owed_at_first(const f32x16 (&S)[KT]) {
    uint32_t bits = 0;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) bits = bits * 5 + __builtin_bit_cast(uint32_t, S[kt][r]);
    return ((float)(bits * 0x9e3779b1u >> 9) - 0x1p22f) * 0x1p-47f;
}

struct LinearUnit {
    SegInfo s;
    int64_t u;
    int first, rows;              // rows of the series in this piece
    bool any, last;
};
__device__ __forceinline__ LinearUnit linear_unit(const LinearArgs& a, uint32_t u) {
    LinearUnit t;
    t.u = u;
    const int slot = find_seg(a.segs, a.n_seg, u, a.piece);
    t.s = a.segs[slot];
    const int k = (int)(u - (t.s.cum / (uint32_t)a.piece + slot));
    const int n = max(1, (int)(((uint32_t)t.s.nq + a.piece - 1) / (uint32_t)a.piece));
    t.any = k < n;
    t.last = k == n - 1;
    t.first = k * a.piece;
    t.rows = min(a.piece, t.s.nq - t.first);
    return t;
}

// One row of each of n series.  Bound by reading and writing the states once, 8 bytes per element: a wave has 4 columns per
// lane of as many state rows as fit side by side (64 lanes over dv / 4 quads), a workgroup all dk rows of a column block
// of one series and head, and joins what the rows add to the output through LDS.  64 series of 32 heads, 128 x 128: 54 us,
// 4.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void linear_step_kernel(LinearArgs a) {
    __shared__ float part[4 * 256];
    __shared__ float kq[2][128];
    const int h = blockIdx.x % a.heads;
    const int64_t row = blockIdx.x / a.heads;
    const int quads = a.dv / 4, across = min(quads, 64);               // lanes of a workgroup row: quads of columns
    const int down = 256 / across;                                     // state rows at a time
    const int x = threadIdx.x % across, y = threadIdx.x / across;
    const bool on = y < down;
    if (threadIdx.x < a.dk) {
        kq[0][threadIdx.x] = (float)((const T*)a.k + row * a.k_row + (int64_t)(h / a.rep) * a.k_head)[threadIdx.x];
        kq[1][threadIdx.x] = (float)((const T*)a.q + row * a.q_row + (int64_t)h * a.q_head)[threadIdx.x];
    }
    const T* v = (const T*)a.v + row * a.v_row + (int64_t)(h / a.rep) * a.v_head + x * 4;
    f32x4 vc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (on)
#pragma unroll
        for (int e = 0; e < 4; ++e) vc[e] = (float)v[e];
    const Decay decay = decay_of(a, h, 1);
    const int64_t sb = (row * a.heads + h) * (int64_t)a.dk * a.dv + x * 4;
    const float* in = a.state_in + sb;
    float* out = a.state_out + sb;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    __syncthreads();
    if (on) {
        constexpr int U = 8;                                           // rows in flight
        for (int r0 = y; r0 < a.dk; r0 += U * down) {
            f32x4 S[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * down;
                if (r < a.dk) S[u] = *(const f32x4*)(in + (int64_t)r * a.dv);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * down;
                if (r < a.dk) {
                    const float kk = kq[0][r], qq = kq[1][r];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // an infinite state stays one
                        const float kept = fabsf(S[u][e]) < INFINITY ? decay(S[u][e]) : S[u][e] * (decay.most ? 1.0f + decay.f : decay.f);
                        S[u][e] = fmaf(kk, vc[e], kept);
                        acc[e] = fmaf(qq, S[u][e], acc[e]);
                    }
                    *(f32x4*)(out + (int64_t)r * a.dv) = S[u];
                }
            }
        }
    }
    if (on) *(f32x4*)&part[(y * across + x) * 4] = acc;
    __syncthreads();
    if (threadIdx.x < a.dv) {
        float s = 0.0f;
        for (int i = 0; i < down; ++i) s += part[i * across * 4 + threadIdx.x];
        ((T*)a.out + row * a.o_row + (int64_t)h * a.o_head)[threadIdx.x] = (T)(s * a.scale);
    }
}

// 2^-e with |x| 2^-e in [2^13, 2^14), for scaling into float16's range; 1 for 0 and what is not finite.  e stops at -112: below,
// the factor would pass float32's range, and a column that dies out would turn into infinities and, where it holds zeros,
// NaN.  What is lost of smaller values, 2^-137, is below float32's own normal range.
__device__ __forceinline__ float into_range(float x, float& back) {
    const int e = x > 0.0f && x < INFINITY ? max(__builtin_amdgcn_frexp_expf(x) - 14, -112) : 0;
    back = __builtin_amdgcn_ldexpf(1.0f, e);
    return __builtin_amdgcn_ldexpf(1.0f, -e);
}

// 16-bit types.  A wave keeps the state's columns of 32 value dimensions in registers, as the accumulator of the state's
// product: rows of the key width along the registers, value dimension along the lanes.  Rounded to 16 bits it is, register
// by register, an operand of the product with q (the inner index may be taken in any order; q is read from LDS
// in that order, and with it k for the scores).  Scores are computed transposed, keys along the registers, and so is the
// output, value dimension along them: a row is a lane throughout, and its factors are one register.  k and v go through LDS
// once and are read as they are for the scores and transposed (ds_read_b64_tr_b16) for the state.
// Rounding: scores and the state's copy are rounded to the inputs' type (relative error eps/2, like the result's own);
// the float32 state itself takes lam^(n-1-j) v_j as the sum of N parts of that type (24 bits of bfloat16 in three, 22 of
// float16 in two), and loses nothing from call to call.  float16 has no range to spare: scores, state columns and
// weighted values are scaled by powers of two before they are rounded, so that what is below 2^-38 of the largest score of a
// row, or value of a column and chunk, is lost.
// Two series of 32,768 rows, 32 heads of 128 x 128, bfloat16, in 16 pieces: 710-745 us by card, 300 for the pieces' states
// (a second reading of k and v), 12 to join them, the rest the outputs; 2.15 GB once are 457 us.  VALU 51 % busy, matrix
// pipe 42 %; LDS 25 % of the time, a third of it rows that meet on a bank.  24 ragged series, 16 heads of 64 x 128, float16:
// 148 us, as long as the longest series' 64 chunks take, two workgroups to a CU; VALU 55 % (scales and splits), matrix pipe
// 17 %, LDS 16 % (a quarter of it rows that meet); 92 us at a copy's rate.  Eight waves of 16 columns instead of four of 32:
// 852 us against 760 at the time.
template <typename T, int KT, int NW, bool STATE>
__global__ __launch_bounds__(NW * 64, STATE ? 3 : 2) void linear_chunk_kernel(LinearArgs a) {
    typedef typename Vec<T>::x8 x8;
    typedef typename Vec<T>::x4 x4;
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    constexpr bool F16 = __is_same(T, f16);
    constexpr int C = 32, N = F16 ? 2 : 3, THREADS = NW * 64;
    constexpr int DP = KT <= 1 ? 32 : KT <= 2 ? 64 : 128, NC = DP / 8;     // key width of an LDS row, in chunks of 8
    constexpr int VP = 32 * NW, VC = VP / 8;
    constexpr int QK = C * DP * 2, VB = C * VP * 2, STAGE = (STATE ? 1 : 2) * QK + VB;
    extern __shared__ __align__(256) char smem[];
    const uint32_t lds = lds_offset(smem), table = lds + 3 * STAGE;
    const int h = blockIdx.x % a.heads, blk = (blockIdx.x / a.heads) % a.blocks;
    const LinearUnit t = linear_unit(a, blockIdx.x / (a.heads * a.blocks));
    if (!t.any || (STATE && t.last)) return;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = blk * VP + wave * 32;                       // this wave's first value dimension
    const bool on = c0 + col < a.dv;
    const float ld2 = decay_log(a, h) * LOG2E;

    const int64_t row0 = t.s.q0 + t.first;
    const char* qp = (const char*)((const T*)a.q + row0 * a.q_row + (int64_t)h * a.q_head);
    const char* kp = (const char*)((const T*)a.k + row0 * a.k_row + (int64_t)(h / a.rep) * a.k_head);
    const char* vp = (const char*)((const T*)a.v + row0 * a.v_row + (int64_t)(h / a.rep) * a.v_head + blk * VP);
    const TileLoad<C, NC, THREADS, Swz<NC>> load_q(threadIdx.x, a.dk * 2, a.q_row * 2), load_k(threadIdx.x, a.dk * 2, a.k_row * 2);
    const TileLoad<C, VC, THREADS, Swz<VC>> load_v(threadIdx.x, min(a.dv - blk * VP, VP) * 2, a.v_row * 2);
    for (int b = 0; b < 3; ++b) {
        load_k.clear(lds + b * STAGE);
        load_v.clear(lds + b * STAGE + QK);
        if (!STATE) load_q.clear(lds + b * STAGE + QK + VB);
    }
    auto stage = [&](int base, int buf) {
        const uint32_t at = lds + buf * STAGE + wave * 1024;
        load_k(kp + base * a.k_row * 2, t.rows - base, at);
        load_v(vp + base * a.v_row * 2, t.rows - base, at + QK);
        if (!STATE) load_q(qp + base * a.q_row * 2, t.rows - base, at + QK + VB);
    };
    if (t.rows > 0) stage(0, 0);
    if (t.rows > C) stage(C, 1);

    // the state
    f32x16 S[KT];
    const float* from = nullptr;
    if (!STATE) from = a.states ? a.states + (t.u * a.heads + h) * (int64_t)a.dk * a.dv
                                : a.state_in ? a.state_in + ((int64_t)t.s.seg * a.heads + h) * (int64_t)a.dk * a.dv : nullptr;
    const uint32_t lane_s = 4 * half * a.dv + c0 + col;         // state element of a register: a row of the wave's plus the lane's
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int d = kt * 32 + acc_row(r, 0);
            S[kt][r] = from && on && d < a.dk ? (from + d * a.dv)[lane_s] : 0.0f;    // dk is a multiple of 8: d + 4 is inside too
        }
    }


    // LDS places: rows in the order of the accumulators' registers (two reads of 4), and transposed.  Chunk c lies at place
    // c ^ swz of its row, so that one place gives the others by an exclusive or (tiles begin at whole rows).
    const int g = (lane >> 4) & 1, i4 = lane & 15, tr = 4 * half + (i4 >> 2), tc = g * 2 + ((i4 & 3) >> 1);
    const uint32_t row4 = col * (DP * 2) + swz<NC>(col) * 16 + half * 8;
    const uint32_t ktr = tr * (DP * 2) + ((tc ^ swz<NC>(tr)) * 16) + (i4 & 1) * 8;
    const uint32_t ktr8 = (tr + 8) * (DP * 2) + ((tc ^ swz<NC>(tr + 8)) * 16) + (i4 & 1) * 8;
    const uint32_t vtr = QK + tr * (VP * 2) + (((wave * 4 + tc) ^ swz<VC>(tr)) * 16) + (i4 & 1) * 8;
    const uint32_t vtr8 = QK + (tr + 8) * (VP * 2) + (((wave * 4 + tc) ^ swz<VC>(tr + 8)) * 16) + (i4 & 1) * 8;
    auto read_tr = [&](uint32_t a0, uint32_t a1) {
        return __builtin_bit_cast(x8, (s16x8)__builtin_shufflevector(lds_read_tr(a0), lds_read_tr(a1), 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto read_row = [&](uint32_t base, int s) {
        const x4 x = lds_read<x4>((base + row4) ^ (s * 32)), y = lds_read<x4>((base + row4) ^ (s * 32 + 16));
        return (x8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };

    // Powers of lam, the same for all waves and chunks, in LDS, four registers' worth side by side: between a row (lane) and a
    // key (register), times the scale, 0 for the keys behind it; of a value's row to the chunk's end; of a row from its
    // start, times the scale.
    const uint32_t inner_at = table + 640 + lane * 16, left_at = table + half * 64, back_at = table + 128 + wave * 128;
    if (wave == 0)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            f32x4 left, inner;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = acc_row(r + e, half);
                left[e] = power(ld2, C - 1 - row);
                inner[e] = col >= row ? a.scale * power(ld2, col - row) : 0.0f;
            }
            lds_write<f32x4>(left_at + r * 4, left);
            if (!STATE) lds_write<f32x4>(inner_at + r * 256, inner);
        }
    const float grown = a.scale * power(ld2, col + 1);         // of this lane's row from the chunk's start
    const Factor whole(a, h, C), part(a, h, t.rows % C);       // over a chunk, and over one that is not full
    float owed = owed_at_first<KT>(S);

    T* op = (T*)a.out + row0 * a.o_row + (int64_t)h * a.o_head + c0;
    // the state has arrived: no wait for it inside the loop, where it would be one for the chunks to come
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) asm volatile("" : "+v"(S[kt]));
    // Loads run two chunks ahead.  AHEAD: how many a wave issues for a chunk, at least; STORES: what it stores of one.
    constexpr int AHEAD = (STATE ? 1 : 2) * (C * NC / THREADS) + C * VC / THREADS, STORES = STATE ? 0 : 2;
    const bool stores = c0 < a.dv;
    int buf = 0, far = 2;
    for (int base = 0; base < t.rows; base += C, far = buf, buf = buf == 2 ? 0 : buf + 1) {
        const int n = min(C, t.rows - base);
        // The chunk has to be here; what was issued after its loads need not be done: the stores of the two chunks before, the
        // next one's loads.
        if (base + C >= t.rows) wait_loads();
        else if (base < 2 * C || !stores) wait_loads_but<AHEAD>();
        else wait_loads_but<AHEAD + 2 * STORES>();
        __syncthreads();
        if (base + 2 * C < t.rows) stage(base + 2 * C, far);
        if (c0 >= a.dv) continue;                              // a wave behind the values' width only loads
        const float lam_n = (n < C ? part : whole)(owed);
        const uint32_t kb = lds + buf * STAGE, qb = kb + QK + VB;

        x8 v[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) v[s] = read_tr(kb + vtr + s * 16 * VP * 2, kb + vtr8 + s * 16 * VP * 2);
        // A value that is not finite must not meet the rows before its own, not even with weight 0: it is taken out, and its
        // column is set to NaN from its row on.
        int bad;
        const bool odd = __any(not_finite<T>(__builtin_bit_cast(u32x4, v[0]), __builtin_bit_cast(u32x4, v[1])));
        if (odd) {
            bad = C;
#pragma unroll
            for (int e = 15; e >= 0; --e)
                if (!(fabsf((float)v[e >> 3][e & 7]) < INFINITY)) {
                    bad = acc_row(e, half);
                    v[e >> 3][e & 7] = (T)0.0f;
                }
            bad = min(bad, __shfl_xor(bad, 32));
            if (bad >= n) bad = C;                             // rows behind the series' last are its last again
        }

        if constexpr (!STATE) {
            f32x16 z, o;
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = o[r] = 0.0f;
            float s_scale = 1.0f, s_back = 1.0f;
            if constexpr (F16) {
                float m = 0.0f;
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) m = fmaxf(m, fabsf(S[kt][r]));
                s_scale = into_range(pair_max(m), s_back);
                if (half == 0) lds_write<float>(back_at + col * 4, s_back);    // the product has the state's columns along its registers
            }
#pragma unroll
            for (int s = 0; s < 2 * KT; ++s) {
                if (s % 2 == 0) keep_reads();                          // two steps' reads in flight, no more: registers
                const x8 q = read_row(qb, s), k = read_row(kb, s);
                z = mfma(k, q, z);
                x8 b;
#pragma unroll
                for (int e = 0; e < 8; ++e) b[e] = (T)(F16 ? S[s >> 1][8 * (s & 1) + e] * s_scale : S[s >> 1][8 * (s & 1) + e]);
                o = mfma(b, q, o);
            }
            float p[16];
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 inner = lds_read<f32x4>(inner_at + r * 256);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[r + e] = mul_legacy(z[r + e], inner[e]);     // 0 where inner is 0, whatever the score
            }
            float p_scale = 1.0f, p_back = 1.0f;
            f32x16 w = o;
            for (int r = 0; r < 16; r += 4) {
                f32x4 back;
                if (F16) back = lds_read<f32x4>(back_at + r * 8 + half * 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r + e] *= F16 ? grown * back[e] : grown;
            }
            if constexpr (F16) {
                float m = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    m = fmaxf(m, fabsf(p[r]));
                    w[r] = 0.0f;
                }
                p_scale = into_range(pair_max(m), p_back);
            } else w = o;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                x8 b;
#pragma unroll
                for (int e = 0; e < 8; ++e) b[e] = (T)(F16 ? p[8 * s + e] * p_scale : p[8 * s + e]);
                w = mfma(v[s], b, w);
            }
            if constexpr (F16)
#pragma unroll
                for (int r = 0; r < 16; ++r) w[r] = fmaf(w[r], p_back, o[r]);
            if (odd) {
                rarely(bad);
#pragma unroll
                for (int r = 0; r < 16; ++r) w[r] = col >= __shfl(bad, acc_row(r, half)) ? NAN : w[r];
            }
            // Four columns of the lane's row are in four registers, the next four those of the lane 32 away: halves are
            // exchanged, and each lane writes eight.
            u32x4 out[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                u32x2 x = __builtin_bit_cast(u32x2, x4{(T)w[8 * g], (T)w[8 * g + 1], (T)w[8 * g + 2], (T)w[8 * g + 3]});
                u32x2 y = __builtin_bit_cast(u32x2, x4{(T)w[8 * g + 4], (T)w[8 * g + 5], (T)w[8 * g + 6], (T)w[8 * g + 7]});
                const auto e0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false), e1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
                out[g] = u32x4{(uint32_t)e0[0], (uint32_t)e1[0], (uint32_t)e0[1], (uint32_t)e1[1]};
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const auto r = __builtin_amdgcn_permlane16_swap(out[0][e], out[1][e], false, false);
                out[0][e] = r[0];
                out[1][e] = r[1];
            }
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int j = m * 16 + (lane & 15), c = (lane & 16) + 8 * half;
                if (j < n && c0 + c < a.dv) *(u32x4*)(op + (int64_t)(base + j) * a.o_row + c) = out[m];
            }
        }

        float x[16], v_scale = 1.0f, v_back = 1.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = (float)v[e >> 3][e & 7];
        if (n == C) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 left = lds_read<f32x4>(left_at + r * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[r + e] *= left[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = acc_row(e, half);
                x[e] = j < n ? x[e] * power(ld2, n - 1 - j) : 0.0f;
            }
        }
        if constexpr (F16) {
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(x[e]));
            v_scale = into_range(pair_max(m), v_back);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] *= v_scale;
        }
        x8 y[2][N];
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            f32x2 r = {x[e], x[e + 1]};
#pragma unroll
            for (int m = 0; m < N; ++m) {
                const typename Vec<T>::x2 c = __builtin_convertvector(r, typename Vec<T>::x2);
                y[e >> 3][m][e & 7] = c[0];
                y[e >> 3][m][(e & 7) + 1] = c[1];
                r[0] -= (float)c[0];
                r[1] -= (float)c[1];
            }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            keep_reads();
            f32x16 acc;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                S[kt][r] *= lam_n;
                acc[r] = F16 ? 0.0f : S[kt][r];
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const x8 k = read_tr(((kb + ktr) ^ (kt * 64)) + s * 16 * DP * 2, ((kb + ktr8) ^ (kt * 64)) + s * 16 * DP * 2);
#pragma unroll
                for (int m = 0; m < N; ++m) acc = mfma(k, y[s][m], acc);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) S[kt][r] = F16 ? fmaf(acc[r], v_back, S[kt][r]) : acc[r];
        }
        if (odd) {
            rarely(bad);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[kt][r] = bad < C ? NAN : S[kt][r];
        }
    }

    float* to = nullptr;
    if (STATE) to = a.states + ((t.u + 1) * a.heads + h) * (int64_t)a.dk * a.dv;       // the next piece's unit
    else if (t.last && a.state_out) to = a.state_out + ((int64_t)t.s.seg * a.heads + h) * (int64_t)a.dk * a.dv;
    if (to && on)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = kt * 32 + acc_row(r, 0);
                if (d < a.dk) (to + d * a.dv)[lane_s] = S[kt][r];
            }
}

// float32: the same on 32x32x2 products; a register of the state or of the scores is an operand as it is, and nothing is
// rounded or split.  24 series of up to 2,048 rows of 16 heads, 64 x 128: 580 us, matrix pipe 58 % busy (112 products of 64
// cycles a chunk and wave, of which 32 are scores that each of a workgroup's waves makes for itself), with the loads one chunk
// ahead; one of 375 rows of 4 heads in 12 pieces: 20 us, of which its three launches take 6, 4 and 10.
template <int KT, int NW, bool STATE>
__global__ __launch_bounds__(NW * 64) void linear_chunk32_kernel(LinearArgs a) {
    constexpr int C = 32, THREADS = NW * 64;
    constexpr int DP = KT <= 1 ? 32 : KT <= 2 ? 64 : 128, NC = DP / 4;
    constexpr int VP = 32 * NW, VC = VP / 4;
    constexpr int QK = C * DP * 4, VB = C * VP * 4, STAGE = (STATE ? 1 : 2) * QK + VB;
    extern __shared__ char smem[];
    const uint32_t lds = lds_offset(smem);
    const int h = blockIdx.x % a.heads, blk = (blockIdx.x / a.heads) % a.blocks;
    const LinearUnit t = linear_unit(a, blockIdx.x / (a.heads * a.blocks));
    if (!t.any || (STATE && t.last)) return;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c0 = blk * VP + wave * 32;
    const bool on = c0 + col < a.dv;
    const float ld2 = decay_log(a, h) * LOG2E;
    const int64_t row0 = t.s.q0 + t.first;
    const char* qp = (const char*)((const float*)a.q + row0 * a.q_row + (int64_t)h * a.q_head);
    const char* kp = (const char*)((const float*)a.k + row0 * a.k_row + (int64_t)(h / a.rep) * a.k_head);
    const char* vp = (const char*)((const float*)a.v + row0 * a.v_row + (int64_t)(h / a.rep) * a.v_head + blk * VP);
    const TileLoad<C, NC, THREADS, Swz32<NC>> load_q(threadIdx.x, a.dk * 4, a.q_row * 4), load_k(threadIdx.x, a.dk * 4, a.k_row * 4);
    const TileLoad<C, VC, THREADS, Swz32<VC>> load_v(threadIdx.x, min(a.dv - blk * VP, VP) * 4, a.v_row * 4);
    for (int b = 0; b < 2; ++b) {
        load_k.clear(lds + b * STAGE);
        load_v.clear(lds + b * STAGE + QK);
        if (!STATE) load_q.clear(lds + b * STAGE + QK + VB);
    }
    auto stage = [&](int base, int buf) {
        const uint32_t at = lds + buf * STAGE + wave * 1024;
        load_k(kp + base * a.k_row * 4, t.rows - base, at);
        load_v(vp + base * a.v_row * 4, t.rows - base, at + QK);
        if (!STATE) load_q(qp + base * a.q_row * 4, t.rows - base, at + QK + VB);
    };
    if (t.rows > 0) stage(0, 0);

    f32x16 S[KT];
    const float* from = nullptr;
    if (!STATE) from = a.states ? a.states + (t.u * a.heads + h) * (int64_t)a.dk * a.dv
                                : a.state_in ? a.state_in + ((int64_t)t.s.seg * a.heads + h) * (int64_t)a.dk * a.dv : nullptr;
    const uint32_t lane_s = 4 * half * a.dv + c0 + col;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int d = kt * 32 + acc_row(r, 0);
            S[kt][r] = from && on && d < a.dk ? (from + d * a.dv)[lane_s] : 0.0f;
        }

    // LDS places as in the attention kernel for float32: rows by exclusive or, columns in four forms (NC = 8: two, at rows
    // 0 and 8), the rest constant; a wave's values lie at chunk 8 wave, which rows 8 .. 15 exchange with its neighbour.
    const uint32_t row4 = lds + col * (DP * 4) + ((half ^ swz32<NC>(col)) * 16);
    uint32_t kcol[4], vcol[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        const int j = NC == 8 ? (m >> 1) * 2 + (m & 1) * 8 : m;
        kcol[m] = lds + 4 * half * (DP * 4) + (((col >> 2) ^ swz32<NC>(j + 4 * half)) * 16) + (col & 3) * 4;
        vcol[m] = lds + QK + 4 * half * (VP * 4) + (((wave * 8 + (col >> 2)) ^ (m + 4 * half)) * 16) + (col & 3) * 4;
    }
    float up[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) up[r] = uniform(power(ld2, acc_row(r, 0)));
    const float lane_up = a.scale * power(ld2, 4 * half + 1), lane_left = power(ld2, 4 - 4 * half);
    const Factor whole(a, h, C), part(a, h, t.rows % C);       // over a chunk, and over one that is not full
    float owed = owed_at_first<KT>(S);
    float* op = (float*)a.out + row0 * a.o_row + (int64_t)h * a.o_head;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) asm volatile("" : "+v"(S[kt]));        // arrived
    int buf = 0;
    for (int base = 0; base < t.rows; base += C, buf ^= 1) {
        const int n = min(C, t.rows - base);
        wait_loads();
        __syncthreads();
        if (base + C < t.rows) stage(base + C, buf ^ 1);
        if (c0 >= a.dv) continue;
        const float lam_n = (n < C ? part : whole)(owed);
        const uint32_t at = buf * STAGE;
        float v[16];
        bool odd = false;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            v[r] = lds_read<float>(((vcol[r & 3] + at) ^ ((r >> 2) & 1) * 128) + acc_row(r, 0) * (VP * 4));
            odd |= !(fabsf(v[r]) < INFINITY);
        }
        int bad = C;                                           // as for the 16-bit types
        odd = __any(odd);
        if (odd) {
#pragma unroll
            for (int r = 15; r >= 0; --r)
                if (!(fabsf(v[r]) < INFINITY)) {
                    bad = acc_row(r, half);
                    v[r] = 0.0f;
                }
            bad = min(bad, __shfl_xor(bad, 32));
            if (bad >= n) bad = C;
        }
        if constexpr (!STATE) {
            f32x16 z, o;
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = o[r] = 0.0f;
#pragma unroll
            for (int s = 0; s < 4 * KT; ++s) {
                const f32x4 q = lds_read<f32x4>((row4 + at + QK + VB) ^ (s * 32)), k = lds_read<f32x4>((row4 + at) ^ (s * 32));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z = mfma(k[e], q[e], z);
                    o = mfma(q[e], S[s >> 2][4 * (s & 3) + e], o);
                }
            }
            int apart = col - 4 * half;
            asm volatile("" : "+v"(apart));
#pragma unroll
            for (int r = 0; r < 16; ++r) o[r] *= lane_up * up[r];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = apart - acc_row(r, 0);
                o = mfma(d >= 0 ? z[r] * a.scale * power(ld2, d) : 0.0f, v[r], o);
            }
            if (on)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = acc_row(r, half);
                    if (j < n) op[(int64_t)(base + j) * a.o_row + c0 + col] = j >= bad ? NAN : o[r];
                }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = acc_row(r, half);
            v[r] *= n == C ? lane_left * up[15 - r] : j < n ? power(ld2, n - 1 - j) : 0.0f;
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            f32x16 sum;                                        // the chunk's own: the state is rounded once per chunk
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[r] = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int eight = (r >> 2) & 1;
                const uint32_t k = kcol[NC == 8 ? (r & 2) + eight : r & 3] + at + (acc_row(r, 0) * (DP * 4) + (NC == 8 ? 0 : (kt ^ eight) * 128));
                sum = mfma(lds_read<float>(k), v[r], sum);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) S[kt][r] = fmaf(S[kt][r], lam_n, sum[r]);
        }
        if (odd && bad < C)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) S[kt][r] = NAN;
    }
    float* to = nullptr;
    if (STATE) to = a.states + ((t.u + 1) * a.heads + h) * (int64_t)a.dk * a.dv;
    else if (t.last && a.state_out) to = a.state_out + ((int64_t)t.s.seg * a.heads + h) * (int64_t)a.dk * a.dv;
    if (to && on)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int d = kt * 32 + acc_row(r, 0);
                if (d < a.dk) (to + d * a.dv)[lane_s] = S[kt][r];
            }
}

// The states before each piece: a unit holds what its predecessor added, from a state of 0.  Bound by reading and writing them
// (2 x 16 pieces of 32 heads of 128 x 128: 12 us).
static __global__ __launch_bounds__(256) void linear_scan_kernel(LinearArgs a) {
    const int slot = blockIdx.x, h = blockIdx.y;
    const int64_t size = (int64_t)a.dk * a.dv, e = ((int64_t)blockIdx.z * 256 + threadIdx.x) * 4;
    if (e >= size) return;
    const SegInfo s = a.segs[slot];
    const int n = max(1, (int)(((uint32_t)s.nq + a.piece - 1) / (uint32_t)a.piece));
    const Decay decay = decay_of(a, h, a.piece);
    f32x4 S = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.state_in) S = *(const f32x4*)(a.state_in + ((int64_t)s.seg * a.heads + h) * size + e);
    float* at = a.states + ((int64_t)(s.cum / (uint32_t)a.piece + slot) * a.heads + h) * size + e;
    const int64_t next = a.heads * size;
    *(f32x4*)at = S;
    constexpr int U = 8;                                       // pieces in flight
    for (int k = 1; k < n; k += U) {
        f32x4 add[U];
#pragma unroll
        for (int u = 0; u < U; ++u) add[u] = *(const f32x4*)(at + next * (min(k + u, n - 1) - k + 1));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + u >= n) break;
            at += next;
#pragma unroll
            for (int c = 0; c < 4; ++c) S[c] = decay(S[c]) + add[u][c];
            *(f32x4*)at = S;
        }
    }
}

}  // namespace seq
