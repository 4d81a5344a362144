// Softmax attention over packed series.
//
//   z_ij = scale q_i.k_j,   out_i = sum_j exp(z_ij) v_j / sum_j exp(z_ij)       over the keys j that row i sees
//
// in one pass over the keys with a running reference m (no running maximum is needed: any m works as long as
// exp(z - m) neither overflows nor loses the largest terms), weights p_j = exp(z_j - m), their sum l and the weighted
// sum o; when the maximum passes m by more than 8 (in powers of two) o and l are multiplied by the ratio and m follows.
//
// A "row" of the products is one (row of q, head) pair: the heads that share a kv head lie side by side, so its keys
// and values are read once for all of them, and a single new row per series still fills part of a tile.
#pragma once
#include "seq_common.hip.h"

#include <type_traits>

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
    // heads of one kv head are cut into `blocks` runs of `rep_b`; a tile holds `per` rows of q of one run; every other
    // `turn` units go backwards
    int kv_blocks, blocks, rep_b, per, turn;
    // the keys are cut into runs of `chunk` (splits > 1): partial results of run y, normalised, and their references (in powers of
    // two) and sums: a log-sum would be rounded to its own last place
    int splits, chunk;
    float* part_o;                 // [splits][rows][heads][dim], rows from the first series' first
    f32x2* part_ml;                // [splits][rows][heads]
    int64_t part_rows, row0;
};

// The keys [lo, hi) that row i of a series may see by position (the key mask apart).
__device__ __forceinline__ void visible(const AttnArgs& a, int i, int nq, int nk, int& lo, int& hi) {
    const int64_t end = (int64_t)i + nk - nq;             // the row's own place among the keys
    hi = a.causal ? (int)max((int64_t)0, min((int64_t)nk, end + 1)) : nk;
    lo = a.window > 0 ? (int)max((int64_t)0, min((int64_t)nk, end + 1 - a.window)) : 0;
}

// Run blockIdx.y of these keys.
__device__ __forceinline__ void run_of(const AttnArgs& a, int& lo, int& hi) {
    const int64_t from = lo + (int64_t)blockIdx.y * a.chunk;
    lo = (int)min(from, (int64_t)hi);
    hi = (int)min(from + a.chunk, (int64_t)hi);
}

__device__ __forceinline__ int keys_of(const AttnArgs& a, const SegInfo& s) {
    return a.k_len ? max(0, min(a.k_len[s.seg], s.nk)) : s.nk;
}

// Which of a tile's BK keys from `base` on are there at all: in front of `end`, and not masked.  The mask's bytes are asked
// for a tile ahead.
template <int BK, bool MASK = true>
__device__ __forceinline__ int ask_keys(const AttnArgs& a, const SegInfo& s, int base, int end) {
    if (!MASK) return 1;
    const int j = base + (threadIdx.x & (BK - 1));
    return a.key_mask && j < end ? a.key_mask[s.k0 + j] : 1;
}
template <int BK, bool MASK = true>
__device__ __forceinline__ uint64_t have_keys(int asked, int base, int end) {
    if (!MASK) return ~0ull >> (64 - min(BK, end - base));
    return __ballot(asked && base + (int)(threadIdx.x & (BK - 1)) < end) & (~0ull >> (64 - BK));
}

// float16 weights are multiplied by 2^7: the largest is 2^15 then (an exponent of 8 above the reference at most), and what
// is lost below float16's smallest, 2^-25 a key, is 2^-32 of the sum; a long flat tail behind one large score counts in full.
template <typename T>
__device__ constexpr float lift() { return __is_same(T, f16) ? 7.0f : 0.0f; }

// Beyond this the reference in powers of two, ref c1, has an error that an exponent shows: z c1 - mc is then up to half of mc's
// last place for z = ref itself, not 0, and from 2^24 on weights pass float16's range, from 2^31 on float32's.  Where a row of the
// wave is there, the reference is subtracted from the scores before the product; elsewhere a branch per tile (ragged batch
// 132.3 -> 133.9 us, the other cases 0 to 1.3 % slower).
constexpr float FAR = 0x1p20f;

// The factor for what was summed with the reference `ref` (mc), when that becomes `now` (mcn).
__device__ __forceinline__ float rescale(float ref, float mc, float now, float mcn, float c1) {
    return ref == -INFINITY ? 0.0f : exp2_fast(fabsf(mcn) > FAR ? (ref - now) * c1 : mc - mcn);
}

// Whether a row of the wave is there; mz is what is subtracted from the product with c1, of scores or of what is left of them.
__device__ __forceinline__ int far_away(float ref, float mc, float c1, float lift, float& mz) {
    const int far = __builtin_amdgcn_readfirstlane(__any(fabsf(mc) > FAR));
    mz = mc;
    if (far) mz = fabsf(mc) > FAR ? -lift : ref == -INFINITY ? 0.0f : -fmaf(ref, c1, -mc);
    return far;
}
__device__ __forceinline__ void from_reference(f32x16& z, float ref) {
    float base = ref == -INFINITY ? 0.0f : ref;
    asm volatile("" : "+v"(base));                           // this stays in its branch
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] -= base;
}

// m and l of a row to its log-sum; l = 0 where nothing was seen.
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.0f ? -INFINITY : m + LN2 * __builtin_amdgcn_logf(l); }

// A result in the inputs' type.  A mean of float16 values is inside the type's range; weights that are rounded up by up to 2^-11
// could carry one of the largest values past it, to infinity.
template <typename T>
__device__ __forceinline__ T result(float x) {
    if constexpr (__is_same(T, f16)) x = fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f) : x;
    return (T)x;
}

// One row and head by one wave, straight from the definition, over the keys [from, to): a lane per key for the scores,
// lanes over the width for the sum.  Touches nothing but the visible keys' rows.  Where a tile holds values that are
// not finite and that some of its rows must not see, its rows are computed like this.
template <typename T>
__device__ __forceinline__ void attn_row(const AttnArgs& a, const SegInfo& s, int nk, int i, int h, int from, int to, int split) {
    const int lane = threadIdx.x & 63;
    const int64_t row = s.q0 + i;
    const T* q = (const T*)a.q + row * a.q_row + (int64_t)h * a.q_head;
    const T* kb = (const T*)a.k + s.k0 * a.k_row + (int64_t)(h / a.rep) * a.k_head;
    const T* vb = (const T*)a.v + s.k0 * a.v_row + (int64_t)(h / a.rep) * a.v_head;
    int lo, hi;
    visible(a, i, s.nq, nk, lo, hi);
    lo = max(lo, from);
    hi = min(hi, to);
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
    if (top == -INFINITY) top = 0.0f;
    if (a.splits > 1) {
        const int64_t at = ((int64_t)split * a.part_rows + row - a.row0) * a.heads + h;
        float* o = a.part_o + at * a.dim;
        if (lane < a.dim) o[lane] = o0 * inv;
        if (lane + 64 < a.dim) o[lane + 64] = o1 * inv;
        if (lane == 0) a.part_ml[at] = f32x2{top * LOG2E, sum};
        return;
    }
    T* o = (T*)a.out + row * a.o_row + (int64_t)h * a.o_head;
    if (lane < a.dim) o[lane] = result<T>(o0 * inv);
    if (lane + 64 < a.dim) o[lane + 64] = result<T>(o1 * inv);
    if (a.lse && lane == 0) a.lse[row * a.heads + h] = log_sum(top, sum);
}

// Which tile of which series a workgroup has: units of `per` rows, the longest series and the last rows (causal: the ones
// with the most keys) first.  The kv head changes fastest, so that with eight of them each XCD's L2 holds one.
struct AttnTile {
    SegInfo s;
    int nk, kv, head0, n_heads, i0, rows;     // rows: (row, head) pairs
    bool any;
};
__device__ __forceinline__ AttnTile attn_tile(const AttnArgs& a, uint32_t id) {
    AttnTile t;
    const uint32_t b = id % (uint32_t)a.kv_blocks;
    uint32_t u = id / (uint32_t)a.kv_blocks;
    if (const uint32_t turn = u / (uint32_t)a.turn; turn & 1) {
        const uint32_t first = turn * a.turn, n = min((uint32_t)a.turn, gridDim.x / (uint32_t)a.kv_blocks - first);
        u = first + n - 1 - (u - first);
    }
    const int slot = find_seg(a.segs, a.n_seg, u, a.per);
    t.s = a.segs[slot];
    t.kv = b / (uint32_t)a.blocks;
    const int first = (int)(b % (uint32_t)a.blocks) * a.rep_b;
    t.head0 = t.kv * a.rep + first;
    t.n_heads = min(a.rep_b, a.rep - first);
    const int n = (int)(((uint32_t)t.s.nq + a.per - 1) / (uint32_t)a.per);
    const int k = (int)(u - (t.s.cum / (uint32_t)a.per + slot));
    t.any = k < n && t.n_heads > 0;
    t.i0 = (n - 1 - k) * a.per;
    t.rows = t.any ? min(a.per, t.s.nq - t.i0) * t.n_heads : 0;
    t.nk = keys_of(a, t.s);
    return t;
}

// A wave's rows: o and l as they were summed, m the reference in powers of two.
template <typename T, int DT>
__device__ __forceinline__ void attn_store(const AttnArgs& a, const AttnTile& t, const f32x16 (&o)[DT], float l, float m, int i, int h, bool row_ok, int half, int first = 0) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;           // a NaN sum stays one
    if (!row_ok) return;
    const int64_t row = t.s.q0 + i;
    if (a.splits > 1) {
        const int64_t at = ((int64_t)blockIdx.y * a.part_rows + row - a.row0) * a.heads + h;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int d = (first + dt) * 32 + acc_row(r, half);
                if (d < a.dim) *(f32x4*)(a.part_o + at * a.dim + d) = f32x4{o[dt][r] * inv, o[dt][r + 1] * inv, o[dt][r + 2] * inv, o[dt][r + 3] * inv};
            }
        if (half == 0 && first == 0) a.part_ml[at] = f32x2{m, l};
        return;
    }
    T* out = (T*)a.out + row * a.o_row + (int64_t)h * a.o_head;
    struct alignas(4 * sizeof(T)) Four { T e[4]; };
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int d = (first + dt) * 32 + acc_row(r, half);
            const Four w = {{result<T>(o[dt][r] * inv), result<T>(o[dt][r + 1] * inv), result<T>(o[dt][r + 2] * inv), result<T>(o[dt][r + 3] * inv)}};
            if (d < a.dim) *(Four*)(out + d) = w;
        }
    if (a.lse && half == 0 && first == 0) a.lse[row * a.heads + h] = log_sum(m * LN2, l);
}

// 16-bit types.  A workgroup of four waves has 128 rows, a wave 32 of them; keys and values go through LDS in tiles of 64
// keys, two of them in turn (64 KiB at dim 128: two workgroups per CU, one wave of each per SIMD, so that one's softmax
// runs beside the other's products).
// Scores are computed transposed, keys x rows: a lane then holds 32 scores of ONE row, half of the tile's keys (the lane 32
// away has the others), the maximum is one exchange away, and the weights, rounded to the inputs' type (relative error
// u = eps/2 each, as the result's own rounding), are as they lie in registers the second operand of values^T x weights: the
// order of the keys inside the product is free, and the values are read with ds_read_b64_tr_b16 in the weights' order.
// Bound by issue: one series of 8,192 rows, 32 heads over 8, dim 128, bfloat16: 525-565 us by card, 0.97-1.05 PFLOP/s (one
// library product of 8,192^3: 1.17), matrix pipe 53 % busy and VALU 50 %, each waiting for the other's results.  24 ragged
// series of up to 2,048 rows, 16 heads over 4, dim 64, float16, a tenth of the keys masked: 134-143 us by card, VALU 71 %,
// matrix pipe 33 %: the exponentials and their sums are the same for half the products.
template <typename T, int DT, bool MASK>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(AttnArgs a) {
    typedef typename Vec<T>::x8 x8;
    constexpr int DP = DT <= 1 ? 32 : DT <= 2 ? 64 : 128;     // elements of a tile row in LDS
    constexpr int NC = DP / 8, KS = 2 * DT, BK = 64;
    constexpr int TILE = BK * DP * 2;                         // bytes of a tile of keys (or values)
    extern __shared__ char smem[];
    const uint32_t lds = lds_offset(smem);
    const AttnTile t = attn_tile(a, blockIdx.x);
    if (!t.any) return;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // this lane's row
    const int pr = wave * 32 + col;
    const bool row_ok = pr < t.rows;
    const int prc = row_ok ? pr : t.rows - 1;
    const int i = t.i0 + prc / t.n_heads, h = t.head0 + prc % t.n_heads;
    int lo, hi;
    visible(a, i, t.s.nq, t.nk, lo, hi);
    int LO, HI, x0, x1;      // what any row of the workgroup sees
    visible(a, t.i0, t.s.nq, t.nk, LO, x0);
    visible(a, t.i0 + (t.rows - 1) / t.n_heads, t.s.nq, t.nk, x1, HI);
    if (a.splits > 1) {
        run_of(a, LO, HI);
    }
    // what any row of the wave sees, and what all of them see: they rise with the lane
    const int wl = __builtin_amdgcn_readfirstlane(__shfl(lo, 0)), wh = __builtin_amdgcn_readfirstlane(__shfl(hi, 31));
    const int all_lo = __builtin_amdgcn_readfirstlane(__shfl(lo, 31)), all_hi = __builtin_amdgcn_readfirstlane(__shfl(hi, 0));

    x8 qf[KS];
    {
        const T* q = (const T*)a.q + (t.s.q0 + i) * a.q_row + (int64_t)h * a.q_head;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * half;
            u32x4 x = {0, 0, 0, 0};
            if (d < a.dim) x = *(const u32x4*)(q + d);
            qf[s] = __builtin_bit_cast(x8, x);
        }
    }

    const char* kp = (const char*)((const T*)a.k + t.s.k0 * a.k_row + (int64_t)t.kv * a.k_head);
    const char* vp = (const char*)((const T*)a.v + t.s.k0 * a.v_row + (int64_t)t.kv * a.v_head);
    const int64_t kr = a.k_row * 2, vr = a.v_row * 2;
    const TileLoad<BK, NC, 256, Swz<NC>> load_k(threadIdx.x, a.dim * 2, kr), load_v(threadIdx.x, a.dim * 2, vr);
    for (int b = 0; b < 4; ++b) load_k.clear(lds + b * TILE);
    auto stage = [&](int base, int buf, uint64_t there) {
        if (!there) return;
        const uint32_t at = lds + buf * 2 * TILE + wave * 1024;
        load_k.pick(kp + base * kr, there, at);
        load_v.pick(vp + base * vr, there, at + TILE);
    };

    // operand reads: keys as rows, values transposed
    uint32_t koff[KS], voff[DT][2];
#pragma unroll
    for (int s = 0; s < KS; ++s) koff[s] = lds + col * (DP * 2) + (((2 * s + half) ^ swz<NC>(col)) * 16);
    {
        const int g = (lane >> 4) & 1, i4 = lane & 15;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 8 * j + 4 * half + (i4 >> 2);
                const int c = dt * 4 + g * 2 + ((i4 & 3) >> 1);
                voff[dt][j] = lds + r * (DP * 2) + ((c ^ swz<NC>(r)) * 16) + (i4 & 1) * 8;
            }
    }

    const float c1 = a.scale * LOG2E;
    constexpr float LIFT = lift<T>();
    // Where all rows see all keys but the masked ones, whose scores are copies of a visible one's, a product with a column
    // that holds the type's lowest value for them takes them away: 16 x -65504 x 65504 for float16, -inf for bfloat16 (which
    // has the range).  A quarter of the time that choosing score by score takes (ragged batch: 140 -> 135 us, with the choice made where there is a mask at all).
    constexpr bool F16 = __is_same(T, f16);
    const bool by_product = !F16 || c1 * 6.8e10f > 1000.0f;
    float ref = -INFINITY, mc = 0.0f;        // the reference, in units of the raw score; mc = ref * c1 - LIFT, 0 while there is none
    float mz = 0.0f;
    int far = 0;
    float l0 = 0.0f, l1 = 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;

    // Keys that are not there are not loaded; a key that is stands in their places, and only what a row does not see has to
    // be kept from it.  A tile that some of a wave's rows see only in part: values that are not finite must not meet the
    // weight 0 of the others; if it holds any, the wave's rows are done one by one.
    bool strange = false;
    uint64_t coming = 0;
    int asked = 1;
    if (LO < HI) {
        coming = have_keys<BK, MASK>(ask_keys<BK, MASK>(a, t.s, LO, HI), LO, HI);
        stage(LO, 0, coming);
        asked = ask_keys<BK, MASK>(a, t.s, LO + BK, HI);
    }
    // q has arrived: no wait for it inside the loop, where it would be one for the keys to come
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
    auto tile = [&](auto which, int base) {                    // one tile, in buffer `which`: its places are constants
        constexpr int buf = decltype(which)::value;
        wait_loads();
        __syncthreads();
        const uint64_t there = coming;
        if (base + BK < HI) {
            coming = have_keys<BK, MASK>(asked, base + BK, HI);
            stage(base + BK, buf ^ 1, coming);
            asked = ask_keys<BK, MASK>(a, t.s, base + 2 * BK, HI);
        }
        if (!there || strange || base >= wh || base + BK <= wl || wave * 32 >= t.rows) return;      // nothing of it for this wave
        constexpr uint32_t kt_ = buf * 2 * TILE, vt_ = kt_ + TILE;
        const bool edge = base < all_lo || base + BK > all_hi;
        if (edge) {
            bool odd = false;
#pragma unroll
            for (int n = 0; n < TILE / 1024; ++n) odd |= not_finite<T>(lds_read<u32x4>(lds + vt_ + (n * 64 + lane) * 16));
            if (__any(odd)) { strange = true; return; }
        }

        // all reads of the first 32 keys, then a read of the others behind each product
        f32x16 z[2];
        {
            __builtin_amdgcn_s_setprio(1);
            x8 kf[2][KS];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int s = 0; s < KS; ++s) kf[kt][s] = lds_read<x8>(koff[s] + (kt_ + kt * 32 * DP * 2));
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int r = 0; r < 16; ++r) z[kt][r] = 0.0f;
#pragma unroll
                for (int s = 0; s < KS; ++s) z[kt] = mfma(kf[kt][s], qf[s], z[kt]);
            }
            sched_reads(KS);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                sched_products(1);
                sched_reads(1);
            }
            sched_products(KS);
            __builtin_amdgcn_s_setprio(0);
        }
        if (MASK && !edge && there != ~0ull >> (64 - BK) && by_product) {
            const T off = (T)(F16 ? -65504.0f : -3.3895314e38f);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                x8 drop, one;
                const T d = ((uint32_t)(there >> (32 * kt)) >> col) & 1 ? (T)0.0f : off;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    drop[e] = d;
                    one[e] = (T)(F16 ? 65504.0f : 1.0f);
                }
                z[kt] = mfma(drop, one, z[kt]);
            }
        } else if (edge || (MASK && there != ~0ull >> (64 - BK))) {
            const int from = max(lo - base, 0), to = min(hi - base, 64);
            uint64_t see = to <= from ? 0 : there & (~0ull << from) & (~0ull >> (64 - to));
            see >>= 4 * half;
            const uint32_t s0 = (uint32_t)see, s1 = (uint32_t)(see >> 32);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                z[0][r] = if_bit(s0, acc_row(r, 0), z[0][r], -INFINITY);
                z[1][r] = if_bit(s1, acc_row(r, 0), z[1][r], -INFINITY);
            }
        }
        s16x4 va[DT][2];                                       // the first values' reads, before the softmax
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 2; ++j) va[dt][j] = lds_read_tr(voff[dt][j] + vt_);
        __builtin_amdgcn_sched_barrier(0);
        const float m = pair_max(fmaxf(max16(z[0]), max16(z[1])));
        if (__any((m - ref) * c1 > 8.0f)) {
            const float now = fmaxf(m, ref);
            const float mcn = now == -INFINITY ? 0.0f : now * c1 - LIFT;
            const float f = rescale(ref, mc, now, mcn, c1);
            ref = now;
            mc = mcn;
            far = far_away(ref, mc, c1, LIFT, mz);
            l0 *= f;
            l1 *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= f;
        }
        if (far) {
            from_reference(z[0], ref);
            from_reference(z[1], ref);
        }
        x8 p[4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float w0 = exp2_fast(fmaf(z[kt][r], c1, -mz)), w1 = exp2_fast(fmaf(z[kt][r + 1], c1, -mz));
                l0 += w0;                     // the sum takes the weights as they are: the log-sum is float32
                l1 += w1;
                const int g = 2 * kt + (r >> 3);
                p[g][r & 7] = (T)w0;
                p[g][(r & 7) + 1] = (T)w1;
            }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const s16x4 v0 = s == 0 ? va[dt][0] : lds_read_tr(voff[dt][0] + (vt_ + s * 16 * DP * 2));
                const s16x4 v1 = s == 0 ? va[dt][1] : lds_read_tr(voff[dt][1] + (vt_ + s * 16 * DP * 2));
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                const s16x8 v = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
                o[dt] = mfma(__builtin_bit_cast(x8, v), p[s], o[dt]);
            }
#pragma unroll
        for (int n = 0; n < 3 * DT; ++n) {                     // a read ahead of each product
            sched_reads(2);
            sched_products(1);
        }
        sched_products(DT);
    };
    for (int base = LO; base < HI; base += 2 * BK) {
        tile(std::integral_constant<int, 0>(), base);
        if (base + BK < HI) tile(std::integral_constant<int, 1>(), base + BK);
    }
    if (strange) {
        wait_loads();
        for (int r = wave * 32; r < min(t.rows, wave * 32 + 32); ++r)
            attn_row<T>(a, t.s, t.nk, t.i0 + r / t.n_heads, t.head0 + r % t.n_heads, LO, HI, blockIdx.y);
        return;
    }

    attn_store<T, DT>(a, t, o, pair_sum(l0 + l1), mc, i, h, row_ok, half);
}

// float32.  The same on 32x32x2 products, with tiles of 32 keys: the matrix pipe is 16 times slower, and what it does takes
// most of the time.  Here a score register is at once an operand of values^T x weights, and nothing is rounded.
// 8 series of 1,000 rows of 8 heads, dim 128: 224 us, matrix pipe 74 % busy; 67 series of 1,421 rows of 8 heads, dim
// 32, windows of 50: 155 us, three tiles to a row of which two are edges, bound by how long one tile takes (matrix pipe 41 %
// busy), with 82 us of reading and writing below it.
template <int DT, bool LONG>
__global__ __launch_bounds__(256, 2) void attn_tile32_kernel(AttnArgs a) {
    constexpr int DP = DT <= 1 ? 32 : DT <= 2 ? 64 : 128, NC = DP / 4, KS = 4 * DT, BK = 32;
    constexpr int TILE = BK * DP * 4;
    extern __shared__ char smem[];
    const uint32_t lds = lds_offset(smem);
    const AttnTile t = attn_tile(a, blockIdx.x);
    if (!t.any) return;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pr = wave * 32 + col;
    const bool row_ok = pr < t.rows;
    const int prc = row_ok ? pr : t.rows - 1;
    const int i = t.i0 + prc / t.n_heads, h = t.head0 + prc % t.n_heads;
    int lo, hi, LO, HI, x0, x1;
    visible(a, i, t.s.nq, t.nk, lo, hi);
    visible(a, t.i0, t.s.nq, t.nk, LO, x0);
    visible(a, t.i0 + (t.rows - 1) / t.n_heads, t.s.nq, t.nk, x1, HI);
    if (a.splits > 1) {
        run_of(a, LO, HI);
    }
    // what any row of the wave sees, and what all of them see: they rise with the lane
    const int wl = __builtin_amdgcn_readfirstlane(__shfl(lo, 0)), wh = __builtin_amdgcn_readfirstlane(__shfl(hi, 31));
    const int all_lo = __builtin_amdgcn_readfirstlane(__shfl(lo, 31)), all_hi = __builtin_amdgcn_readfirstlane(__shfl(hi, 0));

    f32x4 qf[KS];                            // elements 8 s + 4 half .. of this lane's row
    {
        const float* q = (const float*)a.q + (t.s.q0 + i) * a.q_row + (int64_t)h * a.q_head;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 8 * s + 4 * half;
            qf[s] = d < a.dim ? *(const f32x4*)(q + d) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    const char* kp = (const char*)((const float*)a.k + t.s.k0 * a.k_row + (int64_t)t.kv * a.k_head);
    const char* vp = (const char*)((const float*)a.v + t.s.k0 * a.v_row + (int64_t)t.kv * a.v_head);
    const int64_t kr = a.k_row * 4, vr = a.v_row * 4;
    const TileLoad<BK, NC, 256, Swz32<NC>> load_k(threadIdx.x, a.dim * 4, kr), load_v(threadIdx.x, a.dim * 4, vr);
    for (int b = 0; b < 4; ++b) load_k.clear(lds + b * TILE);
    auto stage = [&](int base, int buf, uint64_t there) {
        if (!there) return;
        const uint32_t at = lds + buf * 2 * TILE + wave * 1024;
        load_k.pick(kp + base * kr, there, at);
        load_v.pick(vp + base * vr, there, at + TILE);
    };
    // Operand reads: 32 s bytes on in a row of keys is an exclusive or, since tiles begin at whole rows; in a column of values
    // the lane's part of the place takes four forms, and the rest is constant.
    const uint32_t koff = lds + col * (DP * 4) + ((half ^ swz32<NC>(col)) * 16);
    uint32_t voff[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int j = NC == 8 ? (n >> 1) * 2 + (n & 1) * 8 : n;
        voff[n] = lds + TILE + 4 * half * (DP * 4) + (((col >> 2) ^ swz32<NC>(j + 4 * half)) * 16) + (col & 3) * 4;
    }
    auto value = [&](int r, int d, uint32_t at) {              // this lane's element of part d of the value in register r's place
        const int eight = (r >> 2) & 1;
        return lds_read<float>(voff[NC == 8 ? (r & 2) + eight : r & 3] + at + (acc_row(r, 0) * (DP * 4) + (NC == 8 ? 0 : (d ^ eight) * 128)));
    };
    const float c1 = a.scale * LOG2E;
    float ref = -INFINITY, mc = 0.0f, l = 0.0f;
    float mz = 0.0f;
    int far = 0;
    constexpr int ASIDE = DT > 2 || !LONG ? 0 : DT;
    f32x16 o[DT], aside[ASIDE + 1];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            o[dt][r] = 0.0f;
            if (dt < ASIDE) aside[dt][r] = 0.0f;
        }
    int tiles = 0;

    // Keys that are not there are not loaded; a key that is stands in their places, and only what a row does not see has to
    // be kept from it.  A tile that some of a wave's rows see only in part: values that are not finite must not meet the
    // weight 0 of the others; if it holds any, the wave's rows are done one by one.
    bool strange = false;
    uint64_t coming = 0;
    int asked = 1;
    if (LO < HI) {
        coming = have_keys<BK>(ask_keys<BK>(a, t.s, LO, HI), LO, HI);
        stage(LO, 0, coming);
        asked = ask_keys<BK>(a, t.s, LO + BK, HI);
    }
    // q has arrived: no wait for it inside the loop, where it would be one for the keys to come
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
    int buf = 0;
    for (int base = LO; base < HI; base += BK, buf ^= 1) {
        wait_loads();
        __syncthreads();
        const uint64_t there = coming;
        if (base + BK < HI) {
            coming = have_keys<BK>(asked, base + BK, HI);
            stage(base + BK, buf ^ 1, coming);
            asked = ask_keys<BK>(a, t.s, base + 2 * BK, HI);
        }
        if (!there || strange || base >= wh || base + BK <= wl || wave * 32 >= t.rows) continue;      // nothing of it for this wave
        const uint32_t at = buf * 2 * TILE;
        const bool edge = base < all_lo || base + BK > all_hi;
        if (edge) {
            bool odd = false;
#pragma unroll
            for (int n = 0; n < TILE / 1024; ++n) odd |= not_finite<float>(lds_read<u32x4>(lds + at + TILE + (n * 64 + lane) * 16));
            if (__any(odd)) { strange = true; continue; }
        }

        f32x16 z;
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const f32x4 k = lds_read<f32x4>((koff + at) ^ (s * 32));
#pragma unroll
            for (int e = 0; e < 4; ++e) z = mfma(k[e], qf[s][e], z);
        }
        sched_reads(2);
#pragma unroll
        for (int s = 0; s < KS - 2; ++s) {
            sched_products(4);
            sched_reads(1);
        }
        sched_products(8);
        if (edge || there != ~0ull >> (64 - BK)) {
            const int from = max(lo - base, 0), to = min(hi - base, 32);
            const uint32_t see = (to <= from ? 0 : (uint32_t)there & (~0u << from) & (~0u >> (32 - to))) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = if_bit(see, acc_row(r, 0), z[r], -INFINITY);
        }
        const float m = pair_max(max16(z));
        if (__any((m - ref) * c1 > 8.0f)) {
            const float now = fmaxf(m, ref);
            const float mcn = now == -INFINITY ? 0.0f : now * c1;
            const float f = rescale(ref, mc, now, mcn, c1);
            ref = now;
            mc = mcn;
            far = far_away(ref, mc, c1, 0.0f, mz);
            l *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    o[dt][r] *= f;
                    if (dt < ASIDE) aside[dt][r] *= f;
                }
        }
        if (far) from_reference(z, ref);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            z[r] = exp2_fast(fmaf(z[r], c1, -mz));
            l += z[r];
        }
        // Short chains of sums: added to the running sum, each key would be rounded to its last place (the last of 16,000 rows:
        // 1.7e-6 off, 6.6e-7 like this).  Wide rows sum each tile's products by themselves, two parts of the width at a time;
        // narrow ones, where that would be waited for, put the sum aside now and then if there are more than 1,024 keys, and
        // else not, for the registers (windows of 50 at dim 32: 171 us with, 155 without).
        if constexpr (DT > 2) {
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += 2) {
                f32x16 sum[2];
#pragma unroll
                for (int d = 0; d < 2; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[d][r] = 0.0f;
#pragma unroll
                for (int r = 0; r < 16; ++r)
#pragma unroll
                    for (int d = 0; d < 2; ++d)
                        if (d0 + d < DT) sum[d] = mfma(value(r, d0 + d, at), z[r], sum[d]);
#pragma unroll
                for (int d = 0; d < 2; ++d)
                    if (d0 + d < DT)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d0 + d][r] += sum[d][r];
            }
        } else {
            if (LONG && ++tiles % 16 == 0) {
#pragma unroll
                for (int d = 0; d < ASIDE; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        aside[d][r] += o[d][r];
                        o[d][r] = 0.0f;
                    }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] = mfma(value(r, d, at), z[r], o[d]);
        }
        sched_reads(4);                                        // reads four products ahead
#pragma unroll
        for (int n = 0; n < 16 * DT - 4; ++n) {
            sched_products(1);
            sched_reads(1);
        }
        sched_products(4);
    }
    if (strange) {
        wait_loads();
        for (int r = wave * 32; r < min(t.rows, wave * 32 + 32); ++r)
            attn_row<float>(a, t.s, t.nk, t.i0 + r / t.n_heads, t.head0 + r % t.n_heads, LO, HI, blockIdx.y);
        return;
    }
#pragma unroll
    for (int dt = 0; dt < ASIDE; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] += aside[dt][r];
    attn_store<float, DT>(a, t, o, pair_sum(l), mc, i, h, row_ok, half);
}

// At most 32 rows per kv head (steps).  Reading the cache is what takes the time: every wave has tiles of 32 keys of its
// own, every NW-th, in two LDS buffers of its own, and waits for nothing but its own loads (with a key mask, whose bytes are
// asked for last, for those of the tile to come as well); at the end the waves' sums are joined through LDS.  With 16-bit
// types, what the weights lose by rounding goes into a second product: it is free here. 16 caches of up to 32,768 rows, 8 kv
// heads, dim 128, bfloat16: 256 us, 4.9 TB/s (a copy: 4.7), with a mask 288; 4 of up to 384: 8.6 us in a graph, of which the
// shortest launch is 5.4.  In float32 the products bound it, of 32 rows where 4 are there: 16 caches of up to 16,384 rows,
// 790 us, 1.9 TB/s.
template <typename T, int DT, int NW>
__global__ __launch_bounds__(NW * 64) void attn_step_kernel(AttnArgs a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int E = 16 / sizeof(T);                          // elements of a chunk
    constexpr int DP = DT <= 1 ? 32 : DT <= 2 ? 64 : 128, NC = DP / E, KS = F32 ? 4 * DT : 2 * DT, BK = 32;
    constexpr int ROW = DP * sizeof(T), TILE = BK * ROW, LOADS = BK * NC / 64;
    extern __shared__ char smem[];
    const uint32_t lds = lds_offset(smem);
    const AttnTile t = attn_tile(a, blockIdx.x);
    if (!t.any) return;
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool row_ok = col < t.rows;
    const int prc = row_ok ? col : t.rows - 1;
    const int i = t.i0 + prc / t.n_heads, h = t.head0 + prc % t.n_heads;
    int lo, hi, LO, HI, all_lo, all_hi;
    visible(a, i, t.s.nq, t.nk, lo, hi);
    visible(a, t.i0, t.s.nq, t.nk, LO, all_hi);
    visible(a, t.i0 + (t.rows - 1) / t.n_heads, t.s.nq, t.nk, all_lo, HI);
    if (a.splits > 1) {
        run_of(a, LO, HI);
    }
    auto sw = [](int r) { return F32 ? swz32<NC>(r) : swz<NC>(r); };

    u32x4 qf[KS];
    {
        const T* q = (const T*)a.q + (t.s.q0 + i) * a.q_row + (int64_t)h * a.q_head;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = E * (2 * s + half);
            qf[s] = d < a.dim ? *(const u32x4*)(q + d) : u32x4{0, 0, 0, 0};
        }
    }
    const char* kp = (const char*)((const T*)a.k + t.s.k0 * a.k_row + (int64_t)t.kv * a.k_head);
    const char* vp = (const char*)((const T*)a.v + t.s.k0 * a.v_row + (int64_t)t.kv * a.v_head);
    const int64_t kr = a.k_row * sizeof(T), vr = a.v_row * sizeof(T);
    const uint32_t mine = lds + wave * 4 * TILE;
    const TileLoad<BK, NC, 64, std::conditional_t<F32, Swz32<NC>, Swz<NC>>> load_k(lane, a.dim * sizeof(T), kr), load_v(lane, a.dim * sizeof(T), vr);
    for (int b = 0; b < 4; ++b) load_k.clear(mine + b * TILE);
    auto stage = [&](int base, int buf, uint64_t there) {
        if (!there) return;
        const uint32_t at = mine + buf * 2 * TILE;
        load_k.pick(kp + base * kr, there, at);
        load_v.pick(vp + base * vr, there, at + TILE);
    };
    const float c1 = a.scale * LOG2E;
    constexpr float LIFT = lift<T>();
    float ref = -INFINITY, mc = 0.0f, l = 0.0f;
    float mz = 0.0f;
    int far = 0;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
    int odd = 0;
    const int first = LO + wave * BK, stride = NW * BK;
    auto keys = [&](int base) { return base < HI ? have_keys<BK>(ask_keys<BK>(a, t.s, base, HI), base, HI) : 0; };
    uint64_t there = keys(first), coming = keys(first + stride);
    stage(first, 0, there);
    stage(first + stride, 1, coming);
    // q has arrived: no wait for it inside the loop, where it would be one for the keys to come
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
    int buf = 0;
    for (int base = first; base < HI; base += stride, buf ^= 1) {
        // this tile's loads, not the next one's
        if (coming) wait_loads_but<2 * LOADS>();
        else wait_loads();
        const uint32_t kt_ = mine + buf * 2 * TILE, vt_ = kt_ + TILE;
        const bool edge = base < all_lo || base + BK > all_hi;
        if (edge && there)
#pragma unroll
            for (int n = 0; n < LOADS; ++n) odd |= not_finite<T>(lds_read<u32x4>(vt_ + (n * 64 + lane) * 16));
        if (there) {
        f32x16 z;
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const u32x4 k = lds_read<u32x4>(kt_ + col * ROW + (((2 * s + half) ^ sw(col)) * 16));
            if constexpr (F32) {
                const f32x4 kf = __builtin_bit_cast(f32x4, k), q = __builtin_bit_cast(f32x4, qf[s]);
#pragma unroll
                for (int e = 0; e < 4; ++e) z = mfma(kf[e], q[e], z);
            } else z = mfma(__builtin_bit_cast(typename Vec<T>::x8, k), __builtin_bit_cast(typename Vec<T>::x8, qf[s]), z);
        }
        if (edge || there != 0xffffffffu) {
            const int from = max(lo - base, 0), to = min(hi - base, 32);
            const uint32_t see = (to <= from ? 0 : (uint32_t)there & (~0u << from) & (~0u >> (32 - to))) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = if_bit(see, acc_row(r, 0), z[r], -INFINITY);
        }
        const float m = pair_max(max16(z));
        if (__any((m - ref) * c1 > 8.0f)) {
            const float now = fmaxf(m, ref);
            const float mcn = now == -INFINITY ? 0.0f : now * c1 - LIFT;
            const float f = rescale(ref, mc, now, mcn, c1);
            ref = now;
            mc = mcn;
            far = far_away(ref, mc, c1, LIFT, mz);
            l *= f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= f;
        }
        if (far) from_reference(z, ref);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            z[r] = exp2_fast(fmaf(z[r], c1, -mz));
            l += z[r];
        }
        if constexpr (F32) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = acc_row(r, half);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    o[dt] = mfma(lds_read<float>(vt_ + row * ROW + (((dt * 8 + (col >> 2)) ^ sw(row)) * 16) + (col & 3) * 4), z[r], o[dt]);
            }
        } else {
            typedef typename Vec<T>::x8 x8;
            typedef short s16x8 __attribute__((ext_vector_type(8)));
            const int g = (lane >> 4) & 1, i4 = lane & 15;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                x8 p, p2;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = (T)z[8 * s + e];
                    p2[e] = (T)(z[8 * s + e] - (float)p[e]);
                }
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    s16x4 v[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int r = 8 * j + 4 * half + (i4 >> 2), c = dt * 4 + g * 2 + ((i4 & 3) >> 1);
                        v[j] = lds_read_tr(vt_ + (16 * s + r) * ROW + ((c ^ sw(r)) * 16) + (i4 & 1) * 8);
                    }
                    const x8 vv = __builtin_bit_cast(x8, (s16x8)__builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    o[dt] = mfma(vv, p, o[dt]);
                    o[dt] = mfma(vv, p2, o[dt]);
                }
            }
        }
        }
        // the tile is read: its place may be loaded again
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        there = coming;
        coming = keys(base + 2 * stride);
        stage(base + 2 * stride, buf, coming);
    }
    l = pair_sum(l);
    if (__syncthreads_or(odd)) {
        for (int r = wave; r < t.rows; r += NW)
            attn_row<T>(a, t.s, t.nk, t.i0 + r / t.n_heads, t.head0 + r % t.n_heads, LO, HI, blockIdx.y);
        return;
    }

    // sums of the waves, in units of 2^(m_w - M); a wave takes a 32-wide part of the result (two, where they are fewer)
    float* all = (float*)smem;                               // [NW][DT][16][64], then m and l [NW][2][32]
    float* ml = all + NW * DT * 1024;
    const float m = ref == -INFINITY ? -INFINITY : mc;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) all[((wave * DT + dt) * 16 + r) * 64 + lane] = o[dt][r];
    if (half == 0) {
        ml[wave * 64 + col] = m;
        ml[wave * 64 + 32 + col] = l;
    }
    __syncthreads();
    float M = -INFINITY, f[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w * 64 + col]);
    const float MM = M == -INFINITY ? 0.0f : M;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        f[w] = exp2_fast(ml[w * 64 + col] - MM);
        l = fmaf(f[w], ml[w * 64 + 32 + col], l);
    }
    for (int dt = wave; dt < DT; dt += NW) {
        f32x16 x[1];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            x[0][r] = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) x[0][r] = fmaf(f[w], all[((w * DT + dt) * 16 + r) * 64 + lane], x[0][r]);
        }
        attn_store<T, 1>(a, t, x, l, MM, i, h, row_ok, half, dt);
    }
}

// Joins the runs of keys of a row and head: weights l_y 2^(m_y - max), one wave each.  A run in which nothing is seen (l = 0)
// weighs nothing and its partial result is not read.  5 us for 16 rows of 32 heads: latency.
template <typename T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= a.part_rows * a.heads) return;
    const int lane = threadIdx.x & 63;
    const int64_t stride = a.part_rows * a.heads;
    float m = -INFINITY;
    for (int y = lane; y < a.splits; y += 64) {
        const f32x2 x = a.part_ml[y * stride + id];
        if (x[1] != 0.0f) m = fmaxf(m, x[0]);
    }
    m = wave_max(m);
    const float mm = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int y0 = 0; y0 < a.splits; y0 += 64) {
        const f32x2 x = y0 + lane < a.splits ? a.part_ml[(y0 + lane) * stride + id] : f32x2{0.0f, 0.0f};
        const float w = x[1] == 0.0f ? 0.0f : x[1] * exp2_fast(x[0] - mm);        // a NaN sum stays one
        l += w;
        uint64_t todo = __ballot(x[1] != 0.0f);
        while (todo) {
            int y[4];
            float wy[4], p0[4], p1[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {                    // four loads in flight; the last run again where there are fewer
                y[n] = todo ? __ffsll((unsigned long long)todo) - 1 : y[n ? n - 1 : 0];
                wy[n] = todo ? __shfl(w, y[n]) : 0.0f;
                todo &= todo - 1;
                const float* o = a.part_o + ((y0 + y[n]) * stride + id) * a.dim;
                p0[n] = lane < a.dim ? o[lane] : 0.0f;
                p1[n] = lane + 64 < a.dim ? o[lane + 64] : 0.0f;
            }
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (wy[n] != 0.0f || n == 0) {
                    o0 = fmaf(wy[n], p0[n], o0);
                    o1 = fmaf(wy[n], p1[n], o1);
                }
        }
    }
    l = wave_sum(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t row = a.row0 + id / a.heads;
    const int h = (int)(id % a.heads);
    T* out = (T*)a.out + row * a.o_row + (int64_t)h * a.o_head;
    if (lane < a.dim) out[lane] = result<T>(o0 * inv);
    if (lane + 64 < a.dim) out[lane + 64] = result<T>(o1 * inv);
    if (a.lse && lane == 0) a.lse[row * a.heads + h] = log_sum(mm * LN2, l);
}

}  // namespace seq
