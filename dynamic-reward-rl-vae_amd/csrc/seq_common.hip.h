// What the kernels of the sequence operators share: element types, the layout's tables, small reductions.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace seq {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T> struct Vec;
template <> struct Vec<bf16> { typedef bf16 x8 __attribute__((ext_vector_type(8))); typedef bf16 x4 __attribute__((ext_vector_type(4))); typedef bf16 x2 __attribute__((ext_vector_type(2))); };
template <> struct Vec<f16> { typedef f16 x8 __attribute__((ext_vector_type(8))); typedef f16 x4 __attribute__((ext_vector_type(4))); typedef f16 x2 __attribute__((ext_vector_type(2))); };

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// One series of a layout, in device memory.  The entries are sorted by falling row count, so that the longest series
// are started first; `cum` counts the q rows of the entries before this one, and one more entry behind the last holds
// the total.
struct SegInfo {
    int64_t q0, k0;       // first row in q / k
    uint32_t cum;
    int32_t nq, nk;
    int32_t seg;          // its number in the caller's order
};

// A value that is the same in all lanes, into a scalar register.
__device__ __forceinline__ float uniform(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); }

// What depends on x behind this stays in its branch; the compiler does without the branch otherwise, on every pass.
__device__ __forceinline__ void rarely(int& x) { asm volatile("" : "+v"(x)); }

// Lanes are joined without LDS: what lane l ^ M holds, where the lanes of each M hold the same (so that for 4 and 8 the
// mirrored half row and row will do); 4 to 8 cycles each, where a shuffle through LDS takes a hundred.
template <int M>
__device__ __forceinline__ float other(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    if constexpr (M < 16) {
        constexpr int CTRL = M == 1 ? 0xb1 : M == 2 ? 0x4e : M == 4 ? 0x141 : 0x140;      // quad_perm 1,0,3,2 and 2,3,0,1; mirrors
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, (int)u, CTRL, 0xf, 0xf, true));
    } else {
        const auto r = M == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false) : __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return __builtin_bit_cast(float, (uint32_t)((threadIdx.x & M) ? r[0] : r[1]));
    }
}
// The larger / the sum of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float pair_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, other<1>(x));
    x = fmaxf(x, other<2>(x));
    x = fmaxf(x, other<4>(x));
    x = fmaxf(x, other<8>(x));
    x = fmaxf(x, other<16>(x));
    return pair_max(x);
}
// Over groups of `lanes` lanes, a power of two and the same in the whole wave.
__device__ __forceinline__ float lanes_sum(float x, int lanes) {
    if (lanes > 1) x += other<1>(x);
    if (lanes > 2) x += other<2>(x);
    if (lanes > 4) x += other<4>(x);
    if (lanes > 8) x += other<8>(x);
    if (lanes > 16) x += other<16>(x);
    if (lanes > 32) x = pair_sum(x);
    return x;
}
__device__ __forceinline__ float wave_sum(float x) { return lanes_sum(x, 64); }

// The entry that holds unit `t` when the entries own floor(cum / per) + index .. units (a tiling of each series in
// blocks of `per` rows, at most one empty unit per series): the last s with floor(cum_s / per) + s <= t.  Four entries per
// lane and round: one round of loads up to 256 series.
__device__ __forceinline__ int find_seg(const SegInfo* segs, int n_seg, uint32_t t, uint32_t per) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n_seg;                   // answer in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 255) / 256;
        int below = 0;
        uint32_t cum[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) cum[k] = segs[min(lo + (lane + 64 * k) * step, hi - 1)].cum;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = lo + (lane + 64 * k) * step;
            below += __popcll(__ballot(at < hi && cum[k] / per + at <= t));
        }
        lo = lo + (below - 1) * step;         // the first of them is always below
        hi = min(hi, lo + step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// ---- tiles in LDS ------------------------------------------------------------------------------------------------
// A tile row holds NC chunks of 16 bytes; chunk c of row r lies at place c ^ swz<NC>(r).  With it neither the reads of one
// chunk of 16 consecutive rows (ds_read_b128, an MFMA operand's rows) nor the transposing reads of four consecutive
// rows by 64 bytes (ds_read_b64_tr_b16) meet on a bank: LDS has 64 banks of 4 bytes, so 256 bytes go at once.
// Reads of 8 bytes of 32 rows (linear attention's, in the order of its accumulators) do: rows 16 apart lie alike.
template <int NC>
__device__ __forceinline__ int swz(int r) {
    if constexpr (NC == 4) return (r >> 2) & 3;
    else if constexpr (NC == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return ((r & 3) << 2) | ((r >> 2) & 3);
}

// The same for float32, chunks of 4: reads of one chunk of 16 consecutive rows.
template <int NC>
__device__ __forceinline__ int swz32(int r) {
    if constexpr (NC == 8) return (r >> 1) & 7;
    else return r & 15;
}

typedef __attribute__((address_space(3))) char lds_char;
__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(lds_char*)p; }

// 16 bytes per lane from global memory, `base` (the same for the whole wave) + `offset` bytes, into LDS at `lds` + 16 * lane
// (the same `lds` for the whole wave), without registers between.  Nothing waits for it by itself: wait_loads() does,
// then a barrier shows it to the other waves.  (m0 is written: nothing else in these kernels uses it, and the compiler
// sets it before uses of its own.)
__device__ __forceinline__ void load_lds16(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}

// A tile of ROWS rows of NC 16-byte chunks on its way into LDS, THREADS threads at it: where each of a thread's loads comes
// from and goes to.  Chunks behind the rows' width are not loaded: their places are cleared once, with clear().
// SW::at(row) is where a row's chunks are moved.  Row strides are below 2^26 bytes.
template <int ROWS, int NC, int THREADS, typename SW>
struct TileLoad {
    static constexpr int LOADS = (ROWS * NC + THREADS - 1) / THREADS;
    uint32_t offset[LOADS];
    int width, stride;            // bytes
    int first;                    // this thread's number among those at the tile
    __device__ __forceinline__ int row(int n) const { return (n * THREADS + first) / NC; }
    __device__ __forceinline__ int chunk(int n) const { return (((n * THREADS + first) % NC) ^ SW::at(row(n))) * 16; }
    __device__ __forceinline__ bool has(int n) const { return ROWS * NC % THREADS == 0 || n * THREADS + first < ROWS * NC; }
    __device__ __forceinline__ TileLoad(int first_, int width_, int64_t stride_) : width(width_), stride((int)stride_), first(first_) {
#pragma unroll
        for (int n = 0; n < LOADS; ++n) offset[n] = (uint32_t)row(n) * (uint32_t)stride + chunk(n);
    }
    __device__ __forceinline__ void clear(uint32_t tile) const {
        if (width < NC * 16)
#pragma unroll
            for (int n = 0; n < LOADS; ++n)
                if (has(n) && chunk(n) >= width) *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(tile + (n * THREADS + first) * 16) = u32x4{0, 0, 0, 0};
    }
    // The rows from `base` on, of which there are `rows`: behind them the last one again.  `tile`: where the wave's first
    // lane writes.
    __device__ __forceinline__ void operator()(const void* base, int rows, uint32_t tile) const {
        if (rows >= ROWS && width == NC * 16) {
#pragma unroll
            for (int n = 0; n < LOADS; ++n)
                if (has(n)) load_lds16(base, offset[n], tile + n * THREADS * 16);
        } else {
#pragma unroll
            for (int n = 0; n < LOADS; ++n)
                if (has(n) && chunk(n) < width) load_lds16(base, (uint32_t)min(row(n), rows - 1) * (uint32_t)stride + chunk(n), tile + n * THREADS * 16);
        }
    }
    // The rows whose bit is set in `there` (one at least); in the others' places the first of these.
    __device__ __forceinline__ void pick(const void* base, uint64_t there, uint32_t tile) const {
        constexpr uint64_t ALL = ~0ull >> (64 - ROWS);
        if (there == ALL && width == NC * 16) {
#pragma unroll
            for (int n = 0; n < LOADS; ++n)
                if (has(n)) load_lds16(base, offset[n], tile + n * THREADS * 16);
        } else {
            const uint32_t lo = (uint32_t)there, hi = (uint32_t)(there >> 32), instead = __builtin_ctzll(there) * (uint32_t)stride;
#pragma unroll
            for (int n = 0; n < LOADS; ++n) {
                constexpr int STEP = THREADS / NC;             // rows that go at once
                const uint32_t word = ROWS <= 32 ? lo : STEP <= 32 ? (n * STEP < 32 ? lo : hi) : row(n) < 32 ? lo : hi;
                const uint32_t off = (word >> (row(n) & 31)) & 1 ? offset[n] : instead + chunk(n);
                if (has(n) && chunk(n) < width) load_lds16(base, off, tile + n * THREADS * 16);
            }
        }
    }
};
template <int NC> struct Swz { static __device__ __forceinline__ int at(int r) { return swz<NC>(r); } };
template <int NC> struct Swz32 { static __device__ __forceinline__ int at(int r) { return swz32<NC>(r); } };

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// All but the last N loads.
template <int N>
__device__ __forceinline__ void wait_loads_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Whether 16 (or 32) bytes hold an infinity or NaN: the largest exponent of all.
template <typename T, typename... X>
__device__ __forceinline__ bool not_finite(X... x) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    if constexpr (sizeof(T) == 4) {
        uint32_t top = 0;
        ((top = max(max(top, x[0] & 0x7fffffffu), max(x[1] & 0x7fffffffu, max(x[2] & 0x7fffffffu, x[3] & 0x7fffffffu)))), ...);
        return top >= 0x7f800000u;
    } else {
        constexpr unsigned short E = __is_same(T, bf16) ? 0x7f80 : 0x7c00;
        u16x2 top = {0, 0};
        auto one = [&](uint32_t w) { top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w & 0x7fff7fffu)); };
        ((one(x[0]), one(x[1]), one(x[2]), one(x[3])), ...);
        return max(top[0], top[1]) >= E;
    }
}

template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) { return *(const __attribute__((address_space(3))) V*)(uintptr_t)at; }
template <typename V>
__device__ __forceinline__ void lds_write(uint32_t at, V x) { *(__attribute__((address_space(3))) V*)(uintptr_t)at = x; }

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Lane i of a group of 16 names 8 bytes: row i / 4 of four, columns 4 (i % 4) ..; it gets column i of the four rows.
__device__ __forceinline__ s16x4 lds_read_tr(uint32_t at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)at);
}

// x y, and 0 where one of them is 0, whatever the other holds (v_mul_legacy_f32).
extern "C" __device__ float drl_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float mul_legacy(float x, float y) { return drl_mul_legacy(x, y); }

// The largest of a product's 16 results.  Assembly, because the compiler quietens each NaN first and
// takes three times the instructions; it waits for the products itself (19 states are the most that any needs).
__device__ __forceinline__ float max16(const f32x16& x) {
    float m, n;
    asm("s_nop 15\n\ts_nop 3\n\t"
        "v_max3_f32 %0, %2, %3, %4\n\tv_max3_f32 %1, %5, %6, %7\n\t"
        "v_max3_f32 %0, %0, %8, %9\n\tv_max3_f32 %1, %1, %10, %11\n\t"
        "v_max3_f32 %0, %0, %12, %13\n\tv_max3_f32 %1, %1, %14, %15\n\t"
        "v_max3_f32 %0, %0, %16, %17\n\tv_max_f32 %0, %0, %1"
        : "=&v"(m), "=&v"(n)
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(x[4]), "v"(x[5]), "v"(x[6]), "v"(x[7]), "v"(x[8]), "v"(x[9]), "v"(x[10]),
          "v"(x[11]), "v"(x[12]), "v"(x[13]), "v"(x[14]), "v"(x[15]));
    return m;
}

// x where bit n of `bits` is set, else y: two instructions, and no lane mask between.
__device__ __forceinline__ float if_bit(uint32_t bits, int n, float x, float y) {
    const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)bits, n, 1);
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & m) | (__builtin_bit_cast(uint32_t, y) & ~m));
}

// The next so many LDS reads (matrix products) in this order.
#define sched_reads(n) __builtin_amdgcn_sched_group_barrier(0x100, n, 0)
#define sched_products(n) __builtin_amdgcn_sched_group_barrier(0x008, n, 0)

// LDS reads stay on their side of this; everything else may be moved across.
__device__ __forceinline__ void keep_reads() { __builtin_amdgcn_sched_barrier(0x67f); }

// 32x32x16 product: lane l holds row (column) l & 31 of A (B), elements 8 (l >> 5) .. + 7 of the inner axis; of the result
// column l & 31, rows (r & 3) + 8 (r >> 2) + 4 (l >> 5) in registers r = 0 .. 15.
__device__ __forceinline__ f32x16 mfma(Vec<bf16>::x8 a, Vec<bf16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(Vec<f16>::x8 a, Vec<f16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
// 32x32x2 product: one element of the inner axis per lane half.
__device__ __forceinline__ f32x16 mfma(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ int acc_row(int r, int half) { return (r & 3) + 8 * (r >> 2) + 4 * half; }

}  // namespace seq
