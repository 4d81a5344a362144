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
    int64_t cum;
    int32_t nq, nk;
    int32_t seg;          // its number in the caller's order
    int32_t pad;
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
    return x;
}

// The entry that holds unit `t` when the entries own floor(cum / per) + index .. units (a tiling of each series in
// blocks of `per` rows, at most one empty unit per series): the last s with floor(cum_s / per) + s <= t.  64-ary search,
// one load per lane and round.
__device__ __forceinline__ int find_seg(const SegInfo* segs, int n_seg, int64_t t, int per) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = n_seg;                   // answer in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64;
        const int at = lo + lane * step;
        const bool below = at < hi && segs[at].cum / per + at <= t;
        const int n = __popcll(__ballot(below));      // lane 0 is always below
        lo = lo + (n - 1) * step;
        hi = min(hi, lo + step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace seq
