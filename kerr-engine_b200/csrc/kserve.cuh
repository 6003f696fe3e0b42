// Device helpers shared by the serving kernels (packed prompts, paged cache,
// attention over it): element types, rows of packed sequences, cache places.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kattn_common.cuh"
#include "kattn_launch.h"

namespace kattn {
namespace serve {

template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// 16 bytes of T.
template <class T>
struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    union {
        uint4 raw;
        T x[N];
    };
    __device__ __forceinline__ Vec16() {}
};

// Sequence s's rows [x, y) of N packed ones; an offset outside 0 .. N, or a
// descending pair, is brought inside (the arrays are never left).
__device__ __forceinline__ int2 seq_rows(const int* cu, int s, int N) {
    const int lo = min(max(__ldg(cu + s), 0), N);
    return make_int2(lo, max(lo, min(__ldg(cu + s + 1), N)));
}

// The sequence that owns row r: the last s < S with cu[s] <= r, or -1 for a
// row before the first; the caller checks r against the sequence's end.
__device__ __forceinline__ int seq_of_row(const int* cu, int S, int r) {
    int lo = 0, hi = S;  // cu[s] <= r for all s < lo
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(cu + mid) <= r) lo = mid + 1;
        else hi = mid;
    }
    return lo - 1;
}

// The page of position p, or -1 where the position does not exist.
__device__ __forceinline__ int page_of(const CacheArgs& a, int page_shift, int s, int p) {
    const int i = p >> page_shift;
    if (p < 0 || i >= a.max_pages) return -1;
    const int page = __ldg(a.table + s * a.ld_table + i);
    return page >= 0 && page < a.c.n_pages ? page : -1;
}

__host__ __device__ inline int page_shift_of(int page_size) {
    int s = 0;
    while ((1 << s) < page_size) ++s;
    return s;
}

}  // namespace serve
}  // namespace kattn
