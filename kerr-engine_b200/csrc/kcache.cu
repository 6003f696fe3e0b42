// The 8-bit paged cache (include/kerr_attn.h, kattn_cache_append / _read):
// each row of d values of one key head is held as codes with one f32 scale.
//
//   m = max |x|;  scale = fl(m / L);  code = rn(x * fl(L / m));  value = code * scale
//
// The product is rounded once, straight to the code: for int8 by an FMA onto
// 1.5 * 2^23, whose last place is one; for e4m3 the f32 product is rounded to
// odd first (truncated, its last bit set when anything was cut off), and the
// rounding of such a number to four significant bits is that of the exact one.
//
// Both directions only move bytes.  A block takes a few tokens (their sequences and
// pages are looked up once, by one thread each) and streams their heads: a
// lane holds 16 bytes of a row, d / 4 or d / 8 lanes a row, k and v together.
#include "kserve.cuh"

namespace kattn {

namespace {

using namespace serve;

constexpr int kThreads = 256;
constexpr int kMaxTokens = 32;  // tokens of a block at most

// Looks up tokens t0 .. t0+n-1 into shared memory: whether a sequence owns the
// row, and the cache row of its key head 0, (page * n_kv_head) * page_size +
// place, or -1 where there is no such row or position.
__device__ __forceinline__ void find_places(const CacheArgs& a, int page_shift, int t0, int n, long* place, bool* owned) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int r = t0 + i;
        long at = -1;
        bool mine = false;
        if (r < a.N) {
            const int s = seq_of_row(a.cu, a.S, r);
            if (s >= 0) {
                const int2 rows = seq_rows(a.cu, s, a.N);
                if (r < rows.y) {
                    mine = true;
                    const int p = max(__ldg(a.kv_len + s), 0) - (rows.y - r);
                    const int page = page_of(a, page_shift, s, p);
                    if (page >= 0)
                        at = (static_cast<long>(page) * a.c.n_kv_head << page_shift) + (p & (a.c.page_size - 1));
                }
            }
        }
        place[i] = at;
        owned[i] = mine;
    }
    __syncthreads();
}

template <int FORMAT>
__device__ __forceinline__ uint32_t encode(float x, float inverse) {
    if constexpr (FORMAT == KATTN_CACHE_INT8) {
        // |x * inverse| <= 127 (1 + 2^-23): the sum's low byte is the code.
        return __float_as_uint(__fmaf_rn(x, inverse, 12582912.f)) & 0xFFu;
    } else {
        const float p = __fmul_rz(x, inverse);
        const float rest = __fmaf_rn(x, inverse, -p);
        const float odd = __uint_as_float(__float_as_uint(p) | (rest != 0.f ? 1u : 0u));
        uint16_t two;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.f), "f"(odd));
        return two & 0xFFu;
    }
}

template <class T, int FORMAT>
__global__ void __launch_bounds__(kThreads) cache_append_rows(CacheArgs a, const T* __restrict__ k,
                                                              const T* __restrict__ v, long ld, int page_shift,
                                                              int tokens) {
    constexpr int E = Vec16<T>::N;  // elements of a lane
    constexpr float L = FORMAT == KATTN_CACHE_INT8 ? 127.f : 448.f;
    __shared__ long place[kMaxTokens];
    __shared__ bool owned[kMaxTokens];
    pdl_enter();
    const int t0 = blockIdx.x * tokens;
    const int n = min(tokens, a.N - t0);
    find_places(a, page_shift, t0, n, place, owned);
    const int d = a.c.d, lanes = d / E, heads = a.c.n_kv_head;
    const int units = n * heads * 2 * lanes;  // a multiple of `lanes`, itself a power of two up to 32
    for (int u0 = 0; u0 < units; u0 += kThreads) {
        const int u = u0 + threadIdx.x;
        const bool in = u < units;
        const int c = u % lanes, rest = u / lanes;
        const int head = rest % heads, tk = rest / heads;
        const int token = in ? tk >> 1 : 0;
        const bool is_v = tk & 1;
        const long at = in ? place[token] : -1;
        Vec16<T> x;
        x.raw = make_uint4(0, 0, 0, 0);
        if (at >= 0)
            x.raw = __ldg(reinterpret_cast<const uint4*>((is_v ? v : k) + static_cast<long>(t0 + token) * ld +
                                                         head * d + c * E));
        float f[E], m = 0.f;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            f[i] = to_f32(x.x[i]);
            m = fmaxf(m, fabsf(f[i]));
            nan |= f[i] != f[i];
        }
        if (nan) m = __uint_as_float(0x7F800000u);  // NaN and infinity alike
        for (int o = lanes >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const bool bad = m == __uint_as_float(0x7F800000u);
        const bool usual = !bad && m >= 0x1p-100f;
        const float inverse = usual ? __fdiv_rn(L, m) : 0.f;
        uint32_t w[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            w[i] = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (usual) w[i] |= encode<FORMAT>(f[4 * i + j], inverse) << (8 * j);
        }
        if (at >= 0) {
            const long row = at + (static_cast<long>(head) << page_shift);
            uint8_t* code = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + row * d + c * E;
            if constexpr (E == 4) *reinterpret_cast<uint32_t*>(code) = w[0];
            else *reinterpret_cast<uint2*>(code) = make_uint2(w[0], w[1]);
            if (c == 0)
                (is_v ? a.c.v_scale : a.c.k_scale)[row] =
                    bad ? __uint_as_float(0x7FC00000u) : (usual ? __fdiv_rn(m, L) : 0.f);
        }
    }
}

template <class T, int FORMAT>
__global__ void __launch_bounds__(kThreads) cache_read_rows(CacheArgs a, T* __restrict__ k, T* __restrict__ v, long ld,
                                                            int page_shift, int tokens) {
    constexpr int E = Vec16<T>::N;
    __shared__ long place[kMaxTokens];
    __shared__ bool owned[kMaxTokens];
    pdl_enter();
    const int t0 = blockIdx.x * tokens;
    const int n = min(tokens, a.N - t0);
    find_places(a, page_shift, t0, n, place, owned);
    const int d = a.c.d, lanes = d / E, heads = a.c.n_kv_head;
    const int units = n * heads * 2 * lanes;
    for (int u = threadIdx.x; u < units; u += kThreads) {
        const int c = u % lanes, rest = u / lanes;
        const int head = rest % heads, tk = rest / heads;
        const int token = tk >> 1;
        const bool is_v = tk & 1;
        if (!owned[token]) continue;
        const long at = place[token];
        uint32_t w[E / 4];
#pragma unroll
        for (int i = 0; i < E / 4; ++i) w[i] = 0;
        float scale = 0.f;
        if (at >= 0) {
            const long row = at + (static_cast<long>(head) << page_shift);
            const uint8_t* code = static_cast<const uint8_t*>(is_v ? a.c.v : a.c.k) + row * d + c * E;
            if constexpr (E == 4) {
                w[0] = __ldg(reinterpret_cast<const uint32_t*>(code));
            } else {
                const uint2 t = __ldg(reinterpret_cast<const uint2*>(code));
                w[0] = t.x;
                w[1] = t.y;
            }
            scale = __ldg((is_v ? a.c.v_scale : a.c.k_scale) + row);
        }
        Vec16<T> y;
#pragma unroll
        for (int i = 0; i < E; ++i)
            y.x[i] = from_f32<T>(__fmul_rn(code_value<FORMAT>((w[i / 4] >> (8 * (i % 4))) & 0xFFu), scale));
        *reinterpret_cast<uint4*>((is_v ? v : k) + static_cast<long>(t0 + token) * ld + head * d + c * E) = y.raw;
    }
}

// Tokens of a block: as many as leave four blocks to an SM, up to kMaxTokens.
int block_tokens(int N, int num_sms) {
    int t = 1;
    while (t < kMaxTokens && N / (2 * t) >= 4 * num_sms) t *= 2;
    return t;
}

template <class T, int FORMAT>
ProjStatus launch_append(const CacheArgs& a, const void* k, const void* v, long ld, int num_sms, cudaStream_t s) {
    const int tokens = block_tokens(a.N, num_sms);
    ProjStatus st;
    st.cuda = launch_pdl(cache_append_rows<T, FORMAT>, dim3((a.N + tokens - 1) / tokens), dim3(kThreads), 0, s, a,
                         static_cast<const T*>(k), static_cast<const T*>(v), ld, page_shift_of(a.c.page_size), tokens);
    st.what = "cache append launch";
    return st;
}

template <class T, int FORMAT>
ProjStatus launch_read(const CacheArgs& a, void* k, void* v, long ld, int num_sms, cudaStream_t s) {
    const int tokens = block_tokens(a.N, num_sms);
    ProjStatus st;
    st.cuda = launch_pdl(cache_read_rows<T, FORMAT>, dim3((a.N + tokens - 1) / tokens), dim3(kThreads), 0, s, a,
                         static_cast<T*>(k), static_cast<T*>(v), ld, page_shift_of(a.c.page_size), tokens);
    st.what = "cache read launch";
    return st;
}

}  // namespace

ProjStatus cache_append(const CacheArgs& a, int dtype, const void* k, const void* v, long ld, int num_sms,
                        cudaStream_t s, int* launches) {
    const bool i8 = a.c.format == KATTN_CACHE_INT8;
    auto fn = dtype == KATTN_F32    ? (i8 ? launch_append<float, KATTN_CACHE_INT8> : launch_append<float, KATTN_CACHE_E4M3>)
              : dtype == KATTN_BF16 ? (i8 ? launch_append<__nv_bfloat16, KATTN_CACHE_INT8>
                                          : launch_append<__nv_bfloat16, KATTN_CACHE_E4M3>)
                                    : (i8 ? launch_append<__half, KATTN_CACHE_INT8> : launch_append<__half, KATTN_CACHE_E4M3>);
    const ProjStatus st = fn(a, k, v, ld, num_sms, s);
    if (st.ok()) ++*launches;
    return st;
}

ProjStatus cache_read(const CacheArgs& a, int dtype, void* k, void* v, long ld, int num_sms, cudaStream_t s,
                      int* launches) {
    const bool i8 = a.c.format == KATTN_CACHE_INT8;
    auto fn = dtype == KATTN_F32    ? (i8 ? launch_read<float, KATTN_CACHE_INT8> : launch_read<float, KATTN_CACHE_E4M3>)
              : dtype == KATTN_BF16 ? (i8 ? launch_read<__nv_bfloat16, KATTN_CACHE_INT8>
                                          : launch_read<__nv_bfloat16, KATTN_CACHE_E4M3>)
                                    : (i8 ? launch_read<__half, KATTN_CACHE_INT8> : launch_read<__half, KATTN_CACHE_E4M3>);
    const ProjStatus st = fn(a, k, v, ld, num_sms, s);
    if (st.ok()) ++*launches;
    return st;
}

}  // namespace kattn
