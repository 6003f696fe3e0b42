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
// Both directions move bytes, and are bound by the memory's rate once a row costs few
// instructions: magnitudes are compared as integers (a NaN is larger than
// an infinity is larger than a number; 16-bit ones two at a time), and a lane's place is kept by
// additions.  A block streams groups of tokens, two 16-byte pieces of a row to a lane; its
// ninth warp looks up the next group's sequences and pages (a chain of loads) meanwhile.
//
// Measured: 97k bf16 tokens, 8 heads of 128, written to int8 codes and read back, 999 MB: 230 us,
// 4.3 TB/s, 5.2 with the codes counted as written and as read (343 us with one piece to a lane and the
// lookups in line); 18k f32 positions of 12 heads of 64 read back, 106 MB: 23 us, 4.6 TB/s.
#include <algorithm>
#include <type_traits>

#include "kserve.cuh"
#include "sm100.cuh"

namespace kattn {

namespace {

using namespace serve;
using namespace sm100;

constexpr int kThreads = 256;   // streaming threads
constexpr int kBlock = kThreads + 32;
constexpr int kMaxTokens = 32;  // tokens of a group at most
constexpr int kBlocksPerSm = 7; // resident: 32 registers a thread

// Where a group's tokens are: the cache row of key head 0, (page * n_kv_head)
// * page_size + place; kNowhere: no such position; kNoRow: no sequence owns the row.
constexpr long kNowhere = -1, kNoRow = -2;

__device__ __forceinline__ void find_places(const CacheArgs& a, int page_shift, int t0, int n, long* place) {
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const int r = t0 + i;
        long at = kNoRow;
        const int s = seq_of_row(a.cu, a.S, r);
        if (s >= 0) {
            const int2 rows = seq_rows(a.cu, s, a.N);
            if (r < rows.y) {
                const int p = max(__ldg(a.kv_len + s), 0) - (rows.y - r);
                const int page = page_of(a, page_shift, s, p);
                at = page < 0 ? kNowhere
                              : (static_cast<long>(page) * a.c.n_kv_head << page_shift) + (p & (a.c.page_size - 1));
            }
        }
        place[i] = at;
    }
}

// Runs stream(first token, tokens, places) over the block's groups.
template <class F>
__device__ __forceinline__ void for_groups(const CacheArgs& a, int page_shift, int tokens, F stream) {
    __shared__ long place[2][kMaxTokens];
    const int groups = (a.N + tokens - 1) / tokens;
    int buf = 0;
    for (int g = static_cast<int>(blockIdx.x) - static_cast<int>(gridDim.x); g < groups; g += gridDim.x, buf ^= 1) {
        const int next = g + gridDim.x;
        if (threadIdx.x >= kThreads) {
            if (next < groups) find_places(a, page_shift, next * tokens, min(tokens, a.N - next * tokens), place[buf ^ 1]);
        } else if (g >= 0) {
            stream(g * tokens, min(tokens, a.N - g * tokens), place[buf]);
        }
        __syncthreads();
    }
}

// The largest magnitude among 16 bytes of T, as the bits of an f32.
template <class T>
__device__ __forceinline__ uint32_t magnitude(const uint4& x) {
    if constexpr (sizeof(T) == 4) {
        return max(max(x.x & 0x7FFFFFFFu, x.y & 0x7FFFFFFFu), max(x.z & 0x7FFFFFFFu, x.w & 0x7FFFFFFFu));
    } else {
        const uint32_t m = __vmaxu2(__vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu),
                                    __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
        const uint32_t h = max(m & 0xFFFFu, m >> 16);
        if constexpr (std::is_same_v<T, __nv_bfloat16>) return h << 16;
        else return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(h))));
    }
}

template <class T, int N>
__device__ __forceinline__ void widen(const uint4& x, float (&f)[N]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                f[2 * i] = __uint_as_float(w[i] << 16);
                f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            } else {
                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                f[2 * i] = y.x;
                f[2 * i + 1] = y.y;
            }
        }
    }
}

// Four values' codes in one word.
template <int FORMAT>
__device__ __forceinline__ uint32_t encode4(const float* f, float inverse) {
    if constexpr (FORMAT == KATTN_CACHE_INT8) {
        // |x * inverse| <= 127 (1 + 2^-23): each sum's low byte is the code.
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(__fmaf_rn(f[i], inverse, 12582912.f));
        return __byte_perm(__byte_perm(w[0], w[1], 0x0040u), __byte_perm(w[2], w[3], 0x0040u), 0x5410u);
    } else {
        float odd[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __fmul_rz(f[i], inverse);
            const float rest = __fmaf_rn(f[i], inverse, -p);
            odd[i] = __uint_as_float(__float_as_uint(p) | (rest != 0.f ? 1u : 0u));
        }
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(odd[1]), "f"(odd[0]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(odd[3]), "f"(odd[2]));
        return lo | (static_cast<uint32_t>(hi) << 16);
    }
}

// Four codes' values, their scale applied.
template <int FORMAT>
__device__ __forceinline__ void decode4(uint32_t w, float scale, float* f) {
    if constexpr (FORMAT == KATTN_CACHE_INT8) {
        w ^= 0x80808080u;  // code + 128, the low byte of 2^23 + 128 + code
        const uint64_t back = f2_pack(8388736.f, 8388736.f), s2 = f2_pack(scale, scale);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u + 2 * i));
            const float y = __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7441u + 2 * i));
            f2_unpack(f2_mul(f2_sub(f2_pack(x, y), back), s2), f[2 * i], f[2 * i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t h;
            const uint16_t two = static_cast<uint16_t>(w >> (16 * i));
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h));
            f[2 * i] = __fmul_rn(y.x, scale);
            f[2 * i + 1] = __fmul_rn(y.y, scale);
        }
    }
}

// A thread's rows of the block's: row r is head r % heads of tensor (r / heads)
// % 2 (k, v) of token r / heads / 2; the thread's are `step` apart.
struct Walk {
    int head, tk, heads, step_head, step_tk;
    __device__ __forceinline__ Walk(int first, int step, int heads_)
        : head(first % heads_), tk(first / heads_), heads(heads_), step_head(step % heads_), step_tk(step / heads_) {}
    __device__ __forceinline__ void next() {
        head += step_head;
        tk += step_tk;
        if (head >= heads) {
            head -= heads;
            ++tk;
        }
    }
};

template <class T, int FORMAT>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm) cache_append_rows(CacheArgs a, const T* __restrict__ k,
                                                            const T* __restrict__ v, long ld, int page_shift,
                                                            int tokens) {
    constexpr int E = Vec16<T>::N;  // elements of a piece
    constexpr float L = FORMAT == KATTN_CACHE_INT8 ? 127.f : 448.f;
    pdl_enter();
    const int d = a.c.d, lanes = d / (2 * E), heads = a.c.n_kv_head;  // lanes: a power of two up to 16
    const int c = threadIdx.x & (lanes - 1), first = threadIdx.x / lanes, step = kThreads / lanes;
    for_groups(a, page_shift, tokens, [&](int t0, int n, const long* place) {
        Walk w(first, step, heads);
        // Every thread runs as many rounds: the shuffles want whole warps.
        for (int r = 0; r < n * heads * 2; r += step, w.next()) {
            const int token = w.tk >> 1;
            const bool is_v = w.tk & 1;
            const long at = token < n ? place[token] : -1;
            uint4 x[2];
            x[0] = x[1] = make_uint4(0, 0, 0, 0);
            if (at >= 0) {
                const uint4* src = reinterpret_cast<const uint4*>((is_v ? v : k) + static_cast<long>(t0 + token) * ld +
                                                                  w.head * d) + c;
                x[0] = __ldcs(src);
                x[1] = __ldcs(src + lanes);
            }
            uint32_t m = max(magnitude<T>(x[0]), magnitude<T>(x[1]));
            for (int o = lanes >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (at < 0) continue;
            const float most = __uint_as_float(m);
            const bool bad = m >= 0x7F800000u, usual = !bad && most >= 0x1p-100f;
            const float inverse = usual ? __fdiv_rn(L, most) : 0.f;
            const long row = at + (static_cast<long>(w.head) << page_shift);
            uint8_t* to = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + row * d + c * E;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[E];
                widen<T>(x[h], f);
                uint32_t code[E / 4];
#pragma unroll
                for (int i = 0; i < E / 4; ++i) code[i] = usual ? encode4<FORMAT>(f + 4 * i, inverse) : 0u;
                if constexpr (E == 4) *reinterpret_cast<uint32_t*>(to + h * lanes * E) = code[0];
                else *reinterpret_cast<uint2*>(to + h * lanes * E) = make_uint2(code[0], code[1]);
            }
            if (c == 0)
                (is_v ? a.c.v_scale : a.c.k_scale)[row] =
                    bad ? __uint_as_float(0x7FC00000u) : (usual ? __fdiv_rn(most, L) : 0.f);
        }
    });
}

template <class T, int FORMAT>
__global__ void __launch_bounds__(kBlock, kBlocksPerSm) cache_read_rows(CacheArgs a, T* __restrict__ k, T* __restrict__ v, long ld,
                                                          int page_shift, int tokens) {
    constexpr int E = Vec16<T>::N;
    pdl_enter();
    const int d = a.c.d, lanes = d / (2 * E), heads = a.c.n_kv_head;
    const int c = threadIdx.x & (lanes - 1), first = threadIdx.x / lanes, step = kThreads / lanes;
    for_groups(a, page_shift, tokens, [&](int t0, int n, const long* place) {
        Walk w(first, step, heads);
        for (int r = first; r < n * heads * 2; r += step, w.next()) {
            const int token = w.tk >> 1;
            const bool is_v = w.tk & 1;
            const long at = token < n ? place[token] : kNoRow;
            if (at == kNoRow) continue;
            uint4* to = reinterpret_cast<uint4*>((is_v ? v : k) + static_cast<long>(t0 + token) * ld + w.head * d) + c;
            float scale = 0.f;
            uint32_t code[2][E / 4] = {};
            if (at >= 0) {
                const long row = at + (static_cast<long>(w.head) << page_shift);
                const uint8_t* from = static_cast<const uint8_t*>(is_v ? a.c.v : a.c.k) + row * d + c * E;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (E == 4) {
                        code[h][0] = __ldcs(reinterpret_cast<const uint32_t*>(from + h * lanes * E));
                    } else {
                        const uint2 y = __ldcs(reinterpret_cast<const uint2*>(from + h * lanes * E));
                        code[h][0] = y.x;
                        code[h][1] = y.y;
                    }
                }
                scale = __ldg((is_v ? a.c.v_scale : a.c.k_scale) + row);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float f[E];
#pragma unroll
                for (int i = 0; i < E / 4; ++i) decode4<FORMAT>(code[h][i], scale, f + 4 * i);
                uint4 y;
                if constexpr (sizeof(T) == 4) {
                    y = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                   __float_as_uint(f[3]));
                } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                    y = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                                   pack_bf16(f[6], f[7]));
                } else {
                    y = make_uint4(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]), pack_f16(f[4], f[5]),
                                   pack_f16(f[6], f[7]));
                }
                __stcs(&to[h * lanes], y);
            }
        }
    });
}

// Tokens of a group: up to 16, fewer where they would leave SMs without one (64 tokens of a
// decoding step: a group each, 3.5 us a call; in groups of 16 only four blocks would work); the
// grid is as many blocks as fit at once.
int group_tokens(int N, int num_sms) {
    int t = 1;
    while (t < 16 && N / (2 * t) >= 2 * num_sms) t *= 2;
    return t;
}

template <class T, int FORMAT>
ProjStatus launch_append(const CacheArgs& a, const void* k, const void* v, long ld, int num_sms, cudaStream_t s) {
    const int tokens = group_tokens(a.N, num_sms), groups = (a.N + tokens - 1) / tokens;
    ProjStatus st;
    st.cuda = launch_pdl(cache_append_rows<T, FORMAT>, dim3(std::min(groups, kBlocksPerSm * num_sms)), dim3(kBlock), 0, s,
                         a, static_cast<const T*>(k), static_cast<const T*>(v), ld, page_shift_of(a.c.page_size), tokens);
    st.what = "cache append launch";
    return st;
}

template <class T, int FORMAT>
ProjStatus launch_read(const CacheArgs& a, void* k, void* v, long ld, int num_sms, cudaStream_t s) {
    const int tokens = group_tokens(a.N, num_sms), groups = (a.N + tokens - 1) / tokens;
    ProjStatus st;
    st.cuda = launch_pdl(cache_read_rows<T, FORMAT>, dim3(std::min(groups, kBlocksPerSm * num_sms)), dim3(kBlock), 0, s, a,
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
