// Attention of new tokens over the 8-bit paged cache (include/kerr_attn.h,
// kattn_fwd_cached).
//
//   s_ij = scale (q_i . kc_j) ks_j,  o_i = sum_j softmax_j(s_ij) vs_j vc_j
//
// with the codes kc, vc and scales ks, vs of position j, for the positions
// that row i sees: those before the new tokens, and of the new ones the tree's.
#include <type_traits>

#include "kserve.cuh"

namespace kattn {

namespace {

using namespace serve;

// One warp per (row, query head): a lane holds D / 32 columns, positions one by one.
template <class T, int D, int FORMAT>
__global__ void __launch_bounds__(128) cached_rows(CachedArgs a, int page_shift) {
    constexpr int E = D / 32;
    pdl_enter();
    const CacheArgs& b = a.cache;
    const int lane = threadIdx.x & 31;
    const long units = static_cast<long>(b.N) * a.H;
    const float c = a.scale * kLog2e;
    for (long u = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 5); u < units; u += 4L * gridDim.x) {
        const int r = static_cast<int>(u / a.H), h = static_cast<int>(u % a.H);
        const int s = seq_of_row(b.cu, b.S, r);
        if (s < 0) continue;
        const int2 rows = seq_rows(b.cu, s, b.N);
        if (r >= rows.y) continue;
        const int len = __ldg(b.kv_len + s), base = len - (rows.y - rows.x);
        const unsigned long long bits = a.tree ? __ldg(a.tree + r) : 0;
        const int hk = h / (a.H / b.c.n_kv_head);
        const T* q = static_cast<const T*>(a.q) + static_cast<long>(r) * a.ld_q + h * D + lane * E;
        float x[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_f32(q[i]), acc[i] = 0.f;
        for (int j = 0; j < len; ++j) {
            if (j >= base) {
                const int t = j - base;
                if (a.tree ? t >= 64 || !((bits >> t) & 1) : t > r - rows.x) continue;
            }
            const int page = page_of(b, page_shift, s, j);
            if (page < 0) continue;
            const long row = ((static_cast<long>(page) * b.c.n_kv_head + hk) << page_shift) + (j & (b.c.page_size - 1));
            const uint8_t* k = static_cast<const uint8_t*>(b.c.k) + row * D + lane * E;
            const uint8_t* v = static_cast<const uint8_t*>(b.c.v) + row * D + lane * E;
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) dot = fmaf(x[i], code_value<FORMAT>(k[i]), dot);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            const float y = dot * b.c.k_scale[row] * c, m2 = fmaxf(m, y);
            const float keep = ex2(m - m2), p = ex2(y - m2);
            m = m2;
            l = fmaf(l, keep, p);
            const float w = p * b.c.v_scale[row];
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] = fmaf(w, code_value<FORMAT>(v[i]), acc[i] * keep);
        }
        T* o = static_cast<T*>(a.o) + static_cast<long>(r) * a.ld_o + h * D + lane * E;
        const bool any = l != 0.f;
        const float inv = any ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = from_f32<T>(acc[i] * inv);
        if (lane == 0) a.lse[static_cast<long>(h) * b.N + r] = any ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
}

}  // namespace

ProjStatus cached_forward(const CachedArgs& a, int num_sms, cudaMemPool_t pool, cudaStream_t s, int* launches) {
    (void)pool;
    ProjStatus st;
    st.what = "cached forward launch";
    const long units = static_cast<long>(a.cache.N) * a.H;
    const dim3 grid(static_cast<unsigned>(units / 4 + 1 < 16L * num_sms ? units / 4 + 1 : 16L * num_sms));
    auto pick = [&](auto f32, auto bf16, auto f16) {
        auto k = a.dtype == KATTN_F32 ? f32 : a.dtype == KATTN_BF16 ? bf16 : f16;
        return launch_pdl(k, grid, dim3(128), 0, s, a, page_shift_of(a.cache.c.page_size));
    };
    auto size = [&](auto format) {
        constexpr int F = decltype(format)::value;
        const int d = a.cache.c.d;
        return d == 32   ? pick(cached_rows<float, 32, F>, cached_rows<__nv_bfloat16, 32, F>, cached_rows<__half, 32, F>)
               : d == 64 ? pick(cached_rows<float, 64, F>, cached_rows<__nv_bfloat16, 64, F>, cached_rows<__half, 64, F>)
                         : pick(cached_rows<float, 128, F>, cached_rows<__nv_bfloat16, 128, F>, cached_rows<__half, 128, F>);
    };
    st.cuda = a.cache.c.format == KATTN_CACHE_INT8 ? size(std::integral_constant<int, KATTN_CACHE_INT8>{})
                                                   : size(std::integral_constant<int, KATTN_CACHE_E4M3>{});
    if (st.ok()) ++*launches;
    return st;
}

}  // namespace kattn
