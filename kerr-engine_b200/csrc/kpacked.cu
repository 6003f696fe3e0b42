// Causal attention of packed sequences with grouped heads (include/kerr_attn.h,
// kattn_fwd_packed).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i),
//   j <= i + nk - nq of the row's sequence;  lse_i = m_i + log sum_j p_ij
#include "kserve.cuh"

namespace kattn {

namespace {

using namespace serve;

// One warp per (row, query head): a lane holds D / 32 columns, keys one by one.
template <class T, int D>
__global__ void __launch_bounds__(128) packed_rows(PackedArgs a) {
    constexpr int E = D / 32;
    pdl_enter();
    const int lane = threadIdx.x & 31;
    const long units = static_cast<long>(a.Nq) * a.H;
    const float c = a.scale * kLog2e;
    for (long u = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 5); u < units; u += 4L * gridDim.x) {
        const int r = static_cast<int>(u / a.H), h = static_cast<int>(u % a.H);
        const int s = seq_of_row(a.cu_q, a.S, r);
        if (s < 0) continue;
        const int2 rows = seq_rows(a.cu_q, s, a.Nq), keys = seq_rows(a.cu_k, s, a.Nk);
        if (r >= rows.y) continue;
        const int nk = keys.y - keys.x;
        const int seen = a.causal ? min(nk, nk - (rows.y - 1 - r)) : nk;
        const int hk = h / (a.H / a.Hkv);
        const T* q = static_cast<const T*>(a.q) + static_cast<long>(r) * a.ld_q + h * D + lane * E;
        float x[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_f32(q[i]), acc[i] = 0.f;
        for (int j = 0; j < seen; ++j) {
            const long at = (static_cast<long>(keys.x) + j) * a.ld_kv + hk * D + lane * E;
            const T* k = static_cast<const T*>(a.k) + at;
            const T* v = static_cast<const T*>(a.v) + at;
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) dot = fmaf(x[i], to_f32(k[i]), dot);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            const float y = dot * c, m2 = fmaxf(m, y);
            const float keep = ex2(m - m2), p = ex2(y - m2);
            m = m2;
            l = fmaf(l, keep, p);
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] = fmaf(p, to_f32(v[i]), acc[i] * keep);
        }
        T* o = static_cast<T*>(a.o) + static_cast<long>(r) * a.ld_o + h * D + lane * E;
        const float inv = seen > 0 ? 1.f / l : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = from_f32<T>(acc[i] * inv);
        if (lane == 0) a.lse[static_cast<long>(h) * a.Nq + r] = seen > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
}

}  // namespace

ProjStatus packed_forward(const PackedArgs& a, int num_sms, cudaMemPool_t pool, cudaStream_t s, int* launches) {
    (void)pool;
    ProjStatus st;
    st.what = "packed forward launch";
    const long units = static_cast<long>(a.Nq) * a.H;
    const dim3 grid(static_cast<unsigned>(units / 4 + 1 < 16L * num_sms ? units / 4 + 1 : 16L * num_sms));
    auto pick = [&](auto f32, auto bf16, auto f16) {
        auto k = a.dtype == KATTN_F32 ? f32 : a.dtype == KATTN_BF16 ? bf16 : f16;
        return launch_pdl(k, grid, dim3(128), 0, s, a);
    };
    st.cuda = a.d == 32   ? pick(packed_rows<float, 32>, packed_rows<__nv_bfloat16, 32>, packed_rows<__half, 32>)
              : a.d == 64 ? pick(packed_rows<float, 64>, packed_rows<__nv_bfloat16, 64>, packed_rows<__half, 64>)
                          : pick(packed_rows<float, 128>, packed_rows<__nv_bfloat16, 128>, packed_rows<__half, 128>);
    if (st.ok()) ++*launches;
    return st;
}

}  // namespace kattn
