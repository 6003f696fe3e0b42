// Causal attention of packed sequences with grouped heads (include/kerr_attn.h,
// kattn_fwd_packed), on the tensor cores.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i),
//   j <= i + nk - nq of the row's sequence;  lse_i = m_i + log sum_j p_ij
//
// One pass over the keys with a running row maximum m and sum; the scores and
// weights of a tile never leave the SM.
//
// Rows.  The G = H / Hkv query heads of a key head share its keys, so a
// sequence's nq tokens are nq * G rows per key head (row = token * G + head), and
// a work item is 256 of them: two tiles of 128, which read the same K and V
// tiles.  A group of few tokens then still fills its tile.
//
// Warps (16).  0-3 and 4-7: the softmax of the first and the second row tile,
// one thread a row.  8-11: Q into shared memory (and, for f32, K and V, split into bf16
// hi and lo).  12: issues every MMA.  13: TMA of K and V (16-bit types).  14:
// finds the CTA's items.  While one row tile is in its softmax, the tensor core
// works on the other: O += P V of the tile before, then S = Q K^T of the next.
//
// TMEM.  S of each row tile (BN columns; P is packed over it) and O of each
// (D columns): 512 columns at BN = D = 128.
//
// Types.  16-bit operands enter the MMAs as they are and P is rounded to the type; f32
// ones as bf16 pairs, hi*hi + hi*lo + lo*hi (about 2^-17 of a product, where one
// TF32 product would be off by 2^-11).
//
// Weights are 2^(c s - c mu), c = scale log2(e), with mu raised only when a
// tile's maximum passes it by more than 2^8 (then O and the sum are scaled): weights
// stay below 2^8, which f16 holds, and O is almost never read back.
#include <atomic>

#include <cuda.h>

#include "kserve.cuh"
#include "sm100.cuh"
#include "tma_map.h"

namespace kattn {

namespace {

using namespace serve;
using namespace sm100;

constexpr int BM = 128;          // rows of a row tile
constexpr int ITEM_ROWS = 2 * BM;
constexpr int N_THREADS = 512;
constexpr int LOAD_WARP = 8, MMA_WARP = 12, TMA_WARP = 13, ITEM_WARP = 14;
constexpr int ITEMS = 4;         // item ring
constexpr int HELD = 64;         // columns of a row of S held in registers
constexpr float RESCALE_LOG2 = 8.f;
constexpr uint32_t TMEM_COLS = 512;
constexpr size_t SMEM_MAX = 227 * 1024;

template <class T, int D>
struct Cfg {
    static constexpr bool SPLIT = sizeof(T) == 4;            // operands as bf16 hi / lo pairs
    static constexpr int PARTS = SPLIT ? 2 : 1;
    static constexpr int BN = SPLIT && D == 128 ? 64 : 128;  // keys of a tile (64: Q's pairs leave less room)
    static constexpr int ROW = D == 32 ? 64 : 128;           // bytes of a row of a swizzled block
    static constexpr int BLOCKS = D == 128 ? 2 : 1;          // 64-column blocks (32 at D = 32) of a row
    static constexpr int Q_BLOCK = BM * ROW, Q_PART = BLOCKS * Q_BLOCK, Q_BYTES = PARTS * Q_PART;
    static constexpr int KV_BLOCK = BN * ROW, KV_PART = BLOCKS * KV_BLOCK, KV_BYTES = PARTS * KV_PART;
    static constexpr int FIT = static_cast<int>((SMEM_MAX - 2048 - 2 * Q_BYTES) / KV_BYTES);
    static constexpr int STAGES = FIT < 8 ? FIT : 8;  // K and V tiles in flight
    static constexpr bool BF16 = !std::is_same_v<T, __half>;
    // Registers of a softmax, loader and service thread (512 threads of 128 at launch).
    static constexpr int R_SOFT = SPLIT ? 168 : 184, R_LOAD = SPLIT ? 112 : 80, R_SERV = 64;
    static_assert(2 * R_SOFT + R_LOAD + R_SERV <= 512, "register split");
    __host__ __device__ static constexpr uint32_t col_s(int t) { return t * BN; }
    __host__ __device__ static constexpr uint32_t col_o(int t) { return 2 * BN + t * D; }
    static_assert(2 * BN + 2 * D <= 512, "TMEM columns");
    // P's words of the 16 keys of step s, relative to S: packed, or, for pairs, the hi words of 32 keys and then the lo.
    __host__ __device__ static constexpr uint32_t col_p(int s) { return SPLIT ? 32 * (s >> 1) + 8 * (s & 1) : 8 * s; }
};

struct Item {
    int q0, nq, k0, nk;  // the sequence's rows and keys
    int hk;              // key head
    int r0;              // first row of the item among the sequence's nq * G
    int n0, n1;          // key tiles of each row tile
    int valid;
    __device__ __forceinline__ int n(int t) const { return t ? n1 : n0; }
};

template <class T, int D>
struct Smem {
    using C = Cfg<T, D>;
    alignas(1024) uint8_t q[2][C::Q_BYTES];
    alignas(1024) uint8_t kv[C::STAGES][C::KV_BYTES];
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_ready[2], o_full[2];
    uint64_t kv_full[C::STAGES], kv_empty[C::STAGES];
    uint64_t item_full[ITEMS], item_empty[ITEMS];
    uint64_t tail, drain;
    Item items[ITEMS];
    uint32_t tmem_slot;
};

struct Params {
    CUtensorMap tk, tv;
    PackedArgs a;
    int G;     // query heads of a key head
    float c;   // |scale| log2(e)
    int flip;  // scale < 0: the rows of Q are negated
};

// ---------------------------------------------------------------- items
// A row's keys: the first `seen` of its sequence.
__device__ __forceinline__ int row_seen(const Item& it, int token, int causal) {
    return causal ? min(max(token + it.nk - it.nq + 1, 0), it.nk) : it.nk;
}

// How many of a sequence's items take at least c key tiles.
template <int BN>
__device__ __forceinline__ int items_at_least(int nq, int nk, int G, int causal, int c) {
    const int tiles = (nq * G + ITEM_ROWS - 1) / ITEM_ROWS;
    if (c <= 0) return tiles;
    const int first = (c - 1) * BN;  // some row has to see more than these
    if (first >= nk) return 0;
    const int token = first - (nk - nq);
    if (!causal || token <= 0) return tiles;
    return token >= nq ? 0 : tiles - token * G / ITEM_ROWS;
}

// Items in order of their key tiles, longest first, dealt to the CTAs in
// snake order: item k is in round k / CTAs.  A warp finds the k-th without a list: the
// count of items with at least c tiles is a sum over the sequences, and c
// only falls as k grows.
template <int BN>
struct ItemFinder {
    const PackedArgs& a;
    int G, lane, level, total;

    __device__ __forceinline__ int count(int c) const {
        int n = 0;
        for (int s = lane; s < a.S; s += 32) {
            const int2 q = seq_rows(a.cu_q, s, a.Nq), k = seq_rows(a.cu_k, s, a.Nk);
            n += items_at_least<BN>(q.y - q.x, k.y - k.x, G, a.causal, c);
        }
        return __reduce_add_sync(0xffffffffu, n) * a.Hkv;
    }
    __device__ __forceinline__ void start() {
        int nk = 0;
        for (int s = lane; s < a.S; s += 32) {
            const int2 k = seq_rows(a.cu_k, s, a.Nk);
            nk = max(nk, k.y - k.x);
        }
        level = (__reduce_max_sync(0xffffffffu, nk) + BN - 1) / BN;
        total = count(0);
    }
    // The k-th item (k not below an earlier call's).
    __device__ __forceinline__ Item find(int k) {
        Item it;
        it.valid = k < total;
        if (!it.valid) return it;
        if (count(level) <= k) {
            int lo = 0, hi = level;  // count(lo) > k >= count(hi)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (count(mid) > k) lo = mid;
                else hi = mid;
            }
            level = lo;
        }
        int rank = k - count(level + 1);  // among the items of exactly `level` tiles
        for (int s0 = 0; s0 < a.S; s0 += 32) {
            const int s = s0 + lane;
            int2 q = make_int2(0, 0), kk = make_int2(0, 0);
            int mine = 0, above = 0;
            if (s < a.S) {
                q = seq_rows(a.cu_q, s, a.Nq);
                kk = seq_rows(a.cu_k, s, a.Nk);
                above = items_at_least<BN>(q.y - q.x, kk.y - kk.x, G, a.causal, level + 1);
                mine = items_at_least<BN>(q.y - q.x, kk.y - kk.x, G, a.causal, level) - above;
            }
            int sum = mine * a.Hkv;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, sum > rank);
            if (hit) {
                const int src = __ffs(hit) - 1;
                const int at = rank - (__shfl_sync(0xffffffffu, sum, src) - __shfl_sync(0xffffffffu, mine, src) * a.Hkv);
                const int m = __shfl_sync(0xffffffffu, mine, src);
                it.q0 = __shfl_sync(0xffffffffu, q.x, src);
                it.nq = __shfl_sync(0xffffffffu, q.y, src) - it.q0;
                it.k0 = __shfl_sync(0xffffffffu, kk.x, src);
                it.nk = __shfl_sync(0xffffffffu, kk.y, src) - it.k0;
                const int first = (it.nq * G + ITEM_ROWS - 1) / ITEM_ROWS -
                                  __shfl_sync(0xffffffffu, above, src) - m;
                it.hk = at / m;
                it.r0 = (first + at % m) * ITEM_ROWS;
                break;
            }
            rank -= __shfl_sync(0xffffffffu, sum, 31);
        }
        const int rows = it.nq * G;
        const int end0 = min(rows, it.r0 + BM) - 1, end1 = min(rows, it.r0 + 2 * BM) - 1;  // last rows of the tiles
        it.n0 = (row_seen(it, end0 / G, a.causal) + BN - 1) / BN;
        it.n1 = end1 < it.r0 + BM ? 0 : (row_seen(it, end1 / G, a.causal) + BN - 1) / BN;
        return it;
    }
};

// ---------------------------------------------------------------- operands
template <class T, int D>
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) {  // 16-byte chunk of a block's row
    if constexpr (D == 32) return sw64(row, chunk);
    else return sw128(row, chunk);
}

// 8 values of a row -> the operand's bytes at (row, 8-column chunk ch): one
// 16-byte chunk, two (hi, lo) for f32.
template <class T, int D, int PART, int BLOCK>
__device__ __forceinline__ void put8(uint8_t* base, int row, int ch, const uint4& x0, const uint4& x1) {
    uint8_t* at = base + (ch >> 3) * BLOCK + swizzled<T, D>(row, ch & 7);
    if constexpr (sizeof(T) == 4) {
        uint4 hi, lo;
        split2(__uint_as_float(x0.x), __uint_as_float(x0.y), hi.x, lo.x);
        split2(__uint_as_float(x0.z), __uint_as_float(x0.w), hi.y, lo.y);
        split2(__uint_as_float(x1.x), __uint_as_float(x1.y), hi.z, lo.z);
        split2(__uint_as_float(x1.z), __uint_as_float(x1.w), hi.w, lo.w);
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + PART) = lo;
    } else {
        *reinterpret_cast<uint4*>(at) = x0;
    }
}

// Row tile t of an item's Q -> shared memory, by the 128 loader threads: rows
// past the sequence's are zeros.
template <class T, int D>
__device__ __forceinline__ void load_q(const Params& p, const Item& it, int t, uint8_t* dst, int tid) {
    using C = Cfg<T, D>;
    constexpr int CH = D / 8, N = BM * CH / 128, V = sizeof(T) / 2;  // chunks a row, a thread; 16-byte loads a chunk
    constexpr int BATCH = N * V < 8 ? N : 8 / V;
    const uint32_t flip = p.flip ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
    const int rows = it.nq * p.G;
#pragma unroll
    for (int b = 0; b < N; b += BATCH) {
        uint4 x[BATCH][V];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int u = tid + (b + i) * 128, r = u / CH, ch = u % CH;
            const int row = it.r0 + t * BM + r;
            if (row < rows) {
                const T* src = static_cast<const T*>(p.a.q) + static_cast<long>(it.q0 + row / p.G) * p.a.ld_q +
                               (it.hk * p.G + row % p.G) * D + ch * 8;
#pragma unroll
                for (int v = 0; v < V; ++v) x[i][v] = __ldg(reinterpret_cast<const uint4*>(src) + v);
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) x[i][v] = make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int u = tid + (b + i) * 128, r = u / CH, ch = u % CH;
#pragma unroll
            for (int v = 0; v < V; ++v)
                x[i][v] = make_uint4(x[i][v].x ^ flip, x[i][v].y ^ flip, x[i][v].z ^ flip, x[i][v].w ^ flip);
            put8<T, D, C::Q_PART, C::Q_BLOCK>(dst, r, ch, x[i][0], x[i][V - 1]);
        }
    }
}

// A tile of BN f32 rows (K or V) held in registers by the 128 loader threads
// between its loads and its conversion; rows past the sequence's are zeros.
template <int D, int BN>
struct F32Tile {
    static constexpr int CH = D / 8, N = BN * CH / 128;
    float4 x[N][2];
    __device__ __forceinline__ void load(const float* base, long ld, int rows, int tid) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = tid + i * 128, r = u / CH, ch = u % CH;
            x[i][0] = x[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) {
                const float4* src = reinterpret_cast<const float4*>(base + r * ld + ch * 8);
                x[i][0] = __ldg(src);
                x[i][1] = __ldg(src + 1);
            }
        }
    }
    template <int PART, int BLOCK>
    __device__ __forceinline__ void store(uint8_t* dst, int tid) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = tid + i * 128, r = u / CH, ch = u % CH;
            put8<float, D, PART, BLOCK>(dst, r, ch, *reinterpret_cast<const uint4*>(&x[i][0]),
                                        *reinterpret_cast<const uint4*>(&x[i][1]));
        }
    }
};

template <class T, int D>
__device__ __forceinline__ uint64_t k_major(uint32_t addr) {
    if constexpr (D == 32) return smem_desc_sw64(addr, 512);
    else return smem_desc(addr, 16, 1024);
}

// S_t = Q_t K^T of the K tile at `k`: 16 columns of d a step.
template <class T, int D>
__device__ __forceinline__ void issue_s(uint32_t tm, int t, uint32_t q, uint32_t k) {
    using C = Cfg<T, D>;
    constexpr uint32_t id = C::BF16 ? idesc_bf16(BM, C::BN, 0, 0) : idesc_f16(BM, C::BN, 0, 0);
    const uint32_t out = tm + C::col_s(t);
    const uint64_t qd = k_major<T, D>(q), kd = k_major<T, D>(k);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const uint32_t qo = (s >> 2) * C::Q_BLOCK + (s & 3) * 32, ko = (s >> 2) * C::KV_BLOCK + (s & 3) * 32;
        mma_ss(out, desc_add(qd, qo), desc_add(kd, ko), id, s > 0);
        if constexpr (C::SPLIT) {
            mma_ss(out, desc_add(qd, qo), desc_add(kd, ko + C::KV_PART), id, 1);
            mma_ss(out, desc_add(qd, qo + C::Q_PART), desc_add(kd, ko), id, 1);
        }
    }
}

// O_t (+)= P_t V of the V tile at `v`: 16 keys a step; P's hi (and lo) words over S_t.
template <class T, int D>
__device__ __forceinline__ void issue_pv(uint32_t tm, int t, uint32_t v, bool first) {
    using C = Cfg<T, D>;
    constexpr uint32_t id = C::BF16 ? idesc_bf16(BM, D, 0, 1) : idesc_f16(BM, D, 0, 1);
    const uint32_t out = tm + C::col_o(t), ph = tm + C::col_s(t);
    const uint64_t vd = D == 32 ? smem_desc_sw64(v, 512) : smem_desc(v, C::KV_BLOCK, 1024);
#pragma unroll
    for (int s = 0; s < C::BN / 16; ++s) {
        const uint32_t o = s * 16 * C::ROW, ps = ph + C::col_p(s);
        mma_ts(out, ps, desc_add(vd, o), id, (first && s == 0) ? 0u : 1u);
        if constexpr (C::SPLIT) {
            mma_ts(out, ps, desc_add(vd, o + C::KV_PART), id, 1);
            mma_ts(out, ps + 16, desc_add(vd, o), id, 1);
        }
    }
}

// ---------------------------------------------------------------- softmax
// N columns of this thread's row of S; those from `lim` on are masked where
// `masked` (the same for the warp).
template <int N>
__device__ __forceinline__ void load_scores(uint32_t at, float (&s)[N], bool masked, int lim) {
#pragma unroll
    for (int q = 0; q < N / 32; ++q) tmem_ld32(at + 32 * q, reinterpret_cast<float(&)[32]>(s[32 * q]));
    tmem_wait_ld();
    if (masked) {
#pragma unroll
        for (int q = 0; q < N; ++q) s[q] = q < lim ? s[q] : -INFINITY;
    }
}

template <int N>
__device__ __forceinline__ float row_max(const float (&s)[N]) {
    float mx[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) mx[q] = fmaxf(s[q], s[q + 8]);
#pragma unroll
    for (int q = 16; q < N; q += 16)
#pragma unroll
        for (int u = 0; u < 8; ++u) mx[u] = max3(mx[u], s[q + u], s[q + 8 + u]);
    return fmaxf(max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[4]), max3(mx[5], mx[6], mx[7]));
}

// ---------------------------------------------------------------- kernel
template <class T, int D>
__global__ void __launch_bounds__(N_THREADS, 1) packed_fwd(const __grid_constant__ Params p) {
    using C = Cfg<T, D>;
    constexpr int BN = C::BN;
    extern __shared__ uint8_t smem_raw[];
    Smem<T, D>& sm = *reinterpret_cast<Smem<T, D>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_launch();
    if (warp == MMA_WARP) {
        tmem_alloc(&sm.tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm.q_full[i], 128);
            mbar_init(&sm.q_empty[i], 1);
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_ready[i], 128);
            mbar_init(&sm.o_full[i], 1);
        }
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&sm.kv_full[i], C::SPLIT ? 128 : 1);
            mbar_init(&sm.kv_empty[i], 1);
        }
        for (int i = 0; i < ITEMS; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], C::SPLIT ? 13 : 14);  // softmax 8, loader 4, MMA, TMA
        }
        mbar_init(&sm.tail, 1);
        mbar_init(&sm.drain, 1);
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();
    const uint32_t tm = sm.tmem_slot;
    const uint64_t limit = p.a.wait_ns;
    bool failed = false;

    // The i-th item, for a whole warp.
    auto get_item = [&](int i, Item& it) -> bool {
        const int slot = i % ITEMS;
        if (!mbar_wait_warp(&sm.item_full[slot], (i / ITEMS) & 1, limit)) return false;
        it = sm.items[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[slot]);
        return true;
    };

    if (warp < LOAD_WARP) {
        // ------------------------------------------------------------ softmax
        regs_inc<C::R_SOFT>();
        const int t = warp >> 2;
        const int rl = (warp & 3) * 32 + lane;
        const uint32_t lb = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = lb + tm + C::col_s(t), to = lb + tm + C::col_o(t);
        int g = 0, done = 0;  // tiles and items of this row tile so far
        Item it;
        for (int i = 0;; ++i) {
            if (!get_item(i, it)) {
                failed = true;
                break;
            }
            if (!it.valid) break;
            const int row = it.r0 + t * BM + rl;
            const bool mine = row < it.nq * p.G;
            const int token = row / p.G;
            const int seen = mine ? row_seen(it, token, p.a.causal) : 0;
            const int n = it.n(t);
            float mu = -INFINITY, l = 0.f;
            for (int j = 0; j < n; ++j, ++g) {
                if (!mbar_wait_warp(&sm.s_full[t], g & 1, limit)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                // The row's maximum.  Half of a 128-column row is held in registers from here to its
                // weights, the other half is read twice: the whole row does not fit beside the rest.
                const int lim = seen - j * BN;  // visible columns of the tile
                const bool masked = __any_sync(0xffffffffu, lim < BN);
                float s[HELD], m = -INFINITY;
#pragma unroll
                for (int q = BN / HELD - 1; q >= 0; --q) {
                    load_scores<HELD>(ts + HELD * q, s, masked, lim - HELD * q);
                    m = fmaxf(m, row_max<HELD>(s));
                }
                if (j == 0) {
                    mu = m;
                } else {
                    const bool raise = (m - mu) * p.c > RESCALE_LOG2 || (mu == -INFINITY && m > mu);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float to_mu = raise ? m : mu;
                        const float f = raise ? ex2((mu - m) * p.c) : 1.f;
                        mu = to_mu;
                        l *= f;
#pragma unroll 1
                        for (int q = 0; q < D / 16; ++q) {  // few columns at a time: the row of S is held meanwhile
                            float o[16];
                            uint32_t r[16];
                            tmem_ld16(to + 16 * q, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int u = 0; u < 16; ++u) r[u] = __float_as_uint(o[u] * f);
                            tmem_st16(to + 16 * q, r);
                        }
                    }
                }
                const float off = mu == -INFINITY ? 0.f : -mu * p.c;
                const uint64_t c2 = f2_pack(p.c, p.c), off2 = f2_pack(off, off);
                uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
#pragma unroll
                for (int q = 0; q < BN / 32; ++q) {
                    if (q > 0 && q % (HELD / 32) == 0)
                        load_scores<HELD>(ts + 32 * q, s, masked, lim - 32 * q);
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        const int v = (32 * q) % HELD + 2 * u;
                        float x, y;
                        f2_unpack(f2_fma(f2_pack(s[v], s[v + 1]), c2, off2), x, y);
                        x = ex2(x);
                        y = ex2(y);
                        if (u & 1) sum1 = f2_add(sum1, f2_pack(x, y));
                        else sum0 = f2_add(sum0, f2_pack(x, y));
                        if constexpr (C::SPLIT) split2_x2(x, y, hi[u], lo[u]);
                        else if constexpr (C::BF16) hi[u] = pack_bf16(x, y);
                        else hi[u] = pack_f16(x, y);
                    }
                    // Over columns that have been read for the last time: this chunk's own or an earlier one's.
                    tmem_st16(ts + C::col_p(2 * q), hi);
                    if constexpr (C::SPLIT) tmem_st16(ts + C::col_p(2 * q) + 16, lo);
                }
                float a0, a1;
                f2_unpack(f2_add(sum0, sum1), a0, a1);
                l += a0 + a1;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&sm.p_ready[t]);
            }
            if (failed) break;
            // Output: normalised, rounded once; rows that saw nothing are zeros.
            const float inv = seen > 0 ? 1.f / l : 0.f;
            T* out = nullptr;
            if (mine) {
                const int h = it.hk * p.G + row % p.G;
                out = static_cast<T*>(p.a.o) + static_cast<long>(it.q0 + token) * p.a.ld_o + h * D;
                p.a.lse[static_cast<long>(h) * p.a.Nq + it.q0 + token] =
                    seen > 0 ? (mu * p.c + log2f(l)) * kLn2 : -INFINITY;
            }
            if (n > 0) {
                if (!mbar_wait_warp(&sm.o_full[t], done & 1, limit)) {
                    failed = true;
                    break;
                }
                ++done;
                tc_fence_after();
            }
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
                float o[32];
                if (n > 0) {
                    tmem_ld32(to + 32 * q, o);
                    tmem_wait_ld();
                }
                if (mine) {
#pragma unroll
                    for (int u = 0; u < 32; ++u) o[u] = seen > 0 ? o[u] * inv : 0.f;
                    uint4* dst = reinterpret_cast<uint4*>(out + 32 * q);
                    if constexpr (C::SPLIT) {
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            dst[u] = make_uint4(__float_as_uint(o[4 * u]), __float_as_uint(o[4 * u + 1]),
                                                __float_as_uint(o[4 * u + 2]), __float_as_uint(o[4 * u + 3]));
                    } else {
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            uint32_t w[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                w[x] = C::BF16 ? pack_bf16(o[8 * u + 2 * x], o[8 * u + 2 * x + 1])
                                               : pack_f16(o[8 * u + 2 * x], o[8 * u + 2 * x + 1]);
                            dst[u] = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
        }
    } else if (warp < MMA_WARP) {
        // ------------------------------------------------------------ loaders
        regs_dec<C::R_LOAD>();
        const int lt = tid - 32 * LOAD_WARP;
        int used[2] = {0, 0}, kv = 0;
        Item it;
        for (int i = 0; !failed; ++i) {
            if (!get_item(i, it)) {
                failed = true;
                break;
            }
            if (!it.valid) break;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if (it.n(t) == 0) continue;
                // Q_t is free once the last S of the item that used it is done.
                if (used[t] > 0 && !mbar_wait_warp(&sm.q_empty[t], (used[t] - 1) & 1, limit)) {
                    failed = true;
                    break;
                }
                ++used[t];
                load_q<T, D>(p, it, t, sm.q[t], lt);
                fence_async_smem();
                mbar_arrive(&sm.q_full[t]);
            }
            if constexpr (C::SPLIT) {
                // K_0, V_0, K_1, ...: a tile's loads are in flight while its stage is waited for.
                const int n = max(it.n0, it.n1);
                for (int x = 0; x < 2 * n && !failed; ++x, ++kv) {
                    const int j = x >> 1, st = kv % C::STAGES, turn = kv / C::STAGES;
                    F32Tile<D, BN> tile;
                    tile.load(static_cast<const float*>(x & 1 ? p.a.v : p.a.k) + static_cast<long>(it.k0 + j * BN) * p.a.ld_kv + it.hk * D, p.a.ld_kv,
                              it.nk - j * BN, lt);
                    if (turn > 0 && !mbar_wait_warp(&sm.kv_empty[st], (turn - 1) & 1, limit)) {
                        failed = true;
                        break;
                    }
                    tile.template store<C::KV_PART, C::KV_BLOCK>(sm.kv[st], lt);
                    fence_async_smem();
                    mbar_arrive(&sm.kv_full[st]);
                }
            }
        }
    } else {
        regs_dec<C::R_SERV>();
        if (warp == MMA_WARP) {
            // -------------------------------------------------------- MMA issuer
            int kv = 0, q_used[2] = {0, 0}, p_used[2] = {0, 0};
            Item it;
            for (int i = 0; !failed; ++i) {
                if (!get_item(i, it)) {
                    failed = true;
                    break;
                }
                if (!it.valid) break;
                const int n = max(it.n0, it.n1);
                if (n == 0) continue;
                if (lane == 0) {
                    auto full = [&](int x) { return mbar_wait(&sm.kv_full[x % C::STAGES], (x / C::STAGES) & 1, limit); };
                    failed = !full(kv);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (failed || it.n(t) == 0) continue;
                        failed = !mbar_wait(&sm.q_full[t], q_used[t]++ & 1, limit);
                        if (failed) continue;
                        tc_fence_after();
                        issue_s<T, D>(tm, t, smem_u32(sm.q[t]), smem_u32(sm.kv[kv % C::STAGES]));
                        mma_commit(&sm.s_full[t]);
                        if (it.n(t) == 1) mma_commit(&sm.q_empty[t]);
                    }
                    mma_commit(&sm.kv_empty[kv % C::STAGES]);
                    ++kv;
                    for (int j = 0; j < n && !failed; ++j) {
                        const bool next = j + 1 < n;
                        failed = !full(kv);
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            if (failed || j >= it.n(t)) continue;
                            failed = !mbar_wait(&sm.p_ready[t], p_used[t]++ & 1, limit);
                            if (failed) continue;
                            tc_fence_after();
                            issue_pv<T, D>(tm, t, smem_u32(sm.kv[kv % C::STAGES]), j == 0);
                            if (j + 1 < it.n(t)) {
                                failed = !full(kv + 1);
                                if (failed) continue;
                                tc_fence_after();
                                issue_s<T, D>(tm, t, smem_u32(sm.q[t]), smem_u32(sm.kv[(kv + 1) % C::STAGES]));
                                mma_commit(&sm.s_full[t]);
                                if (j + 2 == it.n(t)) mma_commit(&sm.q_empty[t]);
                            } else {
                                mma_commit(&sm.o_full[t]);
                            }
                        }
                        mma_commit(&sm.kv_empty[kv % C::STAGES]);
                        if (next) mma_commit(&sm.kv_empty[(kv + 1) % C::STAGES]);
                        kv += next ? 2 : 1;
                    }
                }
                failed = __any_sync(0xffffffffu, failed);
            }
            if (lane == 0) {
                // MMAs still in flight complete before the columns are freed.
                mma_commit(&sm.drain);
                mbar_wait(&sm.drain, 0, 10000000ull);
            }
            __syncwarp();
        } else if (warp == TMA_WARP && !C::SPLIT) {
            // -------------------------------------------------------- K / V copies
            if (lane == 0 && p.a.Nk > 0) {
                prefetch_tensormap(&p.tk);
                prefetch_tensormap(&p.tv);
            }
            int kv = 0, tails = 0;
            Item it;
            for (int i = 0; !failed; ++i) {
                if (!get_item(i, it)) {
                    failed = true;
                    break;
                }
                if (!it.valid) break;
                const int n = max(it.n0, it.n1);
                for (int x = 0; x < 2 * n; ++x, ++kv) {
                    const int j = x >> 1, st = kv % C::STAGES, turn = kv / C::STAGES;
                    if (turn > 0 && !mbar_wait_warp(&sm.kv_empty[st], (turn - 1) & 1, limit)) {
                        failed = true;
                        break;
                    }
                    const CUtensorMap* map = x & 1 ? &p.tv : &p.tk;
                    // A V tile past the sequence's end holds rows of the next one, whose weights are zero: those
                    // rows are cleared, as zero times an infinity or a NaN there would not be zero.
                    const int rows = it.nk - j * BN;
                    const bool tail = (x & 1) && rows < BN;
                    uint64_t* bar = tail ? &sm.tail : &sm.kv_full[st];
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar, C::KV_BYTES);
#pragma unroll
                        for (int b = 0; b < C::BLOCKS; ++b)
                            tma_load_2d(sm.kv[st] + b * C::KV_BLOCK, map, it.hk * D + 64 * b, it.k0 + j * BN, bar);
                    }
                    if (tail) {
                        if (!mbar_wait_warp(&sm.tail, tails++ & 1, limit)) {
                            failed = true;
                            break;
                        }
                        for (int b = 0; b < C::BLOCKS; ++b)
                            for (int u = rows * C::ROW + lane * 16; u < C::KV_BLOCK; u += 512)
                                *reinterpret_cast<uint4*>(sm.kv[st] + b * C::KV_BLOCK + u) = make_uint4(0, 0, 0, 0);
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.kv_full[st]);
                    }
                }
            }
            if (failed) {
                // Copies still landing complete before the shared memory is released.
                for (int x = max(0, kv - C::STAGES); x < kv; ++x)
                    mbar_wait(&sm.kv_full[x % C::STAGES], (x / C::STAGES) & 1, 10000000ull);
                if (tails > 0) mbar_wait(&sm.tail, (tails - 1) & 1, 10000000ull);
            }
        } else if (warp == ITEM_WARP) {
            // -------------------------------------------------------- items
            ItemFinder<BN> find{p.a, p.G, lane, 0, 0};
            find.start();
            const int ctas = gridDim.x, b = blockIdx.x;
            for (int i = 0;; ++i) {
                const Item it = find.find(i * ctas + (i & 1 ? ctas - 1 - b : b));
                const int slot = i % ITEMS;
                if (i >= ITEMS && !mbar_wait_warp(&sm.item_empty[slot], (i / ITEMS - 1) & 1, limit)) {
                    failed = true;
                    break;
                }
                if (lane == 0) {
                    sm.items[slot] = it;
                    mbar_arrive(&sm.item_full[slot]);
                }
                if (!it.valid) break;
            }
        }
    }
    if (failed && lane == 0) atomicOr(p.a.status, 1);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tmem_dealloc(tm, TMEM_COLS);
}

template <class T, int D>
cudaError_t launch(const PackedArgs& a, int num_sms, cudaStream_t stream) {
    using C = Cfg<T, D>;
    Params p{};
    p.a = a;
    p.G = a.H / a.Hkv;
    // A scale of zero weighs every key alike; kept positive so that a masked score stays -inf.
    p.c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
    p.flip = a.scale < 0.f;
    if constexpr (!C::SPLIT) {
        if (a.Nk > 0) {
            const CUtensorMapSwizzle sw = D == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
            const long cols = static_cast<long>(a.Hkv) * D;
            const int box = D == 32 ? 32 : 64;
            if (!encode_2d_bf16(&p.tk, static_cast<const uint16_t*>(a.k), cols, a.Nk, a.ld_kv, box, C::BN, sw) ||
                !encode_2d_bf16(&p.tv, static_cast<const uint16_t*>(a.v), cols, a.Nk, a.ld_kv, box, C::BN, sw))
                return cudaErrorInvalidValue;
        }
    }
    auto kernel = packed_fwd<T, D>;
    constexpr size_t smem = sizeof(Smem<T, D>) + 1024;
    static_assert(smem <= SMEM_MAX, "shared memory");
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<uint64_t> attr_done{0};  // one bit per device
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_done.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
        attr_done.fetch_or(bit);
    }
    // No more items than this: each sequence ends at most one item that is not full.
    const long items = (static_cast<long>(a.Nq) * p.G / ITEM_ROWS + a.S) * a.Hkv;
    return launch_pdl(kernel, dim3(static_cast<unsigned>(items < num_sms ? items : num_sms)), dim3(N_THREADS), smem,
                      stream, p);
}

}  // namespace

ProjStatus packed_forward(const PackedArgs& a, int num_sms, cudaStream_t s, int* launches) {
    ProjStatus st;
    st.what = "packed forward launch";
    auto pick = [&](auto f32, auto bf16, auto f16) {
        return (a.dtype == KATTN_F32 ? f32 : a.dtype == KATTN_BF16 ? bf16 : f16)(a, num_sms, s);
    };
    st.cuda = a.d == 32   ? pick(launch<float, 32>, launch<__nv_bfloat16, 32>, launch<__half, 32>)
              : a.d == 64 ? pick(launch<float, 64>, launch<__nv_bfloat16, 64>, launch<__half, 64>)
                          : pick(launch<float, 128>, launch<__nv_bfloat16, 128>, launch<__half, 128>);
    if (st.ok()) ++*launches;
    return st;
}

}  // namespace kattn
