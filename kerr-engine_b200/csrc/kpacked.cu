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
// Work.  Where enough items share the GPU, each CTA takes whole ones, longest first.  A few long
// ones are a line of key tiles cut into equal parts, one a CTA, and packed_join adds the
// parts of cut items; line_pays() has the rule and what both measured.  The search for a whole item
// sweeps all sequences, so it grows with their square and from some hundreds on is what takes the time
// (sequences of 64, 8 heads of 64, bf16: 53 us for 128 of them, 283 for 512, 13.6 ms for 4096).
//
// Bounds.  Long prompts: the tensor core's rate, shared with the exponentials (three bf16 prompts of
// 1500 .. 8192, 32 heads of 128: 580 us, 1110 TFLOP/s, back to back at 1965 MHz; 633 us after other work there; 660 us,
// 980 TFLOP/s, once the power cap has brought the clock to 1.7 GHz).  f32: three products of each, whose operands shared
// memory feeds, 3300 clocks a step.  Short prompts: the chain from launch to first copy
// to store (one f32 prompt of 256, 12 heads: 19 us; 32 bf16 prompts of 9 .. 512, 20 heads on 4: 28 us).
//
// Warps (16).  0-3 and 4-7: the softmax of the first and the second row tile,
// one thread a row.  8-11: Q into shared memory (and, for f32, K and V split
// in place into hi and lo).  12: issues every MMA.  13: TMA of K and V.  14: walks
// the CTA's work.
//
// Steps of 128 keys (64 for f32 at D = 128).  While one row tile is in its softmax,
// the tensor core works on the other: O += P V of its step, then S = Q K^T of its next.
// P goes over the S it came from, 64 keys at a time, and each half's product starts when
// it is written.  (Steps of 64 keys with two S buffers a tile were slower: an MMA
// with both operands in shared memory costs the same at N = 64 as at 128, the rows of Q
// being the larger read.)  TMEM: 2 x 128 columns of S and P, 2 x D of O, 512 at D = 128.
//
// Types.  16-bit operands enter the MMAs as they are and P is rounded to the type; f32
// ones as f16 pairs (22 bits), hi*hi + hi*lo + lo*hi, after powers of two have brought
// them near 2^14: one a row of Q, one a tile of K, one for the V tiles of an item (it
// rises when one needs it, and O follows).  They go back in with the exponent's factor
// and the output.  bf16 pairs need no powers and took 84 us where this took 94 (91 now; chunks
// over cached contexts, f32), but are off by 6e-6; these by 3e-7 to 9e-7, as an f32 product is, and by up to 1.8e-6 at
// D = 128, where TMEM has no room for a second O and every product is cut into the one sum.
//
// Weights are 2^(c s - c mu), c = scale log2(e), with mu raised only when a
// tile's maximum passes it by more than 2^8 (then O and the sum are scaled): weights
// stay below 2^8 (2^15 as f16 holds them), and O is almost never read back.
#include <algorithm>
#include <atomic>
#include <climits>

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
constexpr int HALF = 64;         // keys whose weights are handed over at once
constexpr int N_THREADS = 512, LAUNCH_REGS = 128;
constexpr int LOAD_WARP = 8, MMA_WARP = 12, TMA_WARP = 13, ITEM_WARP = 14;
constexpr int ITEMS = 4;         // item ring
constexpr float RESCALE_LOG2 = 8.f;
constexpr uint32_t GAVE_UP = 0xFFFFFFFFu;  // for a largest magnitude's bits: the warp's wait ran out
constexpr int UNITS = 16;        // ring of the K and V tiles' powers of two: more than tiles can be under way
constexpr int POLY = 1;          // of 8 pairs of weights by the FMA units (16-bit types): 582, 576, 586 us for 0, 1, 2 (long prompts)
constexpr uint32_t TMEM_COLS = 512;
constexpr size_t SMEM_MAX = 227 * 1024;

template <class T, int D>
struct Cfg {
    static constexpr bool SPLIT = sizeof(T) == 4;            // operands as f16 hi / lo pairs
    static constexpr int PARTS = SPLIT ? 2 : 1;
    static constexpr int BN = SPLIT && D == 128 ? 64 : 128;  // keys of a step (64: Q's pairs leave less room)
    static constexpr int HALVES = BN / HALF;
    static constexpr int ROW = D == 32 ? 64 : 128;           // bytes of a row of a swizzled block
    static constexpr int BLOCKS = D == 128 ? 2 : 1;          // 64-column blocks (32 at D = 32) of a row
    static constexpr int Q_BLOCK = BM * ROW, Q_PART = BLOCKS * Q_BLOCK, Q_BYTES = PARTS * Q_PART;
    // A K or V tile: per block its rows (f32: as the copy lands them, then hi rows and lo rows in their place).
    static constexpr int KV_PART = BN * ROW, KV_BLOCK = PARTS * KV_PART, KV_BYTES = BLOCKS * KV_BLOCK;
    // Output rows leave through shared memory, 64 bytes of each of a warp's 32 rows at a time, so that four lanes
    // store one row's stretch (a lane a row takes a request each); at D = 128 the copies' stages need the place.
    static constexpr int OUT_PITCH = 80, OUT_BYTES = D < 128 ? 8 * 32 * OUT_PITCH : 0;
    static constexpr int FIT = static_cast<int>((SMEM_MAX - 2048 - OUT_BYTES - 2 * Q_BYTES) / KV_BYTES);
    static constexpr int STAGES = FIT < 8 ? FIT : 8;  // K and V tiles in flight
    static constexpr bool BF16 = std::is_same_v<T, __nv_bfloat16>;  // the operands' type; else f16
    // f16 weights are held times 2^7 (then at most 2^15), further from f16's subnormals: a weight of 2^-25 of the largest
    // and less would vanish, and tens of thousands of those are more than the output's rounding.
    static constexpr float W_UP = BF16 ? 0.f : 7.f;
    // Registers of a softmax, loader and service thread (LAUNCH_REGS at launch).
    static constexpr int R_SOFT = SPLIT ? 176 : 200, R_LOAD = SPLIT ? 112 : 64, R_SERV = 48;
    static_assert(2 * R_SOFT + R_LOAD + R_SERV <= 4 * LAUNCH_REGS, "register split");
    __host__ __device__ static constexpr uint32_t col_s(int t) { return t * BN; }
    // Pairs at D <= 64: V's hi and lo are one operand of 2 D columns, and O two halves that are added at the end.  An MMA
    // costs the same at N = 64 as at 128, so P V takes two MMAs for 16 keys instead of three.
    static constexpr bool WIDE = SPLIT && D <= 64;
    static constexpr int OW = WIDE ? 2 * D : D;  // TMEM columns of O
    __host__ __device__ static constexpr uint32_t col_o(int t) { return 2 * BN + t * OW; }
    static_assert(2 * BN + 2 * OW <= 512, "TMEM columns");
    // P's words of the 16 keys of k-step s, relative to S: packed, or, for pairs, the hi words of 32 keys and then the lo.
    __host__ __device__ static constexpr uint32_t col_p(int s) { return SPLIT ? 32 * (s >> 1) + 8 * (s & 1) : 8 * s; }
};

// A work item, or, where the line of work was cut, a part of one: the steps
// from the shift-th key on.
struct Item {
    int q0, nq, nk;   // the sequence's first row, its rows and keys
    int k0, shift;    // the first key row here, and how many of the sequence lie before it
    int hk;           // key head
    int r0;           // first row of the item among the sequence's nq * G
    int n0, n1;       // steps of each row tile
    int slot;         // where a part's sums go; -1: the item is whole
    int valid;
    __device__ __forceinline__ int n(int t) const { return t ? n1 : n0; }
};

// An item whose parts packed_join adds.
struct Join {
    int first_cta;  // holds the item's first part; -1: this CTA ends no item that others began
    int q0, nq, hk, r0;
};

// A border of the line of work: before step `tile` of item `item` (numbered
// through the key heads).
struct Border {
    int item, tile;
};

// Small problems: the items of one key head and their running cost, while a
// CTA looks for its part of the line.
constexpr int PLAN = N_THREADS;
struct Plan {
    int2 seq[PLAN];   // rows and keys of each sequence
    int item0[PLAN];  // its first item
    int cost[PLAN];   // running cost of the items
    int warp_sum[N_THREADS / 32];
};

template <class T, int D>
struct Smem {
    using C = Cfg<T, D>;
    alignas(1024) uint8_t q[2][C::Q_BYTES];
    union {
        alignas(1024) uint8_t kv[C::STAGES][C::KV_BYTES];
        Plan plan;  // before the first copy
    };
    uint64_t raw_full[C::STAGES];  // f32: the copy has landed
    uint64_t q_full[2], q_empty[2];
    uint64_t s_full[2], p_ready[2][2], o_full[2];  // by row tile (and half)
    uint64_t kv_full[C::STAGES], kv_empty[C::STAGES];
    uint64_t item_full[ITEMS], item_empty[ITEMS];
    uint64_t tail, drain;
    Item items[ITEMS];
    Border from, to;  // the CTA's part of the line
    int first_cta;    // of the item that `from` cuts
    int head_items;   // items of a key head
    int from_hk, from_seq, from_i;  // the item at `from`: key head, sequence, item of the sequence
    uint8_t unit_q[2][2][BM];   // f32: the exponents that go back into Q's rows, by row tile, of its items in turn
    float unit_kv[UNITS];      // and the factors of the K and V tiles, in their order
    uint32_t most[2][4];         // the loader warps' largest magnitudes of a tile
    alignas(16) uint8_t out[C::OUT_BYTES > 0 ? C::OUT_BYTES : 16];
    uint32_t tmem_slot;
};

struct Params {
    CUtensorMap tk, tv;
    PackedArgs a;
    int G;     // query heads of a key head
    uint32_t inv_g;  // 2^32 / G + 1
    float c;   // |scale| log2(e)
    int flip;  // scale < 0: the rows of Q are negated
    int line;  // a small problem
    float4* part_o;   // [2 * CTAs][D / 4][256 rows]: a CTA's part that began before it (0) or begins in it (1)
    float* part_lse;  // [2 * CTAs][256 rows]: log2 of the rows' sums
    Join* joins;      // [CTAs]
    // x / G: x inv_g / 2^32 is too large by less than x / 2^32, which shows from x = 2^32 / G on, by one.
    __device__ __forceinline__ int div(int x) const {
        if (G == 1) return x;
        const uint32_t y = __umulhi(x, inv_g);
        return static_cast<int>(y - (y * G > static_cast<uint32_t>(x) ? 1u : 0u));
    }
};

// ---------------------------------------------------------------- items
// A row's keys: the first of its sequence, so many.
__device__ __forceinline__ int row_seen(int nq, int nk, int token, int causal) {
    return causal ? min(max(token + nk - nq + 1, 0), nk) : nk;
}

// Steps of the row tile of rows r .. r + 127 of a sequence's nq * G.
template <int BN>
__device__ __forceinline__ int key_tiles(int nq, int nk, int G, int causal, int r) {
    const int last = min(nq * G, r + BM) - 1;
    return last < r ? 0 : (row_seen(nq, nk, last / G, causal) + BN - 1) / BN;
}

// How many of a sequence's items take at least c steps.
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

// Items in order of their steps, longest first, dealt to the CTAs in
// snake order: item k is in round k / CTAs.  A warp finds the k-th without a list: the
// count of items with at least c steps is a sum over the sequences, and c
// only falls as k grows.
template <int BN>
struct ItemFinder {
    const PackedArgs& a;
    int G, lane, level, total;

    __device__ __forceinline__ int count(int c) const {
        int n = 0;
#pragma unroll 1
        for (int s = lane; s < a.S; s += 32) {
            const int2 q = seq_rows(a.cu_q, s, a.Nq), k = seq_rows(a.cu_k, s, a.Nk);
            n += items_at_least<BN>(q.y - q.x, k.y - k.x, G, a.causal, c);
        }
        return __reduce_add_sync(0xffffffffu, n) * a.Hkv;
    }
    __device__ __forceinline__ void start() {
        int nk = 0;
        long items = 0;
#pragma unroll 1
        for (int s = lane; s < a.S; s += 32) {
            const int2 q = seq_rows(a.cu_q, s, a.Nq), k = seq_rows(a.cu_k, s, a.Nk);
            nk = max(nk, k.y - k.x);
            items += static_cast<long>(items_at_least<BN>(q.y - q.x, k.y - k.x, G, a.causal, 0)) * a.Hkv;
        }
        level = (__reduce_max_sync(0xffffffffu, nk) + BN - 1) / BN;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) items += __shfl_xor_sync(0xffffffffu, items, o);
        total = items <= INT_MAX ? static_cast<int>(items) : 0;  // (ascending offsets make no more)
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
        int rank = k - count(level + 1);  // among the items of exactly `level` steps
#pragma unroll 1
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
        it.shift = 0;
        it.slot = -1;
        it.n0 = key_tiles<BN>(it.nq, it.nk, G, a.causal, it.r0);
        it.n1 = key_tiles<BN>(it.nq, it.nk, G, a.causal, it.r0 + BM);
        return it;
    }
};

// All items as one line of steps, ITEM_COST more for each (its rows, its output), cut
// into equal parts of at least MIN_PART.  A border moves to an item's edge that is near.
constexpr int ITEM_COST = 3, MIN_PART = 5;

// Whether the line pays, by the lengths that the host knows, in steps of 128 keys.  Whole items
// end with the longest: an average prompt (a longer one has more items too, which hide it) behind
// three times the average context, as contexts differ.  Parts end with the mean, but plan
// and join cost what 5 steps do.  Dealt whole and in parts, us: one bf16 prompt of 1024 and of
// 2048, 12 heads of 64, 20.6 and 23.4, 34.3 and 29.3; 16 of 512, 12 heads on 4, 29.2 and 37.5; 8 f32
// chunks of 100 .. 1000 behind up to 3096 positions 112 and 94; three bf16 prompts of 1500 ..
// 8192, 32 heads of 128 on 8, 576 and 644 (when the rule was set).  It knows averages only: one prompt of 8192 is
// 66 us in parts, but 124 us beside 31 of 64, whole (2 heads of 64).
inline bool line_pays(const PackedArgs& a, long items, int num_sms) {
    const double nk = static_cast<double>(a.Nk) / a.S, nq = std::min(static_cast<double>(a.Nq) / a.S, nk);
    const double mean = items / static_cast<double>(num_sms) * (nk - (a.causal ? nq / 2 : 0)) / 128;
    const double longest = std::min(nq + 3 * (nk - nq), static_cast<double>(a.Nk)) / 128;
    return longest - std::max<double>(mean, MIN_PART) > 5;
}

template <int BN>
__device__ __forceinline__ int item_cost(int2 seq, int G, int causal, int item) {
    const int r = item * ITEM_ROWS;
    return ITEM_COST + max(key_tiles<BN>(seq.x, seq.y, G, causal, r), key_tiles<BN>(seq.x, seq.y, G, causal, r + BM));
}

// Running sum of x over the block's threads.
__device__ __forceinline__ int block_scan(int x, int* warp_sum, int tid) {
    const int lane = tid & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sum[tid >> 5] = x;
    __syncthreads();
    const int before = __reduce_add_sync(0xffffffffu, lane < (tid >> 5) ? warp_sum[lane] : 0);
    __syncthreads();
    return x + before;
}

// The last element of the ascending v[0 .. n-1] that is <= x (v[0] is).
__device__ __forceinline__ int last_up_to(const int* v, int n, int x) {
    int lo = 0, hi = n;
#pragma unroll 1
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The CTA's part of the line, by the whole block: fills from, to, first_cta and head_items.
template <int BN, class S>
__device__ __forceinline__ void plan_line(S& sm, const Params& p, int tid) {
    const PackedArgs& a = p.a;
    Plan& pl = sm.plan;
    int own = 0;
    if (tid < a.S) {
        const int2 q = seq_rows(a.cu_q, tid, a.Nq), k = seq_rows(a.cu_k, tid, a.Nk);
        pl.seq[tid] = make_int2(q.y - q.x, k.y - k.x);
        own = ((q.y - q.x) * p.G + ITEM_ROWS - 1) / ITEM_ROWS;
    }
    int sum = block_scan(own, pl.warp_sum, tid);
    if (tid < a.S) pl.item0[tid] = sum - own;
    if (tid == N_THREADS - 1) sm.head_items = min(sum, PLAN);  // (ascending offsets make no more)
    __syncthreads();
    const int items = sm.head_items;
    own = 0;
    if (tid < items) {
        const int s = last_up_to(pl.item0, a.S, tid);
        own = item_cost<BN>(pl.seq[s], p.G, a.causal, tid - pl.item0[s]);
    }
    sum = block_scan(own, pl.warp_sum, tid);
    if (tid < items) pl.cost[tid] = sum;
    __syncthreads();
    if (tid < 2) {  // the CTA's first border and its last; 32 bits hold the line (checked at launch)
        const int head = items > 0 ? pl.cost[items - 1] : 0, total = head * a.Hkv;
        const int ctas = min(static_cast<int>(gridDim.x), max(total / MIN_PART, 1));
        const int share = total / ctas, left = total % ctas, near = max(share / 4, 1);
        auto border = [&](int b) -> Border {
            if (b >= ctas || total == 0) return Border{items * a.Hkv, 0};
            const int at = b * share + b * left / ctas;
            const int hk = at / head, in = at - hk * head;
            int lo = -1, hi = items - 1;  // the first item whose running cost passes `in`
#pragma unroll 1
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pl.cost[mid] > in) hi = mid;
                else lo = mid;
            }
            const int start = hi > 0 ? pl.cost[hi - 1] : 0, cost = pl.cost[hi] - start, off = in - start;
            if (off <= max(near, ITEM_COST)) return Border{hk * items + hi, 0};
            if (cost - off <= near) return Border{hk * items + hi + 1, 0};
            return Border{hk * items + hi, off - ITEM_COST};
        };
        // Thread 0 goes on to the CTA where the item that its border cuts begins.
        int b = blockIdx.x + tid;
        Border y = border(b);
        if (tid == 1) sm.to = y;
        else sm.from = y;
        if (tid == 0) {
            const Border from = y;
#pragma unroll 1
            while (y.tile > 0 && y.item == from.item) y = border(--b);
            sm.first_cta = b;
            const int e = items > 0 ? from.item % items : 0;
            const int s = items > 0 && from.item < items * a.Hkv ? last_up_to(pl.item0, a.S, e) : 0;
            sm.from_seq = s;
            sm.from_i = items > 0 ? e - pl.item0[s] : 0;
            sm.from_hk = items > 0 ? from.item / items : 0;
        }
    }
    fence_async_smem();  // the plan's place is the copies' next
    __syncthreads();
}

// Walks the CTA's part of the line; a whole warp, every lane alike.
template <int BN>
struct LineWalker {
    const Params& p;
    Border at, to;
    int cta, first_cta, head_items;
    int hk, s, i, tiles;  // key head, sequence, item of the sequence and of how many
    int2 q, k;

    __device__ __forceinline__ void load(int seq) {
        s = seq;
        q = seq_rows(p.a.cu_q, s, p.a.Nq);
        k = seq_rows(p.a.cu_k, s, p.a.Nk);
        tiles = ((q.y - q.x) * p.G + ITEM_ROWS - 1) / ITEM_ROWS;
    }
    __device__ __forceinline__ void start(int hk_, int seq, int i_) {
        hk = hk_;
        i = i_;
        load(seq);
    }
    __device__ __forceinline__ Item next() {
        Item it;
        it.valid = at.item < to.item || (at.item == to.item && at.tile < to.tile);
        if (!it.valid) return it;
        it.q0 = q.x;
        it.nq = q.y - q.x;
        it.nk = k.y - k.x;
        it.hk = hk;
        it.r0 = i * ITEM_ROWS;
        const int n0 = key_tiles<BN>(it.nq, it.nk, p.G, p.a.causal, it.r0);
        const int n1 = key_tiles<BN>(it.nq, it.nk, p.G, p.a.causal, it.r0 + BM);
        const int all = max(n0, n1), t0 = at.tile, t1 = at.item == to.item ? to.tile : all;
        it.shift = t0 * BN;
        it.k0 = k.x + it.shift;
        it.n0 = max(min(n0, t1) - t0, 0);
        it.n1 = max(min(n1, t1) - t0, 0);
        it.slot = t0 == 0 && t1 == all ? -1 : 2 * cta + (t0 == 0 ? 1 : 0);
        if (t0 > 0 && t1 == all && (threadIdx.x & 31) == 0)
            p.joins[cta] = Join{first_cta, it.q0, it.nq, it.hk, it.r0};
        at = Border{at.item + 1, 0};
        ++i;
        if (at.item < to.item || (at.item == to.item && to.tile > 0)) {
            // A key head's items end by their number: offsets that descend may make more than the plan took, and
            // its last item then lies inside a sequence.  Before it, a sequence with items follows.
            const bool head_end = at.item % head_items == 0;
            if (head_end || i == tiles) {
                hk += head_end ? 1 : 0;
                i = 0;
                load(head_end ? 0 : s + 1);
                while (tiles == 0 && s + 1 < p.a.S) load(s + 1);
            }
        }
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
// 16-byte chunk, two (hi, lo, times `up`) for f32.
template <class T, int D, int PART, int BLOCK>
__device__ __forceinline__ void put8(uint8_t* base, int row, int ch, const uint4& x0, const uint4& x1, float up) {
    uint8_t* at = base + (ch >> 3) * BLOCK + swizzled<T, D>(row, ch & 7);
    if constexpr (sizeof(T) == 4) {
        uint4 hi, lo;
        const uint64_t up2 = f2_pack(up, up);
        split2_f16(f2_mul(f2_pack(__uint_as_float(x0.x), __uint_as_float(x0.y)), up2), hi.x, lo.x);
        split2_f16(f2_mul(f2_pack(__uint_as_float(x0.z), __uint_as_float(x0.w)), up2), hi.y, lo.y);
        split2_f16(f2_mul(f2_pack(__uint_as_float(x1.x), __uint_as_float(x1.y)), up2), hi.z, lo.z);
        split2_f16(f2_mul(f2_pack(__uint_as_float(x1.z), __uint_as_float(x1.w)), up2), hi.w, lo.w);
        *reinterpret_cast<uint4*>(at) = hi;
        *reinterpret_cast<uint4*>(at + PART) = lo;
    } else {
        *reinterpret_cast<uint4*>(at) = x0;
    }
}

// Row tile t of an item's Q -> shared memory, by the 128 loader threads: rows
// past the sequence's are zeros.  The first loads are in flight while free() waits
// for the place; false: it did not become free.
template <class T, int D, class F>
__device__ __forceinline__ bool load_q(const Params& p, const Item& it, int t, uint8_t* dst, uint8_t* unit_q, int tid, F free) {
    using C = Cfg<T, D>;
    constexpr int CH = D / 8, N = BM * CH / 128, V = sizeof(T) / 2;  // chunks a row, a thread; 16-byte loads a chunk
    constexpr int BATCH = N < 8 / V ? N : 8 / V;
    static_assert(N % BATCH == 0, "whole batches");
    const uint32_t flip = p.flip ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
    const int r0 = it.r0 + t * BM, rows = it.nq * p.G - r0;
    const int token0 = r0 / p.G, head0 = r0 % p.G;
    const T* base = static_cast<const T*>(p.a.q) + static_cast<long>(it.q0 + token0) * p.a.ld_q + it.hk * p.G * D;
#pragma unroll
    for (int b = 0; b < N; b += BATCH) {
        uint4 x[BATCH][V];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int u = tid + (b + i) * 128, r = u / CH, ch = u % CH;
            const int k = head0 + r, token = p.div(k);
            const T* src = base + static_cast<long>(token) * p.a.ld_q + (k - token * p.G) * D + ch * 8;
#pragma unroll
            for (int v = 0; v < V; ++v)
                x[i][v] = r < rows ? __ldg(reinterpret_cast<const uint4*>(src) + v) : make_uint4(0, 0, 0, 0);
        }
        if (b == 0 && !free()) return false;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int u = tid + (b + i) * 128, r = u / CH, ch = u % CH;
#pragma unroll
            for (int v = 0; v < V; ++v)
                x[i][v] = make_uint4(x[i][v].x ^ flip, x[i][v].y ^ flip, x[i][v].z ^ flip, x[i][v].w ^ flip);
            float up = 1.f;
            if constexpr (C::SPLIT) {
                uint32_t most = 0;
#pragma unroll
                for (int v = 0; v < V; ++v)
                    most = max(most, max(max(x[i][v].x & 0x7FFFFFFFu, x[i][v].y & 0x7FFFFFFFu),
                                         max(x[i][v].z & 0x7FFFFFFFu, x[i][v].w & 0x7FFFFFFFu)));
#pragma unroll
                for (int o = CH / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                const float unit = unit_2_14(most);
                up = inverse_of_power(unit);
                if (ch == 0) unit_q[r] = static_cast<uint8_t>(__float_as_uint(unit) >> 23);
            }
            put8<T, D, C::Q_PART, C::Q_BLOCK>(dst, r, ch, x[i][0], x[i][V - 1], up);
        }
    }
    return true;
}

// A K or V tile of f32 rows as the copy lands it (blocks of 64 columns, 32 at
// D = 32, row-major) -> the same bytes as swizzled f16 hi rows and lo rows, by the
// 128 loader threads: all read before any writes.  Rows from `rows` on, the next
// sequence's, become zeros: their weights are zero, and zero times an infinity is not.
template <int D>
struct F32Tile {
    using C = Cfg<float, D>;
    static constexpr int W = D < 64 ? D : 64, Q4 = W / 4;           // columns and float4 of a block's row
    static constexpr int N = C::BN * Q4 / 128;                      // float4 of a block for a thread
    float4 x[C::BLOCKS][N];
    __device__ __forceinline__ void read(const uint8_t* tile, int rows, int tid) {
#pragma unroll
        for (int b = 0; b < C::BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int f = tid + i * 128;
                x[b][i] = reinterpret_cast<const float4*>(tile + b * C::KV_BLOCK)[f];
                if (f / Q4 >= rows) x[b][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
    }
    __device__ __forceinline__ uint32_t most() const {  // the bits of the largest magnitude but NaN
        float m = 0.f;
#pragma unroll
        for (int b = 0; b < C::BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                m = fmaxf(m, fmaxf(fabsf(x[b][i].x), fabsf(x[b][i].y)));
                m = fmaxf(m, fmaxf(fabsf(x[b][i].z), fabsf(x[b][i].w)));
            }
        return __float_as_uint(m);
    }
    __device__ __forceinline__ void write(uint8_t* tile, float up, int tid) const {
        const uint64_t up2 = f2_pack(up, up);
#pragma unroll
        for (int b = 0; b < C::BLOCKS; ++b)
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int f = tid + i * 128, r = f / Q4, c4 = f % Q4;
                uint2 h, l;
                split2_f16(f2_mul(f2_pack(x[b][i].x, x[b][i].y), up2), h.x, l.x);
                split2_f16(f2_mul(f2_pack(x[b][i].z, x[b][i].w), up2), h.y, l.y);
                uint8_t* at = tile + b * C::KV_BLOCK + swizzled<float, D>(r, c4 >> 1) + (c4 & 1) * 8;
                *reinterpret_cast<uint2*>(at) = h;
                *reinterpret_cast<uint2*>(at + C::KV_PART) = l;
            }
    }
};

template <class T, int D>
__device__ __forceinline__ uint64_t k_major(uint32_t addr) {
    if constexpr (D == 32) return smem_desc_sw64(addr, 512);
    else return smem_desc(addr, 16, 1024);
}

// S = Q_t K^T of the K tile at `k`: 16 columns of d a k-step.
template <class T, int D>
__device__ __forceinline__ void issue_s(uint32_t out, uint32_t q, uint32_t k, uint32_t elected) {
    using C = Cfg<T, D>;
    constexpr uint32_t id = C::BF16 ? idesc_bf16(BM, C::BN, 0, 0) : idesc_f16(BM, C::BN, 0, 0);
    const uint64_t qd = k_major<T, D>(q), kd = k_major<T, D>(k);
    // The products with a lo first: each sum is rounded to the size that it has by then.
#pragma unroll
    for (int part = C::SPLIT ? 2 : 0; part >= 0; --part)
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            const uint32_t qo = (s >> 2) * C::Q_BLOCK + (s & 3) * 32 + (part == 2 ? C::Q_PART : 0);
            const uint32_t ko = (s >> 2) * C::KV_BLOCK + (s & 3) * 32 + (part == 1 ? C::KV_PART : 0);
            if (s == 0 && part == (C::SPLIT ? 2 : 0)) mma_ss_elected<false>(out, desc_add(qd, qo), desc_add(kd, ko), id, elected);
            else mma_ss_elected<true>(out, desc_add(qd, qo), desc_add(kd, ko), id, elected);
        }
}

// O_t (+)= P V of half h of the V tile at `v`: 16 keys a k-step; P's hi (and lo) words lie over S, at `ph`.  Of a
// wide O the first half takes hi hi, the second the products with a lo, so that the larger is rounded less often.
template <class T, int D>
__device__ __forceinline__ void issue_pv(uint32_t out, uint32_t ph, uint32_t v, int h, bool first, uint32_t elected) {
    using C = Cfg<T, D>;
    constexpr uint32_t id = C::BF16 ? idesc_bf16(BM, C::OW, 0, 1) : idesc_f16(BM, C::OW, 0, 1);
    constexpr uint32_t id_lo = idesc_f16(BM, D, 0, 1), to_lo = C::WIDE ? D : 0;
    constexpr uint32_t lbo = C::WIDE ? C::KV_PART : C::KV_BLOCK;
    const uint64_t vd = D == 32 ? smem_desc_sw64(v, 512, lbo) : smem_desc(v, lbo, 1024);
#pragma unroll
    for (int k = 0; k < HALF / 16; ++k) {
        const int s = h * (HALF / 16) + k;
        const uint32_t o = s * 16 * C::ROW, ps = ph + C::col_p(s);
        mma_ts_elected(out, ps, desc_add(vd, o), id, s > 0 ? 1u : first ? 0u : 1u, elected);
        if constexpr (C::SPLIT && !C::WIDE) mma_ts_elected(out, ps, desc_add(vd, o + C::KV_PART), id, 1, elected);
        if constexpr (C::SPLIT) mma_ts_elected(out + to_lo, ps + 16, desc_add(vd, o), id_lo, 1, elected);
    }
}

// ---------------------------------------------------------------- softmax
// O's columns times f, few at a time: the scores are held meanwhile.
template <int N>
__device__ __forceinline__ void scale_o(uint32_t at, float f) {
#pragma unroll 1
    for (int q = 0; q < N; q += 16) {
        float o[16];
        uint32_t r[16];
        tmem_ld16(at + q, o);
        tmem_wait_ld();
#pragma unroll
        for (int u = 0; u < 16; ++u) r[u] = __float_as_uint(o[u] * f);
        tmem_st16(at + q, r);
    }
}

// The largest, or a NaN.
template <int N>
__device__ __forceinline__ float row_max(const float (&s)[N]) {
    float mx[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) mx[q] = max_nan(s[q], s[q + 8]);
#pragma unroll
    for (int q = 16; q < N; q += 16)
#pragma unroll
        for (int u = 0; u < 8; ++u) mx[u] = max3_nan(mx[u], s[q + u], s[q + 8 + u]);
    return max_nan(max3_nan(max3_nan(mx[0], mx[1], mx[2]), mx[3], mx[4]), max3_nan(mx[5], mx[6], mx[7]));
}

// N columns of this thread's row of O; of a wide O, the sum of its halves.
template <bool WIDE, int D, int N>
__device__ __forceinline__ void load_o(uint32_t at, float (&o)[N]) {
    float y[WIDE ? N : 1];
    if constexpr (N == 32) tmem_ld32(at, o);
    else tmem_ld16(at, o);
    if constexpr (WIDE) {
        if constexpr (N == 32) tmem_ld32(at + D, y);
        else tmem_ld16(at + D, y);
    }
    tmem_wait_ld();
    if constexpr (WIDE) {
#pragma unroll
        for (int u = 0; u < N; ++u) o[u] += y[u];
    }
}

// N neighbouring columns of an output row, rounded once.
template <class T, int N>
__device__ __forceinline__ void store_row(void* out, const float (&o)[N]) {
    uint4* dst = reinterpret_cast<uint4*>(out);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int u = 0; u < N / 4; ++u)
            dst[u] = make_uint4(__float_as_uint(o[4 * u]), __float_as_uint(o[4 * u + 1]), __float_as_uint(o[4 * u + 2]),
                                __float_as_uint(o[4 * u + 3]));
    } else {
#pragma unroll
        for (int u = 0; u < N / 8; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                w[x] = std::is_same_v<T, __half> ? pack_f16(o[8 * u + 2 * x], o[8 * u + 2 * x + 1])
                                                 : pack_bf16(o[8 * u + 2 * x], o[8 * u + 2 * x + 1]);
            dst[u] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
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
            for (int h = 0; h < 2; ++h) mbar_init(&sm.p_ready[i][h], 4);
            mbar_init(&sm.o_full[i], 1);
        }
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&sm.kv_full[i], C::SPLIT ? 128 : 1);
            mbar_init(&sm.raw_full[i], 1);
            mbar_init(&sm.kv_empty[i], 1);
        }
        for (int i = 0; i < ITEMS; ++i) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], 14);  // softmax 8, loader 4, MMA, TMA
        }
        mbar_init(&sm.tail, 1);
        mbar_init(&sm.drain, 1);
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();
    if (p.line) plan_line<BN>(sm, p, tid);
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
        regs_to<C::R_SOFT, LAUNCH_REGS>();
        const int t = warp >> 2;
        const int rl = (warp & 3) * 32 + lane;
        const uint32_t lb = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = lb + tm + C::col_s(t), to = lb + tm + C::col_o(t);
        int g = 0, done = 0;  // steps and items of this row tile so far
        int kv = 0;           // f32: K and V tiles before the item's
        for (int i = 0;; ++i) {
            Item it;
            if (!get_item(i, it)) {
                failed = true;
                break;
            }
            if (!it.valid) break;
            const int row = it.r0 + t * BM + rl;
            const bool mine = row < it.nq * p.G;
            const int token = row / p.G;
            const int seen = mine ? row_seen(it.nq, it.nk, token, p.a.causal) - it.shift : 0;
            const int n = it.n(t);
            float mu = -INFINITY, l = 0.f;  // mu in the exponent's units
            float c = p.c;     // f32: times the power of two of the row of Q
            float unit = 1.f;  // f32: the power of two that V and O are counted in
            for (int j = 0; j < n; ++j, ++g) {
                if (!mbar_wait_busy_warp(&sm.s_full[t], g & 1, limit)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                float s[BN];
#pragma unroll
                for (int q = 0; q < BN / 32; ++q) tmem_ld32(ts + 32 * q, reinterpret_cast<float(&)[32]>(s[32 * q]));
                tmem_wait_ld();
                const int lim = seen - j * BN;  // visible columns of these
                if (__any_sync(0xffffffffu, lim < BN)) {
#pragma unroll
                    for (int q = 0; q < BN; ++q) s[q] = q < lim ? s[q] : -INFINITY;
                }
                float cs = c;
                if constexpr (C::SPLIT) {
                    if (j == 0) c = p.c * __uint_as_float(static_cast<uint32_t>(sm.unit_q[t][done & 1][rl]) << 23);
                    cs = fmaxf(c * sm.unit_kv[(kv + 2 * j) % UNITS], 1e-37f);  // positive: a masked score stays -inf
                }
                const float m = row_max<BN>(s) * cs;
                float f = 1.f;  // for O, before this step's products join it
                if (j == 0) {
                    mu = m;
                } else {
                    const bool raise = !(m <= mu + RESCALE_LOG2);  // a NaN too
                    if (__any_sync(0xffffffffu, raise)) {
                        f = raise ? ex2(mu - m) : 1.f;
                        mu = raise ? m : mu;
                        l *= f;
                    }
                }
                // A row of nothing yet has zeros; one with an infinite score is a NaN throughout.
                const float off = mu == -INFINITY ? 0.f : mu == INFINITY ? __uint_as_float(0x7FC00000u) : C::W_UP - mu;
                const uint64_t c2 = f2_pack(cs, cs), off2 = f2_pack(off, off);
                uint64_t sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
#pragma unroll
                for (int q = 0; q < BN / 32; ++q) {
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        const uint64_t z = f2_fma(f2_pack(s[32 * q + 2 * u], s[32 * q + 2 * u + 1]), c2, off2);
                        float x, y;
                        if (!C::SPLIT && u % 8 < POLY) {
                            exp2_poly(z, x, y);
                        } else {
                            f2_unpack(z, x, y);
                            x = ex2(x);
                            y = ex2(y);
                        }
                        if (u & 1) sum1 = f2_add(sum1, f2_pack(x, y));
                        else sum0 = f2_add(sum0, f2_pack(x, y));
                        if constexpr (C::SPLIT) split2_f16(f2_pack(x, y), hi[u], lo[u]);
                        else if constexpr (C::BF16) hi[u] = pack_bf16(x, y);
                        else hi[u] = pack_f16(x, y);
                    }
                    const uint32_t at = ts + C::col_p(2 * q);
                    tmem_st16(at, hi);
                    if constexpr (C::SPLIT) tmem_st16(at + 16, lo);
                    if ((q + 1) % (HALF / 32) == 0) {
                        if constexpr (C::SPLIT) {
                            // V's unit may have risen.
                            if (q == HALF / 32 - 1) {
                                const int x = kv + 2 * j + 1;
                                if (!mbar_wait_busy_warp(&sm.kv_full[x % C::STAGES], x / C::STAGES & 1, limit)) failed = true;
                                const float now = sm.unit_kv[x % UNITS];
                                if (j > 0) f *= unit * inverse_of_power(now);
                                unit = now;
                            }
                        }
                        if (q == HALF / 32 - 1 && __any_sync(0xffffffffu, f != 1.f)) scale_o<C::OW>(to, f);
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.p_ready[t][q / (HALF / 32)]);
                    }
                }
                float a0, a1;
                f2_unpack(f2_add(sum0, sum1), a0, a1);
                l += a0 + a1;
                if (failed) break;
            }
            if (failed) break;
            kv += 2 * max(it.n0, it.n1);
            if (n > 0) {
                if (!mbar_wait_busy_warp(&sm.o_full[t], done & 1, limit)) {
                    failed = true;
                    break;
                }
                ++done;
                tc_fence_after();
            }
            const float inv = l == 0.f ? 0.f : unit / l;
            const float lse = l == 0.f ? -INFINITY : mu - C::W_UP + log2f(l);
            if (it.slot >= 0) {
                // A part: normalised, columns in fours so that neighbouring rows' stores touch.
                const int r = t * BM + rl;
                float4* dst = p.part_o + static_cast<long>(it.slot) * (D / 4) * ITEM_ROWS + r;
                p.part_lse[static_cast<long>(it.slot) * ITEM_ROWS + r] = lse;
                if (n > 0) {
#pragma unroll 1
                    for (int q = 0; q < D / 32; ++q) {
                        float o[32];
                        load_o<C::WIDE, D>(to + 32 * q, o);
#pragma unroll
                        for (int u = 0; u < 8; ++u)
                            dst[(8 * q + u) * ITEM_ROWS] =
                                make_float4(o[4 * u] * inv, o[4 * u + 1] * inv, o[4 * u + 2] * inv, o[4 * u + 3] * inv);
                    }
                }
                continue;
            }
            // Output: normalised, rounded once; rows that saw nothing are zeros.
            const int h = it.hk * p.G + row % p.G;
            T* out = static_cast<T*>(p.a.o) + static_cast<long>(it.q0 + token) * p.a.ld_o + h * D;
            if (mine)
                p.a.lse[static_cast<long>(h) * p.a.Nq + it.q0 + token] = lse * kLn2;
            if constexpr (C::OUT_BYTES > 0) {
                constexpr int W = 64 / static_cast<int>(sizeof(T));  // columns of a stretch
                uint8_t* stage = sm.out + warp * 32 * C::OUT_PITCH;
                const uint64_t mine_at = mine ? reinterpret_cast<uint64_t>(out) : 0;
                uint64_t at[4];  // rows 8 k + lane / 4, whose stretches this lane stores a quarter of
#pragma unroll
                for (int k = 0; k < 4; ++k) at[k] = __shfl_sync(0xffffffffu, mine_at, 8 * k + (lane >> 2));
#pragma unroll 1
                for (int q = 0; q < D / W; ++q) {
                    float o[W];
                    if (n > 0) load_o<C::WIDE, D>(to + W * q, o);
#pragma unroll
                    for (int u = 0; u < W; ++u) o[u] = l == 0.f ? 0.f : o[u] * inv;
                    store_row<T, W>(stage + lane * C::OUT_PITCH, o);
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint4 x = *reinterpret_cast<const uint4*>(stage + (8 * k + (lane >> 2)) * C::OUT_PITCH + 16 * (lane & 3));
                        if (at[k]) reinterpret_cast<uint4*>(at[k] + 64 * q)[lane & 3] = x;
                    }
                    __syncwarp();
                }
            } else {
#pragma unroll 1
                for (int q = 0; q < D / 32; ++q) {
                    float o[32];
                    if (n > 0) load_o<C::WIDE, D>(to + 32 * q, o);
                    if (mine) {
#pragma unroll
                        for (int u = 0; u < 32; ++u) o[u] = l == 0.f ? 0.f : o[u] * inv;
                        store_row<T, 32>(out + 32 * q, o);
                    }
                }
            }
        }
    } else if (warp < MMA_WARP) {
        // ------------------------------------------------------------ loaders
        regs_to<C::R_LOAD, LAUNCH_REGS>();
        const int lt = tid - 32 * LOAD_WARP;
        uint32_t used = 0, phase = 0, turn = 0;  // by row tile: whether Q_t was used before, its phase, its scales' turn
        int kv = 0;
        Item it;
        for (int i = 0; !failed; ++i) {
            if (!get_item(i, it)) {
                failed = true;
                break;
            }
            if (!it.valid) break;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
                if (it.n(t) == 0) continue;
                // Q_t is free once the last S of the item that used it is done.
                const bool again = (used >> t) & 1;
                const uint32_t ph = (phase >> t) & 1;
                if (!load_q<T, D>(p, it, t, sm.q[t], sm.unit_q[t][turn >> t & 1], lt, [&] {
                        return !again || mbar_wait_busy_warp(&sm.q_empty[t], ph, limit);
                    })) {
                    failed = true;
                    break;
                }
                if (again) phase ^= 1u << t;
                used |= 1u << t;
                turn ^= 1u << t;
                fence_async_smem();
                mbar_arrive(&sm.q_full[t]);
            }
            if constexpr (C::SPLIT) {
                // K_0, V_0, K_1, ...: each converted in place once it has landed.
                const int n = max(it.n0, it.n1);
                float unit_v = 0.f;  // rises only, with room for V tiles up to four times the first
                for (int x = 0; x < 2 * n && !failed; ++x, ++kv) {
                    const int st = kv % C::STAGES;
                    const bool ok = mbar_wait_busy(&sm.raw_full[st], (kv / C::STAGES) & 1, limit);
                    F32Tile<D> tile;
                    tile.read(sm.kv[st], it.nk - it.shift - (x >> 1) * BN, lt);
                    const uint32_t own = __reduce_max_sync(0xffffffffu, ok ? tile.most() : GAVE_UP);
                    if (lane == 0) sm.most[kv & 1][warp - LOAD_WARP] = own;
                    named_sync(1, 128);
                    const uint32_t* w = sm.most[kv & 1];
                    const uint32_t most = max(max(w[0], w[1]), max(w[2], w[3]));
                    if (most == GAVE_UP) {
                        failed = true;
                        break;
                    }
                    float unit = unit_2_14(most);
                    if (x & 1) unit = unit_v = x == 1 || unit > unit_v ? 4.f * unit : unit_v;
                    if (lt == 0) sm.unit_kv[kv % UNITS] = unit;
                    tile.write(sm.kv[st], inverse_of_power(unit), lt);
                    fence_async_smem();
                    mbar_arrive(&sm.kv_full[st]);
                }
            }
        }
    } else {
        regs_to<C::R_SERV, LAUNCH_REGS>();
        if (warp == MMA_WARP) {
            // -------------------------------------------------------- MMA issuer
            // The whole warp walks in step and one lane issues; counts come from reductions, whose results are
            // uniform to the compiler too.
            const uint32_t one = elect_one();
            const uint32_t q0 = smem_u32(sm.q[0]), q1 = smem_u32(sm.q[1]), kv0 = smem_u32(sm.kv[0]);
            //
            // Per step and row tile: O += P V of the step before, then S of the step.  One copy of that code, for code
            // size: short calls are bound by fetching instructions.
            int st = 0;          // ring: the stage of V(j - 1), or of K(0), and its phase
            uint32_t phase = 0, q_phase = 0, p_phase = 0;  // the latter two by row tile
            auto stage_full = [&](int at, uint32_t ph) { return mbar_wait_busy_warp(&sm.kv_full[at], ph, limit); };
#pragma unroll 1
            for (int i = 0; !failed; ++i) {
                Item it;
                if (!get_item(i, it)) {
                    failed = true;
                    break;
                }
                if (!__reduce_max_sync(0xffffffffu, it.valid)) break;
                const int n0 = __reduce_max_sync(0xffffffffu, it.n0), n1 = __reduce_max_sync(0xffffffffu, it.n1);
                const int n = max(n0, n1);
#pragma unroll 1
                for (int j = 0; j <= n && n > 0 && !failed; ++j) {
                    // j = 0: K(0) at st.  j > 0: V(j - 1) at st and, for j < n, K(j) behind it.
                    int ks = st;
                    uint32_t k_phase = phase;
                    if (j > 0) {
                        failed = !stage_full(st, phase);
                        if (++ks == C::STAGES) ks = 0, k_phase ^= 1;
                    }
                    if (j < n && !failed) failed = !stage_full(ks, k_phase);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const int nt = t ? n1 : n0;
                        if (failed || j > nt || nt == 0) continue;
                        if (j > 0) {
#pragma unroll
                            for (int h = 0; h < C::HALVES; ++h) {
                                if (!failed) failed = !mbar_wait_busy_warp(&sm.p_ready[t][h], (p_phase >> t) & 1, limit);
                                if (failed) continue;
                                tc_fence_after();
                                issue_pv<T, D>(tm + C::col_o(t), tm + C::col_s(t), kv0 + st * C::KV_BYTES, h,
                                               h == 0 && j == 1, one);
                            }
                            if (failed) continue;
                            p_phase ^= 1u << t;
                        } else {
                            failed = !mbar_wait_busy_warp(&sm.q_full[t], (q_phase >> t) & 1, limit);
                            if (failed) continue;
                            q_phase ^= 1u << t;
                            tc_fence_after();
                        }
                        if (j < nt) {
                            issue_s<T, D>(tm + C::col_s(t), t ? q1 : q0, kv0 + ks * C::KV_BYTES, one);
                            mma_commit_elected(&sm.s_full[t], one);
                            if (j + 1 == nt) mma_commit_elected(&sm.q_empty[t], one);
                        } else {
                            mma_commit_elected(&sm.o_full[t], one);
                        }
                    }
                    // After a wait that ran out no stage goes back: its copy may still be on its way, and a second
                    // copy's arrival in the same phase of its barrier would be one too many.
                    if (failed) break;
                    if (j > 0) {
                        mma_commit_elected(&sm.kv_empty[st], one);
                        if (++st == C::STAGES) st = 0, phase ^= 1;
                    }
                    if (j < n) {
                        mma_commit_elected(&sm.kv_empty[st], one);
                        if (++st == C::STAGES) st = 0, phase ^= 1;
                    }
                }
            }
            // MMAs still in flight complete before the columns are freed.
            mma_commit_elected(&sm.drain, one);
            mbar_wait(&sm.drain, 0, 10000000ull);
            __syncwarp();
        } else if (warp == TMA_WARP) {
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
                    if (turn > 0 && !mbar_wait_busy_warp(&sm.kv_empty[st], (turn - 1) & 1, limit)) {
                        failed = true;
                        break;
                    }
                    const CUtensorMap* map = x & 1 ? &p.tv : &p.tk;
                    // A V tile past the sequence's end holds rows of the next one, whose weights are zero: those
                    // rows are cleared, as zero times an infinity or a NaN there would not be zero.
                    const int rows = it.nk - it.shift - j * BN;
                    const bool tail = !C::SPLIT && (x & 1) && rows < BN;
                    uint64_t* bar = C::SPLIT ? &sm.raw_full[st] : tail ? &sm.tail : &sm.kv_full[st];
                    if (lane == 0) {
                        mbar_arrive_expect_tx(bar, C::KV_BYTES);
#pragma unroll
                        for (int b = 0; b < C::BLOCKS; ++b)
                            if (kv != 0 || !p.a.withhold_first_key_load)
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
            // Copies still landing complete before the shared memory is released, also where it is another warp that gave
            // up (elsewhere the last tiles are waited for in any case).
#pragma unroll 1
            for (int x = max(0, kv - C::STAGES); x < kv; ++x)
                mbar_wait(C::SPLIT ? &sm.raw_full[x % C::STAGES] : &sm.kv_full[x % C::STAGES], (x / C::STAGES) & 1,
                          10000000ull);
            if (failed && tails > 0) mbar_wait(&sm.tail, (tails - 1) & 1, 10000000ull);
        } else if (warp == ITEM_WARP) {
            // -------------------------------------------------------- items
            const int ctas = gridDim.x, b = blockIdx.x;
            if (p.line && lane == 0) p.joins[b].first_cta = -1;
            ItemFinder<BN> find{p.a, p.G, lane, 0, 0};
            LineWalker<BN> walk{p, sm.from, sm.to, b, sm.first_cta, sm.head_items};
            if (p.line) walk.start(sm.from_hk, sm.from_seq, sm.from_i);
            else find.start();
            for (int i = 0;; ++i) {
                const Item it = p.line ? walk.next() : find.find(i * ctas + (i & 1 ? ctas - 1 - b : b));
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
    if (failed) {
        if (lane == 0) atomicOr(p.a.status, 1);
        if (C::SPLIT && warp >= LOAD_WARP && warp < MMA_WARP) {
            // The loaders meet at every tile: one whose wait ran out elsewhere lets the others out of their next meeting.
            if (lane < 2) sm.most[lane][warp - LOAD_WARP] = GAVE_UP;
            __syncwarp();
            named_arrive(1, 128);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA_WARP) tmem_dealloc(tm, TMEM_COLS);
}

// Adds the parts of the items that borders cut: block (c, y) the rows 32y ..
// 32y + 31, one lane each, of the item that CTA c ended.  The parts lie in the CTAs
// from the join's first to c, one each, and are added in that order; the
// block's four warps share the columns.
template <class T, int D>
__global__ void __launch_bounds__(128) packed_join(const __grid_constant__ Params p) {
    constexpr int E = D / 4;  // columns of a warp
    pdl_enter();
    const int c = blockIdx.x, r = 32 * blockIdx.y + (threadIdx.x & 31), w = threadIdx.x >> 5;
    const Join j = p.joins[c];
    const int row = j.r0 + r;
    if (j.first_cta < 0 || row >= j.nq * p.G) return;
    float acc[E], big = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int q = j.first_cta; q <= c; ++q) {
        const long slot = 2L * q + (q == j.first_cta ? 1 : 0);
        const float lse = p.part_lse[slot * ITEM_ROWS + r];
        if (lse == -INFINITY) continue;  // the row saw none of the part's keys
        const float top = fmaxf(big, lse);
        float keep = l * ex2(big - top), mine = ex2(lse - top);
        big = top;
        l = keep + mine;
        const float inv = 1.f / l;  // normalised at every step: nothing passes the largest |v|
        keep *= inv;
        mine *= inv;
        const float4* src = p.part_o + (slot * (D / 4) + w * (E / 4)) * ITEM_ROWS + r;
#pragma unroll
        for (int e = 0; e < E / 4; ++e) {
            const float4 v = src[e * ITEM_ROWS];
            acc[4 * e] = fmaf(acc[4 * e], keep, v.x * mine);
            acc[4 * e + 1] = fmaf(acc[4 * e + 1], keep, v.y * mine);
            acc[4 * e + 2] = fmaf(acc[4 * e + 2], keep, v.z * mine);
            acc[4 * e + 3] = fmaf(acc[4 * e + 3], keep, v.w * mine);
        }
    }
    const int h = j.hk * p.G + row % p.G;
    const long at = j.q0 + row / p.G;
    T* out = static_cast<T*>(p.a.o) + at * p.a.ld_o + h * D + w * E;
#pragma unroll
    for (int e = 0; e < E; e += 16 / static_cast<int>(sizeof(T))) {
        Vec16<T> y;
#pragma unroll
        for (int i = 0; i < Vec16<T>::N; ++i) y.x[i] = from_f32<T>(acc[e + i]);
        *reinterpret_cast<uint4*>(out + e) = y.raw;
    }
    if (w == 0) p.a.lse[static_cast<long>(h) * p.a.Nq + at] = l == 0.f ? -INFINITY : (big + log2f(l)) * kLn2;
}

template <class T, int D>
ProjStatus launch(const PackedArgs& a, int num_sms, cudaMemPool_t pool, cudaStream_t stream, int* launches) {
    using C = Cfg<T, D>;
    ProjStatus st;
    st.what = "packed forward launch";
    Params p{};
    p.a = a;
    p.G = a.H / a.Hkv;
    p.inv_g = p.G > 1 ? static_cast<uint32_t>((1ull << 32) / p.G) + 1 : 0;
    // A scale of zero weighs every key alike; kept positive so that a masked score stays -inf.
    p.c = fmaxf(fabsf(a.scale) * kLog2e, 1e-30f);
    p.flip = a.scale < 0.f;
    if (a.Nk > 0) {
        const long cols = static_cast<long>(a.Hkv) * D;
        const int box = D == 32 ? 32 : 64;
        bool ok;
        if constexpr (C::SPLIT) {
            ok = encode_2d(&p.tk, static_cast<const float*>(a.k), cols, a.Nk, a.ld_kv, box, C::BN) &&
                 encode_2d(&p.tv, static_cast<const float*>(a.v), cols, a.Nk, a.ld_kv, box, C::BN);
        } else {
            const CUtensorMapSwizzle sw = D == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
            ok = encode_2d_bf16(&p.tk, static_cast<const uint16_t*>(a.k), cols, a.Nk, a.ld_kv, box, C::BN, sw) &&
                 encode_2d_bf16(&p.tv, static_cast<const uint16_t*>(a.v), cols, a.Nk, a.ld_kv, box, C::BN, sw);
        }
        if (!ok) {
            st.cuda = cudaErrorInvalidValue;
            return st;
        }
    }
    auto kernel = packed_fwd<T, D>;
    constexpr size_t smem = sizeof(Smem<T, D>) + 1024;
    static_assert(smem <= SMEM_MAX, "shared memory");
    int dev = 0;
    st.cuda = cudaGetDevice(&dev);
    if (!st.ok()) return st;
    static std::atomic<uint64_t> attr_done{0};  // one bit per device
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_done.load(std::memory_order_relaxed) & bit)) {
        st.cuda = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (!st.ok()) return st;
        attr_done.fetch_or(bit);
    }
    // Each sequence ends at most one item that is not full.
    const long head_items = static_cast<long>(a.Nq) * p.G / ITEM_ROWS + a.S;
    p.line = head_items <= PLAN && line_pays(a, head_items * a.Hkv, num_sms) &&
             PLAN * static_cast<long>(a.Hkv) * (a.Nk / C::BN + ITEM_COST + 1) <= INT_MAX;
    const int ctas = p.line || head_items * a.Hkv > num_sms ? num_sms : static_cast<int>(head_items * a.Hkv);
    char* ws = nullptr;
    const size_t o_bytes = sizeof(float) * 2 * ctas * ITEM_ROWS * D, lse_bytes = sizeof(float) * 2 * ctas * ITEM_ROWS;
    if (p.line) {
        st.cuda = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&ws), o_bytes + lse_bytes + sizeof(Join) * ctas, pool, stream);
        if (!st.ok()) return st;
        p.part_o = reinterpret_cast<float4*>(ws);
        p.part_lse = reinterpret_cast<float*>(ws + o_bytes);
        p.joins = reinterpret_cast<Join*>(ws + o_bytes + lse_bytes);
    }
    st.cuda = launch_pdl(kernel, dim3(ctas), dim3(N_THREADS), smem, stream, p);
    if (st.ok()) ++*launches;
    if (p.line) {
        if (st.ok()) {
            st.cuda = launch_pdl(packed_join<T, D>, dim3(ctas, ITEM_ROWS / 32), dim3(128), 0, stream, p);
            if (st.ok()) ++*launches;
        }
        const cudaError_t freed = cudaFreeAsync(ws, stream);
        if (st.ok()) st.cuda = freed;
    }
    return st;
}

}  // namespace

ProjStatus packed_forward(const PackedArgs& a, int num_sms, cudaMemPool_t pool, cudaStream_t s, int* launches) {
    auto pick = [&](auto f32, auto bf16, auto f16) {
        return (a.dtype == KATTN_F32 ? f32 : a.dtype == KATTN_BF16 ? bf16 : f16)(a, num_sms, pool, s, launches);
    };
    return a.d == 32   ? pick(launch<float, 32>, launch<__nv_bfloat16, 32>, launch<__half, 32>)
           : a.d == 64 ? pick(launch<float, 64>, launch<__nv_bfloat16, 64>, launch<__half, 64>)
                       : pick(launch<float, 128>, launch<__nv_bfloat16, 128>, launch<__half, 128>);
}

}  // namespace kattn
