// Attention of new tokens over the 8-bit paged cache (include/kerr_attn.h,
// kattn_fwd_cached).
//
//   s_ij = scale (q_i . kc_j) ks_j,  o_i = sum_j softmax_j(s_ij) vs_j vc_j
//
// with the codes kc, vc and scales ks, vs of position j, for the positions
// that row i sees: those before the new tokens, and of the new ones the tree's.
//
// What bounds it is the cache: each byte is read once for a handful of rows,
// so the work is to keep enough copies in flight and to turn codes into
// MMA operands with few instructions.  64 bf16 sequences' one token over up to 8191
// positions, 8 key heads of 128, int8 codes, 347 MB: 86 us, 4.0 TB/s.  With more rows
// the products' instructions bound it: trees of 8 tokens, 32 rows a key head, of two
// sequences of up to 131k positions, 370 MB of e4m3: 130 us, 175 TFLOP/s.
//
// Rows.  The G query heads of a key head share its positions: a sequence's n
// tokens are n * G rows, in row tiles of 8 * NB.  Positions are the m of
// mma.m16n8k16 and rows its n, so that a tile of few rows wastes few products:
// S^T = K q^T, then O^T = V^T P^T with P^T turned in registers.
//
// Split.  The (sequence, key head, row tile) items and their tiles of positions
// are one line of work, cut into as many equal parts as there are CTAs
// (two to an SM), whatever the lengths; an item cut by a border leaves parts
// (row maxima, sums, O) in a workspace, which cached_join adds in order.  An item
// counts as EXTRA tiles more than it has: 85, 88 and 91 us for 1, 2 and 3 (the 64 sequences), 98
// and 88 for 0 and 1 when the line came in.
//
// Operands.  Codes are exact in f16, so
// only q and the weights are rounded: q to f16 after a power of two per row has
// brought its largest element near 2^13 (exact for bf16 and f16 but for elements 2^-37
// of it; f32 as a hi / lo pair), the weights p_j vs_j to f16 after a power of two
// per warp (f32: as a pair).  The scale ks_j multiplies the score.
// A weight's step is 2^-24 (f16's subnormals, a pair's too) where its largest, by the power of two, is 2^7 for
// a row's first score: with codes up to the limit L and that power at most twice the largest scale, a position
// is off by 2^-25 2^-7 2 max|v| = 2^-31 max|v| at most, whoever sees the largest.
//
// Lanes read whole 16-byte chunks of codes: the order of d in the first product
// is free (q is permuted alike), and in the second a lane's chunk spreads over
// the m of 8 MMAs, which leaves it 16 neighbouring columns of O.  tau() orders eight
// positions so that both reads meet no bank twice under the copy's swizzle.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include <cuda.h>

#include "kserve.cuh"
#include "sm100.cuh"
#include "tma_map.h"

namespace kattn {

namespace {

using namespace serve;
using namespace sm100;

constexpr int TK = 128;              // positions of a tile
constexpr int WARPS = 4;             // computing warps, 32 positions of a tile each
// A warpgroup computes; of the other, a warp walks the line of work and issues the copies, one writes results and two
// bring q into shared memory (so an item's start and end cost the computing warps little), and registers are lent.
// Two such CTAs to an SM.
constexpr int N_THREADS = 256;
constexpr int COPY_WARP = WARPS, OUT_WARP = WARPS + 1, Q_WARP = WARPS + 2, Q_WARPS = 2;
constexpr int PIECES = 4;            // ring of pieces
constexpr float RAISE = 8.f;         // a row's reference is raised when its maximum passes it by 2^8
constexpr int EXTRA = 1;             // what an item's rows, joins and stores cost, in tiles
constexpr float W_UP = 128.f;        // weights are held times 2^7: at most 2^15 with RAISE, far from f16's subnormals

// A part's place in the line of work, and what joins it.
struct Join {
    int first_cta;  // holds the item's first part; -1: this CTA ends no item that others began
    int row0, rows; // the item's first row among the sequence's n * G, and how many
    int q0, hk;
};

struct Params {
    CUtensorMap tk, tv;
    CachedArgs a;
    int page_shift, G;
    uint32_t inv_g;  // (2^32 - 1) / G
    float* part_o;   // [2 * CTAs][rows][D]: a CTA's part that began before it (0) or begins in it (1)
    float2* part_ml; // [2 * CTAs][rows]
    Join* joins;     // [CTAs]
    // x / G: the product is at most one too small.
    __device__ __forceinline__ int div(int x) const {
        const int y = static_cast<int>(__umulhi(static_cast<uint32_t>(x), inv_g));
        return y + (x - y * G >= G ? 1 : 0);
    }
};

template <int D, int NB, bool SPLIT>
struct Cfg {
    static constexpr int MR = 8 * NB;
    static constexpr int KS = D / 16;                          // k steps of the first product
    static constexpr int GR = NB * D > 256 ? 1 : 2;            // groups of 16 positions a warp takes at once (registers)
    // Registers of a computing and of another thread: 256 together (of 128 each at launch).
    static constexpr int R_COMPUTE = NB * D > 256 ? 224 : 184, R_SERVE = 256 - R_COMPUTE;
    static constexpr bool Q_SMEM = NB * D * (SPLIT ? 2 : 1) > 256;  // q in shared memory rather than registers
    static constexpr int Q_WORDS = KS * NB * (SPLIT ? 2 : 1) * 32;  // of a piece
    static constexpr int Q_SLOTS = Q_WORDS >= 1024 ? 1 : 2;
    static constexpr int FIT = (110 * 1024 - WARPS / 2 * MR * D * 4 - 8 * Q_WORDS * Q_SLOTS) / (2 * TK * (D + 4));
    static constexpr int STAGES = FIT < 6 ? FIT : 6;
    static_assert(STAGES >= 2, "stages");
};

// A stretch of an item's tiles.
struct Piece {
    int s, q0, n, len;   // sequence, its first row, rows and length
    int base;            // the first new position
    int hk, row0, rows;  // key head, first row of the row tile and how many
    int t0, t1, tiles;   // its tiles t0 .. t1-1 of the item's
    int first_cta;       // the CTA of the item's first tile
    int valid;
};

template <int D, int NB, bool SPLIT>
struct Smem {
    using C = Cfg<D, NB, SPLIT>;
    alignas(1024) uint8_t k[C::STAGES][TK * D];
    alignas(1024) uint8_t v[C::STAGES][TK * D];
    alignas(16) float ks[C::STAGES][TK];
    alignas(16) float vs[C::STAGES][TK];
    alignas(16) uint2 q[C::Q_SLOTS][C::Q_WORDS];
    alignas(16) float4 o[WARPS / 2][C::MR * D / 4];  // the warps' O on its way to one
    float f[C::Q_SLOTS][C::MR];                      // factors of the rows' scores
    float2 ml[WARPS][C::MR];                         // the warps' row maxima and sums
    float2 row[C::MR];                               // the piece's
    Piece pieces[PIECES];
    uint32_t valid[C::STAGES];  // a bit for each 16 positions: they exist
    uint64_t full[C::STAGES], empty[C::STAGES];
    uint64_t piece_full[PIECES], piece_empty[PIECES];
    uint64_t q_full[C::Q_SLOTS], q_empty[C::Q_SLOTS];
    uint64_t meet, o_full, o_empty;
};

// The position, of 8, behind column n = 2t + b of an n8 tile.
template <int D>
__device__ __forceinline__ int tau(int n) {
    const int b = n & 1, lo = (n >> 1) & 1, hi = n >> 2;
    if constexpr (D == 128) return ((b ^ hi) << 2) | (lo << 1) | hi;
    else if constexpr (D == 64) return (hi << 2) | (lo << 1) | (b ^ lo);
    else return (hi << 2) | ((b ^ hi) << 1) | lo;
}

// Byte offset of the 16-byte chunk ch of row r in a tile as the copy swizzles it.
template <int D>
__device__ __forceinline__ int chunk_at(int r, int ch) {
    if constexpr (D == 128) return r * 128 + ((ch ^ (r & 7)) << 4);
    else if constexpr (D == 64) return r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
    else return r * 32 + ((ch ^ ((r >> 2) & 1)) << 4);
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8x8 matrix of 16-bit elements whose row lane / 4 has its columns 2 (lane % 4)
// and the next in x, transposed.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}

// Codes as f16 pairs.  int8: code + 128 under 1024's exponent is 1152 + code.
// e4m3 has an instruction.  Codes arrive through prepare(), one word of four.
template <int FORMAT>
struct Codes {
    static __device__ __forceinline__ uint32_t prepare(uint32_t w) {
        return FORMAT == KATTN_CACHE_INT8 ? w ^ 0x80808080u : w;
    }
    // Bytes I and J of w (a prepared word, or two of them interleaved).
    template <int I, int J>
    static __device__ __forceinline__ uint32_t pair(uint32_t w) {
        if constexpr (FORMAT == KATTN_CACHE_INT8) {
            return sub2(prmt(w, 0x64646464u, 0x4040u | I | (J << 8)), 0x64806480u);
        } else {
            static_assert(J == I + 1 && I % 2 == 0, "a half of the word");
            uint32_t x;
            const uint16_t two = static_cast<uint16_t>(I == 0 ? w : w >> 16);
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(x) : "h"(two));
            return x;
        }
    }
};

// ---------------------------------------------------------------- the line of work
// An item counts EXTRA tiles before its own.
template <int MR>
struct Line {
    const CachedArgs& a;
    int G, lane, capacity;  // positions that the tables hold
    long at, end, total;    // the CTA's tiles, all tiles
    int ctas;
    int s, row_tiles, tiles, q0, n, len;  // current sequence
    long base;                            // its first tile

    __device__ __forceinline__ long load(int i) {  // sequence i's tiles
        const int2 r = seq_rows(a.cache.cu, i, a.cache.N);
        q0 = r.x;
        n = r.y - r.x;
        len = min(max(__ldg(a.cache.kv_len + i), 0), capacity);
        row_tiles = (n * G + MR - 1) / MR;
        tiles = max(1, (len + TK - 1) / TK);
        return sequence();
    }
    __device__ __forceinline__ long sequence() const {
        return static_cast<long>(row_tiles) * a.cache.c.n_kv_head * (tiles + EXTRA);
    }
    // Finds the CTA's part; whole warps.  The first 128 sequences are loaded once, all at the same time.
    __device__ __forceinline__ bool start(int cta, int grid) {
        constexpr int ONCE = 4;
        const int S = a.cache.S;
        long mine[ONCE], sum = 0;
#pragma unroll
        for (int c = 0; c < ONCE; ++c) mine[c] = 32 * c + lane < S ? load(32 * c + lane) : 0;
#pragma unroll
        for (int c = 0; c < ONCE; ++c) sum += mine[c];
#pragma unroll 1
        for (int i = 32 * ONCE + lane; i < S; i += 32) sum += load(i);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        total = sum;
        ctas = static_cast<int>(min(static_cast<long>(grid), total));
        if (cta >= ctas) return false;
        if (total <= 0x7FFFFFFFL / 1024) {  // 32-bit divisions
            const unsigned n = static_cast<unsigned>(total), c = static_cast<unsigned>(ctas);
            at = cta * n / c;
            end = (cta + 1) * n / c;
        } else {
            at = cta * total / ctas;
            end = (cta + 1) * total / ctas;
        }
        long before = 0;
#pragma unroll 1
        for (int i0 = 0;; i0 += 32) {
            const int i = i0 + lane;
            long run = 0;
            if (i0 < 32 * ONCE) {
#pragma unroll
                for (int c = 0; c < ONCE; ++c) run = i0 == 32 * c ? mine[c] : run;
            } else if (i < S) {
                run = load(i);
            }
            const long own = run;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long x = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += x;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, before + run > at);
            if (hit) {
                const int src = __ffs(hit) - 1;
                s = i0 + src;
                base = before + __shfl_sync(0xffffffffu, run - own, src);
                break;
            }
            before += __shfl_sync(0xffffffffu, run, 31);
        }
        load(s);
        return true;
    }
    // The next piece of the CTA's part; false: none is left.
    __device__ __forceinline__ bool next(Piece& p) {
        while (at < end) {
            long mine = sequence();
            while (at >= base + mine) {
                base += mine;
                mine = load(++s);
            }
            const long into = at - base;
            const int item = into <= 0x7FFFFFFFL ? static_cast<int>(into) / (tiles + EXTRA)
                                                 : static_cast<int>(into / (tiles + EXTRA));
            p.s = s;
            p.q0 = q0;
            p.n = n;
            p.len = len;
            p.hk = item / row_tiles;
            p.row0 = (item % row_tiles) * MR;
            p.rows = min(n * G - p.row0, MR);
            p.base = max(__ldg(a.cache.kv_len + s), 0) - n;
            p.tiles = tiles;
            const long first = base + static_cast<long>(item) * (tiles + EXTRA) + EXTRA;  // the place of its first tile
            p.t0 = static_cast<int>(max(at - first, 0L));
            p.t1 = static_cast<int>(min(static_cast<long>(tiles), end - first));
            p.first_cta = owner(first);
            at = first + p.t1;
            if (p.t1 > p.t0) return true;
            at = end;  // the border lies before the item's first tile
        }
        return false;
    }
    // The CTA that holds the line's tile g.
    __device__ __forceinline__ int owner(long g) const {
        if (total <= 0x7FFFFFFFL / 1024) {
            const unsigned n = static_cast<unsigned>(total);
            return static_cast<int>((static_cast<unsigned>(g + 1) * ctas + n - 1) / n) - 1;
        }
        return static_cast<int>(((g + 1) * ctas + total - 1) / total) - 1;
    }
};

// ---------------------------------------------------------------- rows
// Four neighbouring elements of q, as they lie (16-byte rows, so 8-byte pieces are aligned).
__device__ __forceinline__ float4 widened(const uint4& w, int) {
    return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ float4 widened(const uint2& w, int dtype) {
    if (dtype == KATTN_BF16) return make_float4(bf16_lo_f(w.x), bf16_hi_f(w.x), bf16_lo_f(w.y), bf16_hi_f(w.y));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(x.x, x.y, y.x, y.y);
}

// The largest magnitude (a NaN or an infinity above all).
template <int N>
__device__ __forceinline__ float largest(const uint4 (&w)[N], int) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < N; ++k)
        m = max(m, max(max(w[k].x & 0x7FFFFFFFu, w[k].y & 0x7FFFFFFFu), max(w[k].z & 0x7FFFFFFFu, w[k].w & 0x7FFFFFFFu)));
    return __uint_as_float(min(m, 0x7F800000u));
}
template <int N>
__device__ __forceinline__ float largest(const uint2 (&w)[N], int dtype) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) m = __vmaxu2(m, __vmaxu2(w[k].x & 0x7FFF7FFFu, w[k].y & 0x7FFF7FFFu));
    m = max(m & 0xFFFFu, m >> 16);
    if (dtype == KATTN_BF16) return __uint_as_float(min(m << 16, 0x7F800000u));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(min(m, 0x7C00u))));
}

// N (a multiple of 4) neighbouring outputs, rounded once.
template <int N>
__device__ __forceinline__ void store_out(const CachedArgs& a, long i, const float (&x)[N]) {
    if (a.dtype == KATTN_F32) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(a.o) + i);
#pragma unroll
        for (int u = 0; u < N / 4; ++u) p[u] = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
    } else {
        uint2* p = reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + i);
#pragma unroll
        for (int u = 0; u < N / 4; ++u)
            p[u] = a.dtype == KATTN_BF16
                       ? make_uint2(pack_bf16(x[4 * u], x[4 * u + 1]), pack_bf16(x[4 * u + 2], x[4 * u + 3]))
                       : make_uint2(pack_f16(x[4 * u], x[4 * u + 1]), pack_f16(x[4 * u + 2], x[4 * u + 3]));
    }
}

// ---------------------------------------------------------------- kernel
template <int D, int FORMAT, int NB, bool SPLIT>
__global__ void __launch_bounds__(N_THREADS, 2) cached_fwd(const __grid_constant__ Params p) {
    using C = Cfg<D, NB, SPLIT>;
    using Code = Codes<FORMAT>;
    constexpr int MR = C::MR, KS = C::KS, GR = C::GR;
    constexpr int CH = D >= 64 ? 16 : 8;  // bytes of K that a lane reads at once
    constexpr int KY = D / (4 * CH);      // such reads of a row
    constexpr int VB = D / 8;             // bytes of V that a lane reads of a row, columns of O that it keeps
    constexpr int NJ = VB / 2;            // MMAs of the second product, two of those columns each
    extern __shared__ uint8_t smem_raw[];
    Smem<D, NB, SPLIT>& sm =
        *reinterpret_cast<Smem<D, NB, SPLIT>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const CachedArgs& a = p.a;
    const CacheArgs& b = a.cache;

    pdl_launch();
    if (tid == 0) {
        for (int i = 0; i < C::STAGES; ++i) {
            mbar_init(&sm.full[i], 33);  // the copies' issuer and every lane's scales
            mbar_init(&sm.empty[i], WARPS);
        }
        for (int i = 0; i < PIECES; ++i) {
            mbar_init(&sm.piece_full[i], 1);
            mbar_init(&sm.piece_empty[i], WARPS + 1 + Q_WARPS);
        }
        for (int i = 0; i < C::Q_SLOTS; ++i) {
            mbar_init(&sm.q_full[i], Q_WARPS);
            mbar_init(&sm.q_empty[i], WARPS);
        }
        mbar_init(&sm.meet, WARPS);
        mbar_init(&sm.o_full, 2);
        mbar_init(&sm.o_empty, 1);
        fence_barrier_init();
    }
    __syncthreads();
    pdl_wait();

    // A wait that runs out sets the status word, and the warp leaves; the others' waits then run out too.
    auto await = [&](uint64_t* bar, uint32_t parity) {
        const bool ok = mbar_wait_warp(bar, parity, a.wait_ns);
        if (!ok && lane == 0) atomicOr(a.status, 1);
        return ok;
    };
    auto arrive = [&](uint64_t* bar) {  // once for the warp
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    const Piece* piece = nullptr;
    auto next_piece = [&](int i) {  // the i-th, for a warp that reads them
        if (!await(&sm.piece_full[i % PIECES], (i / PIECES) & 1)) return false;
        piece = &sm.pieces[i % PIECES];
        return piece->valid != 0;
    };

    if (warp >= WARPS) {
        regs_dec<C::R_SERVE>();
        if (warp == COPY_WARP) {
            // -------------------------------------------------------- the line of work, copies
            if (tid == 32 * COPY_WARP) p.joins[blockIdx.x].first_cta = -1;
            if (lane == 0 && b.c.n_pages > 0 && b.max_pages > 0) {
                prefetch_tensormap(&p.tk);
                prefetch_tensormap(&p.tv);
            }
            const int capacity = b.max_pages << p.page_shift;
            Line<MR> line{a, p.G, lane, capacity};
            const int frag_shift = min(p.page_shift, 7), frag = 1 << frag_shift;  // a stretch of a page that a copy takes
            bool more = line.start(blockIdx.x, gridDim.x);
            int st = 0, turn = 0;
            for (int i = 0;; ++i) {
                Piece x;
                more = more && line.next(x);
                x.valid = more;
                if (i >= PIECES && !await(&sm.piece_empty[i % PIECES], (i / PIECES - 1) & 1)) break;
                if (lane == 0) {
                    sm.pieces[i % PIECES] = x;
                    mbar_arrive(&sm.piece_full[i % PIECES]);
                }
                if (!more) break;
                // Lane f looks up the page of the f-th stretch, a tile ahead.
                auto page_at = [&](int tile) {
                    const int pos = tile * TK + lane * frag;
                    return lane < (TK >> frag_shift) && pos < x.len ? page_of(b, p.page_shift, x.s, pos) : -1;
                };
                int next = page_at(x.t0);
                bool ok = true;
                for (int j = x.t0; j < x.t1; ++j) {
                    const int page = next;
                    if (j + 1 < x.t1) next = page_at(j + 1);
                    const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
                    const int page16 = __shfl_sync(0xffffffffu, page, ((lane & 7) * 16) >> frag_shift);
                    const unsigned bits = __ballot_sync(0xffffffffu, page16 >= 0) & 0xFFu;
                    const int page4 = __shfl_sync(0xffffffffu, page, (lane * 4) >> frag_shift);
                    if (turn > 0 && !await(&sm.empty[st], (turn - 1) & 1)) {
                        ok = false;
                        break;
                    }
                    if (lane == 0) {
                        sm.valid[st] = bits;
                        mbar_arrive_expect_tx(&sm.full[st], __popc(there) * 2 * frag * D);
                    }
                    __syncwarp();
                    if (page >= 0 && !(a.withhold_first_key_load && i == 0 && j == x.t0)) {
                        const int row = (x.hk << p.page_shift) + ((j * TK + lane * frag) & (b.c.page_size - 1));
                        tma_load_3d(sm.k[st] + lane * frag * D, &p.tk, 0, row, page, &sm.full[st]);
                        tma_load_3d(sm.v[st] + lane * frag * D, &p.tv, 0, row, page, &sm.full[st]);
                    }
                    if (page4 >= 0) {  // scales, four of each a lane
                        const long row = ((static_cast<long>(page4) * b.c.n_kv_head + x.hk) << p.page_shift) +
                                         ((j * TK + lane * 4) & (b.c.page_size - 1));
                        cp_async16(&sm.ks[st][lane * 4], b.c.k_scale + row, 16);
                        cp_async16(&sm.vs[st][lane * 4], b.c.v_scale + row, 16);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sm.full[st]))
                                 : "memory");
                    if (++st == C::STAGES) st = 0, ++turn;
                }
                if (!ok) break;
            }
            // Copies still landing complete before the shared memory is released, also where it is another warp that gave
            // up (elsewhere they are waited for in any case).
            for (int f = 0; f < C::STAGES; ++f) {
                if (turn > 0) mbar_wait(&sm.full[st], (turn - 1) & 1, 10000000ull);
                if (++st == C::STAGES) st = 0, ++turn;
            }
        } else if (warp >= Q_WARP) {
            // -------------------------------------------------------- q
            using Raw = std::conditional_t<SPLIT, uint4, uint2>;  // four elements
            using Element = std::conditional_t<SPLIT, uint32_t, uint16_t>;
            // Operand B, row 8 nb + g: k slots (2t, 2t+1) and (2t+8, 2t+9) of step k are four neighbouring columns.
            for (int i = 0; next_piece(i); ++i) {
                const int slot = i % C::Q_SLOTS, use = i / C::Q_SLOTS;
                // The rows' lines start on their way before they are needed one by one.
                for (int r = 8 * (warp - Q_WARP) + g; r < piece->rows; r += 8 * Q_WARPS) {
                    const int row = piece->row0 + r, token = p.div(row);
                    const long at = static_cast<long>(piece->q0 + token) * a.ld_q + (piece->hk * p.G + row - token * p.G) * D;
                    const int size = SPLIT ? 4 : 2;
                    if (t * 128 < D * size)
                        asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const char*>(a.q) + at * size + t * 128));
                }
                if (use > 0 && !await(&sm.q_empty[slot], (use - 1) & 1)) return;
#pragma unroll 1
                for (int nb = warp - Q_WARP; nb < NB; nb += Q_WARPS) {
                    const int r = 8 * nb + g, row = piece->row0 + r, token = p.div(row);
                    const bool in = r < piece->rows;
                    const long at = static_cast<long>(piece->q0 + token) * a.ld_q + (piece->hk * p.G + row - token * p.G) * D;
                    Raw w[KS];
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const long i = at + 4 * CH * (k / (CH / 4)) + CH * t + 4 * (k % (CH / 4));
                        w[k] = in ? __ldg(reinterpret_cast<const Raw*>(static_cast<const Element*>(a.q) + i)) : Raw{};
                    }
                    float most = largest(w, a.dtype);
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    // The row times 2^(13 - e), e the exponent of its largest element.
                    const int e = most < INFINITY ? max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -100) : 13;
                    const float up = __uint_as_float(static_cast<uint32_t>(127 + min(13 - e, 127)) << 23);
                    const float down = __uint_as_float(static_cast<uint32_t>(127 + max(e - 13, -126)) << 23);
                    if (t == 0) sm.f[slot][r] = down * (a.scale * kLog2e);
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const float4 x = widened(w[k], a.dtype);
                        const float4 v = make_float4(x.x * up, x.y * up, x.z * up, x.w * up);
                        const uint2 hi = make_uint2(pack_f16(v.x, v.y), pack_f16(v.z, v.w));
                        sm.q[slot][(k * NB + nb) * 32 + lane] = hi;
                        if constexpr (SPLIT) {
                            const float2 h0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
                            const float2 h1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                            sm.q[slot][((KS + k) * NB + nb) * 32 + lane] =
                                make_uint2(pack_f16(v.x - h0.x, v.y - h0.y), pack_f16(v.z - h1.x, v.w - h1.y));
                        }
                    }
                }
                arrive(&sm.q_full[slot]);
                arrive(&sm.piece_empty[i % PIECES]);
            }
        } else if (warp == OUT_WARP) {
            // -------------------------------------------------------- results
            // Column VB g + 2j + u of row 8 nb + 2t + c is component 2u + c of o[.][nb, j].
            for (int i = 0; next_piece(i); ++i) {
                if (!await(&sm.o_full, i & 1)) return;
                const Piece x = *piece;
                const bool whole = x.t0 == 0 && x.t1 == x.tiles;
                const int slot = 2 * blockIdx.x + (x.t0 == 0 ? 1 : 0);
#pragma unroll 1
                for (int nb = 0; nb < NB; ++nb) {
                    const int r0 = 8 * nb + 2 * t;
                    const float2 ml[2] = {sm.row[r0], sm.row[r0 + 1]};
                    constexpr int JS = NJ < 4 ? NJ : 4;  // two columns each
#pragma unroll 1
                    for (int j0 = 0; j0 < NJ; j0 += JS) {
                        float y[2][2 * JS];
#pragma unroll
                        for (int j = 0; j < JS; ++j) {
                            const float4 v0 = sm.o[0][(nb * NJ + j0 + j) * 32 + lane];
                            const float4 v1 = sm.o[1][(nb * NJ + j0 + j) * 32 + lane];
                            y[0][2 * j] = v0.x + v1.x;
                            y[1][2 * j] = v0.y + v1.y;
                            y[0][2 * j + 1] = v0.z + v1.z;
                            y[1][2 * j + 1] = v0.w + v1.w;
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int r = r0 + c;
                            if (r >= x.rows) continue;
                            if (whole) {
                                const int row = x.row0 + r, token = p.div(row), h = x.hk * p.G + row - token * p.G;
                                const float inv = ml[c].y == 0.f ? 0.f : 1.f / ml[c].y;
#pragma unroll
                                for (int q = 0; q < 2 * JS; ++q) y[c][q] *= inv;
                                store_out<2 * JS>(a, static_cast<long>(x.q0 + token) * a.ld_o + h * D + VB * g + 2 * j0, y[c]);
                            } else {
                                float4* dst = reinterpret_cast<float4*>(p.part_o + (static_cast<long>(slot) * MR + r) * D + VB * g + 2 * j0);
#pragma unroll
                                for (int q = 0; q < JS / 2; ++q)
                                    dst[q] = make_float4(y[c][4 * q], y[c][4 * q + 1], y[c][4 * q + 2], y[c][4 * q + 3]);
                            }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int r = r0 + c;
                        if (g != 0 || r >= x.rows) continue;
                        if (whole) {
                            const int row = x.row0 + r, token = p.div(row), h = x.hk * p.G + row - token * p.G;
                            a.lse[static_cast<long>(h) * b.N + x.q0 + token] =
                                ml[c].y == 0.f ? -INFINITY : (ml[c].x + log2f(ml[c].y)) * kLn2;
                        } else {
                            p.part_ml[static_cast<long>(slot) * MR + r] = ml[c];
                        }
                    }
                }
                if (lane == 0 && x.t0 > 0 && x.t1 == x.tiles)
                    p.joins[blockIdx.x] = Join{x.first_cta, x.row0, x.rows, x.q0, x.hk};
                arrive(&sm.o_empty);
                arrive(&sm.piece_empty[i % PIECES]);
            }
        }
        return;
    }

    // ---------------------------------------------------------------- products
    regs_inc<C::R_COMPUTE>();
    // This lane's rows are 8 nb + 2t + c; the statistics of a row are the same in its eight lanes.
    int st = 0, turn = 0;  // ring of tiles
    uint32_t met = 0;      // meetings of the computing warps, their parity
    for (int i = 0; next_piece(i); ++i) {
        const int row0 = piece->row0, rows = piece->rows, base = piece->base, len = piece->len, q0 = piece->q0;
        const int t0 = piece->t0, t1 = piece->t1;
        const int slot = i % C::Q_SLOTS;
        if (!await(&sm.q_full[slot], (i / C::Q_SLOTS) & 1)) return;
        uint2 qh[C::Q_SMEM ? 1 : KS][NB], ql[SPLIT && !C::Q_SMEM ? KS : 1][NB];
        float f[NB][2];  // factors of the rows' scores
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int c = 0; c < 2; ++c) f[nb][c] = sm.f[slot][8 * nb + 2 * t + c];
            if constexpr (!C::Q_SMEM) {
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    qh[k][nb] = sm.q[slot][(k * NB + nb) * 32 + lane];
                    if constexpr (SPLIT) ql[k][nb] = sm.q[slot][((KS + k) * NB + nb) * 32 + lane];
                }
            }
        }
        if constexpr (!C::Q_SMEM) arrive(&sm.q_empty[slot]);

        float o[NB][NJ][4], m[NB][2], l[NB][2];
        float unit = 0.f, w_in = 0.f;  // a power of two, at least the largest value scale so far; 2^7 / unit
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nb][j][i] = 0.f;
        }

        for (int tile = t0; tile < t1; ++tile) {
            if (!await(&sm.full[st], turn & 1)) return;
#pragma unroll 1
            for (int step = 0; step < 2 / GR; ++step) {
                const int group = warp * 2 + step * GR;  // of 16 positions
                const int pos0 = tile * TK + group * 16;
                const uint32_t here = (sm.valid[st] >> group) & ((1u << GR) - 1u);
                if (here == 0 || pos0 >= len) continue;
                const uint8_t* kt = sm.k[st] + group * 16 * D;
                const uint8_t* vt = sm.v[st] + group * 16 * D;
                // ---- S^T = codes of K . q
                float s[GR][NB][4];
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 4; ++c) s[gr][nb][c] = 0.f;
                    uint32_t kw[2][KS];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int r = 16 * gr + 8 * u + tau<D>(g);
#pragma unroll
                        for (int y = 0; y < KY; ++y) {
                            if constexpr (CH == 16) {
                                const uint4 w = *reinterpret_cast<const uint4*>(kt + chunk_at<D>(r, 4 * y + t));
                                kw[u][4 * y] = w.x;
                                kw[u][4 * y + 1] = w.y;
                                kw[u][4 * y + 2] = w.z;
                                kw[u][4 * y + 3] = w.w;
                            } else {
                                const uint2 w = *reinterpret_cast<const uint2*>(kt + chunk_at<D>(r, t >> 1) + 8 * (t & 1));
                                kw[u][0] = w.x;
                                kw[u][1] = w.y;
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KS; ++k) {
                        const uint32_t w0 = Code::prepare(kw[0][k]), w1 = Code::prepare(kw[1][k]);
                        const uint32_t ka[4] = {Code::template pair<0, 1>(w0), Code::template pair<0, 1>(w1),
                                                Code::template pair<2, 3>(w0), Code::template pair<2, 3>(w1)};
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const uint2 h = C::Q_SMEM ? sm.q[slot][(k * NB + nb) * 32 + lane] : qh[C::Q_SMEM ? 0 : k][nb];
                            mma16816(s[gr][nb], ka, h.x, h.y);
                            if constexpr (SPLIT) {
                                const uint2 e = C::Q_SMEM ? sm.q[slot][((KS + k) * NB + nb) * 32 + lane] : ql[C::Q_SMEM ? 0 : k][nb];
                                mma16816(s[gr][nb], ka, e.x, e.y);
                            }
                        }
                    }
                }
                // ---- scores and masks
                const bool seen_all = pos0 + 16 * GR <= min(base, len) && here == (1u << GR) - 1u;
                float vs[GR][2];
                bool raise = false;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int r = 16 * gr + 8 * u + tau<D>(g);
                        const float k_s = sm.ks[st][group * 16 + r];
                        vs[gr][u] = sm.vs[st][group * 16 + r];
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                            for (int c = 0; c < 2; ++c) s[gr][nb][2 * u + c] *= k_s * f[nb][c];
                        if (!seen_all && !(pos0 + r < len && ((here >> gr) & 1))) vs[gr][u] = 0.f;  // no such position
                        raise |= vs[gr][u] > unit;
                    }
                if (!seen_all) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int mine = 8 * nb + 2 * t + c, token = p.div(row0 + mine);
                            // The new tokens that the row sees: a tree's, or all up to its own.
                            unsigned long long bits = 0;
                            if (a.tree && mine < rows && pos0 + 16 * GR > base) bits = __ldg(a.tree + q0 + token);
#pragma unroll
                            for (int gr = 0; gr < GR; ++gr)
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    const int pos = pos0 + 16 * gr + 8 * u + tau<D>(g), j = pos - base;
                                    const bool see = mine < rows && pos < len && ((here >> gr) & 1) &&
                                                     (j < 0 || (a.tree ? j < 64 && ((bits >> j) & 1) : j <= token));
                                    if (!see) s[gr][nb][2 * u + c] = -INFINITY;
                                }
                        }
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float y = fmaxf(s[0][nb][c], s[0][nb][2 + c]);
                        if constexpr (GR == 2) y = fmaxf(y, fmaxf(s[GR - 1][nb][c], s[GR - 1][nb][2 + c]));
                        raise |= y > m[nb][c] + RAISE;  // from -inf: any score
                    }
                // The references rise seldom, so only then are the warp's maxima formed.
                if (__any_sync(0xffffffffu, raise)) {
                    float most = 0.f;
#pragma unroll
                    for (int gr = 0; gr < GR; ++gr) most = fmaxf(most, fmaxf(vs[gr][0], vs[gr][1]));
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                    // unit: the next power of two.
                    const float to = most > unit ? __uint_as_float((__float_as_uint(most) + 0x7FFFFFu) & 0x7F800000u) : unit;
                    const float turn_unit = to > 0.f ? unit / to : 1.f;
                    unit = to;
                    w_in = to > 0.f ? W_UP / to : 0.f;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float y = fmaxf(s[0][nb][c], s[0][nb][2 + c]);
                            if constexpr (GR == 2) y = fmaxf(y, fmaxf(s[GR - 1][nb][c], s[GR - 1][nb][2 + c]));
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, d));
                            float r = 1.f;
                            if (y > m[nb][c] + RAISE) {
                                r = ex2(m[nb][c] - y);
                                m[nb][c] = y;
                            }
                            l[nb][c] *= r;
                            r *= turn_unit;
#pragma unroll
                            for (int j = 0; j < NJ; ++j) {
                                o[nb][j][c] *= r;
                                o[nb][j][2 + c] *= r;
                            }
                        }
                }
                // ---- weights as operand B
                uint2 ph[GR][NB], pl[SPLIT ? GR : 1][NB];
#pragma unroll
                for (int gr = 0; gr < GR; ++gr)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        uint32_t h[2], e[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float w[2];
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const float ref = m[nb][c] == -INFINITY ? 0.f : m[nb][c];
                                const float q = ex2(s[gr][nb][2 * u + c] - ref);
                                l[nb][c] += q;
                                w[c] = q * (vs[gr][u] * w_in);
                                if (!seen_all && q == 0.f) w[c] = 0.f;  // an unseen position's scale may be a NaN
                            }
                            h[u] = pack_f16(w[0], w[1]);
                            if constexpr (SPLIT) {
                                const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h[u]));
                                e[u] = pack_f16(w[0] - y.x, w[1] - y.y);
                            }
                        }
                        ph[gr][nb] = make_uint2(turned(h[0]), turned(h[1]));
                        if constexpr (SPLIT) pl[gr][nb] = make_uint2(turned(e[0]), turned(e[1]));
                    }
                // ---- O^T += codes of V^T . weights
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    uint32_t vw[4][VB / 4];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int r = 16 * gr + 8 * u + tau<D>(2 * t + c);
                            uint32_t(&to)[VB / 4] = vw[2 * u + c];
                            if constexpr (VB == 16) {
                                const uint4 w = *reinterpret_cast<const uint4*>(vt + chunk_at<D>(r, g));
                                to[0] = w.x, to[1] = w.y, to[2] = w.z, to[3] = w.w;
                            } else if constexpr (VB == 8) {
                                const uint2 w = *reinterpret_cast<const uint2*>(vt + chunk_at<D>(r, g >> 1) + 8 * (g & 1));
                                to[0] = w.x, to[1] = w.y;
                            } else {
                                to[0] = *reinterpret_cast<const uint32_t*>(vt + chunk_at<D>(r, g >> 2) + 4 * (g & 3));
                            }
                            // A place that no position has may hold e4m3's NaN, which a weight of zero does not remove.
                            if (FORMAT == KATTN_CACHE_E4M3 && !seen_all && (pos0 + r >= len || !((here >> gr) & 1))) {
#pragma unroll
                                for (int q = 0; q < VB / 4; ++q) to[q] = 0;
                            }
                        }
#pragma unroll
                    for (int q = 0; q < VB / 4; ++q) {
                        uint32_t z[2][2];  // two positions' bytes side by side: columns 4q, 4q+1 and 4q+2, 4q+3
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint32_t w0 = Code::prepare(vw[2 * u][q]), w1 = Code::prepare(vw[2 * u + 1][q]);
                            z[u][0] = prmt(w0, w1, 0x5140u);
                            z[u][1] = prmt(w0, w1, 0x7362u);
                        }
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const uint32_t va[4] = {Code::template pair<0, 1>(z[0][y]), Code::template pair<2, 3>(z[0][y]),
                                                    Code::template pair<0, 1>(z[1][y]), Code::template pair<2, 3>(z[1][y])};
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                mma16816(o[nb][2 * q + y], va, ph[gr][nb].x, ph[gr][nb].y);
                                if constexpr (SPLIT) mma16816(o[nb][2 * q + y], va, pl[gr][nb].x, pl[gr][nb].y);
                            }
                        }
                    }
                }
            }
            arrive(&sm.empty[st]);
            if (++st == C::STAGES) st = 0, ++turn;
        }
        if constexpr (C::Q_SMEM) arrive(&sm.q_empty[slot]);

        // ---- the four warps' parts into one: each scaled to the common maximum, then added in order
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nb][c] += __shfl_xor_sync(0xffffffffu, l[nb][c], d);
                if (g == 0) sm.ml[warp][8 * nb + 2 * t + c] = make_float2(m[nb][c], l[nb][c]);
            }
        arrive(&sm.meet);
        if (!await(&sm.meet, met)) return;
        met ^= 1;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float big = -INFINITY, sum = 0.f;
                float2 e[WARPS];
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    e[w] = sm.ml[w][8 * nb + 2 * t + c];
                    big = fmaxf(big, e[w].x);
                }
                const float ref = big == -INFINITY ? 0.f : big;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) sum += e[w].y * ex2(e[w].x - ref);
                const float r = ex2(m[nb][c] - ref) * unit * (1.f / W_UP);
                m[nb][c] = big;
                l[nb][c] = sum;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    o[nb][j][c] *= r;
                    o[nb][j][2 + c] *= r;
                }
            }
        // Warps 2 and 3 hand theirs to 0 and 1, whose sums the result warp adds.
        if (i > 0 && !await(&sm.o_empty, (i - 1) & 1)) return;
        float4* mine = sm.o[warp & 1];
        if (warp >= 2) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
                    mine[(nb * NJ + j) * 32 + lane] = make_float4(o[nb][j][0], o[nb][j][1], o[nb][j][2], o[nb][j][3]);
        }
        arrive(&sm.meet);
        if (!await(&sm.meet, met)) return;
        met ^= 1;
        if (warp < 2) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                if (warp == 0 && g == 0) {
                    sm.row[8 * nb + 2 * t] = make_float2(m[nb][0], l[nb][0]);
                    sm.row[8 * nb + 2 * t + 1] = make_float2(m[nb][1], l[nb][1]);
                }
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float4 y = mine[(nb * NJ + j) * 32 + lane];
                    y.x += o[nb][j][0];
                    y.y += o[nb][j][1];
                    y.z += o[nb][j][2];
                    y.w += o[nb][j][3];
                    mine[(nb * NJ + j) * 32 + lane] = y;
                }
            }
            arrive(&sm.o_full);
        }
        arrive(&sm.piece_empty[i % PIECES]);
    }
}

// Adds the parts of the items that CTAs cut: block (c, y) the rows 4y .. 4y+3,
// one warp each, of the item that CTA c ended.  The parts lie in the CTAs from
// the join's first to c, one each, and are added in that order.
template <int D, int MR>
__global__ void __launch_bounds__(128) cached_join(const __grid_constant__ Params p) {
    pdl_enter();
    const CachedArgs& a = p.a;
    const int c = blockIdx.x;
    const Join j = p.joins[c];
    const int r = 4 * blockIdx.y + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (j.first_cta < 0 || r >= j.rows) return;
    constexpr int E = D / 32;
    float acc[E], big = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int q0 = j.first_cta; q0 <= c; q0 += 32) {
        // 32 parts at a time: a lane holds one's maximum and sum.
        const int q = q0 + lane;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (q <= c) ml = p.part_ml[(2L * q + (q == j.first_cta ? 1 : 0)) * MR + r];
        float top = ml.x;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, big);
        const float ref = top == -INFINITY ? 0.f : top;
        const float keep = ex2(big - ref), w = ex2(ml.x - ref);
        big = top;
        float sum = ml.y * w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, keep, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= keep;
        const int n = min(32, c + 1 - q0);
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
            const float* src = p.part_o + ((2L * (q0 + i) + (q0 + i == j.first_cta ? 1 : 0)) * MR + r) * D + lane * E;
            float v[E];
            if constexpr (E == 4) {
                const float4 y = *reinterpret_cast<const float4*>(src);
                v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
            } else if constexpr (E == 2) {
                const float2 y = *reinterpret_cast<const float2*>(src);
                v[0] = y.x, v[1] = y.y;
            } else {
                v[0] = *src;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(wi, v[e], acc[e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int row = j.row0 + r, h = j.hk * p.G + row % p.G;
    const long at = j.q0 + row / p.G;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float y = acc[e] * inv;
        const long i = at * a.ld_o + h * D + lane * E + e;
        if (a.dtype == KATTN_F32) static_cast<float*>(a.o)[i] = y;
        else if (a.dtype == KATTN_BF16) static_cast<__nv_bfloat16*>(a.o)[i] = __float2bfloat16_rn(y);
        else static_cast<__half*>(a.o)[i] = __float2half_rn(y);
    }
    if (lane == 0) a.lse[static_cast<long>(h) * a.cache.N + at] = l == 0.f ? -INFINITY : (big + log2f(l)) * kLn2;
}

template <int D, int FORMAT, int NB, bool SPLIT>
cudaError_t launch(Params& p, int ctas, bool join, cudaStream_t stream, int* launches) {
    constexpr size_t smem = sizeof(Smem<D, NB, SPLIT>) + 1024;
    static_assert(2 * (smem + 1024) <= 228 * 1024, "two CTAs to an SM");
    auto kernel = cached_fwd<D, FORMAT, NB, SPLIT>;
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
    e = launch_pdl(kernel, dim3(ctas), dim3(N_THREADS), smem, stream, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (!join) return cudaSuccess;
    e = launch_pdl(cached_join<D, 8 * NB>, dim3(ctas, 2 * NB), dim3(128), 0, stream, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace

ProjStatus cached_forward(const CachedArgs& a, int num_sms, cudaMemPool_t pool, cudaStream_t s, int* launches) {
    const CacheArgs& b = a.cache;
    const int D = b.c.d;
    Params p{};
    p.a = a;
    p.page_shift = page_shift_of(b.c.page_size);
    p.G = a.H / b.c.n_kv_head;
    p.inv_g = 0xFFFFFFFFu / p.G;
    // Row tiles of 8, 16 or 32, the smallest that holds a sequence's rows on average: fewer row tiles read
    // the cache less often, smaller ones leave fewer idle rows.  (350 MB read for one row tile of
    // 8, 16, 32 rows: 75, 103 and 188 us when the rule was set; four tiles of 8 would read it four times.)
    const long per_seq = (static_cast<long>(b.N) * p.G + b.S - 1) / b.S;
    // (f32 rows of 128 columns stop at 16: pairs of q and O of 32 would leave no second stage.)
    const int NB = per_seq <= 8 ? 1 : per_seq <= 16 || (a.dtype == KATTN_F32 && D == 128) ? 2 : 4;
    const int MR = 8 * NB, ctas = 2 * num_sms;
    const bool join = (static_cast<long>(b.max_pages) << p.page_shift) > TK;  // else no item has two tiles
    ProjStatus st;
    const size_t o_bytes = sizeof(float) * 2 * ctas * MR * D, ml_bytes = sizeof(float2) * 2 * ctas * MR;
    char* ws = nullptr;
    st.what = "cached forward workspace";
    st.cuda = cudaMallocFromPoolAsync(reinterpret_cast<void**>(&ws), o_bytes + ml_bytes + sizeof(Join) * ctas, pool, s);
    if (!st.ok()) return st;
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(ws + o_bytes);
    p.joins = reinterpret_cast<Join*>(ws + o_bytes + ml_bytes);
    st.what = "cached forward launch";
    if (b.c.n_pages > 0 && b.max_pages > 0) {
        const CUtensorMapSwizzle sw = D == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                      : D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                : CU_TENSOR_MAP_SWIZZLE_32B;
        const int rows = std::min(b.c.page_size, TK);
        if (!encode_pages(&p.tk, b.c.k, b.c.n_pages, b.c.n_kv_head * b.c.page_size, D, rows, sw) ||
            !encode_pages(&p.tv, b.c.v, b.c.n_pages, b.c.n_kv_head * b.c.page_size, D, rows, sw))
            st.cuda = cudaErrorInvalidValue;
    }
    if (st.ok()) {
        auto pick = [&](auto d, auto fmt, auto nb, auto split) {
            if constexpr (decltype(split)::value && decltype(d)::value == 128 && decltype(nb)::value == 4)
                return cudaErrorInvalidValue;
            else
                return launch<decltype(d)::value, decltype(fmt)::value, decltype(nb)::value, decltype(split)::value>(
                    p, ctas, join, s, launches);
        };
        auto by_split = [&](auto d, auto fmt, auto nb) {
            return a.dtype == KATTN_F32 ? pick(d, fmt, nb, std::true_type{}) : pick(d, fmt, nb, std::false_type{});
        };
        auto by_nb = [&](auto d, auto fmt) {
            return NB == 1   ? by_split(d, fmt, std::integral_constant<int, 1>{})
                   : NB == 2 ? by_split(d, fmt, std::integral_constant<int, 2>{})
                             : by_split(d, fmt, std::integral_constant<int, 4>{});
        };
        auto by_format = [&](auto d) {
            return b.c.format == KATTN_CACHE_INT8 ? by_nb(d, std::integral_constant<int, KATTN_CACHE_INT8>{})
                                                  : by_nb(d, std::integral_constant<int, KATTN_CACHE_E4M3>{});
        };
        st.cuda = D == 32   ? by_format(std::integral_constant<int, 32>{})
                  : D == 64 ? by_format(std::integral_constant<int, 64>{})
                            : by_format(std::integral_constant<int, 128>{});
    }
    const cudaError_t freed = cudaFreeAsync(ws, s);
    if (st.ok()) st.cuda = freed;
    return st;
}

}  // namespace kattn
