// C ABI of the serving calls (include/kerr_attn.h): argument checking and
// dispatch of packed prompts, the 8-bit paged cache and attention over it.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>

#include "kattn_internal.h"
#include "kattn_launch.h"
#include "kerr_attn.h"

using namespace kattn_abi;

namespace {

#define KATTN_TRY(expr)                \
    do {                               \
        const int _s = (expr);         \
        if (_s != KATTN_OK) return _s; \
    } while (0)

int check_dtype(int dtype) {
    if (dtype != KATTN_F32 && dtype != KATTN_BF16 && dtype != KATTN_F16)
        return fail(KATTN_ERR_UNSUPPORTED, "dtype %d unsupported (KATTN_F32, KATTN_BF16 or KATTN_F16)", dtype);
    return KATTN_OK;
}

int check_heads(int H, int Hkv, int d) {
    if (H <= 0 || Hkv <= 0) return fail(KATTN_ERR_INVALID_ARGUMENT, "head counts must be positive (%d, %d)", H, Hkv);
    if (H % Hkv != 0) return fail(KATTN_ERR_INVALID_ARGUMENT, "%d query heads do not divide into %d key heads", H, Hkv);
    if (d != 32 && d != 64 && d != 128)
        return fail(KATTN_ERR_UNSUPPORTED, "head_dim %d unsupported (32, 64 or 128)", d);
    if (static_cast<long>(H) * d > INT_MAX / 4) return fail(KATTN_ERR_INVALID_ARGUMENT, "H*d too large");
    return KATTN_OK;
}

// A [rows][cols] array of `dtype` at row stride ld.
int check_rows(const char* name, const void* p, long ld, long cols, int dtype) {
    const int size = dtype == KATTN_F32 ? 4 : 2;
    if (!p) return fail(KATTN_ERR_INVALID_ARGUMENT, "%s is NULL", name);
    if (ld < cols) return fail(KATTN_ERR_INVALID_ARGUMENT, "%s row stride %ld < %ld columns", name, ld, cols);
    if (ld > LONG_MAX / 4 / INT_MAX) return fail(KATTN_ERR_INVALID_ARGUMENT, "%s row stride %ld too large", name, ld);
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return fail(KATTN_ERR_MISALIGNED, "%s is not 16-byte aligned", name);
    if (ld * size % 16 != 0)
        return fail(KATTN_ERR_MISALIGNED, "%s row stride %ld is not a multiple of 16 bytes", name, ld);
    return KATTN_OK;
}

int check_array(const char* name, const void* p, int align) {
    if (!p) return fail(KATTN_ERR_INVALID_ARGUMENT, "%s is NULL", name);
    if (reinterpret_cast<uintptr_t>(p) % align != 0)
        return fail(KATTN_ERR_MISALIGNED, "%s is not %d-byte aligned", name, align);
    return KATTN_OK;
}

int check_counts(int S, int N) {
    if (S < 0 || N < 0) return fail(KATTN_ERR_INVALID_ARGUMENT, "negative size (S=%d N=%d)", S, N);
    if (S > INT_MAX - 256 || N > INT_MAX - 256)
        return fail(KATTN_ERR_INVALID_ARGUMENT, "problem too large (S=%d N=%d)", S, N);
    return KATTN_OK;
}

int check_cache(const kattn_kv_cache* c) {
    if (!c) return fail(KATTN_ERR_INVALID_ARGUMENT, "cache is NULL");
    if (c->format != KATTN_CACHE_INT8 && c->format != KATTN_CACHE_E4M3)
        return fail(KATTN_ERR_UNSUPPORTED, "cache format %d unsupported", c->format);
    if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)) != 0)
        return fail(KATTN_ERR_UNSUPPORTED, "page_size %d unsupported (16, 32, 64, 128 or 256)", c->page_size);
    if (c->n_pages < 0) return fail(KATTN_ERR_INVALID_ARGUMENT, "negative n_pages");
    KATTN_TRY(check_heads(c->n_kv_head, c->n_kv_head, c->d));
    if (static_cast<long>(c->n_kv_head) * c->page_size > INT_MAX)
        return fail(KATTN_ERR_INVALID_ARGUMENT, "n_kv_head * page_size too large");
    if (c->n_pages > 0) {
        KATTN_TRY(check_array("cache k", c->k, 16));
        KATTN_TRY(check_array("cache v", c->v, 16));
        KATTN_TRY(check_array("cache k_scale", c->k_scale, 16));
        KATTN_TRY(check_array("cache v_scale", c->v_scale, 16));
    }
    return KATTN_OK;
}

int check_batch(const int* cu, const int* kv_len, const int* table, long ld_table, int max_pages, int page_size) {
    KATTN_TRY(check_array("cu", cu, 4));
    KATTN_TRY(check_array("kv_len", kv_len, 4));
    if (max_pages < 0 || ld_table < max_pages)
        return fail(KATTN_ERR_INVALID_ARGUMENT, "table row stride %ld < max_pages %d", ld_table, max_pages);
    if (static_cast<long>(max_pages) * page_size > INT_MAX - 256)
        return fail(KATTN_ERR_INVALID_ARGUMENT, "max_pages * page_size too large (%d, %d)", max_pages, page_size);
    if (max_pages > 0) KATTN_TRY(check_array("table", table, 4));
    return KATTN_OK;
}

int result(const kattn::ProjStatus& st, int launches) {
    if (!st.ok()) return cuda_fail(st.cuda, st.what);
    return ok_with_launches(launches);
}

int cache_rows_checks(const kattn_ctx* ctx, const kattn_kv_cache* cache, int dtype, const void* k, const void* v,
                      long ld_kv, const int* cu, const int* kv_len, const int* table, long ld_table, int max_pages,
                      int S, int N) {
    if (!ctx) return fail(KATTN_ERR_INVALID_ARGUMENT, "ctx is NULL");
    KATTN_TRY(check_cache(cache));
    KATTN_TRY(check_dtype(dtype));
    KATTN_TRY(check_counts(S, N));
    if (S == 0 || N == 0) return KATTN_OK;
    const long cols = static_cast<long>(cache->n_kv_head) * cache->d;
    KATTN_TRY(check_rows("k", k, ld_kv, cols, dtype));
    KATTN_TRY(check_rows("v", v, ld_kv, cols, dtype));
    return check_batch(cu, kv_len, table, ld_table, max_pages, cache->page_size);
}

}  // namespace

extern "C" {
#pragma GCC visibility push(default)

int kattn_fwd_packed(kattn_ctx* ctx, int dtype, const void* q, long ld_q, const void* k, const void* v, long ld_kv,
                     void* o, long ld_o, float* lse, const int* cu_q, const int* cu_k, int S, int Nq, int Nk, int H,
                     int Hkv, int d, float scale, int causal, void* stream) {
    g_last_launches = 0;
    if (!ctx) return fail(KATTN_ERR_INVALID_ARGUMENT, "ctx is NULL");
    KATTN_TRY(check_dtype(dtype));
    KATTN_TRY(check_heads(H, Hkv, d));
    KATTN_TRY(check_counts(S, Nq));
    if (Nk < 0) return fail(KATTN_ERR_INVALID_ARGUMENT, "negative size (Nk=%d)", Nk);
    if (static_cast<long>(Nq) * H > INT_MAX - 256 || Nk > INT_MAX - 256 || static_cast<long>(S) * Hkv > INT_MAX / 2)
        return fail(KATTN_ERR_INVALID_ARGUMENT, "problem too large (Nq=%d H=%d Nk=%d S=%d)", Nq, H, Nk, S);
    if (!std::isfinite(scale)) return fail(KATTN_ERR_INVALID_ARGUMENT, "scale is not finite");
    if (causal != 0 && causal != 1) return fail(KATTN_ERR_INVALID_ARGUMENT, "causal must be 0 or 1");
    if (S == 0 || Nq == 0) return ok_with_launches(0);
    KATTN_TRY(check_rows("q", q, ld_q, static_cast<long>(H) * d, dtype));
    KATTN_TRY(check_rows("o", o, ld_o, static_cast<long>(H) * d, dtype));
    if (Nk > 0) {
        KATTN_TRY(check_rows("k", k, ld_kv, static_cast<long>(Hkv) * d, dtype));
        KATTN_TRY(check_rows("v", v, ld_kv, static_cast<long>(Hkv) * d, dtype));
    }
    KATTN_TRY(check_array("lse", lse, 4));
    KATTN_TRY(check_array("cu_q", cu_q, 4));
    KATTN_TRY(check_array("cu_k", cu_k, 4));
    DeviceScope scope(ctx->device);
    if (scope.err != cudaSuccess) return cuda_fail(scope.err, "cudaSetDevice");
    const kattn::PackedArgs a{dtype, q,  ld_q, k, v, ld_kv, o, ld_o, lse, cu_q, cu_k, S, Nq, Nk, H, Hkv, d,
                              scale, causal, ctx->d_status, ctx->wait_ns.load(std::memory_order_relaxed),
                              ctx->withhold_next_load.exchange(0)};
    int launches = 0;
    const kattn::ProjStatus st =
        kattn::packed_forward(a, ctx->num_sms, ctx->pool, static_cast<cudaStream_t>(stream), &launches);
    return result(st, launches);
}

int kattn_cache_append(kattn_ctx* ctx, const kattn_kv_cache* cache, int dtype, const void* k, const void* v,
                       long ld_kv, const int* cu, const int* kv_len, const int* table, long ld_table, int max_pages,
                       int S, int N, void* stream) {
    g_last_launches = 0;
    KATTN_TRY(cache_rows_checks(ctx, cache, dtype, k, v, ld_kv, cu, kv_len, table, ld_table, max_pages, S, N));
    if (S == 0 || N == 0) return ok_with_launches(0);
    DeviceScope scope(ctx->device);
    if (scope.err != cudaSuccess) return cuda_fail(scope.err, "cudaSetDevice");
    const kattn::CacheArgs a{*cache, cu, kv_len, table, ld_table, max_pages, S, N};
    int launches = 0;
    const kattn::ProjStatus st =
        kattn::cache_append(a, dtype, k, v, ld_kv, ctx->num_sms, static_cast<cudaStream_t>(stream), &launches);
    return result(st, launches);
}

int kattn_cache_read(kattn_ctx* ctx, const kattn_kv_cache* cache, int dtype, void* k, void* v, long ld_kv,
                     const int* cu, const int* kv_len, const int* table, long ld_table, int max_pages, int S, int N,
                     void* stream) {
    g_last_launches = 0;
    KATTN_TRY(cache_rows_checks(ctx, cache, dtype, k, v, ld_kv, cu, kv_len, table, ld_table, max_pages, S, N));
    if (S == 0 || N == 0) return ok_with_launches(0);
    DeviceScope scope(ctx->device);
    if (scope.err != cudaSuccess) return cuda_fail(scope.err, "cudaSetDevice");
    const kattn::CacheArgs a{*cache, cu, kv_len, table, ld_table, max_pages, S, N};
    int launches = 0;
    const kattn::ProjStatus st =
        kattn::cache_read(a, dtype, k, v, ld_kv, ctx->num_sms, static_cast<cudaStream_t>(stream), &launches);
    return result(st, launches);
}

int kattn_fwd_cached(kattn_ctx* ctx, const kattn_kv_cache* cache, int dtype, const void* q, long ld_q, void* o,
                     long ld_o, float* lse, const int* cu, const int* kv_len, const int* table, long ld_table,
                     int max_pages, const unsigned long long* tree, int S, int N, int H, float scale, void* stream) {
    g_last_launches = 0;
    if (!ctx) return fail(KATTN_ERR_INVALID_ARGUMENT, "ctx is NULL");
    KATTN_TRY(check_cache(cache));
    KATTN_TRY(check_dtype(dtype));
    KATTN_TRY(check_heads(H, cache->n_kv_head, cache->d));
    KATTN_TRY(check_counts(S, N));
    if (static_cast<long>(N) * H > INT_MAX - 256)
        return fail(KATTN_ERR_INVALID_ARGUMENT, "problem too large (N=%d H=%d)", N, H);
    if (!std::isfinite(scale)) return fail(KATTN_ERR_INVALID_ARGUMENT, "scale is not finite");
    if (S == 0 || N == 0) return ok_with_launches(0);
    KATTN_TRY(check_rows("q", q, ld_q, static_cast<long>(H) * cache->d, dtype));
    KATTN_TRY(check_rows("o", o, ld_o, static_cast<long>(H) * cache->d, dtype));
    KATTN_TRY(check_array("lse", lse, 4));
    KATTN_TRY(check_batch(cu, kv_len, table, ld_table, max_pages, cache->page_size));
    if (tree) KATTN_TRY(check_array("tree", tree, 8));
    DeviceScope scope(ctx->device);
    if (scope.err != cudaSuccess) return cuda_fail(scope.err, "cudaSetDevice");
    const kattn::CachedArgs a{{*cache, cu, kv_len, table, ld_table, max_pages, S, N}, dtype, q, ld_q, o, ld_o, lse,
                              tree, H, scale, ctx->d_status, ctx->wait_ns.load(std::memory_order_relaxed),
                              ctx->withhold_next_load.exchange(0)};
    int launches = 0;
    const kattn::ProjStatus st =
        kattn::cached_forward(a, ctx->num_sms, ctx->pool, static_cast<cudaStream_t>(stream), &launches);
    return result(st, launches);
}

#pragma GCC visibility pop
}  // extern "C"
