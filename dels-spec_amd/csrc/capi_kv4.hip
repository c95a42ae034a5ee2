// C ABI of the 4-bit key/value cache (declared in include/dels.h): argument
// checks and dispatch.  Nothing here allocates device memory or synchronises.
#include <algorithm>

#include "capi_paged.h"

using namespace dels;

extern "C" {

size_t dels_kv4_page_bytes(int64_t head_dim) {
    return head_dim == 64 || head_dim == 128 ? (size_t)(66 * head_dim + 128) : 0;
}

int dels_kv4_append(const dels_kv4_cache* p, const void* k, int64_t k_batch, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_batch, int64_t v_token, int64_t v_head, int dtype,
                    const int32_t* lengths, const int32_t* counts, int64_t T, void* stream) {
    PagedCache c{};
    int rc = cache_of(p, c);
    if (rc != DELS_OK) return rc;
    if ((rc = check_type(dtype, true)) != DELS_OK) return rc;
    if (!extent_ok(T)) return fail(DELS_ERR_INVALID_ARGUMENT, "bad block length %lld", (long long)T);
    if (!grid_ok({c.batch, c.heads, T / 8 + 2}) || c.batch > 65535 || c.heads > 65535)
        return fail(DELS_ERR_UNSUPPORTED, "shape past the supported extents");
    if (c.batch == 0 || T == 0) return DELS_OK;
    if ((rc = check_rows(k, k_batch, k_token, k_head, dtype, "k")) != DELS_OK) return rc;
    if ((rc = check_rows(v, v_batch, v_token, v_head, dtype, "v")) != DELS_OK) return rc;
    if (!lengths) return fail(DELS_ERR_INVALID_ARGUMENT, "lengths is NULL");
    if (c.max_pages == 0 || c.num_pages == 0) return DELS_OK;
    const hipError_t e = launch_kv4_append(c, {k, k_batch, k_token, k_head}, {v, v_batch, v_token, v_head}, dtype,
                                           lengths, counts, (int)T, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache append launch");
}

int dels_kv4_read(const dels_kv4_cache* p, const int32_t* starts, const int32_t* counts, int64_t T, void* k, void* v,
                  int dtype, void* stream) {
    PagedCache c{};
    int rc = cache_of(p, c);
    if (rc != DELS_OK) return rc;
    if ((rc = check_type(dtype, true)) != DELS_OK) return rc;
    if (!extent_ok(T)) return fail(DELS_ERR_INVALID_ARGUMENT, "bad block length %lld", (long long)T);
    if (!grid_ok({c.batch, c.heads, T / 8 + 2}) || c.batch > 65535 || c.heads > 65535)
        return fail(DELS_ERR_UNSUPPORTED, "shape past the supported extents");
    if (c.batch == 0 || T == 0) return DELS_OK;
    if (!starts || !k || !v) return fail(DELS_ERR_INVALID_ARGUMENT, "starts, k or v is NULL");
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(DELS_ERR_ALIGNMENT, "k and v must be 16-byte aligned");
    const hipError_t e = launch_kv4_read(c, starts, counts, (int)T, k, v, dtype, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache read launch");
}

size_t dels_kv4_attention_ws_bytes(int64_t batch, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t max_pages) {
    if (!attention_ok(batch, T, q_heads, kv_heads, max_pages) || (head_dim != 64 && head_dim != 128)) return 0;
    return kDataOff + kv4_attention_data_bytes(batch, T, q_heads, kv_heads, head_dim, max_pages);
}

int dels_kv4_attention(const dels_kv4_cache* p, const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                       int dtype, int64_t q_heads, int64_t T, const int32_t* lengths, const int32_t* counts,
                       int block, const int64_t* mask, int64_t ld_mask, float scale, void* out, int64_t out_batch,
                       int64_t out_token, int64_t out_head, float* lse, void* ws, size_t ws_bytes, void* stream) {
    Kv4AttentionArgs a{};
    int rc = cache_of(p, a.cache);
    if (rc != DELS_OK) return rc;
    if (a.cache.batch == 0 || T == 0) return DELS_OK;
    rc = check_block(a.cache, q, q_batch, q_token, q_head, dtype, q_heads, T, lengths, block, mask, ld_mask, scale);
    if (rc != DELS_OK) return rc;
    if ((rc = check_rows(out, out_batch, out_token, out_head, dtype, "out")) != DELS_OK) return rc;
    if (!lse) return fail(DELS_ERR_INVALID_ARGUMENT, "lse is NULL");
    if (a.cache.num_pages == 0) a.cache.max_pages = 0;       // nothing to see
    const size_t need = dels_kv4_attention_ws_bytes(a.cache.batch, T, q_heads, a.cache.heads, a.cache.head_dim,
                                                    a.cache.max_pages);
    if ((rc = check_ws(ws, ws_bytes, need)) != DELS_OK) return rc;
    a.block = {lengths, counts, (int)T, block, mask, ld_mask};
    a.q = {q, q_batch, q_token, q_head};
    a.dtype = dtype, a.q_heads = (int)q_heads, a.scale = scale;
    a.out = out, a.out_batch = out_batch, a.out_token = out_token, a.out_head = out_head, a.lse = lse;
    const hipError_t e = launch_kv4_attention(a, ws, kDataOff, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache attention launch");
}

int dels_kv4_weights(const dels_kv4_cache* p, const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                     int dtype, int64_t q_heads, int64_t T, const int32_t* lengths, const int32_t* counts,
                     const int32_t* accepted, int block, const int64_t* mask, int64_t ld_mask, float scale,
                     const float* lse, const float* weights, float* out, void* stream) {
    Kv4WeightsArgs a{};
    int rc = cache_of(p, a.cache);
    if (rc != DELS_OK) return rc;
    if (a.cache.batch == 0 || a.cache.max_pages == 0) return DELS_OK;
    if (T == 0) {                                             // no rows: neither queries nor lse are there
        if (!lengths) return fail(DELS_ERR_INVALID_ARGUMENT, "lengths is NULL");
        if (!grid_ok({a.cache.batch, a.cache.heads, a.cache.max_pages}))
            return fail(DELS_ERR_UNSUPPORTED, "shape past the supported extents");
    } else {
        rc = check_block(a.cache, q, q_batch, q_token, q_head, dtype, q_heads, T, lengths, block, mask, ld_mask, scale);
        if (rc != DELS_OK) return rc;
        if (!lse) return fail(DELS_ERR_INVALID_ARGUMENT, "lse is NULL");
    }
    if (!weights || !out) return fail(DELS_ERR_INVALID_ARGUMENT, "weights or out is NULL");
    a.block = {lengths, counts, (int)T, block, mask, ld_mask};
    a.q = {q, q_batch, q_token, q_head};
    a.dtype = dtype, a.q_heads = (int)q_heads, a.scale = scale;
    a.accepted = accepted, a.lse = lse, a.weights = weights, a.out = out;
    const hipError_t e = launch_kv4_weights(a, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "attention weights launch");
}

size_t dels_kv4_evict_ws_bytes(int64_t batch, int64_t kv_heads, int64_t keep) {
    if (!extent_ok(batch) || !extent_ok(kv_heads) || keep < 0 || keep >= INT32_MAX ||
        !grid_ok({batch, kv_heads, keep / 8 + 1}))
        return 0;
    return kDataOff + kv4_evict_data_bytes(batch, kv_heads, keep);
}

int dels_kv4_evict(const dels_kv4_cache* p, const int32_t* lengths, const float* weights, int64_t keep, int64_t recent,
                   int32_t* out_lengths, float* out_weights, int32_t* source, void* ws, size_t ws_bytes,
                   void* stream) {
    Kv4EvictArgs a{};
    int rc = cache_of(p, a.cache);
    if (rc != DELS_OK) return rc;
    if (keep < 1 || keep >= INT32_MAX || recent < 0)
        return fail(DELS_ERR_INVALID_ARGUMENT, "bad budget keep=%lld recent=%lld", (long long)keep, (long long)recent);
    if (a.cache.batch == 0) return DELS_OK;
    if (!lengths || !out_lengths || !source || (a.cache.max_pages && (!weights || !out_weights)))
        return fail(DELS_ERR_INVALID_ARGUMENT, "lengths, weights or an output is NULL");
    if (lengths == out_lengths || (weights && weights == out_weights))
        return fail(DELS_ERR_INVALID_ARGUMENT, "an output is one of the inputs");
    if (!grid_ok({a.cache.batch, a.cache.heads, a.cache.max_pages}) || a.cache.batch > 65535 || a.cache.heads > 65535)
        return fail(DELS_ERR_UNSUPPORTED, "shape past the supported extents");
    const size_t need = dels_kv4_evict_ws_bytes(a.cache.batch, a.cache.heads, keep);
    if ((rc = check_ws(ws, ws_bytes, need)) != DELS_OK) return rc;
    a.lengths = lengths, a.weights = weights, a.keep = (int)keep;
    a.recent = (int)std::min<int64_t>(recent, keep);
    a.out_lengths = out_lengths, a.out_weights = out_weights, a.source = source;
    const hipError_t e = launch_kv4_evict(a, ws, kDataOff, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache eviction launch");
}

}  // extern "C"
