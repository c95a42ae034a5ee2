// C ABI of the 4-bit key/value cache (declared in include/dels.h): argument
// checks and dispatch.  Nothing here allocates device memory or synchronises.
#include <algorithm>
#include <initializer_list>

#include "../../include/dels.h"
#include "dels_internal.h"

namespace dels {

namespace {

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool extent_ok(int64_t x) { return x >= 0 && x < (int64_t(1) << 24); }

// Workgroups of a launch over these extents stay far below 2^31.
bool grid_ok(std::initializer_list<int64_t> xs) {
    int64_t total = 1;
    for (int64_t x : xs) {
        if (x > 0 && total > (int64_t(1) << 30) / x) return false;
        total *= std::max<int64_t>(x, 1);
    }
    return true;
}

int cache_of(const dels_kv4_cache* p, Kv4Cache& c) {
    if (!p) return fail(DELS_ERR_INVALID_ARGUMENT, "cache is NULL");
    if (p->head_dim != 64 && p->head_dim != 128)
        return fail(DELS_ERR_UNSUPPORTED, "cache head size must be 64 or 128 (got %lld)", (long long)p->head_dim);
    if (p->num_pages < 0 || p->num_pages >= INT32_MAX || !extent_ok(p->kv_heads) || p->kv_heads == 0 ||
        !extent_ok(p->batch) || p->max_pages < 0 || p->max_pages > (int64_t(1) << 24))
        return fail(DELS_ERR_INVALID_ARGUMENT, "bad cache extents pages=%lld heads=%lld batch=%lld max_pages=%lld",
                    (long long)p->num_pages, (long long)p->kv_heads, (long long)p->batch, (long long)p->max_pages);
    if ((p->ld_table < p->max_pages && p->ld_table != 0) || p->ld_table >= (int64_t(1) << 40))
        return fail(DELS_ERR_INVALID_ARGUMENT, "table row stride %lld out of range", (long long)p->ld_table);
    if (p->batch && p->max_pages && !p->table) return fail(DELS_ERR_INVALID_ARGUMENT, "page table is NULL");
    if (p->num_pages && !p->data) return fail(DELS_ERR_INVALID_ARGUMENT, "cache data is NULL");
    if (!aligned(p->data, 128)) return fail(DELS_ERR_ALIGNMENT, "cache data must be 128-byte aligned");
    c.data = static_cast<uint8_t*>(p->data);
    c.num_pages = (int)p->num_pages, c.heads = (int)p->kv_heads, c.head_dim = (int)p->head_dim;
    c.table = p->table, c.ld_table = p->ld_table, c.batch = (int)p->batch, c.max_pages = (int)p->max_pages;
    return DELS_OK;
}

// A [batch, tokens, heads, D] operand whose rows are read in 16-byte pieces.
int check_rows(const void* p, int64_t sb, int64_t st, int64_t sh, int dtype, const char* name) {
    if (!p) return fail(DELS_ERR_INVALID_ARGUMENT, "%s is NULL", name);
    const int64_t per16 = dtype == DELS_DTYPE_F32 ? 4 : 8;
    for (int64_t s : {sb, st, sh}) {
        if (s < 0 || s >= (int64_t(1) << 40)) return fail(DELS_ERR_INVALID_ARGUMENT, "%s: stride out of range", name);
        if (s % per16) return fail(DELS_ERR_ALIGNMENT, "%s: strides must be multiples of 16 bytes", name);
    }
    if (!aligned(p, 16)) return fail(DELS_ERR_ALIGNMENT, "%s must be 16-byte aligned", name);
    return DELS_OK;
}

int check_type(int dtype, bool single) {
    if (dtype == DELS_DTYPE_BF16 || dtype == DELS_DTYPE_F16 || (single && dtype == DELS_DTYPE_F32)) return DELS_OK;
    return fail(DELS_ERR_INVALID_ARGUMENT, "unknown or unsupported element type %d", dtype);
}

// Extents that attention and its weights take: the pages of all rows stay below 2^30.
bool attention_ok(int64_t batch, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t max_pages) {
    return extent_ok(batch) && extent_ok(T) && extent_ok(q_heads) && extent_ok(kv_heads) && kv_heads > 0 &&
           q_heads % kv_heads == 0 && max_pages >= 0 && grid_ok({T, q_heads / kv_heads, 64}) &&
           grid_ok({batch, kv_heads, T * (q_heads / kv_heads) / 16 + 1, max_pages});
}

// The arguments that attention and its weights share.
int check_block(const Kv4Cache& c, const void* q, int64_t qb, int64_t qt, int64_t qh, int dtype, int64_t q_heads,
                int64_t T, const int32_t* lengths, int block, const int64_t* mask, int64_t ld_mask, float scale) {
    int rc = check_type(dtype, false);
    if (rc != DELS_OK) return rc;
    if (!extent_ok(T)) return fail(DELS_ERR_INVALID_ARGUMENT, "bad block length %lld", (long long)T);
    if (q_heads <= 0 || !extent_ok(q_heads) || q_heads % c.heads)
        return fail(DELS_ERR_INVALID_ARGUMENT, "%lld query heads over %d key/value heads", (long long)q_heads, c.heads);
    if (block < DELS_KV4_CAUSAL || block > DELS_KV4_MASK)
        return fail(DELS_ERR_INVALID_ARGUMENT, "unknown block mode %d", block);
    if (block == DELS_KV4_MASK) {
        if (!mask) return fail(DELS_ERR_INVALID_ARGUMENT, "block mask is NULL");
        if (T > 64) return fail(DELS_ERR_UNSUPPORTED, "a block mask holds 64 slots (T = %lld)", (long long)T);
        if ((ld_mask < T && ld_mask != 0) || ld_mask >= (int64_t(1) << 40))
            return fail(DELS_ERR_INVALID_ARGUMENT, "mask row stride %lld out of range", (long long)ld_mask);
    }
    if (!(scale == scale) || scale == __builtin_inff() || scale == -__builtin_inff())
        return fail(DELS_ERR_INVALID_ARGUMENT, "scale must be finite");
    if (!lengths) return fail(DELS_ERR_INVALID_ARGUMENT, "lengths is NULL");
    if (!attention_ok(c.batch, T, q_heads, c.heads, c.max_pages))
        return fail(DELS_ERR_UNSUPPORTED, "shape past the supported extents");
    return check_rows(q, qb, qt, qh, dtype, "q");
}

}  // namespace

}  // namespace dels

using namespace dels;

extern "C" {

size_t dels_kv4_page_bytes(int64_t head_dim) {
    return head_dim == 64 || head_dim == 128 ? (size_t)(66 * head_dim + 128) : 0;
}

int dels_kv4_append(const dels_kv4_cache* p, const void* k, int64_t k_batch, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_batch, int64_t v_token, int64_t v_head, int dtype,
                    const int32_t* lengths, const int32_t* counts, int64_t T, void* stream) {
    Kv4Cache c{};
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
    Kv4Cache c{};
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
