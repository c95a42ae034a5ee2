// C ABI of the 8-bit key/value cache (declared in include/dels.h): argument
// checks and dispatch.  Nothing here allocates device memory or synchronises.
#include "capi_paged.h"

using namespace dels;

namespace {

// A row of positions for each sequence, or one for all.
int check_positions(const int32_t* positions, int64_t ld, int64_t T) {
    if (positions && ((ld < T && ld != 0) || ld >= (int64_t(1) << 40)))
        return fail(DELS_ERR_INVALID_ARGUMENT, "positions row stride %lld out of range", (long long)ld);
    return DELS_OK;
}

int check_rotary(const dels_rotary* p, const PagedCache& c, int64_t T, const int32_t* positions, int64_t ld_positions,
                 KvRotary& r) {
    if (!p) return positions ? fail(DELS_ERR_INVALID_ARGUMENT, "positions without a rotary table") : DELS_OK;
    if (p->channels < 16 || p->channels % 16 || p->channels > c.head_dim)
        return fail(DELS_ERR_INVALID_ARGUMENT, "%lld rotated channels of %d", (long long)p->channels, c.head_dim);
    if (p->positions < 0 || p->positions >= (int64_t(1) << 40) || p->ld < p->channels / 2 ||
        p->ld >= (int64_t(1) << 24))
        return fail(DELS_ERR_INVALID_ARGUMENT, "bad rotary extents positions=%lld ld=%lld", (long long)p->positions,
                    (long long)p->ld);
    if (p->positions == 0) return fail(DELS_ERR_INVALID_ARGUMENT, "a rotary table of no positions");
    if (!p->cos || !p->sin) return fail(DELS_ERR_INVALID_ARGUMENT, "cos or sin is NULL");
    if (!aligned(p->cos, 16) || !aligned(p->sin, 16) || p->ld % 4)
        return fail(DELS_ERR_ALIGNMENT, "rotary rows must be 16-byte aligned");
    const int rc = check_positions(positions, ld_positions, T);
    if (rc != DELS_OK) return rc;
    r = {p->cos, p->sin, p->ld, p->positions, (int)p->channels, p->interleaved != 0, positions, ld_positions};
    return DELS_OK;
}

}  // namespace

extern "C" {

size_t dels_kv8_page_bytes(int64_t head_dim) {
    return head_dim == 64 || head_dim == 128 ? (size_t)(128 * head_dim + 128) : 0;
}

int dels_kv8_append(const dels_kv8_cache* p, const void* k, int64_t k_batch, int64_t k_token, int64_t k_head,
                    const void* v, int64_t v_batch, int64_t v_token, int64_t v_head, int dtype,
                    const int32_t* lengths, const int32_t* counts, int64_t T, const dels_rotary* rotary,
                    const int32_t* positions, int64_t ld_positions, const void* q, int64_t q_batch, int64_t q_token,
                    int64_t q_head, int64_t q_heads, void* q_out, int64_t out_batch, int64_t out_token,
                    int64_t out_head, void* stream) {
    PagedCache c{};
    int rc = cache_of(p, c);
    if (rc != DELS_OK) return rc;
    if ((rc = check_type(dtype, true)) != DELS_OK) return rc;
    if (!extent_ok(T)) return fail(DELS_ERR_INVALID_ARGUMENT, "bad block length %lld", (long long)T);
    if (!grid_ok({c.batch, c.heads, T / 8 + 2}) || c.batch > 65535 || c.heads > 65535)
        return fail(DELS_ERR_UNSUPPORTED, "shape past the supported extents");
    if (c.batch == 0 || T == 0) return DELS_OK;
    KvRotary r{};
    if ((rc = check_rotary(rotary, c, T, positions, ld_positions, r)) != DELS_OK) return rc;
    if ((rc = check_rows(k, k_batch, k_token, k_head, dtype, "k")) != DELS_OK) return rc;
    if ((rc = check_rows(v, v_batch, v_token, v_head, dtype, "v")) != DELS_OK) return rc;
    if (!lengths) return fail(DELS_ERR_INVALID_ARGUMENT, "lengths is NULL");
    if (!q) q_heads = 0;
    if (q) {
        if (!rotary) return fail(DELS_ERR_INVALID_ARGUMENT, "q without a rotary table");
        if (q_heads <= 0 || !extent_ok(q_heads) || q_heads % c.heads || !grid_ok({q_heads / c.heads, 32, 8}))
            return fail(DELS_ERR_INVALID_ARGUMENT, "%lld query heads over %d key/value heads", (long long)q_heads,
                        c.heads);
        if ((rc = check_rows(q, q_batch, q_token, q_head, dtype, "q")) != DELS_OK) return rc;
        if ((rc = check_rows(q_out, out_batch, out_token, out_head, dtype, "q_out")) != DELS_OK) return rc;
    }
    const hipError_t e = launch_kv8_append(c, {k, k_batch, k_token, k_head}, {v, v_batch, v_token, v_head}, dtype,
                                           lengths, counts, (int)T, r, {q, q_batch, q_token, q_head}, (int)q_heads,
                                           {q_out, out_batch, out_token, out_head}, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache append launch");
}

int dels_kv8_read(const dels_kv8_cache* p, const int32_t* starts, const int32_t* counts, int64_t T, void* k, void* v,
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
    if (c.num_pages == 0) c.max_pages = 0;                    // nothing is held
    const hipError_t e = launch_kv8_read(c, starts, counts, (int)T, k, v, dtype, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache read launch");
}

size_t dels_kv8_attention_ws_bytes(int64_t batch, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                   int64_t max_pages) {
    if (!attention_ok(batch, T, q_heads, kv_heads, max_pages) || (head_dim != 64 && head_dim != 128)) return 0;
    return kDataOff + kv8_attention_data_bytes(batch, T, q_heads, kv_heads, head_dim, max_pages);
}

int dels_kv8_attention(const dels_kv8_cache* p, const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                       int dtype, int64_t q_heads, int64_t T, const int32_t* lengths, const int32_t* counts,
                       int block, const int64_t* mask, int64_t ld_mask, float scale, int64_t window, int64_t sinks,
                       void* out, int64_t out_batch, int64_t out_token, int64_t out_head, float* lse, void* ws,
                       size_t ws_bytes, void* stream) {
    return dels_kv8_attention_ex(p, q, q_batch, q_token, q_head, dtype, q_heads, T, lengths, counts, block, mask,
                                 ld_mask, scale, window, sinks, nullptr, out, out_batch, out_token, out_head, lse, ws,
                                 ws_bytes, stream);
}

int dels_kv8_attention_ex(const dels_kv8_cache* p, const void* q, int64_t q_batch, int64_t q_token, int64_t q_head,
                          int dtype, int64_t q_heads, int64_t T, const int32_t* lengths, const int32_t* counts,
                          int block, const int64_t* mask, int64_t ld_mask, float scale, int64_t window, int64_t sinks,
                          const dels_kv8_options* options, void* out, int64_t out_batch, int64_t out_token,
                          int64_t out_head, float* lse, void* ws, size_t ws_bytes, void* stream) {
    const dels_kv8_options given = options ? *options : dels_kv8_options{};
    Kv8AttentionArgs a{};
    int rc = cache_of(p, a.cache);
    if (rc != DELS_OK) return rc;
    if (window < 0 || sinks < 0 || (sinks && !window))
        return fail(DELS_ERR_INVALID_ARGUMENT, "bad window %lld with %lld sinks", (long long)window, (long long)sinks);
    if (given.positions && (!window || block != DELS_KV4_MASK))
        return fail(DELS_ERR_INVALID_ARGUMENT, "positions are for a window over a block mask");
    if (given.weight_parts < 0 || given.weight_parts > 2)
        return fail(DELS_ERR_INVALID_ARGUMENT, "weights in %d parts", given.weight_parts);
    if (a.cache.batch == 0 || T == 0) return DELS_OK;
    rc = check_block(a.cache, q, q_batch, q_token, q_head, dtype, q_heads, T, lengths, block, mask, ld_mask, scale);
    if (rc != DELS_OK) return rc;
    if ((rc = check_positions(given.positions, given.ld_positions, T)) != DELS_OK) return rc;
    if ((rc = check_rows(out, out_batch, out_token, out_head, dtype, "out")) != DELS_OK) return rc;
    if (!lse) return fail(DELS_ERR_INVALID_ARGUMENT, "lse is NULL");
    if (a.cache.num_pages == 0) a.cache.max_pages = 0;       // nothing to see
    const size_t need = dels_kv8_attention_ws_bytes(a.cache.batch, T, q_heads, a.cache.heads, a.cache.head_dim,
                                                    a.cache.max_pages);
    if ((rc = check_ws(ws, ws_bytes, need)) != DELS_OK) return rc;
    // wider than everything is no window
    const int64_t all = (int64_t)a.cache.slots() + T;
    a.window = window > all ? 0 : window, a.sinks = std::min<int64_t>(sinks, all);
    if (a.window) a.at = given.positions, a.ld_at = given.ld_positions;
    a.block = {lengths, counts, (int)T, block, mask, ld_mask};
    a.q = {q, q_batch, q_token, q_head};
    a.dtype = dtype, a.q_heads = (int)q_heads, a.scale = scale, a.split = given.weight_parts == 2;
    a.out = out, a.out_batch = out_batch, a.out_token = out_token, a.out_head = out_head, a.lse = lse;
    const hipError_t e = launch_kv8_attention(a, ws, kDataOff, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? DELS_OK : hip_fail(e, "cache attention launch");
}

}  // extern "C"
