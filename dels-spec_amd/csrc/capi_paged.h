// Argument checks that the entry points of the paged key/value caches share.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "../../include/dels.h"
#include "dels_internal.h"

namespace dels {

inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline bool extent_ok(int64_t x) { return x >= 0 && x < (int64_t(1) << 24); }

// Workgroups of a launch over these extents stay far below 2^31.
inline bool grid_ok(std::initializer_list<int64_t> xs) {
    int64_t total = 1;
    for (int64_t x : xs) {
        if (x > 0 && total > (int64_t(1) << 30) / x) return false;
        total *= std::max<int64_t>(x, 1);
    }
    return true;
}

inline int cache_of(const dels_kv4_cache* p, PagedCache& c) {
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
inline int check_rows(const void* p, int64_t sb, int64_t st, int64_t sh, int dtype, const char* name) {
    if (!p) return fail(DELS_ERR_INVALID_ARGUMENT, "%s is NULL", name);
    const int64_t per16 = dtype == DELS_DTYPE_F32 ? 4 : 8;
    for (int64_t s : {sb, st, sh}) {
        if (s < 0 || s >= (int64_t(1) << 40)) return fail(DELS_ERR_INVALID_ARGUMENT, "%s: stride out of range", name);
        if (s % per16) return fail(DELS_ERR_ALIGNMENT, "%s: strides must be multiples of 16 bytes", name);
    }
    if (!aligned(p, 16)) return fail(DELS_ERR_ALIGNMENT, "%s must be 16-byte aligned", name);
    return DELS_OK;
}

inline int check_type(int dtype, bool single) {
    if (dtype == DELS_DTYPE_BF16 || dtype == DELS_DTYPE_F16 || (single && dtype == DELS_DTYPE_F32)) return DELS_OK;
    return fail(DELS_ERR_INVALID_ARGUMENT, "unknown or unsupported element type %d", dtype);
}

// Extents that attention and its weights take: the pages of all rows stay below 2^30.
inline bool attention_ok(int64_t batch, int64_t T, int64_t q_heads, int64_t kv_heads, int64_t max_pages) {
    return extent_ok(batch) && extent_ok(T) && extent_ok(q_heads) && extent_ok(kv_heads) && kv_heads > 0 &&
           q_heads % kv_heads == 0 && max_pages >= 0 && grid_ok({T, q_heads / kv_heads, 64}) &&
           grid_ok({batch, kv_heads, T * (q_heads / kv_heads) / 16 + 1, max_pages});
}

// The arguments that attention and its weights share.
inline int check_block(const PagedCache& c, const void* q, int64_t qb, int64_t qt, int64_t qh, int dtype,
                       int64_t q_heads, int64_t T, const int32_t* lengths, int block, const int64_t* mask,
                       int64_t ld_mask, float scale) {
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

}  // namespace dels
