// The 4-bit key/value cache: format and device helpers shared by its kernels.
//
// A page holds 64 slots of one key/value head of D channels (D = 64 or 128):
//   [0, 32 D)          key codes: 64 rows of D/2 bytes, channel 2c in the low half of byte c
//   [32 D, 34 D)       key scales, one byte e (2^(e-127)) per slot and 32 channels: slot
//                      32 s + 8 rh + 4 a + rl of block m at byte 64 m + 16 rh + 4 rl + 2 s + a
//   [34 D, 66 D)       value codes: 8 rows (8 slots each) of D words, slot 8 g + i in bits
//                      4 i .. 4 i + 3 of its channel's word in row g
//   [66 D, 66 D + 128) value scales: 64 bf16 numbers
// Codes are e2m1: 0, .5, 1, 1.5, 2, 3, 4, 6 with a sign bit.
//
// Why so: an MFMA's 16-bit operand is eight consecutive elements of the
// contraction per lane.  For q.k that is eight channels of a slot -- one word of a
// key row -- and a block of 32 channels has one scale, which the conversion
// instruction (v_cvt_scalef32_pk_*_fp4) applies for nothing.  For p.v it is eight
// slots of a channel -- one word of a value row -- and there the scale is the
// slot's, which multiplies p.  The slots in the order that the scales show are the
// ones whose scores a lane holds after the first product, so p never leaves its lane.
#pragma once

#include "dels_device.h"
#include "dels_internal.h"

namespace dels {

template <int D> struct Kv4 {
    static_assert(D == 64 || D == 128, "head sizes of the cache");
    static constexpr int kKeyRow = D / 2;
    static constexpr int kKeyScale = 32 * D;
    static constexpr int kValue = 34 * D;
    static constexpr int kValueScale = 66 * D;
    static constexpr int kBytes = 66 * D + 128;
    // byte of the key scale of `slot` (0..63), channel block `blk`, within the page
    __device__ static int scale_byte(int slot, int blk) {
        return kKeyScale + 64 * blk + 16 * ((slot >> 3) & 3) + 4 * (slot & 3) + 2 * (slot >> 5) + ((slot >> 2) & 1);
    }
};

// Page of (b, h) that holds slots 64 p .. 64 p + 63, or null where the table
// names no page.
__device__ __forceinline__ uint8_t* kv4_page(const Kv4Cache& c, int b, int h, int p, int page_bytes) {
    const int id = c.table[(int64_t)b * c.ld_table + p];
    if (id < 0 || id >= c.num_pages) return nullptr;
    return c.data + ((int64_t)id * c.heads + h) * page_bytes;
}

// Sum over the lanes up to this one: within rows of 16 lanes, then from row to row.
__device__ __forceinline__ int sum_upto(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);     // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // row_bcast:31 into rows 2 and 3
    return x;
}

// Context length and valid block rows of sequence b, within the table's slots.
__device__ __forceinline__ int kv4_length(const int32_t* lengths, int b, int slots) {
    return min(max(lengths[b], 0), slots);
}
__device__ __forceinline__ int kv4_count(const int32_t* counts, int b, int T) {
    return counts ? min(max(counts[b], 0), T) : T;
}

__device__ __forceinline__ float kv4_pow2(uint32_t e) { return __uint_as_float(e << 23); }

}  // namespace dels
