// The 8-bit key/value cache: format and device helpers shared by its kernels.
//
// A page holds 64 slots of one key/value head of D channels (D = 64 or 128), two blocks of
// 32 slots:
//   [0, 64 D)      keys, e4m3: channel 16 c + i of slot s of block u at 32 D u + 512 c + 16 pos(s) + i,
//                  pos(s) = 8 (s % 16 / 4) + 4 (s / 16) + s % 4
//   [64 D, 128 D)  values, e4m3: channel c of slot 16 h + i of block u at 64 D + 32 D u + 16 D h + 16 c + i
//   [128 D, + 16)  8 bytes a block: exponents of its keys and of its values (2^(e - 127)), two bytes
//                  of 0, and a word with the bits of the slots whose row was not finite
//   [.., 128 D + 128)  nothing
//
// Why so: the rows of a block are the columns of both products of attention, and what a
// lane holds of S^T = K Q^T has to be what it needs of P^T in O^T = V^T P^T.  With the keys in
// this order a lane's accumulators hold sixteen consecutive slots, so its weights are
// operands as they are, and every load of keys or values is 16 bytes a lane from whole
// lines: keys in pieces of 16 channels of 32 slots, values in pieces of 16 slots of all channels.
#pragma once

#include "fp8.h"
#include "paged_attention.h"

namespace dels {

constexpr int kKv8Block = 32;                    // slots that share a scale
constexpr int kKv8Low = 63, kKv8High = 191;      // exponents that a block may have: 2^-64 .. 2^64

template <int D> struct Kv8 {
    static_assert(D == 64 || D == 128, "head sizes of the cache");
    static constexpr int kValue = 64 * D;
    static constexpr int kHead = 128 * D;
    static constexpr int kBytes = 128 * D + 128;
    __device__ static int place(int slot) { return 8 * (slot % 16 / 4) + 4 * (slot / 16) + slot % 4; }
};

// What a block says of itself.
struct Kv8Head {
    uint32_t exponents, bad;
    __device__ uint32_t key() const { return exponents & 255u; }
    __device__ uint32_t value() const { return (exponents >> 8) & 255u; }
};

// Page of (b, h) that holds slots 64 p .. 64 p + 63, or null where the table names no page.
template <int D> __device__ __forceinline__ uint8_t* kv8_page(const PagedCache& c, int b, int h, int p) {
    const int id = c.table[(int64_t)b * c.ld_table + p];
    if (id < 0 || id >= c.num_pages) return nullptr;
    return c.data + ((int64_t)id * c.heads + h) * Kv8<D>::kBytes;
}

__device__ __forceinline__ float kv8_pow2(uint32_t e) { return __uint_as_float(e << 23); }

// f(element type, head size) as types.
template <typename F> hipError_t kv8_by_type(int dtype, int head_dim, F&& f) {
    auto by_size = [&](auto tag) {
        if (head_dim == 64) f(tag, std::integral_constant<int, 64>{});
        else f(tag, std::integral_constant<int, 128>{});
    };
    if (dtype == DELS_DTYPE_BF16) by_size(bf16_t{});
    else if (dtype == DELS_DTYPE_F16) by_size(f16_t{});
    else by_size(float{});
    return hipGetLastError();
}

}  // namespace dels
