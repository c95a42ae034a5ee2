// Writing and reading the 4-bit key/value cache (format: kv4.h).
//
// One wave per (sequence, head, 8 slots): the eight slots share the value words
// of a page row, so no two waves write one word, whatever the block's start.
// Both kernels are bound by memory where they are long, by the launch where short.
#include <algorithm>

#include "kv4.h"

namespace dels {

namespace {

constexpr int kCacheThreads = 256;
constexpr float kBig = 3.0e38f;                    // magnitudes are clamped here: six steps stay finite
constexpr float kSixth = 0.16666667163372040f;

// N consecutive elements widened to fp32; NaN counts as 0.
template <typename T, int N>
__device__ __forceinline__ void load_clean(const T* p, float (&x)[N]) {
    u32x4 w[N * sizeof(T) / 16];
#pragma unroll
    for (size_t i = 0; i < N * sizeof(T) / 16; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float f;
        if constexpr (sizeof(T) == 4) {
            f = __uint_as_float(w[i / 4][i % 4]);
        } else {
            f = widen_raw<T>((w[i / 8][(i % 8) / 2] >> (16 * (i & 1))) & 0xffffu);
        }
        x[i] = f != f ? 0.f : fminf(fmaxf(f, -kBig), kBig);
    }
}

// Code of x at this step: the nearest magnitude, ties to the even code.  A step
// has at most 8 significant bits, so every threshold is exact and the result is
// the same on every machine; no division.
__device__ __forceinline__ uint32_t encode(float x, float step) {
    const float a = fabsf(x);
    uint32_t c = a > 0.25f * step ? 1u : 0u;
    c += a >= 0.75f * step ? 1u : 0u;
    c += a > 1.25f * step ? 1u : 0u;
    c += a >= 1.75f * step ? 1u : 0u;
    c += a > 2.5f * step ? 1u : 0u;
    c += a >= 3.5f * step ? 1u : 0u;
    c += a > 5.0f * step ? 1u : 0u;
    return c | (x < 0.f ? 8u : 0u);
}

// Lanes: slot i = lane / 8 of the group, channels N * (lane % 8) .. + N - 1 (N = D / 8).
template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void kv4_append_kernel(
    Kv4Cache c, const T* __restrict__ k, int64_t kb, int64_t kt, int64_t kh, const T* __restrict__ v, int64_t vb,
    int64_t vt, int64_t vh, const int32_t* lengths, const int32_t* counts, int T_rows, int groups) {
    constexpr int N = D / 8;
    const int lane = threadIdx.x & 63;
    int64_t unit = (int64_t)blockIdx.x * (kCacheThreads / 64) + (threadIdx.x >> 6);
    if (unit >= (int64_t)c.batch * c.heads * groups) return;
    const int h = (int)(unit % c.heads);
    unit /= c.heads;
    const int grp = (int)(unit % groups), b = (int)(unit / groups);
    const int slots = c.slots();
    const int n = kv4_length(lengths, b, slots);
    const int end = (int)min((int64_t)slots, (int64_t)n + kv4_count(counts, b, T_rows));
    const int s0 = (n & ~7) + 8 * grp;             // the group's first slot
    if (max(s0, n) >= end) return;
    uint8_t* page = kv4_page(c, b, h, s0 / kKv4Page, Kv4<D>::kBytes);
    if (!page) return;
    const int i = lane >> 3, ch = (lane & 7) * N;
    const int slot = s0 + i, in_page = slot % kKv4Page;
    const bool mine = slot >= n && slot < end;
    const int64_t t = mine ? slot - n : max(n, s0) - n;   // a row that exists, for lanes without one
    float x[N];

    load_clean(k + (int64_t)b * kb + t * kt + (int64_t)h * kh + ch, x);
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(x[j]));
    for (int off = 1; off < 32 / N; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
    // the smallest exponent whose sevenfold holds the largest magnitude: then no
    // element is off by more than half the widest step
    const uint32_t bits = __float_as_uint(amax);
    const int e = min(max((int)(bits >> 23) - 2 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 1), 252);
    uint32_t w[N / 8];
#pragma unroll
    for (int q = 0; q < N / 8; ++q) {
        w[q] = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[q] |= encode(x[8 * q + j], kv4_pow2(e)) << (4 * j);
    }
    if (mine) {
        uint32_t* row = reinterpret_cast<uint32_t*>(page + in_page * Kv4<D>::kKeyRow) + ch / 8;
#pragma unroll
        for (int q = 0; q < N / 8; ++q) row[q] = w[q];
        if (ch % 32 == 0) page[Kv4<D>::scale_byte(in_page, ch / 32)] = (uint8_t)e;
    }

    load_clean(v + (int64_t)b * vb + t * vt + (int64_t)h * vh + ch, x);
    amax = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(x[j]));
    for (int off = 1; off < 8; off <<= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
    const float step = fmaxf(round_bf16(amax * kSixth), 0x1p-126f);
    uint32_t words[N];                             // this slot's nibble of each channel's word
#pragma unroll
    for (int j = 0; j < N; ++j) words[j] = mine ? encode(x[j], step) << (4 * i) : 0u;
    if (mine && ch == 0)
        *reinterpret_cast<uint16_t*>(page + Kv4<D>::kValueScale + 2 * in_page) = f32_to_bf16_bits(step);
    // the eight slots' nibbles of a word are in the lanes 8 apart: each exchange
    // halves the channels that a lane goes on with
    int base = 0;
#pragma unroll
    for (int half = N / 2, off = 8; off < 64; half >>= 1, off <<= 1) {
        const bool hi = lane & off;
#pragma unroll
        for (int j = 0; j < half; ++j) {
            const uint32_t send = hi ? words[j] : words[j + half];
            words[j] = (hi ? words[j + half] : words[j]) | (uint32_t)__shfl_xor((int)send, off, 64);
        }
        base += hi ? half : 0;
    }
    uint32_t valid = 0u;
#pragma unroll
    for (int q = 0; q < 8; ++q) valid |= s0 + q >= n && s0 + q < end ? 15u << (4 * q) : 0u;
    uint32_t* row = reinterpret_cast<uint32_t*>(page + Kv4<D>::kValue) + (s0 % kKv4Page / 8) * D + ch + base;
#pragma unroll
    for (int j = 0; j < N / 8; ++j) row[j] = valid == ~0u ? words[j] : (row[j] & ~valid) | words[j];
}

template <typename T> __device__ __forceinline__ void store_value(T* p, float x);
template <> __device__ __forceinline__ void store_value(float* p, float x) { *p = x; }
template <> __device__ __forceinline__ void store_value(bf16_t* p, float x) { p->bits = f32_to_bf16_bits(x); }
template <> __device__ __forceinline__ void store_value(f16_t* p, float x) {
    const _Float16 h = (_Float16)x;
    __builtin_memcpy(&p->bits, &h, 2);
}

// One wave per (b, h, 8 slots), a lane D / 64 channels of all of them.
template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void kv4_read_kernel(Kv4Cache c, const int32_t* starts,
                                                                 const int32_t* counts, int T_rows, int groups,
                                                                 T* __restrict__ k, T* __restrict__ v) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63, ch = lane * N;
    int64_t unit = (int64_t)blockIdx.x * (kCacheThreads / 64) + (threadIdx.x >> 6);
    if (unit >= (int64_t)c.batch * c.heads * groups) return;
    const int h = (int)(unit % c.heads);
    unit /= c.heads;
    const int grp = (int)(unit % groups), b = (int)(unit / groups);
    const int slots = c.slots();
    const int n = kv4_length(starts, b, slots);
    const int64_t end = min((int64_t)slots, (int64_t)n + kv4_count(counts, b, T_rows));
    const int64_t s0 = (n & ~7) + 8 * (int64_t)grp;
    if (s0 >= (int64_t)n + T_rows) return;
    const uint8_t* page = s0 < end ? kv4_page(c, b, h, (int)(s0 / kKv4Page), Kv4<D>::kBytes) : nullptr;
    uint32_t words[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        words[j] = 0u;
        if (page)
            words[j] = reinterpret_cast<const uint32_t*>(page + Kv4<D>::kValue)[(s0 % kKv4Page / 8) * D + ch + j];
    }
    for (int i = 0; i < 8; ++i) {
        const int64_t slot = s0 + i;
        if (slot < n || slot >= (int64_t)n + T_rows) continue;
        const int in_page = (int)(slot % kKv4Page);
        const bool have = page && slot < end;
        float ks = 0.f, vs = 0.f;
        uint32_t code = 0u;
        if (have) {
            ks = kv4_pow2(page[Kv4<D>::scale_byte(in_page, ch / 32)]);
            vs = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(page + Kv4<D>::kValueScale + 2 * in_page));
            code = page[in_page * Kv4<D>::kKeyRow + ch / 2];
        }
        const int64_t at = (((int64_t)b * T_rows + (slot - n)) * c.heads + h) * D + ch;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t kc = (code >> (4 * ((ch + j) & 1))) & 15u;
            store_value(k + at + j, have ? kv4_level(kc) * ks : 0.f);
            store_value(v + at + j, have ? kv4_level((words[j] >> (4 * i)) & 15u) * vs : 0.f);
        }
    }
}

template <typename F> hipError_t by_type(int dtype, int head_dim, F&& f) {
    auto by_size = [&](auto tag) {
        if (head_dim == 64) f(tag, std::integral_constant<int, 64>{});
        else f(tag, std::integral_constant<int, 128>{});
    };
    if (dtype == 1) by_size(bf16_t{});
    else if (dtype == 2) by_size(f16_t{});
    else by_size(float{});
    return hipGetLastError();
}

// Groups of 8 slots that T rows can touch, whatever their first slot.
int groups_of(int T) { return (T + 7 + 7) / 8; }

}  // namespace

hipError_t launch_kv4_append(const Kv4Cache& c, const Kv4Rows& k, const Kv4Rows& v, int dtype, const int32_t* lengths,
                             const int32_t* counts, int T, hipStream_t s) {
    const int groups = groups_of(T), waves = kCacheThreads / 64;
    const int64_t units = (int64_t)c.batch * c.heads * groups;
    return by_type(dtype, c.head_dim, [&](auto tag, auto size) {
        using E = decltype(tag);
        hipLaunchKernelGGL((kv4_append_kernel<E, decltype(size)::value>), dim3((units + waves - 1) / waves),
                           dim3(kCacheThreads), 0, s, c, static_cast<const E*>(k.p), k.batch, k.token, k.head,
                           static_cast<const E*>(v.p), v.batch, v.token, v.head, lengths, counts, T, groups);
    });
}

hipError_t launch_kv4_read(const Kv4Cache& c, const int32_t* starts, const int32_t* counts, int T, void* k, void* v,
                           int dtype, hipStream_t s) {
    const int groups = groups_of(T), waves = kCacheThreads / 64;
    const int64_t units = (int64_t)c.batch * c.heads * groups;
    return by_type(dtype, c.head_dim, [&](auto tag, auto size) {
        using E = decltype(tag);
        hipLaunchKernelGGL((kv4_read_kernel<E, decltype(size)::value>), dim3((units + waves - 1) / waves),
                           dim3(kCacheThreads), 0, s, c, starts, counts, T, groups, static_cast<E*>(k),
                           static_cast<E*>(v));
    });
}

}  // namespace dels
