// Writing and reading the 4-bit key/value cache (format: kv4.h).
//
// One wave per (sequence, head, 8 slots): the eight slots share the value words
// of a page row, so no two waves write one word, whatever the block's start.
// A lane has one slot's D / 8 channels, as eight-nibble words; the value words, eight
// slots of a channel, are those transposed over the eight lanes of a channel group
// (three exchanges of halves, bytes and nibbles).  Long calls run at two thirds of a copy's
// rate (4 x 2039 rows of 8 heads of 128, fp16, 6629 of 8156 valid: 34 MB written in 11.0 us,
// 3.1 TB/s, a wave's values being loaded after its keys are done; 40 MB read in 11.9 us,
// 3.4 TB/s); short ones are bound by latency (8 x 16 rows: 4.6 and 4.5 us).
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
// has at most 8 significant bits, so every threshold is exact.
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

// Codes of eight numbers over a power of two, by the conversion instruction: it divides
// exactly, rounds as encode() does and saturates; -0 is made 0 for it.
__device__ __forceinline__ uint32_t encode8_pow2(const float* x, float scale) {
    uint32_t w = 0u;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0] + 0.f, x[1] + 0.f, scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2] + 0.f, x[3] + 0.f, scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4] + 0.f, x[5] + 0.f, scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6] + 0.f, x[7] + 0.f, scale, 3);
}

// Codes of eight numbers over any step.  Numbers of 16 bits: the quotient by the step's
// reciprocal is within 2^-22, and a number that is not a threshold times the step is at
// least 2^-11 off it (11 significant bits each), so the quotient rounded to 16
// significant bits is on the right side of every threshold and on it for a tie.
// Numbers of 32 bits are compared with the thresholds themselves.
template <typename T> __device__ __forceinline__ uint32_t encode8(const float* x, float step) {
    if constexpr (sizeof(T) == 4) {
        uint32_t w = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= encode(x[j], step) << (4 * j);
        return w;
    } else {
        const float r = 1.0f / step;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = __uint_as_float((__float_as_uint(x[j] * r) + 0x80u) & ~0xffu);
        return encode8_pow2(y, 1.f);
    }
}

// Nibble j of lane group i (lanes 8 i ..) goes to nibble i of lane group j.
__device__ __forceinline__ uint32_t transpose8(uint32_t w) {
    const int lane = threadIdx.x & 63;
    uint32_t o = (uint32_t)__shfl_xor((int)w, 32, 64);
    w = lane & 32 ? (w & 0xffff0000u) | (o >> 16) : (w & 0x0000ffffu) | (o << 16);
    o = (uint32_t)__shfl_xor((int)w, 16, 64);
    w = lane & 16 ? (w & 0xff00ff00u) | (o >> 8 & 0x00ff00ffu) : (w & 0x00ff00ffu) | (o << 8 & 0xff00ff00u);
    o = (uint32_t)__shfl_xor((int)w, 8, 64);
    return lane & 8 ? (w & 0xf0f0f0f0u) | (o >> 4 & 0x0f0f0f0fu) : (w & 0x0f0f0f0fu) | (o << 4 & 0xf0f0f0f0u);
}

// Lanes: slot i = lane / 8 of the group, channels N * (lane % 8) .. + N - 1 (N = D / 8).
template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void kv4_append_kernel(
    Kv4Cache c, const T* __restrict__ k, int64_t kb, int64_t kt, int64_t kh, const T* __restrict__ v, int64_t vb,
    int64_t vt, int64_t vh, const int32_t* lengths, const int32_t* counts, int T_rows, int groups) {
    constexpr int N = D / 8;
    const int lane = threadIdx.x & 63;
    const int grp = blockIdx.x * (kCacheThreads / 64) + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    if (grp >= groups) return;
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
    for (int q = 0; q < N / 8; ++q) w[q] = encode8_pow2(x + 8 * q, kv4_pow2(e));
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
    if (mine && ch == 0)
        *reinterpret_cast<uint16_t*>(page + Kv4<D>::kValueScale + 2 * in_page) = f32_to_bf16_bits(step);
    uint32_t valid = 0u;
#pragma unroll
    for (int q = 0; q < 8; ++q) valid |= s0 + q >= n && s0 + q < end ? 15u << (4 * q) : 0u;
    // lane group i then holds channel 8 q + i of its sixteen (eight)
    uint32_t* row = reinterpret_cast<uint32_t*>(page + Kv4<D>::kValue) + (s0 % kKv4Page / 8) * D + ch + i;
#pragma unroll
    for (int q = 0; q < N / 8; ++q) {
        const uint32_t words = transpose8(encode8<T>(x + 8 * q, step));
        row[8 * q] = valid == ~0u ? words : (row[8 * q] & ~valid) | (words & valid);
    }
}

// Numbers that eight codes stand for, times `by`, as two or four words of type T.
template <typename T> __device__ __forceinline__ void store8(T* p, uint32_t codes, float scale, float by) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
    const float x[8] = {a[0] * by, a[1] * by, b[0] * by, b[1] * by, c[0] * by, c[1] * by, d[0] * by, d[1] * by};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            reinterpret_cast<f32x4*>(p)[h] = f32x4{x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]};
    } else {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (std::is_same<T, bf16_t>::value) {
                w[j] = (uint32_t)f32_to_bf16_bits(x[2 * j]) | (uint32_t)f32_to_bf16_bits(x[2 * j + 1]) << 16;
            } else {
                const _Float16 l = (_Float16)x[2 * j], u = (_Float16)x[2 * j + 1];
                uint16_t lb, ub;
                __builtin_memcpy(&lb, &l, 2);
                __builtin_memcpy(&ub, &u, 2);
                w[j] = (uint32_t)lb | (uint32_t)ub << 16;
            }
        }
        *reinterpret_cast<u32x4*>(p) = w;
    }
}

// Lanes as in the append kernel: slot i = lane / 8, channels N * (lane % 8) .. + N - 1.
template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void kv4_read_kernel(Kv4Cache c, const int32_t* starts,
                                                                 const int32_t* counts, int T_rows, int groups,
                                                                 T* __restrict__ k, T* __restrict__ v) {
    constexpr int N = D / 8;
    const int lane = threadIdx.x & 63;
    const int grp = blockIdx.x * (kCacheThreads / 64) + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    if (grp >= groups) return;
    const int slots = c.slots();
    const int n = kv4_length(starts, b, slots);
    const int64_t end = min((int64_t)slots, (int64_t)n + kv4_count(counts, b, T_rows));
    const int64_t s0 = (n & ~7) + 8 * (int64_t)grp;
    if (s0 >= (int64_t)n + T_rows) return;
    const uint8_t* page = s0 < end ? kv4_page(c, b, h, (int)(s0 / kKv4Page), Kv4<D>::kBytes) : nullptr;
    const int i = lane >> 3, ch = (lane & 7) * N;
    const int64_t slot = s0 + i;
    const bool wanted = slot >= n && slot < (int64_t)n + T_rows, have = page && slot >= n && slot < end;
    const int in_page = (int)(slot % kKv4Page);
    uint32_t kw[N / 8], vw[N / 8];
    float ks = 0.f, vs = 0.f;
#pragma unroll
    for (int q = 0; q < N / 8; ++q) kw[q] = vw[q] = 0u;
    if (page) {
        const uint32_t* row = reinterpret_cast<const uint32_t*>(page + Kv4<D>::kValue) + (s0 % kKv4Page / 8) * D + ch + i;
#pragma unroll
        for (int q = 0; q < N / 8; ++q) vw[q] = row[8 * q];
    }
    if (have) {
        const uint32_t* row = reinterpret_cast<const uint32_t*>(page + in_page * Kv4<D>::kKeyRow) + ch / 8;
#pragma unroll
        for (int q = 0; q < N / 8; ++q) kw[q] = row[q];
        ks = kv4_pow2(page[Kv4<D>::scale_byte(in_page, ch / 32)]);
        vs = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(page + Kv4<D>::kValueScale + 2 * in_page));
    }
    const int64_t at = (((int64_t)b * T_rows + (slot - n)) * c.heads + h) * D + ch;
#pragma unroll
    for (int q = 0; q < N / 8; ++q) {
        const uint32_t codes = transpose8(vw[q]);
        if (wanted) {
            store8(k + at + 8 * q, have ? kw[q] : 0u, have ? ks : 1.f, 1.f);
            store8(v + at + 8 * q, have ? codes : 0u, 1.f, have ? vs : 0.f);
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
    const dim3 grid((groups + waves - 1) / waves, c.heads, c.batch);
    return by_type(dtype, c.head_dim, [&](auto tag, auto size) {
        using E = decltype(tag);
        hipLaunchKernelGGL((kv4_append_kernel<E, decltype(size)::value>), grid,
                           dim3(kCacheThreads), 0, s, c, static_cast<const E*>(k.p), k.batch, k.token, k.head,
                           static_cast<const E*>(v.p), v.batch, v.token, v.head, lengths, counts, T, groups);
    });
}

hipError_t launch_kv4_read(const Kv4Cache& c, const int32_t* starts, const int32_t* counts, int T, void* k, void* v,
                           int dtype, hipStream_t s) {
    const int groups = groups_of(T), waves = kCacheThreads / 64;
    const dim3 grid((groups + waves - 1) / waves, c.heads, c.batch);
    return by_type(dtype, c.head_dim, [&](auto tag, auto size) {
        using E = decltype(tag);
        hipLaunchKernelGGL((kv4_read_kernel<E, decltype(size)::value>), grid,
                           dim3(kCacheThreads), 0, s, c, starts, counts, T, groups, static_cast<E*>(k),
                           static_cast<E*>(v));
    });
}

}  // namespace dels
