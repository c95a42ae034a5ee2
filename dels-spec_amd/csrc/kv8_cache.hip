// Writing and reading the 8-bit key/value cache (format: kv8.h), with the position
// rotation of keys and queries on the way.
//
// A workgroup takes one block of 32 slots of one (sequence, head): the block's rows share
// their scales, so no other workgroup writes there.  A thread has 16 channels of one slot.
//     e = max(exponent of the rows that the block keeps, smallest e with 448 2^e >= |new rows|)
// and where rows are kept under a smaller exponent their codes are rounded once more.  Keys are
// stored as the threads have them, values go through LDS, from rows of channels to columns
// of slots.  Queries are rotated by workgroups of their own behind those of the blocks.
//
// Memory bounds both at a prompt's size (4 x 2039 fp16 rows of 8 heads of 128, 32 query heads, kernel times:
// append 29.5 us, 5.8 TB/s by the 170 MB that it moves; read 10.1 us, 47 MB at 4.7 TB/s), latency at a block's
// (8 x 16 rows: 5.3 and 4.2 us, a launch of nothing 3.6).
#include <algorithm>

#include "kv8.h"

namespace dels {

namespace {

constexpr int kCacheThreads = 256;
constexpr float kMost = 448.f * 0x1p64f;           // magnitudes above are not held

// Eight consecutive elements widened to fp32.
template <typename T> __device__ __forceinline__ void load8(const T* p, float* x) {
    u32x4 w[sizeof(T) / 2];
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i / 4][i % 4]);
        else x[i] = widen_raw<T>((w[0][i / 2] >> (16 * (i & 1))) & 0xffffu);
    }
}

// N consecutive numbers, N a multiple of 8, rounded to T.
template <typename T, int N> __device__ __forceinline__ void store(T* p, const float* x) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<f32x4*>(p + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            u32x4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = (uint32_t)round_to<T>(x[i + 2 * j]) | (uint32_t)round_to<T>(x[i + 2 * j + 1]) << 16;
            *reinterpret_cast<u32x4*>(p + i) = w;
        }
    }
}

// A row of D channels lies with D / 16 threads, two pieces of 8 channels each: those that a
// rotation pairs (i with i + rot / 2), or neighbours.
struct Pieces { int first, second; };
__device__ __forceinline__ Pieces pieces_of(int u, const KvRotary& r) {
    if (!r.interleaved && 16 * u < r.rot) return {8 * u, 8 * u + r.rot / 2};
    return {16 * u, 16 * u + 8};
}

// Rotates the thread's 16 channels by the angles of position p: every product, sum and
// difference rounded to fp32.  NaN for a position that the table does not have.
__device__ __forceinline__ void rotate(const KvRotary& r, int u, int64_t p, float* x) {
#pragma clang fp contract(off)
    if (16 * u >= r.rot) return;
    const bool have = p >= 0 && p < r.positions;
    const int64_t at = (have ? p : 0) * r.ld + 8 * u;
    float c[8], s[8];
    load8(r.cos + at, c);
    load8(r.sin + at, s);
    const float bad = have ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float& a = r.interleaved ? x[2 * i] : x[i];
        float& b = r.interleaved ? x[2 * i + 1] : x[8 + i];
        const float y = a * c[i] - b * s[i], z = b * c[i] + a * s[i];
        a = have ? y : bad;
        b = have ? z : bad;
    }
}

// Position of row t of sequence b, whose context is n.
__device__ __forceinline__ int64_t position_of(const KvRotary& r, int b, int64_t t, int n) {
    return r.at ? (int64_t)r.at[(int64_t)b * r.ld_at + t] : (int64_t)n + t;
}

__device__ __forceinline__ float top_of(const float* x) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(x[i]));
    return m;
}
__device__ __forceinline__ bool held(const float* x) {      // false for NaN too
    bool ok = true;
#pragma unroll
    for (int i = 0; i < 16; ++i) ok &= fabsf(x[i]) <= kMost;
    return ok;
}

// Exponent byte of the smallest power of two whose 448-fold holds `top`.
__device__ __forceinline__ uint32_t exponent_of(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int e = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)min(max(e, kKv8Low), kKv8High);
}

// What codes under the exponent `was` are multiplied by under a larger one.  Exponents lie up to 128
// apart, and from 127 on the power of two is no normal float: 0, and far above that no code leaves
// anything but its sign.
__device__ __forceinline__ float shrink_factor(uint32_t was, uint32_t now) {
    return kv8_pow2((uint32_t)max(127 + (int)was - (int)now, 0));
}

// Four codes rounded under a larger exponent.
__device__ __forceinline__ uint32_t shrink(uint32_t w, float by) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    return f32x4_to_e4m3(lo[0] * by, lo[1] * by, hi[0] * by, hi[1] * by);
}

struct AppendArgs {
    PagedCache cache;
    PagedRows k, v, q;
    KvRotary rotary;
    void* q_out; int64_t out_batch, out_token, out_head;
    const int32_t *lengths, *counts;
    int T, group;              // tokens, query heads per key/value head
    int blocks;                // workgroups in x that take blocks; those behind them take queries
};

// Rotated queries of 32 tokens of the group's heads.
template <typename T, int D>
__device__ __forceinline__ void rotate_queries(const AppendArgs& a, int chunk, int h, int b) {
    constexpr int U = D / 16;
    const int n = paged_length(a.lengths, b, a.cache.slots()), count = paged_count(a.counts, b, a.T);
    const int t0 = kKv8Block * chunk, tokens = min(kKv8Block, a.T - t0);
    for (int e = threadIdx.x; e < tokens * a.group * U; e += kCacheThreads) {
        const int u = e % U, g = e / U % a.group, t = t0 + e / (U * a.group);
        const int64_t hq = (int64_t)h * a.group + g;
        const Pieces at = pieces_of(u, a.rotary);
        float x[16];
        const T* from = static_cast<const T*>(a.q.p) + (int64_t)b * a.q.batch + (int64_t)t * a.q.token + hq * a.q.head;
        load8(from + at.first, x);
        load8(from + at.second, x + 8);
        if (t < count) {
            rotate(a.rotary, u, position_of(a.rotary, b, t, n), x);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = 0.f;
        }
        T* to = static_cast<T*>(a.q_out) + (int64_t)b * a.out_batch + (int64_t)t * a.out_token + hq * a.out_head;
        store<T, 8>(to + at.first, x);
        store<T, 8>(to + at.second, x + 8);
    }
}

template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void kv8_append_kernel(AppendArgs a) {
    constexpr int U = D / 16;                          // threads of a row
    constexpr int kPitch = D + 16;                     // bytes from one slot's values to the next in LDS
    __shared__ __attribute__((aligned(16))) uint8_t s_v[kKv8Block][kPitch];
    __shared__ float s_top[2][kCacheThreads / 64];
    __shared__ uint32_t s_bad;
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    if ((int)blockIdx.x >= a.blocks) return rotate_queries<T, D>(a, blockIdx.x - a.blocks, h, b);
    const PagedCache& c = a.cache;
    const int slots = c.slots(), n = paged_length(a.lengths, b, slots);
    const int end = (int)min((int64_t)slots, (int64_t)n + paged_count(a.counts, b, a.T));
    const int s0 = (n & ~(kKv8Block - 1)) + kKv8Block * (int)blockIdx.x;    // the block's first slot
    const int from = max(s0, n), to = min(s0 + kKv8Block, end);
    if (from >= to) return;
    uint8_t* page = kv8_page<D>(c, b, h, s0 / kCachePage);
    if (!page) return;
    const int u = s0 / kKv8Block % 2;                  // which of the page's blocks
    uint8_t* keys = page + 32 * D * u;
    uint8_t* values = page + Kv8<D>::kValue + 32 * D * u;
    auto* head = reinterpret_cast<uint2*>(page + Kv8<D>::kHead + 8 * u);
    const int kept = from - s0;                        // rows that the block keeps: slots below
    if (tid == 0) s_bad = 0u;
    uint2 was = {0u, 0u};
    if (kept) was = *head;
    __syncthreads();

    const int row = tid / U, part = tid % U, slot = s0 + row;
    const bool mine = row < kKv8Block && slot >= from && slot < to;
    const Pieces at = pieces_of(part, a.rotary);
    float kx[16], vx[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) kx[i] = vx[i] = 0.f;
    if (mine) {
        const int64_t t = slot - n;
        const T* kp = static_cast<const T*>(a.k.p) + (int64_t)b * a.k.batch + t * a.k.token + (int64_t)h * a.k.head;
        const T* vp = static_cast<const T*>(a.v.p) + (int64_t)b * a.v.batch + t * a.v.token + (int64_t)h * a.v.head;
        load8(kp + at.first, kx);
        load8(kp + at.second, kx + 8);
        load8(vp + 16 * part, vx);
        load8(vp + 16 * part + 8, vx + 8);
        if (a.rotary.rot) rotate(a.rotary, part, position_of(a.rotary, b, t, n), kx);
    }
    // a row of which something is not finite (or too large) is held as none of it
    int ok = held(kx) && held(vx);
#pragma unroll
    for (int off = 1; off < U; off <<= 1) ok &= __shfl_xor(ok, off, 64);
    if (!ok) {
#pragma unroll
        for (int i = 0; i < 16; ++i) kx[i] = vx[i] = 0.f;
        if (part == 0) atomicOr(&s_bad, 1u << (row % kKv8Block));
    }
    float kt = top_of(kx), vt = top_of(vx);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        kt = fmaxf(kt, __shfl_xor(kt, off, 64));
        vt = fmaxf(vt, __shfl_xor(vt, off, 64));
    }
    if (tid % 64 == 0) {
        s_top[0][tid / 64] = kt;
        s_top[1][tid / 64] = vt;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kCacheThreads / 64; ++w) {
        kt = fmaxf(kt, s_top[0][w]);
        vt = fmaxf(vt, s_top[1][w]);
    }
    const Kv8Head old = {was.x, was.y};
    uint32_t ke = exponent_of(kt), ve = exponent_of(vt);
    const uint32_t old_ke = min(max(old.key(), (uint32_t)kKv8Low), (uint32_t)kKv8High);
    const uint32_t old_ve = min(max(old.value(), (uint32_t)kKv8Low), (uint32_t)kKv8High);
    if (kept) ke = max(ke, old_ke), ve = max(ve, old_ve);
    if (tid == 0) {
        const uint32_t stay = kept ? old.bad & ((1u << kept) - 1u) : 0u;
        *head = uint2{ke | ve << 8, stay | s_bad};
    }

    const float kinv = kv8_pow2(254u - ke), vinv = kv8_pow2(254u - ve);
    if (mine) {
        uint8_t* p = keys + 16 * Kv8<D>::place(row);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int ch = half ? at.second : at.first;
            const float* x = kx + 8 * half;
            *reinterpret_cast<u32x2*>(p + 512 * (ch / 16) + ch % 16) =
                u32x2{f32x4_to_e4m3(x[0] * kinv, x[1] * kinv, x[2] * kinv, x[3] * kinv),
                      f32x4_to_e4m3(x[4] * kinv, x[5] * kinv, x[6] * kinv, x[7] * kinv)};
        }
    }
    if (row < kKv8Block) {                             // zeros where the slot is not new
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = f32x4_to_e4m3(vx[4 * i] * vinv, vx[4 * i + 1] * vinv, vx[4 * i + 2] * vinv, vx[4 * i + 3] * vinv);
        *reinterpret_cast<u32x4*>(&s_v[row][16 * part]) = w;
    }
    if (kept && ke > old_ke) {                         // a thread: 16 channels of a kept slot
        const float by = shrink_factor(old_ke, ke);
        const int place = tid % 32;
        const int s = 16 * (place / 4 % 2) + 4 * (place / 8) + place % 4;
        for (int piece = tid / 32; s < kept && piece < U; piece += kCacheThreads / 32) {
            auto* p = reinterpret_cast<u32x4*>(keys + 512 * piece + 16 * place);
            u32x4 w = *p;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = shrink(w[i], by);
            *p = w;
        }
    }
    __syncthreads();

    // a thread: 16 slots of a channel
    const int half = tid / D, ch = tid % D;
    if (half >= 2) return;
    const bool moves = kept && ve > old_ve && 16 * half < kept;
    // slots of the half that are new, and those that stay
    const int lo = min(max(from - s0 - 16 * half, 0), 16), hi = min(max(to - s0 - 16 * half, 0), 16);
    const int stay = min(max(kept - 16 * half, 0), 16);
    // a block that keeps nothing is written whole: what lies behind its rows is then numbers,
    // which attention may multiply by 0
    if (kept && lo >= hi && !moves) return;
    auto* p = reinterpret_cast<u32x4*>(values + 16 * D * half + 16 * ch);
    u32x4 w = {0u, 0u, 0u, 0u};
    if (kept) w = *p;
    if (moves) {
        const float by = shrink_factor(old_ve, ve);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = shrink(w[i], by);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t fresh = 0u, take = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = 4 * i + j;
            fresh |= (uint32_t)s_v[16 * half + s][ch] << (8 * j);
            take |= s >= stay ? 255u << (8 * j) : 0u;  // zeros behind the new rows, too
        }
        w[i] = (w[i] & ~take) | (fresh & take);
    }
    *p = w;
}

// Rows s0 .. of a block, as append's threads have them.
template <typename T, int D>
__global__ __launch_bounds__(kCacheThreads) void kv8_read_kernel(PagedCache c, const int32_t* starts,
                                                                 const int32_t* counts, int T_rows, T* __restrict__ k,
                                                                 T* __restrict__ v) {
    constexpr int U = D / 16, kPitch = D + 16;
    __shared__ __attribute__((aligned(16))) uint8_t s_v[kKv8Block][kPitch];
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int slots = c.slots(), n = paged_length(starts, b, slots);
    const int64_t end = min((int64_t)slots, (int64_t)n + paged_count(counts, b, T_rows));
    const int64_t s0 = (n & ~(kKv8Block - 1)) + kKv8Block * (int64_t)blockIdx.x;
    if (s0 >= (int64_t)n + T_rows) return;
    const uint8_t* page = s0 < end ? kv8_page<D>(c, b, h, (int)(s0 / kCachePage)) : nullptr;
    const int u = (int)(s0 / kKv8Block % 2);
    const int row = tid / U, part = tid % U;
    const int64_t slot = s0 + row;
    const bool wanted = row < kKv8Block && slot >= n && slot < (int64_t)n + T_rows;
    bool have = wanted && page && slot < end;
    u32x4 kw = {0u, 0u, 0u, 0u}, vw = {0u, 0u, 0u, 0u};
    float ks = 1.f, vs = 1.f;
    if (page) {
        const auto head = *reinterpret_cast<const uint2*>(page + Kv8<D>::kHead + 8 * u);
        const Kv8Head of = {head.x, head.y};
        ks = kv8_pow2(of.key());
        vs = kv8_pow2(of.value());
        const int half = tid / D, ch = tid % D;
        u32x4 column = {0u, 0u, 0u, 0u};
        if (half < 2)
            column = *reinterpret_cast<const u32x4*>(page + Kv8<D>::kValue + 32 * D * u + 16 * D * half + 16 * ch);
        if (have)
            kw = *reinterpret_cast<const u32x4*>(page + 32 * D * u + 512 * part + 16 * Kv8<D>::place(row));
        if (half < 2)
#pragma unroll
            for (int s = 0; s < 16; ++s) s_v[16 * half + s][ch] = (uint8_t)(column[s / 4] >> (8 * (s % 4)));
        if (have && (of.bad >> row & 1u)) {            // a row that was not finite
            ks = vs = __builtin_nanf("");
            have = false;
        }
    }
    __syncthreads();
    if (!wanted) return;
    if (have) vw = *reinterpret_cast<const u32x4*>(&s_v[row][16 * part]);
    float x[16], y[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const auto a0 = __builtin_amdgcn_cvt_pk_f32_fp8(kw[i], false);
        const auto a1 = __builtin_amdgcn_cvt_pk_f32_fp8(kw[i], true);
        const auto b0 = __builtin_amdgcn_cvt_pk_f32_fp8(vw[i], false);
        const auto b1 = __builtin_amdgcn_cvt_pk_f32_fp8(vw[i], true);
        x[4 * i] = a0[0] * ks, x[4 * i + 1] = a0[1] * ks, x[4 * i + 2] = a1[0] * ks, x[4 * i + 3] = a1[1] * ks;
        y[4 * i] = b0[0] * vs, y[4 * i + 1] = b0[1] * vs, y[4 * i + 2] = b1[0] * vs, y[4 * i + 3] = b1[1] * vs;
    }
    const int64_t at = (((int64_t)b * T_rows + (slot - n)) * c.heads + h) * D + 16 * part;
    store<T, 16>(k + at, x);
    store<T, 16>(v + at, y);
}

// Blocks that T rows can touch, whatever their first slot.
int blocks_of(int T) { return (T + kKv8Block - 2) / kKv8Block + 1; }

}  // namespace

hipError_t launch_kv8_append(const PagedCache& c, const PagedRows& k, const PagedRows& v, int dtype,
                             const int32_t* lengths, const int32_t* counts, int T, const KvRotary& rotary,
                             const PagedRows& q, int q_heads, const PagedRows& q_out, hipStream_t s) {
    AppendArgs a{c, k, v, q, rotary, const_cast<void*>(q_out.p), q_out.batch, q_out.token, q_out.head, lengths, counts,
                 T, q_heads / c.heads, 0};
    a.blocks = c.max_pages && c.num_pages ? blocks_of(T) : 0;
    const int chunks = q_heads ? (T + kKv8Block - 1) / kKv8Block : 0;
    if (a.blocks + chunks == 0) return hipSuccess;
    return kv8_by_type(dtype, c.head_dim, [&](auto tag, auto size) {
        hipLaunchKernelGGL((kv8_append_kernel<decltype(tag), decltype(size)::value>),
                           dim3(a.blocks + chunks, c.heads, c.batch), dim3(kCacheThreads), 0, s, a);
    });
}

hipError_t launch_kv8_read(const PagedCache& c, const int32_t* starts, const int32_t* counts, int T, void* k, void* v,
                           int dtype, hipStream_t s) {
    return kv8_by_type(dtype, c.head_dim, [&](auto tag, auto size) {
        using E = decltype(tag);
        hipLaunchKernelGGL((kv8_read_kernel<E, decltype(size)::value>), dim3(blocks_of(T), c.heads, c.batch),
                           dim3(kCacheThreads), 0, s, c, starts, counts, T, static_cast<E*>(k), static_cast<E*>(v));
    });
}

}  // namespace dels
