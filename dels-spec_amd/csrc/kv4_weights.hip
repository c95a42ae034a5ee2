// The attention weights that a block's accepted rows gave to each slot of the 4-bit
// key/value cache (format: kv4.h).
//
//     out[b, h, j] = (j < lengths[b] ? weights[b, h, j] : 0) + sum_t,hq exp(scale * q[t, hq] . k[j] - lse[t, hq])
#include <algorithm>

#include "../../include/dels.h"
#include "kv4.h"

namespace dels {

namespace {

__device__ __forceinline__ float load_q(const bf16_t* p) { return bf16_bits_to_f32(p->bits); }
__device__ __forceinline__ float load_q(const f16_t* p) { return lds_f32(p); }

// Whether row t of the block sees slot j; n and count as the block's sequence has them.
__device__ __forceinline__ bool kv4_sees(int j, int n, int count, int t, int mode, int64_t bits) {
    const int i = j - n;
    if (i < 0) return true;
    if (i >= count || mode == DELS_KV4_NONE) return false;
    if (mode == DELS_KV4_CAUSAL) return i <= t;
    if (mode == DELS_KV4_FULL) return true;
    return i < 64 && ((bits >> i) & 1) != 0;
}

// Dot product of a key row with q (in LDS, fp32).
template <int D>
__device__ __forceinline__ float dot_key(const uint8_t* page, int in_page, const float* q) {
    const uint32_t* row = reinterpret_cast<const uint32_t*>(page + in_page * Kv4<D>::kKeyRow);
    float sum = 0.f;
    for (int blk = 0; blk < D / 32; ++blk) {
        float part = 0.f;
        for (int w = 0; w < 4; ++w) {
            const uint32_t word = row[4 * blk + w];
            for (int i = 0; i < 8; ++i) part += kv4_level((word >> (4 * i)) & 15u) * q[32 * blk + 8 * w + i];
        }
        sum += part * kv4_pow2(page[Kv4<D>::scale_byte(in_page, blk)]);
    }
    return sum;
}

// One workgroup per (sequence, head, page), a thread per slot.
template <typename T, int D>
__global__ __launch_bounds__(kKv4Page) void kv4_weights_kernel(Kv4WeightsArgs a) {
    __shared__ float s_q[D];
    const int tid = threadIdx.x;
    const int p = blockIdx.x % a.cache.max_pages, bh = blockIdx.x / a.cache.max_pages;
    const int h = bh % a.cache.heads, b = bh / a.cache.heads;
    const int slots = a.cache.slots();
    const int n = kv4_length(a.block.lengths, b, slots), count = kv4_count(a.block.counts, b, a.block.T);
    const int rows = min(kv4_count(a.accepted, b, a.block.T), count), group = a.q_heads / a.cache.heads;
    const int j = p * kKv4Page + tid;
    const int end = (int)min((int64_t)slots, (int64_t)n + count);
    const uint8_t* page = p * kKv4Page < end ? kv4_page(a.cache, b, h, p, Kv4<D>::kBytes) : nullptr;
    float sum = 0.f;
    for (int r = 0; page && r < rows * group; ++r) {
        const int t = r / group, hq = h * group + r % group;
        const T* q = static_cast<const T*>(a.q.p) + (int64_t)b * a.q.batch + (int64_t)t * a.q.token +
                     (int64_t)hq * a.q.head;
        __syncthreads();
        for (int i = tid; i < D; i += kKv4Page) s_q[i] = load_q(q + i) * a.scale;
        __syncthreads();
        const float lse = a.lse[((int64_t)b * a.block.T + t) * a.q_heads + hq];
        const int64_t bits = a.block.mode == DELS_KV4_MASK ? a.block.mask[(int64_t)b * a.block.ld_mask + t] : 0;
        if (lse > -__builtin_inff() && j < end && kv4_sees(j, n, count, t, a.block.mode, bits))
            sum += expf(dot_key<D>(page, tid, s_q) - lse);
    }
    const int64_t at = (int64_t)bh * slots + j;
    a.out[at] = (j < n ? a.weights[at] : 0.f) + sum;
}

template <typename F> hipError_t by_type(int dtype, int head_dim, F&& f) {
    auto by_size = [&](auto tag) {
        if (head_dim == 64) f(tag, std::integral_constant<int, 64>{});
        else f(tag, std::integral_constant<int, 128>{});
    };
    if (dtype == DELS_DTYPE_BF16) by_size(bf16_t{});
    else by_size(f16_t{});
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_weights(const Kv4WeightsArgs& a, hipStream_t s) {
    return by_type(a.dtype, a.cache.head_dim, [&](auto tag, auto size) {
        hipLaunchKernelGGL((kv4_weights_kernel<decltype(tag), decltype(size)::value>),
                           dim3((unsigned)a.cache.batch * a.cache.heads * a.cache.max_pages), dim3(kKv4Page), 0, s, a);
    });
}

}  // namespace dels
