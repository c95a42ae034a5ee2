// Eviction from the 4-bit key/value cache by accumulated attention weight.
//
// For a (sequence, head) of n slots, n > keep: the last `recent` slots stay, and
// of the others the keep - recent of largest weight, equal weights by lowest
// slot.  The slots that stay from `keep` on move, in ascending order, into the
// places below `keep` that are given up, in ascending order: what moves is read
// from one side of `keep` and written on the other, so the move needs no order,
// works in place and touches no slot that stays where it is.  (Attention does not
// depend on the order of the slots.)
#include <algorithm>

#include "kv4.h"

namespace dels {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kMoveThreads = 256;

// A larger key is a larger weight; NaN counts as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
    return f32_order_key(w != w ? -__builtin_inff() : w);
}

// One workgroup per (sequence, head).  The threshold is found eight bits of the
// key at a time (a histogram in LDS of the weights that share the bits so far),
// then slots are walked in order: an equal weight's rank among equals, a hole's
// and a mover's rank come from ballots.
__global__ __launch_bounds__(kSelectThreads) void kv4_select_kernel(Kv4EvictArgs a, int32_t* hole_list) {
    __shared__ uint32_t s_hist[256];
    __shared__ uint32_t s_pick, s_left;
    __shared__ int s_wave[3][kSelectThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = blockIdx.x, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const int slots = a.cache.slots(), keep = a.keep;
    const int n = kv4_length(a.lengths, b, slots);
    const float* w = a.weights + (int64_t)bh * slots;
    float* out = a.out_weights + (int64_t)bh * slots;
    int32_t* source = a.source + (int64_t)bh * keep;
    if (h == 0 && tid == 0) a.out_lengths[b] = min(n, keep);
    for (int j = min(n, keep) + tid; j < slots; j += kSelectThreads) out[j] = 0.f;
    for (int64_t j = tid; j < keep; j += kSelectThreads) source[j] = j < n ? (int32_t)j : -1;
    if (n <= keep) {
        for (int j = tid; j < n; j += kSelectThreads) out[j] = w[j];
        return;
    }
    const int recent = min(a.recent, keep), cand = n - recent;
    uint32_t left = keep - recent;                 // candidates still to choose among the equal prefixes
    uint32_t prefix = 0u;
    for (int shift = 24; shift >= 0 && left > 0; shift -= 8) {
        if (tid < 256) s_hist[tid] = 0u;
        __syncthreads();
        for (int j = tid; j < cand; j += kSelectThreads) {
            const uint32_t key = weight_key(w[j]);
            if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&s_hist[(key >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t l = left;
            int d = 255;
            while (d > 0 && s_hist[d] < l) l -= s_hist[d--];
            s_pick = (uint32_t)d;
            s_left = l;
        }
        __syncthreads();
        prefix = (prefix << 8) | s_pick;
        left = s_left;
        __syncthreads();
    }
    // keys above `prefix` are kept, and `left` of those equal to it
    const bool none = keep == recent;
    int32_t* holes = hole_list + (int64_t)bh * keep;
    int equal_before = 0, hole_before = 0, mover_before = 0;
    for (int j0 = 0; j0 < n; j0 += kSelectThreads) {
        const int j = j0 + tid;
        const uint32_t key = j < cand ? weight_key(w[j]) : 0u;
        const bool equal = j < cand && !none && key == prefix;
        const unsigned long long eq = __ballot(equal);
        if (lane == 0) s_wave[0][wave] = __popcll(eq);
        __syncthreads();
        int rank = equal_before + __popcll(eq & ((1ull << lane) - 1));
        for (int v = 0; v < kSelectThreads / 64; ++v) {
            rank += v < wave ? s_wave[0][v] : 0;
            equal_before += s_wave[0][v];
        }
        const bool kept = j < n && (j >= cand || (!none && (key > prefix || (equal && rank < (int)left))));
        const bool hole = j < keep && !kept, mover = j >= keep && kept;
        const unsigned long long hb = __ballot(hole), mb = __ballot(mover);
        if (lane == 0) s_wave[1][wave] = __popcll(hb), s_wave[2][wave] = __popcll(mb);
        __syncthreads();
        int hr = hole_before + __popcll(hb & ((1ull << lane) - 1)), mr = mover_before + __popcll(mb & ((1ull << lane) - 1));
        for (int v = 0; v < kSelectThreads / 64; ++v) {
            hr += v < wave ? s_wave[1][v] : 0;
            mr += v < wave ? s_wave[2][v] : 0;
            hole_before += s_wave[1][v];
            mover_before += s_wave[2][v];
        }
        if (hole) holes[hr] = j;
        if (j < keep && kept) out[j] = w[j];
        __syncthreads();                           // also orders the holes before the movers that read them
        if (mover) {
            const int to = holes[mr];
            source[to] = j;
            out[to] = w[j];
        }
    }
}

// One wave per (sequence, head, 8 places): the places share the value words of
// their row.  Lanes as in the append kernel for the keys; D / 64 channels each for
// the values.
template <int D>
__global__ __launch_bounds__(kMoveThreads) void kv4_move_kernel(Kv4Cache c, const int32_t* lengths,
                                                                const int32_t* __restrict__ sources, int keep,
                                                                int groups) {
    constexpr int N = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * (kMoveThreads / 64) + (threadIdx.x >> 6);
    if (unit >= (int64_t)c.batch * c.heads * groups) return;
    const int g = (int)(unit % groups), bh = (int)(unit / groups), h = bh % c.heads, b = bh / c.heads;
    const int n = kv4_length(lengths, b, c.slots());
    if (n <= keep || 8 * g >= n) return;
    const int mine = 8 * g + (lane & 7) < keep ? sources[(int64_t)bh * keep + 8 * g + (lane & 7)] : -1;
    const bool moves = mine >= keep && mine < n;
    const uint32_t todo = (uint32_t)__ballot(moves) & 0xffu;
    if (!todo) return;
    uint8_t* page = kv4_page(c, b, h, 8 * g / kKv4Page, Kv4<D>::kBytes);
    if (!page) return;
    uint32_t* row = reinterpret_cast<uint32_t*>(page + Kv4<D>::kValue) + (8 * g % kKv4Page / 8) * D + lane * N;
    uint32_t words[N];
#pragma unroll
    for (int j = 0; j < N; ++j) words[j] = row[j];
    for (int i = 0; i < 8; ++i) {
        if (!(todo >> i & 1u)) continue;
        const int from = __shfl(mine, i, 64), in_from = from % kKv4Page, in_to = (8 * g + i) % kKv4Page;
        const uint8_t* old = kv4_page(c, b, h, from / kKv4Page, Kv4<D>::kBytes);
        if (!old) continue;
        if (lane < Kv4<D>::kKeyRow / 4)
            reinterpret_cast<uint32_t*>(page + in_to * Kv4<D>::kKeyRow)[lane] =
                reinterpret_cast<const uint32_t*>(old + in_from * Kv4<D>::kKeyRow)[lane];
        if (lane < D / 32) page[Kv4<D>::scale_byte(in_to, lane)] = old[Kv4<D>::scale_byte(in_from, lane)];
        if (lane == 0)
            *reinterpret_cast<uint16_t*>(page + Kv4<D>::kValueScale + 2 * in_to) =
                *reinterpret_cast<const uint16_t*>(old + Kv4<D>::kValueScale + 2 * in_from);
        const uint32_t* src = reinterpret_cast<const uint32_t*>(old + Kv4<D>::kValue) + (in_from >> 3) * D + lane * N;
#pragma unroll
        for (int j = 0; j < N; ++j)
            words[j] = (words[j] & ~(15u << (4 * i))) | (((src[j] >> (4 * (in_from & 7))) & 15u) << (4 * i));
    }
#pragma unroll
    for (int j = 0; j < N; ++j) row[j] = words[j];
}

}  // namespace

size_t kv4_evict_data_bytes(int64_t batch, int64_t heads, int64_t keep) {
    return align256((size_t)batch * heads * keep * 4);
}

hipError_t launch_kv4_evict(const Kv4EvictArgs& a, void* ws, size_t data_off, hipStream_t s) {
    const Kv4Cache& c = a.cache;
    auto* holes = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + data_off);
    hipLaunchKernelGGL(kv4_select_kernel, dim3(c.batch * c.heads), dim3(kSelectThreads), 0, s, a, holes);
    const int groups = (std::min(a.keep, c.slots()) + 7) / 8, waves = kMoveThreads / 64;
    const dim3 grid((unsigned)(((int64_t)c.batch * c.heads * groups + waves - 1) / waves));
    if (c.head_dim == 64)
        hipLaunchKernelGGL(kv4_move_kernel<64>, grid, dim3(kMoveThreads), 0, s, c, a.lengths, a.source, a.keep, groups);
    else
        hipLaunchKernelGGL(kv4_move_kernel<128>, grid, dim3(kMoveThreads), 0, s, c, a.lengths, a.source, a.keep, groups);
    return hipGetLastError();
}

}  // namespace dels
