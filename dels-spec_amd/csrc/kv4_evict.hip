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

constexpr int kPerLane = 16;                               // slots of a lane per tile
constexpr int kBins = 2048;                                // 11 bits of the key at a time
constexpr int kMoveThreads = 256;

// A larger key is a larger weight; NaN counts as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
    return f32_order_key(w != w ? -__builtin_inff() : w);
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int scan_wave(int x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(x, off, 64);
        x += lane >= off ? o : 0;
    }
    return x;
}
// Sum of `x` (one value per wave) over the waves before this one, and over all.
template <int WAVES> __device__ __forceinline__ int2 over_waves(const int* x) {
    const int wave = threadIdx.x >> 6;
    int before = 0, all = 0;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
        before += v < wave ? x[v] : 0;
        all += x[v];
    }
    return {before, all};
}

// One workgroup per (sequence, head).  The threshold is found 11 bits of the key at a
// time (a histogram in LDS of the weights that share the bits so far, scanned from
// its top); then the slots are walked in order, 16 THREADS at a time and 1024 of them a
// wave: ranks among equal weights, holes and movers come from ballots, and from the
// waves' counts in three exchanges a tile.  Bound by latency: the weights are read
// four times, all but the first from L2.  COPIES of the histogram: lanes of one digit
// meet on fewer words.
template <int THREADS, int COPIES>
__global__ __launch_bounds__(THREADS) void kv4_select_kernel(Kv4EvictArgs a, int32_t* hole_list) {
    constexpr int kWaves = THREADS / 64, kTile = THREADS * kPerLane, kOwn = kBins / THREADS;
    __shared__ uint32_t s_hist[COPIES][kBins];
    __shared__ int s_wave[kWaves];
    __shared__ uint32_t s_pick, s_left, s_held;
    __shared__ int s_count[3][kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = blockIdx.x, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const int slots = a.cache.slots(), keep = a.keep;
    const int n = kv4_length(a.lengths, b, slots);
    const float* w = a.weights + (int64_t)bh * slots;
    float* out = a.out_weights + (int64_t)bh * slots;
    int32_t* source = a.source + (int64_t)bh * keep;
    if (h == 0 && tid == 0) a.out_lengths[b] = min(n, keep);
    for (int j = min(n, keep) + tid; j < slots; j += THREADS) out[j] = 0.f;
    if (n <= keep) {
        for (int j = tid; j < n; j += THREADS) out[j] = w[j];
        for (int64_t j = tid; j < keep; j += THREADS) source[j] = j < n ? (int32_t)j : -1;
        return;
    }
    const int recent = min(a.recent, keep), cand = n - recent;
    uint32_t left = keep - recent;                 // candidates still to choose among the equal prefixes
    uint32_t prefix = 0u;
    int bits_left = 32;
    while (bits_left > 0 && left > 0) {
        const int digit_bits = min(bits_left, 11), shift = bits_left - digit_bits;
        for (int i = tid; i < COPIES * kBins; i += THREADS) (&s_hist[0][0])[i] = 0u;
        __syncthreads();
        for (int j0 = 0; j0 < cand; j0 += kTile) {
            float x[kPerLane];
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const int j = j0 + i * THREADS + tid;
                x[i] = j < cand ? w[j] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const uint32_t key = weight_key(x[i]);
                const bool mine = bits_left == 32 || (key >> bits_left) == prefix;
                if (j0 + i * THREADS + tid < cand && mine)
                    atomicAdd(&s_hist[lane % COPIES][(key >> shift) & ((1u << digit_bits) - 1)], 1u);
            }
        }
        __syncthreads();
        // bins from the top, kOwn a thread: the one in which the count of larger keys reaches `left`
        uint32_t c[kOwn], own = 0u;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            c[i] = 0u;
#pragma unroll
            for (int q = 0; q < COPIES; ++q) c[i] += s_hist[q][kBins - 1 - (kOwn * tid + i)];
            own += c[i];
        }
        const int upto = scan_wave((int)own);
        if (lane == 63) s_wave[wave] = upto;
        __syncthreads();
        uint32_t before = (uint32_t)(over_waves<kWaves>(s_wave).x + upto) - own;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
            if (before < left && left <= before + c[i])
                s_pick = kBins - 1 - (kOwn * tid + i), s_left = left - before, s_held = c[i];
            before += c[i];
        }
        __syncthreads();
        prefix = (prefix << digit_bits) | s_pick;
        left = s_left;
        bits_left = shift;
        const bool all = s_held == left;           // every key of the prefix is kept: its other bits do not matter
        __syncthreads();
        if (all) break;
    }
    // keys whose bits so far are above `prefix` are kept, and the first `left` of those equal to it
    const bool none = keep == recent;
    int32_t* holes = hole_list + (int64_t)bh * keep;
    int equal_before = 0, hole_before = 0, mover_before = 0;
    for (int j0 = 0; j0 < n; j0 += kTile) {
        // this wave's 1024 slots of the tile, lane by lane
        const int first = j0 + wave * 64 * kPerLane + lane;
        float x[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) x[i] = first + 64 * i < n ? w[first + 64 * i] : 0.f;
        uint32_t kept = 0u, equal = 0u;            // bit i: slot first + 64 i
        int equals = 0;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int j = first + 64 * i;
            const uint32_t key = weight_key(x[i]) >> bits_left;
            const bool eq = j < cand && !none && key == prefix;
            if (j < n && (j >= cand || (!none && key > prefix))) kept |= 1u << i;
            if (eq) equal |= 1u << i;
            equals += __popcll(__ballot(eq));
        }
        if (lane == 0) s_count[0][wave] = equals;
        __syncthreads();
        const int2 e = over_waves<kWaves>(s_count[0]);
        int rank = equal_before + e.x, hole_count = 0, mover_count = 0;
        equal_before += e.y;
        const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int j = first + 64 * i;
            const bool eq = equal >> i & 1u;
            const unsigned long long m = __ballot(eq);
            if (eq && rank + __popcll(m & below) < (int)left) kept |= 1u << i;
            rank += __popcll(m);
            const bool k = kept >> i & 1u;
            hole_count += __popcll(__ballot(j < keep && !k));
            mover_count += __popcll(__ballot(j >= keep && k));
        }
        if (lane == 0) s_count[1][wave] = hole_count, s_count[2][wave] = mover_count;
        __syncthreads();
        const int2 hc = over_waves<kWaves>(s_count[1]), mc = over_waves<kWaves>(s_count[2]);
        int hr = hole_before + hc.x, mr = mover_before + mc.x;
        hole_before += hc.y;
        mover_before += mc.y;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int j = first + 64 * i;
            const bool k = kept >> i & 1u, hole = j < keep && !k;
            const unsigned long long m = __ballot(hole);
            if (hole) holes[hr + __popcll(m & below)] = j;
            hr += __popcll(m);
            if (j < keep && k) {
                source[j] = j;
                out[j] = x[i];
            }
        }
        __syncthreads();                           // the holes before the movers that go there
        if (mc.y) {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const int j = first + 64 * i;
                const bool mover = j >= keep && (kept >> i & 1u);
                const unsigned long long m = __ballot(mover);
                if (mover) {
                    const int to = holes[mr + __popcll(m & below)];
                    source[to] = j;
                    out[to] = x[i];
                }
                mr += __popcll(m);
            }
        }
    }
}

// One wave per (sequence, head, 8 places): the places share the value words of their
// row, so that no two waves write one word.  What moves is loaded for all eight
// places before any of it is written: K words 16 (8) lanes a slot, value words of D / 64
// channels a lane.  A moved slot's value codes lie in D words of eight slots each, so
// eight times what moves is read: consecutive movers are often neighbours, whose
// words the caches still hold.
template <int D>
__global__ __launch_bounds__(kMoveThreads) void kv4_move_kernel(Kv4Cache c, const int32_t* lengths,
                                                                const int32_t* __restrict__ sources, int keep,
                                                                int groups) {
    constexpr int N = D / 64;
    constexpr int kRowLanes = Kv4<D>::kKeyRow / 4, kSlotsPerLoad = 64 / kRowLanes, kLoads = 8 / kSlotsPerLoad;
    using P = Kv4<D>;
    const int lane = threadIdx.x & 63;
    const int g = blockIdx.x * (kMoveThreads / 64) + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    if (g >= groups) return;
    const int64_t bh = (int64_t)b * c.heads + h;
    // lane i < 8 (and i + 8, ...): the slot that place i takes, and its page.  All of this is
    // loaded before any of it is looked at.
    const int i8 = lane & 7;
    const int mine = 8 * g + i8 < keep ? sources[bh * keep + 8 * g + i8] : -1;
    const int n = kv4_length(lengths, b, c.slots());
    uint8_t* page = kv4_page(c, b, h, 8 * g / kKv4Page, P::kBytes);
    if (n <= keep || 8 * g >= n) return;
    const int64_t page_stride = (int64_t)c.heads * P::kBytes;
    const bool comes = mine >= keep && mine < n;
    const int32_t* ids = c.table + (int64_t)b * c.ld_table;
    int from_id = comes ? ids[mine / kKv4Page] : -1;
    const bool moves = comes && from_id >= 0 && from_id < c.num_pages;
    const uint32_t todo = (uint32_t)__ballot(moves) & 0xffu;
    if (!todo || !page) return;
    const int in_page = 8 * g % kKv4Page;
    // a place that takes nothing reads its own content
    const uint8_t* own_head = c.data + (int64_t)h * P::kBytes;
    if (!moves) from_id = ids[8 * g / kKv4Page];
    const int from_slot = moves ? mine % kKv4Page : in_page + i8;

    uint32_t* row = reinterpret_cast<uint32_t*>(page + P::kValue) + (in_page / 8) * D + lane * N;
    uint32_t words[N], src[8][N], key[kLoads];
#pragma unroll
    for (int j = 0; j < N; ++j) words[j] = row[j];
    int slot[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        slot[i] = __builtin_amdgcn_readlane(from_slot, i);
        const uint8_t* from = own_head + __builtin_amdgcn_readlane(from_id, i) * page_stride;
        const uint32_t* at = reinterpret_cast<const uint32_t*>(from + P::kValue) + (slot[i] >> 3) * D + lane * N;
#pragma unroll
        for (int j = 0; j < N; ++j) src[i][j] = at[j];
    }
    // place i's source, for lanes that differ in i
    auto far = [&](int i) { return own_head + (int64_t)__shfl(from_id, i, 64) * page_stride; };
    const int sub = lane / kRowLanes, word = lane % kRowLanes;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
        const int i = q * kSlotsPerLoad + sub;
        key[q] = reinterpret_cast<const uint32_t*>(far(i) + __shfl(from_slot, i, 64) * P::kKeyRow)[word];
    }
    // scales: a lane per (place, block) and per place
    constexpr int kBlocks = D / 32;
    const int si = lane / kBlocks & 7, blk = lane % kBlocks;
    const uint8_t ks = far(si)[P::scale_byte(__shfl(from_slot, si, 64), blk)];
    const uint16_t vs = *reinterpret_cast<const uint16_t*>(own_head + from_id * page_stride + P::kValueScale + 2 * from_slot);

#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
        const int i = q * kSlotsPerLoad + sub;
        if (todo >> i & 1u) reinterpret_cast<uint32_t*>(page + (in_page + i) * P::kKeyRow)[word] = key[q];
    }
    if (lane < 8 * kBlocks && (todo >> si & 1u)) page[P::scale_byte(in_page + si, blk)] = ks;
    if (lane < 8 && (todo >> i8 & 1u)) *reinterpret_cast<uint16_t*>(page + P::kValueScale + 2 * (in_page + i8)) = vs;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (todo >> i & 1u) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                words[j] = (words[j] & ~(15u << (4 * i))) | (((src[i][j] >> (4 * (slot[i] & 7))) & 15u) << (4 * i));
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
    // few slots: a short tile and a small workgroup, whose barriers and histogram take less
    const dim3 grid_select(c.batch * c.heads);
    if (c.slots() <= 256 * kPerLane)
        hipLaunchKernelGGL((kv4_select_kernel<256, 1>), grid_select, dim3(256), 0, s, a, holes);
    else
        hipLaunchKernelGGL((kv4_select_kernel<1024, 4>), grid_select, dim3(1024), 0, s, a, holes);
    const int groups = (std::min(a.keep, c.slots()) + 7) / 8, waves = kMoveThreads / 64;
    const dim3 grid((groups + waves - 1) / waves, c.heads, c.batch);
    if (c.head_dim == 64)
        hipLaunchKernelGGL(kv4_move_kernel<64>, grid, dim3(kMoveThreads), 0, s, c, a.lengths, a.source, a.keep, groups);
    else
        hipLaunchKernelGGL(kv4_move_kernel<128>, grid, dim3(kMoveThreads), 0, s, c, a.lengths, a.source, a.keep, groups);
    return hipGetLastError();
}

}  // namespace dels
