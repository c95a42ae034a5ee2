// Eviction from the 4-bit key/value cache by accumulated attention weight.
//
// For a (sequence, head) of n slots, n > keep: the last `recent` slots stay, and
// of the others the keep - recent of largest weight, equal weights by lowest
// slot.  The slots that stay from `keep` on move, in ascending order, into the
// places below `keep` that are given up, in ascending order: what moves is read
// from one side of `keep` and written on the other, so the move needs no order,
// works in place and touches no slot that stays where it is.  (Attention does not
// depend on the order of the slots.)
//
// Slots of an entry that names no page hold nothing: none of them is moved, and as
// places below `keep` they take nothing, so that a (sequence, head) keeps fewer slots,
// `room` of them: as many as there are places.
#include <algorithm>

#include "kv4.h"

namespace dels {

namespace {

constexpr int kPerLane = 16;                               // consecutive slots of a lane per tile
constexpr int kBins = 2048;                                // 11 bits of the key at a time
constexpr int kMoveThreads = 256;

// A larger key is a larger weight; NaN counts as -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
    return f32_order_key(w != w ? -__builtin_inff() : w);
}

// A lane's slots of a row's weights, those past n whatever follows (a row is whole pages).
__device__ __forceinline__ void load_slots(const float* w, int first, int n, float (&x)[kPerLane]) {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) x[i] = 0.f;
    if (first < n) __builtin_memcpy(x, w + first, sizeof(x));
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
// its top); then the slots are walked in order, 16 THREADS at a time and 16 a lane: the
// ranks among equal weights, of holes and of movers are sums over lanes and waves, in
// two exchanges a tile.  Bound by latency; rows of more than one tile are read up to
// four times, all but the first from L2.  COPIES of the histogram: lanes of one digit
// meet on fewer words.
// 16 x 8 rows of up to 16300 slots: 22 us (30 with 64 slots at a time, ranks by ballots), of
// which the first histogram takes 4.6, the two others 4.6 more and the walk the rest; the 128
// workgroups leave half of the CUs idle.
template <int THREADS, int COPIES>
__global__ __launch_bounds__(THREADS) void kv4_select_kernel(Kv4EvictArgs a, int32_t* hole_list) {
    constexpr int kWaves = THREADS / 64, kTile = THREADS * kPerLane, kOwn = kBins / THREADS;
    __shared__ uint32_t s_hist[COPIES][kBins];
    __shared__ int s_wave[kWaves];
    __shared__ uint32_t s_pick, s_left, s_held;
    __shared__ int s_named[2];
    __shared__ int s_count[2][kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int bh = blockIdx.x, h = bh % a.cache.heads, b = bh / a.cache.heads;
    const int slots = a.cache.slots(), keep = a.keep;
    const int n = paged_length(a.lengths, b, slots);
    const float* w = a.weights + (int64_t)bh * slots;
    float* out = a.out_weights + (int64_t)bh * slots;
    int32_t* source = a.source + (int64_t)bh * keep;
    if (h == 0 && tid == 0) a.out_lengths[b] = min(n, keep);
    if (n <= keep) {
        for (int j = n + tid; j < slots; j += THREADS) out[j] = 0.f;
        for (int j = tid; j < n; j += THREADS) out[j] = w[j];
        for (int64_t j = tid; j < keep; j += THREADS) source[j] = j < n ? (int32_t)j : -1;
        return;
    }
    // the first tile (of many rows the only one) is read once
    const int own_first = tid * kPerLane;
    float held[kPerLane];
    load_slots(w, own_first, n, held);
    auto tile_of = [&](int first, float (&x)[kPerLane]) {
        if (first == own_first) {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) x[i] = held[i];
        } else {
            load_slots(w, first, n, x);
        }
    };
    auto clear = [&]() {
        for (int i = tid; i < COPIES * kBins; i += THREADS) (&s_hist[0][0])[i] = 0u;
    };
    // whether any slot lies in no page (a lane's slots lie in one page)
    const int32_t* ids = a.cache.table + (int64_t)b * a.cache.ld_table;
    auto in_page = [&](int page) { return ids[page] >= 0 && ids[page] < a.cache.num_pages; };
    bool gap = false;
    for (int p = tid; p * kCachePage < n; p += THREADS) gap |= !in_page(p);
    clear();
    if (__any(gap)) gap = true;
    if (lane == 0) s_wave[wave] = gap;
    if (tid < 2) s_named[tid] = 0;
    __syncthreads();
    const bool gaps = over_waves<kWaves>(s_wave).y != 0;
    int recent = min(a.recent, keep), chosen = keep - recent;      // chosen by weight
    if (gaps) {
        auto slots_in_pages = [&](int from, int to, int* sum) {
            int mine = 0;
            for (int p = from / kCachePage + tid; p * kCachePage < to; p += THREADS)
                mine += in_page(p) ? min(to, (p + 1) * kCachePage) - max(from, p * kCachePage) : 0;
            atomicAdd(sum, mine);
            __syncthreads();
            return *sum;
        };
        const int room = slots_in_pages(0, keep, &s_named[0]);
        recent = min(recent, room);
        chosen = room - slots_in_pages(n - recent, n, &s_named[1]);
    }
    auto held_at = [&](int first) { return !gaps || (first < n && in_page(first / kCachePage)); };
    const int cand = n - recent;
    uint32_t left = chosen;                        // candidates still to choose among the equal prefixes
    uint32_t prefix = 0u;
    int bits_left = 32;
    while (bits_left > 0 && left > 0) {
        const int digit_bits = min(bits_left, 11), shift = bits_left - digit_bits;
        if (bits_left < 32) {
            clear();
            __syncthreads();
        }
        for (int j0 = 0; j0 < cand; j0 += kTile) {
            const int first = j0 + own_first;
            float x[kPerLane];
            tile_of(first, x);
            const int end = held_at(first) ? cand : 0;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const uint32_t key = weight_key(x[i]);
                const bool mine = bits_left == 32 || (key >> bits_left) == prefix;
                if (first + i < end && mine)
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
        const int upto = sum_upto((int)own);
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
    const bool none = chosen == 0;
    const int unread = none ? 0 : bits_left;       // low bits of the key that did not matter: below 32
    int32_t* holes = hole_list + (int64_t)bh * keep;
    int equal_before = 0, hole_before = 0, mover_before = 0;
    for (int j0 = 0; j0 < n; j0 += kTile) {
        const int first = j0 + own_first;
        float x[kPerLane];
        tile_of(first, x);
        uint32_t kept = 0u, equal = 0u;            // bit i: slot first + i
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int j = first + i;
            const uint32_t key = weight_key(x[i]) >> unread;
            kept |= (uint32_t)(j < n && (j >= cand || (!none && key > prefix))) << i;
            equal |= (uint32_t)(j < cand && !none && key == prefix) << i;
        }
        const bool held_here = held_at(first);
        if (!held_here) kept = equal = 0u;
        const int equals = __popc(equal), e_upto = sum_upto(equals);
        if (lane == 63) s_count[0][wave] = e_upto;
        __syncthreads();
        const int2 e = over_waves<kWaves>(s_count[0]);
        int rank = equal_before + e.x + e_upto - equals;
        equal_before += e.y;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            if ((equal >> i & 1u) && rank < (int)left) kept |= 1u << i;
            rank += equal >> i & 1u;
        }
        // every place below `keep` starts as its own; what moves in comes after
        const uint32_t below = (1u << min(max(keep - first, 0), kPerLane)) - 1u;
        const uint32_t hole = held_here ? below & ~kept : 0u, mover = kept & ~below;
        if (below == (1u << kPerLane) - 1u) {
            int own[kPerLane];
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) own[i] = first + i;
            __builtin_memcpy(out + first, x, sizeof(x));
            __builtin_memcpy(source + first, own, sizeof(own));
        } else {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i)
                if (below >> i & 1u) out[first + i] = x[i], source[first + i] = first + i;
        }
        // holes in the low half, movers in the high half: at most kTile of each
        const int both = __popc(hole) | __popc(mover) << 16, upto = sum_upto(both);
        if (lane == 63) s_count[1][wave] = upto;
        __syncthreads();
        const int2 c = over_waves<kWaves>(s_count[1]);
        const int at = c.x + upto - both;
        int hr = hole_before + (at & 0xffff), mr = mover_before + (at >> 16);
        hole_before += c.y & 0xffff;
        mover_before += c.y >> 16;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
            if (hole >> i & 1u) holes[hr++] = first + i;
        __syncthreads();                           // the holes before the movers that go there
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            if (mover >> i & 1u) {
                const int to = holes[mr++];
                source[to] = first + i;
                out[to] = x[i];
            }
        }
    }
    for (int j = keep + tid; j < slots; j += THREADS) out[j] = 0.f;
}

// One wave per (sequence, head, 8 places): the places share the value words of their
// row, so that no two waves write one word.  What moves is loaded for all eight
// places before any of it is written: K words 16 (8) lanes a slot, value words of D / 64
// channels a lane.  A moved slot's value codes lie in D words of eight slots each, so
// eight times what moves is read: consecutive movers are often neighbours, whose
// words the caches still hold.  16 x 8 rows of up to 16300 slots to 4096, head size 128: 62 us,
// 62 MB written; 30 us without the values, 45 without the keys, 55 without the scales, 23
// without any of them (sources, page numbers and addresses, one after the other).
template <int D>
__global__ __launch_bounds__(kMoveThreads) void kv4_move_kernel(PagedCache c, const int32_t* lengths,
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
    const int n = paged_length(lengths, b, c.slots());
    uint8_t* page = kv4_page(c, b, h, 8 * g / kCachePage, P::kBytes);
    if (n <= keep || 8 * g >= n) return;
    const int64_t page_stride = (int64_t)c.heads * P::kBytes;
    const bool comes = mine >= keep && mine < n;
    const int32_t* ids = c.table + (int64_t)b * c.ld_table;
    int from_id = comes ? ids[mine / kCachePage] : -1;
    const bool moves = comes && from_id >= 0 && from_id < c.num_pages;
    const uint32_t todo = (uint32_t)__ballot(moves) & 0xffu;
    if (!todo || !page) return;
    const int in_page = 8 * g % kCachePage;
    // a place that takes nothing reads its own content
    const uint8_t* own_head = c.data + (int64_t)h * P::kBytes;
    if (!moves) from_id = ids[8 * g / kCachePage];
    const int from_slot = moves ? mine % kCachePage : in_page + i8;

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
    const PagedCache& c = a.cache;
    auto* holes = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + data_off);
    // one tile of a small workgroup where that holds a row: its barriers and histogram take less
    // (600 slots: 10.6 us, 14.2 by the large one)
    const dim3 grid_select(c.batch * c.heads);
    if (c.slots() <= 256 * kPerLane)
        hipLaunchKernelGGL((kv4_select_kernel<256, 1>), grid_select, dim3(256), 0, s, a, holes);
    else
        hipLaunchKernelGGL((kv4_select_kernel<1024, 4>), grid_select, dim3(1024), 0, s, a, holes);
    if (c.slots() == 0) return hipGetLastError();  // nothing to move, and no grid to do it
    const int groups = (std::min(a.keep, c.slots()) + 7) / 8, waves = kMoveThreads / 64;
    const dim3 grid((groups + waves - 1) / waves, c.heads, c.batch);
    if (c.head_dim == 64)
        hipLaunchKernelGGL(kv4_move_kernel<64>, grid, dim3(kMoveThreads), 0, s, c, a.lengths, a.source, a.keep, groups);
    else
        hipLaunchKernelGGL(kv4_move_kernel<128>, grid, dim3(kMoveThreads), 0, s, c, a.lengths, a.source, a.keep, groups);
    return hipGetLastError();
}

}  // namespace dels
