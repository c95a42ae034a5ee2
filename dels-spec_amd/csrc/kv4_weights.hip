// The attention weights that a block's accepted rows gave to each slot of the 4-bit
// key/value cache (format: kv4.h).
//
//     out[b, h, j] = (j < lengths[b] ? weights[b, h, j] : 0) + sum_t,hq exp(scale * q[t, hq] . k[j] - lse[t, hq])
//
// The keys are read once, the values not at all: S [rows x slots] = Q K^T on the
// matrix cores, a slot per lane and rows along its registers, so that the sum over
// rows is an addition per score and one exchange between lane groups per slot.  A
// wave turns 32 slots' codes into operands once and takes all row tiles over them.
// Rows beyond 128 go in further rounds over the piece's pages.  Every slot belongs to
// one wave: no atomics, one order of additions.
//
// Tiles of 16 rows whatever their number: the products are few enough that the shorter
// chains of the 16-row instruction count for more than its rate (64 rows: 8 x 4000
// slots 17.8 us with tiles of 32, 14.1 with 16; 64 x 8000 slots 110 and 101; 4 x 2000 slots
// of 2048 rows 196 and 175).  Long caches are bound by the read of their keys (32 x 16k
// slots, one token: 66 us, 4.3 TB/s), short ones by latency.
#include <algorithm>

#include "kv4_mma.h"

namespace dels {

namespace {

constexpr int kMinPages = kKv4Waves;             // fewest pages of a part
constexpr int MT = 16;                           // rows of a tile
constexpr int kRows = 128;                       // rows whose queries fit LDS at a time

template <typename T, int D>
__global__ __launch_bounds__(kKv4Threads, 4) void kv4_weights_kernel(Kv4WeightsArgs a, int pieces) {
    using S = Shape<D, MT>;
    using F = typename Frag<T>::type;
    __shared__ F s_q[kRows / MT][S::KS][64];
    __shared__ __align__(16) float s_lse[kRows];             // binary logarithms, +inf for a row that does not count
    __shared__ __align__(16) int s_lim[kRows];               // of the block's slots a row sees those below,
    __shared__ uint64_t s_bits[kRows];                       // and those whose bits are set

    const Kv4Cache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane % MT, g = lane / MT;
    const int slots = c.slots(), group = a.q_heads / c.heads;
    const LaneOffsets<D, MT> at_lane(col, g);
    Scan scan(a.block, c, c.heads);
    const Cuts cuts(scan, Line{1, pieces, kMinPages}, INT32_MAX);
    const float mag = fabsf(a.scale);
    const float unit = (mag == 0.f ? 1.f : mag) * kLog2e * (float)(1 << kKeyShift<T>);
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, zero = mag == 0.f ? 0u : ~0u;

    Scan::Place at{};
    const int2 piece = cuts.piece(scan, blockIdx.x, at);
    int u = piece.x;
    const int u_end = piece.y;
    while (u < u_end) {
        if (u >= at.start + at.pages * scan.per) at = scan.place(u);
        const int b = at.b, rel = u - at.start, h = divide(rel, at.pages), first = rel - h * at.pages;
        const int last = min(at.pages, first + (u_end - u));
        const int n = at.n, count = at.count;
        const int first_page = first + wave;
        const int filled = seq_end(a.block, n, count, slots);
        const int32_t* ids = c.table + (int64_t)b * c.ld_table;
        auto id_at = [&](int p) { return p < last && p * kKv4Page < filled ? ids[p] : -1; };
        const int first_id = id_at(first_page);
        const int rows = uniform(min(kv4_count(a.accepted, b, a.block.T), count)) * group;
        const uint8_t* heads = c.data + (int64_t)h * Kv4<D>::kBytes;
        const int64_t page_stride = (int64_t)c.heads * Kv4<D>::kBytes;
        const int64_t out_row = ((int64_t)b * c.heads + h) * slots;
        auto named = [&](int id) { return id >= 0 && id < c.num_pages; };

        int r0 = 0;
        do {                                                 // once without rows too: the old weights move
            const int tiles = (min(rows - r0, kRows) + MT - 1) / MT;
            KeyWords<D, MT> keys, next_keys;                 // the first are on their way with the queries
            int p = first_page, id = uniform(first_id);
            if (p < last) keys.load(heads + (named(id) ? id : 0) * page_stride, at_lane);
            __syncthreads();
            for (int i = wave; i < tiles * S::KS; i += kKv4Waves) {
                const int tile = i / S::KS, k = i % S::KS, r = r0 + tile * MT + col;
                u32x4 w = {0u, 0u, 0u, 0u};
                if (r < rows) {
                    const int t = divide(r, group), hq = h * group + r - t * group;
                    w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q.p) + (int64_t)b * a.q.batch +
                                                        (int64_t)t * a.q.token + (int64_t)hq * a.q.head + g * S::DL + 8 * k);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) w[x] = (w[x] ^ flip) & zero;
                s_q[tile][k][lane] = __builtin_bit_cast(F, w);
            }
            if ((int)threadIdx.x < kRows) {
                const int r = r0 + threadIdx.x, t = divide(r, group);
                float lse = __builtin_inff();
                int lim = 0;
                uint64_t bits = 0;
                if (r < rows) {
                    lim = a.block.mode == DELS_KV4_CAUSAL ? t + 1 : a.block.mode == DELS_KV4_FULL ? count : 0;
                    if (a.block.mode == DELS_KV4_MASK)
                        bits = (uint64_t)a.block.mask[(int64_t)b * a.block.ld_mask + t] &
                               (count >= 64 ? ~0ull : (1ull << count) - 1);
                    lse = a.lse[((int64_t)b * a.block.T + t) * a.q_heads + h * group + r - t * group] * kLog2e;
                    if (lse == -__builtin_inff()) lse = __builtin_inff();   // an empty row gave nothing
                }
                s_lse[threadIdx.x] = lse;
                s_lim[threadIdx.x] = lim;
                s_bits[threadIdx.x] = bits;
            }
            __syncthreads();

            for (; p < last; p += kKv4Waves) {
                const int next = uniform(id_at(p + kKv4Waves));
                next_keys.load(heads + (named(next) ? next : 0) * page_stride, at_lane);
                asm volatile("" ::: "memory");
                // the slot that this lane writes, of the four it has sums for: by its group
                const int mine = p * kKv4Page + 32 * (g >> 1) + S::slot_of(g & 1, col);
                float sum = r0 > 0 ? a.out[out_row + mine] : mine < n ? a.weights[out_row + mine] : 0.f;
                if (named(id) && tiles > 0) {
                    const bool masked = (p + 1) * kKv4Page > n;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        F kf[S::KT][S::KS];
#pragma unroll
                        for (int t = 0; t < S::KT; ++t)
#pragma unroll
                            for (int k = 0; k < S::KS; ++k) {
                                const uint32_t scales = keys.scale[k * 8 / 32 % S::KB] >> (8 * t);
                                kf[t][k] = decode8<T>(keys.code[s][t][k], key_scale<T>(scales, 2 * s));
                            }
                        float part[S::KT] = {};
                        for (int tile = 0; tile < tiles; ++tile) {
                            typename S::Acc acc[S::KT];
#pragma unroll
                            for (int t = 0; t < S::KT; ++t)
#pragma unroll
                                for (int i = 0; i < S::ACC; ++i) acc[t][i] = 0.f;
#pragma unroll
                            for (int k = 0; k < S::KS; ++k) {
                                const F qk = s_q[tile][k][lane];
#pragma unroll
                                for (int t = 0; t < S::KT; ++t) acc[t] = mma(qk, kf[t][k], acc[t]);
                            }
                            // a lane's registers are rows 4 g .. 4 g + 3 of the tile
                            const int row = tile * MT + 4 * g;
                            const f32x4 lse = *reinterpret_cast<const f32x4*>(&s_lse[row]);
#pragma unroll
                            for (int t = 0; t < S::KT; ++t)
#pragma unroll
                                for (int x = 0; x < 4; ++x) acc[t][x] = __builtin_fmaf(acc[t][x], unit, -lse[x]);
                            if (masked) {                    // after the sum: a slot unseen gets 0 of a NaN row too
                                asm volatile("");            // a branch, not a selection on every page
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const int lim = s_lim[row + x];
                                    const uint64_t bits = s_bits[row + x];
#pragma unroll
                                    for (int t = 0; t < S::KT; ++t) {
                                        const int i = p * kKv4Page + 32 * s + S::slot_of(t, col) - n;
                                        const uint32_t bit = i < 0 || i > 63 ? 0u : (uint32_t)(bits >> (i & 63)) & 1u;
                                        acc[t][x] = i < lim || bit ? acc[t][x] : -__builtin_inff();
                                    }
                                }
                            }
#pragma unroll
                            for (int t = 0; t < S::KT; ++t)
#pragma unroll
                                for (int x = 0; x < 4; ++x)
                                    part[t] += __builtin_amdgcn_exp2f(acc[t][x]);
                        }
#pragma unroll
                        for (int t = 0; t < S::KT; ++t) {
                            const float all = sum_over_groups<MT>(part[t]);
                            if (g == 2 * s + t) sum += all;
                        }
                    }
                }
                a.out[out_row + mine] = sum;
                keys = next_keys;
                id = next;
            }
            r0 += kRows;
        } while (r0 < rows);
        u += last - first;
    }

    // slots past the pages of a sequence are 0
    const int rest = c.batch * c.heads;
    for (int bh = blockIdx.x; bh < rest; bh += gridDim.x) {
        const int pages = uniform(seq_pages(a.block, bh / c.heads, slots));
        for (int j = pages * kKv4Page + threadIdx.x; j < slots; j += kKv4Threads) a.out[(int64_t)bh * slots + j] = 0.f;
    }
}

// A cache of no pages, or a block of no rows: the old weights, cut off at the lengths.
__global__ void kv4_no_weights_kernel(Kv4WeightsArgs a) {
    const int slots = a.cache.slots(), rows = a.cache.batch * a.cache.heads;
    for (int bh = blockIdx.y; bh < rows; bh += gridDim.y) {
        const int n = kv4_length(a.block.lengths, bh / a.cache.heads, slots);
        const int64_t row = (int64_t)bh * slots;
        for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < slots; j += gridDim.x * blockDim.x)
            a.out[row + j] = j < n ? a.weights[row + j] : 0.f;
    }
}

}  // namespace

hipError_t launch_kv4_weights(const Kv4WeightsArgs& a, hipStream_t s) {
    const Kv4Cache& c = a.cache;
    if (c.num_pages == 0 || a.block.T == 0) {
        const int rows = (int)std::min<int64_t>((int64_t)c.batch * c.heads, 65535);
        hipLaunchKernelGGL(kv4_no_weights_kernel, dim3((c.slots() + 1023) / 1024, rows), dim3(256), 0, s, a);
        return hipGetLastError();
    }
    const int64_t units = (int64_t)c.batch * c.heads * c.max_pages;
    // two workgroups a CU: 32 x 16k slots 74 us with one, 68 with two (66 with the first keys ahead of the queries)
    const int pieces = (int)std::min<int64_t>(2 * device_cu_count(), std::max<int64_t>((int64_t)c.batch * c.heads,
                                                                                       (units + kMinPages - 1) / kMinPages));
    return kv4_by_type(a.dtype, c.head_dim, [&](auto tag, auto size) {
        hipLaunchKernelGGL((kv4_weights_kernel<decltype(tag), decltype(size)::value>), dim3(pieces), dim3(kKv4Threads), 0, s,
                           a, pieces);
    });
}

}  // namespace dels
