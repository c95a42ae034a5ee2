// Attention over the 4-bit key/value cache (format: kv4.h).
//
//     x[t, j] = scale * q[t] . k[j]          j a slot that row t sees
//     lse[t]  = log sum_j exp(x[t, j])
//     o[t]    = sum_j exp(x[t, j] - lse[t]) v[j]
// A row that sees nothing has o = 0 and lse = -inf.
//
// One pass over the slots with the running maximum and sum of each row's softmax.
// The rows that share a cache head (block tokens x query heads of the group) are
// the columns of both products:
//     S^T [slots x rows] = K Q^T          O^T [channels x rows] += V^T P^T
// so a lane holds scores of eight consecutive slots of one row, which is the
// operand of the second product: P stays in its lane.  Key codes become bf16 (or
// f16) by the conversion instruction with their block's scale, value codes bf16 with
// scale 2^-20 for all; the value scale of a slot multiplies its weight.  That product enters the
// matrix cores as two bf16 parts (2^-17 of each weight, whatever its size: one part
// alone would round every weight by 2^-8, as much as a bf16 output itself, and f16
// would lose the small ones).  Scores, maxima, sums and outputs are fp32.
//
// A wave takes a page of 64 slots at a time.  WAYS of the 8 waves of a workgroup share a
// row tile and take every WAYS-th page, and their states are joined through LDS; 8 / WAYS
// row tiles go over the same pages at the same time.  The pages of all (sequence,
// head, tiles) are numbered in one line and cut into pieces, one for each workgroup
// (Cuts, kv4_mma.h): a piece that covers all pages of its rows writes their output, others
// write their state, and the last of them to arrive joins the states in their order, so
// that results do not depend on who that is.
//
// Head size 128, 32 query heads on 8.  One token, 32 sequences of up to 16300 slots: 95 us,
// bound by memory (5.1 TB/s over the whole, 6 in the loop).  16 tokens over 131k slots:
// 75 us = 0.46 PFLOP/s, 2 x 512 tokens over up to 3500 slots: 103 us; bound by vector
// instructions, 650 a page and wave against 48 matrix ones of 32 cycles.  One token over
// 700 slots: 9 us, bound by latency: 4 until the first page is there.
#include <algorithm>

#include "kv4_mma.h"

namespace dels {

namespace {

// What a row's weights are relative to lies this many binary orders above its largest score
// when it moves, and moves when a score passes it: until then the outputs need no rescaling,
// no weight is above 1, and its product with a value scale stays finite.
constexpr float kLag = 8.f;
// Values enter their product at 2^-20 of their size (the conversion scales for nothing), so
// that sums over 2^20 slots of the largest values that the cache holds, 3e38, stay finite;
// the reciprocal of the weights' sum makes up for it.
constexpr float kShrink = 0x1p-20f, kGrow = 0x1p20f;

// Two numbers rounded to bf16, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

constexpr int kMinPages = 2 * kKv4Waves;      // fewest pages of a part (one row over 700 slots: 10.6 us in two of eight, 9.2 in one)
constexpr int kCounterWords = 16;      // words from one arrival counter to the next
// Most parts of one tile group (Cuts, kv4_mma.h; even cuts know no limit but the number of
// workgroups): their states are joined by one workgroup, about 0.25 us each (one row over
// 94k slots: 45 us in 184 parts, 29 in 32).
constexpr int kMostParts = 32;

template <typename T> __device__ __forceinline__ uint16_t round_to(float x);
template <> __device__ __forceinline__ uint16_t round_to<bf16_t>(float x) { return f32_to_bf16_bits(x); }
template <> __device__ __forceinline__ uint16_t round_to<f16_t>(float x) {
    const _Float16 h = (_Float16)x;
    uint16_t b;
    __builtin_memcpy(&b, &h, 2);
    return b;
}

// A row tile's row of this lane: token, query head, whether it is a valid row.
struct Row { int t, hq; bool in_block, valid; };
__device__ __forceinline__ Row row_of(int r, int group, int h, int T, int count) {
    Row x;
    x.t = divide(r, group);
    x.hq = h * group + (r - x.t * group);
    x.in_block = x.t < T;
    x.valid = x.t < count;
    return x;
}

template <typename T, int VW>
__device__ __forceinline__ void store_out(const Kv4AttentionArgs& a, int b, const Row& row, int ch, const float* o,
                                          float inv) {
    if (!row.in_block) return;
    uint16_t* p = static_cast<uint16_t*>(a.out) + (int64_t)b * a.out_batch + (int64_t)row.t * a.out_token +
                  (int64_t)row.hq * a.out_head + ch;
    uint32_t w[VW / 2];
#pragma unroll
    for (int i = 0; i < VW / 2; ++i) {
        const float x = row.valid ? o[2 * i] * inv : 0.f, y = row.valid ? o[2 * i + 1] * inv : 0.f;
        w[i] = (uint32_t)round_to<T>(x) | ((uint32_t)round_to<T>(y) << 16);
    }
    if constexpr (VW == 4) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// `ref`: binary logarithm of the unit that `total` counts in.  A sum of 0 is a row that saw
// nothing (the largest score's weight is at least 2^-kLag, or nearly); NaN is a row of scores that are none.
__device__ __forceinline__ void store_lse(const Kv4AttentionArgs& a, int b, const Row& row, float ref, float total) {
    if (!row.in_block) return;
    const float x = row.valid && total != 0.f ? (ref + __builtin_amdgcn_logf(total)) * 0.693147180559945309f
                                             : -__builtin_inff();
    a.lse[((int64_t)b * a.block.T + row.t) * a.q_heads + row.hq] = x;
}

// exp2(m - ref), 0 for m = -inf, whatever ref is.
__device__ __forceinline__ float fade(float m, float ref) {
    return m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - ref);
}

// Floats of a piece's state in the workspace: outputs as the lanes hold them, then references and sums.
template <int D, int MT> constexpr int kStateFloats = MT * D + 2 * MT;

template <int D, int MT> struct ValueWords {
    using S = Shape<D, MT>;
    uint32_t code[2][S::PF][S::CT];
    u32x4 scale[2][S::PF];
    __device__ __forceinline__ void load(const uint8_t* page, const LaneOffsets<D, MT>& at) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int f = 0; f < S::PF; ++f) {
                const int kg = 4 * s + 2 * f;  // past the lane group's own
#pragma unroll
                for (int l = 0; l < S::VL; ++l)
#pragma unroll
                    for (int i = 0; i < S::VW; ++i)
                        code[s][f][l * S::VW + i] = page_word(page, at.value, 4 * (kg * D + l * MT * S::VW))[i];
                scale[s][f] = *reinterpret_cast<const u32x4*>(page_word(page, at.value_scale, 16 * kg));
            }
    }
};

// The rows' state of a wave, and one page's part in it.
template <typename T, int D, int MT> struct Rows {
    using S = Shape<D, MT>;
    using F = typename Frag<T>::type;
    typename S::Acc o[S::CT];
    float top, total;          // what weights are relative to (in raw products) and this lane's part of their sum
    int lim;                   // the row sees slots below it,
    uint64_t bits;             // and those of the block whose bits are set

    // n, filled: context, and the slots that hold anything; unit: binary logarithms per raw
    // product; lag: kLag in raw products
    // q: this lane's operands of the queries in LDS, 64 apart
    __device__ __forceinline__ void page(const F* q, const KeyWords<D, MT>& keys, ValueWords<D, MT>& values, uint32_t half,
                                         int first_slot, int n, int filled, int slots, int g, float unit, float lag) {
        // a page that reaches past the context (a branch: the statement keeps the compiler from
        // computing the masks of every page and selecting)
        const bool masked = first_slot + kKv4Page > n;
        if (masked) {
            asm volatile("");
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int f = 0; f < S::PF; ++f) {
                    const int j = first_slot + 32 * s + 8 * (MT == 16 ? g : 2 * f + g);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        values.scale[s][f][i] &= (j + 2 * i < filled ? 0xffffu : 0u) |
                                                  (j + 2 * i + 1 < filled ? 0xffff0000u : 0u);
                }
        }
        // scores of the page's 64 slots; unit u = (half, operand) holds slots 32 s + 8 kg .. + 7
        typename S::Acc acc[2][S::KT];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < S::KT; ++t)
#pragma unroll
                for (int i = 0; i < S::ACC; ++i) acc[s][t][i] = 0.f;
        F next_q = q[0];
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
            const F qk = next_q;
            if (k + 1 < S::KS) next_q = q[64 * (k + 1)];       // read a step ahead
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < S::KT; ++t) {
                    const uint32_t scales = keys.scale[k * 8 / 32 % S::KB] >> (MT == 16 ? 8 * t : half);
                    acc[s][t] = mma(decode8<T>(keys.code[s][t][k], key_scale<T>(scales, 2 * s)), qk, acc[s][t]);
                }
        }
        float x[2 * S::PF][8];
#pragma unroll
        for (int u = 0; u < 2 * S::PF; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[u][i] = MT == 16 ? acc[u / S::PF][i >> 2 & (S::KT - 1)][i & 3]
                                   : acc[u / S::PF][0][(8 * (u % S::PF) + i) % S::ACC];
        // without this fence the scheduler decodes values ahead of the scores and spills
        __builtin_amdgcn_sched_barrier(0);
        if (masked) {
            asm volatile("");
#pragma unroll
            for (int u = 0; u < 2 * S::PF; ++u) {
                const int j0 = first_slot + 32 * (u / S::PF) + 8 * (MT == 16 ? g : 2 * (u % S::PF) + g);
                // the slots that the row sees by its mask, the first one in bit 0
                const int d = j0 - n;
                uint32_t by_bit = d >= 64 || d <= -8 ? 0u : (uint32_t)(d >= 0 ? bits >> d : bits << -d) & 255u;
                by_bit &= slots - j0 >= 8 ? 255u : (1u << max(slots - j0, 0)) - 1u;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (j0 + i >= lim && !(by_bit >> i & 1u)) x[u][i] = -__builtin_inff();
            }
        }
        float best = x[0][0];
#pragma unroll
        for (int u = 0; u < 2 * S::PF; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) best = fmaxf(best, x[u][i]);
        best = max_over_groups<MT>(best);
        if (__any(best > top)) {
            const float now = fmaxf(top, best + lag), f = fade(top * unit, now * unit);
            top = now;
            total *= f;
#pragma unroll
            for (int t = 0; t < S::CT; ++t)
#pragma unroll
                for (int i = 0; i < S::ACC; ++i) o[t][i] *= f;
        }
        const float ref = top == -__builtin_inff() ? 0.f : top * unit;
        // The weights of a unit are made while the one before multiplies the values: between
        // two matrix instructions stand about as many cycles of vector ones, in this order
        // (the fences keep it), so that neither waits for the other.
        u32x4 hi[2], lo[2];
        float even = 0.f;
        auto weigh = [&](int u, int i) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], unit, -ref));
            total += e;
            const uint32_t vs = values.scale[u / S::PF][u % S::PF][i / 2];
            const float v = e * __uint_as_float(i & 1 ? vs & 0xffff0000u : vs << 16);
            if (i % 2 == 0) {
                even = v;
            } else {
                const uint32_t h = pack_bf16(even, v);
                hi[u & 1][i / 2] = h;
                lo[u & 1][i / 2] = pack_bf16(even - __uint_as_float(h << 16), v - __uint_as_float(h & 0xffff0000u));
            }
        };
#pragma unroll
        for (int i = 0; i < 8; ++i) weigh(0, i);
#pragma unroll
        for (int u = 0; u < 2 * S::PF; ++u) {
            const bool more = u + 1 < 2 * S::PF;
            constexpr int kFirst = S::CT >= 8 ? 0 : 4 / S::CT;     // weights before a tile's first product,
            constexpr int kBoth = 8 / S::CT;                       // and before its second
#pragma unroll
            for (int t = 0; t < S::CT; ++t) {
                const bf16x8 vf = decode8<bf16_t>(values.code[u / S::PF][u % S::PF][t], kShrink);
#pragma unroll
                for (int i = t * kBoth; more && i < t * kBoth + kFirst; ++i) weigh(u + 1, i);
                __builtin_amdgcn_sched_barrier(0);
                o[t] = mma(vf, __builtin_bit_cast(bf16x8, hi[u & 1]), o[t]);
#pragma unroll
                for (int i = t * kBoth + kFirst; more && i < (t + 1) * kBoth; ++i) weigh(u + 1, i);
                __builtin_amdgcn_sched_barrier(0);
                o[t] = mma(vf, __builtin_bit_cast(bf16x8, lo[u & 1]), o[t]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
};

template <typename T, int D, int MT, int WAYS>
__global__ __launch_bounds__(kKv4Threads, 2) void kv4_attention_kernel(Kv4AttentionArgs a, Line line, float* states,
                                                                       unsigned int* counters) {
    using S = Shape<D, MT>;
    constexpr int kRegs = S::CT * S::ACC;                   // output registers
    constexpr int kRound = 32;                              // registers joined at a time
    __shared__ float s_o[kKv4Waves][kRound][64];
    __shared__ float s_m[kKv4Waves][MT], s_l[kKv4Waves][MT];
    constexpr int kTiles = kKv4Waves / WAYS;
    __shared__ typename Frag<T>::type s_q[kTiles][S::KS][64];
    __shared__ bool s_last;

    const Kv4Cache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane % MT, g = lane / MT, tile = wave / WAYS, way = wave % WAYS;
    const int slots = c.slots(), group = a.q_heads / c.heads;
    // pieces that follow each other on one XCD: they share pages where a head has several row tiles
    const int piece = (int)gridDim.x % 8 ? (int)blockIdx.x
                                         : (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
    const LaneOffsets<D, MT> at_lane(col, g);
    Scan scan(a.block, c, c.heads * line.tiles);
    const Cuts cuts(scan, line, kMostParts);
    Scan::Place at{};
    const int2 mine = cuts.piece(scan, piece, at);
    int u = mine.x;
    const int u_end = mine.y;
    if (u >= u_end) return;
    // scores in units of the maximum: |scale| and the query's sign
    const float mag = fabsf(a.scale);
    const float unit = (mag == 0.f ? 1.f : mag) * kLog2e * (float)(1 << kKeyShift<T>);
    const float lag = fminf(kLag / unit, 1e37f);           // finite where the scale is next to nothing
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, zero = mag == 0.f ? 0u : ~0u;

    while (u < u_end) {
        if (u >= at.start + at.pages * scan.per) at = scan.place(u);
        const int b = at.b;
        const int rel = u - at.start, ht = divide(rel, at.pages), first = rel - ht * at.pages;
        const int h = divide(ht, line.tiles), rt0 = (ht - h * line.tiles) * kTiles, rt = rt0 + tile;
        const int last = min(at.pages, first + (u_end - u));
        const int n = at.n, count = at.count;
        const int filled = seq_end(a.block, n, count, slots);     // slots past it may hold anything
        int end = filled;
        if (a.block.mode == DELS_KV4_CAUSAL)                  // no row of the tile sees past its last token
            end = (int)min((int64_t)end, (int64_t)n + divide(rt * MT + MT - 1, group) + 1);
        if (rt * MT >= a.block.T * group) end = 0;            // past the block's rows
        const int stop = min(last, (end + kKv4Page - 1) / kKv4Page);

        // the wave's pages, the next one loaded while one is worked on
        const int32_t* ids = c.table + (int64_t)b * c.ld_table;
        const uint8_t* heads = c.data + (int64_t)h * Kv4<D>::kBytes;
        const int64_t page_stride = (int64_t)c.heads * Kv4<D>::kBytes;
        int p = first + way;
        // the numbers of the wave's next 64 pages, one a lane: a load per page would be
        // waited for with the first read of LDS
        int ids64, base;
        auto fetch_ids = [&](int from) {
            base = from;
            const int at_page = from + lane * WAYS;
            ids64 = at_page < stop ? ids[at_page] : -1;
        };
        auto id_at = [&](int at_page) {
            if (at_page - base >= 64 * WAYS) fetch_ids(at_page);
            return __builtin_amdgcn_readlane(ids64, (at_page - base) / WAYS);
        };
        fetch_ids(p);

        // the queries of all tiles, in operand order
        constexpr int kPerWave = (kTiles * S::KS + kKv4Waves - 1) / kKv4Waves;
        u32x4 qw[kPerWave];
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int e = wave + i * kKv4Waves, k = e % S::KS;
            const Row of = row_of((rt0 + e / S::KS) * MT + col, group, h, a.block.T, count);
            qw[i] = u32x4{0u, 0u, 0u, 0u};
            if (of.valid && e < kTiles * S::KS)
                qw[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q.p) + (int64_t)b * a.q.batch +
                                                        (int64_t)of.t * a.q.token + (int64_t)of.hq * a.q.head +
                                                        g * S::DL + 8 * k);
        }
        const Row row = row_of(rt * MT + col, group, h, a.block.T, count);
        Rows<T, D, MT> rows;
        rows.bits = 0;
        rows.lim = 0;
        if (row.valid) {
            rows.lim = a.block.mode == DELS_KV4_CAUSAL ? n + row.t + 1 : a.block.mode == DELS_KV4_FULL ? n + count : n;
            if (a.block.mode == DELS_KV4_MASK)
                rows.bits = (uint64_t)a.block.mask[(int64_t)b * a.block.ld_mask + row.t] &
                            (count >= 64 ? ~0ull : (1ull << count) - 1);
        }
        rows.lim = min(rows.lim, slots);
        rows.top = -__builtin_inff();
        rows.total = 0.f;
#pragma unroll
        for (int t = 0; t < S::CT; ++t)
#pragma unroll
            for (int i = 0; i < S::ACC; ++i) rows.o[t][i] = 0.f;

        // Pages p, p + WAYS, ... below `stop`; one that the table does not name is passed over.
        // Keys are loaded a page ahead, values at the start of their page's work.  The
        // loads are unconditional (of page 0 where there is none to load) and in this
        // order, so that each wait covers only what it needs.  One copy of the work: two
        // that swap the keys' registers take longer to fetch than their moves.
        auto named = [&](int id) { return id >= 0 && id < c.num_pages; };
        auto address = [&](int id) { return heads + (named(id) ? id : 0) * page_stride; };
        KeyWords<D, MT> keys, next_keys;
        ValueWords<D, MT> values;
        int id = id_at(p), next = id_at(p + WAYS);
        if (p < stop) keys.load(address(id), at_lane);
#pragma unroll
        for (int i = 0; i < kPerWave; ++i) {
            const int e = wave + i * kKv4Waves;
#pragma unroll
            for (int x = 0; x < 4; ++x) qw[i][x] = (qw[i][x] ^ flip) & zero;
            if (e < kTiles * S::KS) s_q[e / S::KS][e % S::KS][lane] = __builtin_bit_cast(typename Frag<T>::type, qw[i]);
        }
        lds_barrier();                                        // the keys stay in flight
        for (; p < stop; p += WAYS) {
            values.load(address(id), at_lane);
            asm volatile("" ::: "memory");
            next_keys.load(address(next), at_lane);
            asm volatile("" ::: "memory");
            if (named(id))
                rows.page(&s_q[tile][0][lane], keys, values, at_lane.half, p * kKv4Page, n, filled, slots, g, unit, lag);
            keys = next_keys;
            id = next;
            next = id_at(p + 2 * WAYS);
        }

        // ---- join the waves
        const float ref = rows.top * unit;
        const float total = sum_over_groups<MT>(rows.total);
        if (g == 0) {
            s_m[wave][col] = ref;
            s_l[wave][col] = total;
        }
        __syncthreads();
        const bool whole = first == 0 && last == at.pages;
        // a piece has at most one state of rows that it begins and one of rows that it goes on with
        auto state_of = [&](int w, bool begins) {
            return states + ((int64_t)(2 * w + (begins ? 1 : 0)) * kTiles + tile) * kStateFloats<D, MT>;
        };
        float* state = state_of(piece, first == 0);
        float m = -__builtin_inff(), l = 0.f;
#pragma unroll
        for (int w = tile * WAYS; w < (tile + 1) * WAYS; ++w) m = fmaxf(m, s_m[w][col]);
#pragma unroll
        for (int w = tile * WAYS; w < (tile + 1) * WAYS; ++w) l += s_l[w][col] * fade(s_m[w][col], m);
        const float f = fade(ref, m), inv = l != 0.f ? kGrow / l : 0.f;
#pragma unroll
        for (int r0 = 0; r0 < kRegs; r0 += kRound) {
            // register (vl, i, v): channel block, row of the tile, channel of the VW
#pragma unroll
            for (int j = 0; j < kRound && r0 + j < kRegs; ++j) {
                const int r = r0 + j, v = r % S::VW, i = r / S::VW % S::ACC, vl = r / S::VW / S::ACC;
                s_o[wave][j][lane] = rows.o[vl * S::VW + v][i] * f;
            }
            __syncthreads();
            for (int jg = way; jg * S::VW < kRound && r0 + jg * S::VW < kRegs; jg += WAYS) {
                float sum[S::VW];
#pragma unroll
                for (int v = 0; v < S::VW; ++v) {
                    sum[v] = 0.f;
#pragma unroll
                    for (int w = 0; w < WAYS; ++w) sum[v] += s_o[tile * WAYS + w][jg * S::VW + v][lane];
                }
                const int gi = r0 / S::VW + jg;
                if (whole) {
                    store_out<T, S::VW>(a, b, row, S::channel_of(gi / S::ACC, gi % S::ACC, g), sum, inv);
                } else {
                    auto* to = reinterpret_cast<unsigned long long*>(state + (gi * 64 + lane) * S::VW);
#pragma unroll
                    for (int v = 0; v < S::VW; v += 2)
                        atomic_store_u64(to + v / 2, (unsigned long long)__float_as_uint(sum[v + 1]) << 32 |
                                                         __float_as_uint(sum[v]));
                }
            }
            __syncthreads();
        }
        if (way == 0 && g == 0) {
            if (whole) {
                store_lse(a, b, row, m, l);
            } else {
                auto* to = reinterpret_cast<unsigned int*>(state + MT * D + col);
                atomic_store_u32(to, __float_as_uint(m));
                atomic_store_u32(to + MT, __float_as_uint(l));
            }
        }
        if (!whole) {
            // The states are written and read with device-coherent stores and loads, and every
            // store is waited for before the arrival is counted: no cache fences.
            const int lo = at.start + ht * at.pages;
            const int2 held = cuts.holders(scan, b, ht, lo, lo + at.pages);
            __builtin_amdgcn_s_waitcnt(0);
            asm volatile("" ::: "memory");
            __syncthreads();
            if (threadIdx.x == 0) {
                unsigned int* counter = counters + held.x * kCounterWords;
                const unsigned prev = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                s_last = prev == (unsigned)(held.y - held.x) - 1u;
                if (s_last) __hip_atomic_exchange(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (s_last) {
                auto load = [&](const float* p) {
                    return __uint_as_float(__hip_atomic_load(reinterpret_cast<const unsigned int*>(p), __ATOMIC_RELAXED,
                                                             __HIP_MEMORY_SCOPE_AGENT));
                };
                constexpr int kMine = (kRegs / S::VW + WAYS - 1) / WAYS;
                float sum[kMine][S::VW];
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int v = 0; v < S::VW; ++v) sum[i][v] = 0.f;
                m = -__builtin_inff(), l = 0.f;
                // several states in flight: their loads go to memory (131k slots, 16 states: 91 us one
                // at a time, 76 eight)
                constexpr int kFlight = WAYS;
                for (int w0 = held.x; w0 < held.y; w0 += kFlight) {
                    float tops[kFlight], sums[kFlight];
                    unsigned long long two[kFlight][kMine][S::VW / 2];
#pragma unroll
                    for (int e = 0; e < kFlight; ++e) {
                        const int w = min(w0 + e, held.y - 1);
                        const float* st = state_of(w, w == held.x);
                        tops[e] = load(st + MT * D + col);
                        sums[e] = load(st + MT * D + MT + col);
#pragma unroll
                        for (int i = 0; i < kMine; ++i) {
                            const int gi = min(way + i * WAYS, kRegs / S::VW - 1);
                            auto* from = reinterpret_cast<unsigned long long*>(
                                const_cast<float*>(st + (gi * 64 + lane) * S::VW));
#pragma unroll
                            for (int v = 0; v < S::VW / 2; ++v) two[e][i][v] = atomic_load_u64(from + v);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < kFlight; ++e) {
                        if (w0 + e >= held.y) break;
                        const float now = fmaxf(m, tops[e]), old = fade(m, now), f = fade(tops[e], now);
                        m = now;
                        l = l * old + sums[e] * f;
#pragma unroll
                        for (int i = 0; i < kMine; ++i)
#pragma unroll
                            for (int v = 0; v < S::VW; ++v)
                                sum[i][v] = sum[i][v] * old +
                                            __uint_as_float((uint32_t)(two[e][i][v / 2] >> (32 * (v & 1)))) * f;
                    }
                }
                const float inv = l != 0.f ? kGrow / l : 0.f;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int gi = way + i * WAYS;
                    if (gi < kRegs / S::VW)
                        store_out<T, S::VW>(a, b, row, S::channel_of(gi / S::ACC, gi % S::ACC, g), sum[i], inv);
                }
                if (way == 0 && g == 0) store_lse(a, b, row, m, l);
            }
        }
        u += last - first;
    }
}

struct Plan { int rows, ways; Line line; };

Plan plan(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t max_pages) {
    Plan p{};
    const int64_t rows = T * (q_heads / heads);
    // Up to 16 rows in a tile of 16 (4 rows, 32 x 16k slots: 96 us, 122 in a tile of 32), more in
    // tiles of 32, each of which turns the codes into operands for itself (64 rows, 8 x 4000
    // slots: 25 us, 28.5 in tiles of 16).
    p.rows = rows <= 16 ? 16 : 32;
    const int64_t tiles = (rows + p.rows - 1) / p.rows, cus = device_cu_count();
    // Many row tiles: four of them a workgroup, two waves each, once that fills the GPU
    // (and hardly a wave is without a tile): a wave has more pages to itself and one state
    // to be joined with.  2 x 512 rows of 4 heads a group over 4000 slots: 138 us with
    // eight waves on a tile, 131 so.
    const int64_t fours = (tiles + 3) / 4;
    p.ways = p.rows == 32 && batch * heads * fours >= cus && 8 * tiles >= 7 * 4 * fours ? 2 : 8;
    const int per = kKv4Waves / p.ways;
    p.line.tiles = (int)((tiles + per - 1) / per);
    p.line.least = kMinPages;
    const int64_t units = batch * heads * p.line.tiles * std::max<int64_t>(max_pages, 1);
    p.line.pieces = (int)std::min<int64_t>({cus, kMaxCounters / kCounterWords,
                                            std::max(batch * heads * p.line.tiles, (units + kMinPages - 1) / kMinPages)});
    return p;
}

}  // namespace

size_t kv4_attention_data_bytes(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t head_dim,
                                int64_t max_pages) {
    const Plan p = plan(batch, T, q_heads, heads, max_pages);
    // four tiles a piece where this or a shorter block has them, so that a workspace for the
    // longest block serves every shorter one
    const int64_t tiles = (T * (q_heads / heads) + p.rows - 1) / p.rows;
    const bool four = p.ways == 2 || (p.rows == 32 && batch * heads * (tiles / 4) >= device_cu_count());
    return align256((size_t)p.line.pieces * 2 * (four ? 4 : 1) * sizeof(float) * (p.rows * head_dim + 2 * p.rows));
}

hipError_t launch_kv4_attention(const Kv4AttentionArgs& a, void* ws, size_t data_off, hipStream_t s) {
    const Kv4Cache& c = a.cache;
    const Plan p = plan(c.batch, a.block.T, a.q_heads, c.heads, c.max_pages);
    auto* states = reinterpret_cast<float*>(static_cast<char*>(ws) + data_off);
    auto* counters = reinterpret_cast<unsigned int*>(static_cast<char*>(ws) + kCountersOff);
    return kv4_by_type(a.dtype, c.head_dim, [&](auto tag, auto size) {
        using T = decltype(tag);
        constexpr int D = decltype(size)::value;
        auto go = [&](auto rows, auto ways) {
            hipLaunchKernelGGL((kv4_attention_kernel<T, D, decltype(rows)::value, decltype(ways)::value>),
                               dim3(p.line.pieces), dim3(kKv4Threads), 0, s, a, p.line, states, counters);
        };
        using std::integral_constant;
        if (p.rows == 16) go(integral_constant<int, 16>{}, integral_constant<int, 8>{});
        else if (p.ways == 8) go(integral_constant<int, 32>{}, integral_constant<int, 8>{});
        else go(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    });
}

}  // namespace dels
