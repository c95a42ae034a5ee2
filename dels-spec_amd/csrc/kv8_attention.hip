// Attention over the 8-bit key/value cache (format: kv8.h), whole or through a window.
//
//     x[t, j] = scale * q[t] . k[j]          j a slot that row t sees
//     lse[t]  = log sum_j exp(x[t, j])
//     o[t]    = sum_j exp(x[t, j] - lse[t]) v[j]
// A row that sees nothing has o = 0 and lse = -inf.  With a window, row t sees of those slots
// the ones from lengths + t - window + 1 on and the first `sinks`.
//
// One pass over the slots with the running maximum and sum of each row's softmax.
// The rows that share a cache head (block tokens x query heads of the group) are
// the columns of both products:
//     S^T [slots x rows] = K Q^T          O^T [channels x rows] += V^T P^T
// and a lane holds scores of sixteen consecutive slots of one row, which are two operands
// of the second product: P stays in its lane.  Codes become the queries' type by
// the conversion instruction, exactly; a block's key scale joins the factor of its
// scores, its value scale is applied by the conversion.  Both products are 16-bit ones: the
// 8-bit matrix instructions add products at 2^-12 of the largest of a group (measured),
// which a float32 lse would show.  Weights enter as f16 numbers (2^-11 of each, an eighth of half a
// step of a bf16 output), for f16 outputs in two parts.  Scores, maxima, sums and outputs are
// fp32.
#include <algorithm>

#include "kv8.h"

namespace dels {

namespace {

constexpr int kWaves = kLineWaves, kThreads = 64 * kWaves;
// What a row's weights are relative to lies this many binary orders above its largest score
// when it moves, and moves when a score passes it: until then the outputs need no rescaling
// and no weight is above 1.
constexpr float kLag = 8.f;
// Weights enter the second product as f16 numbers of up to 2^kLift (below 2^-14 their steps
// are 2^-24, so a weight 2^-31 of the largest still counts), values as f16 numbers of up to 448 * 2^7: a
// block's scale is relative to the largest of the blocks so far, with kHead binary orders to spare
// when it moves.  Once the scales of a wave's blocks lie more than kSpan orders apart, neither
// small values nor small weights of large ones are safe there, and further products are of bf16
// numbers, whose range knows no such bounds, with weights in two parts.
constexpr float kLift = 15.f;
constexpr int kHead = 2, kSpan = 12;
constexpr int kMinPages = 2 * kWaves;  // fewest pages of a part
// Most parts of one tile group: their states are joined by one workgroup.
constexpr int kMostParts = 32;

// Shapes of a wave's work on MT rows: MT x MT tiles of the matrix instructions.  A step is
// 32 * 32 / MT slots, so that a lane has scores of 16 consecutive slots: a page's two blocks at
// once for 16 rows, one after the other for 32.
template <int D, int MT_> struct Shape8 {
    static constexpr int MT = MT_;
    static constexpr int NG = 64 / MT;              // lane groups: lane = MT * group + row
    static constexpr int KS = D / NG / 8;           // steps of the first product's contraction: 8 channels a lane
    static constexpr int KL = KS / 2;               // loads of a key tile: 16 channels a lane
    static constexpr int STEPS = MT / 16;           // steps of a page
    static constexpr int NT = 64 / MT / STEPS;      // key tiles of a step
    static constexpr int ACC = MT == 16 ? 4 : 16;   // accumulator registers of a tile
    static constexpr int CT = D / MT;               // channel tiles of the output
    using Acc = typename std::conditional<MT == 16, f32x4, f32x16>::type;
    // first slot of a lane group's run in a step, within the page
    __device__ static int run_slot(int step, int g) { return MT == 16 ? 16 * g : 32 * step + 16 * g; }
    // first of the four channels of registers 4 j .. 4 j + 3 of channel tile `t`
    __device__ static int channel_of(int t, int j, int g) { return MT * t + (MT == 16 ? 4 * g : 8 * j + 4 * g); }
};

// Eight codes, times a power of two.
template <typename T>
__device__ __forceinline__ typename Frag<T>::type widen8(uint32_t lo, uint32_t hi, float scale) {
    if constexpr (std::is_same<T, bf16_t>::value) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
        const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
        const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
        const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
        return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    } else {
        const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false);
        const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true);
        const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false);
        const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true);
        return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
}

// Two numbers rounded to a 16-bit type, the first in the low half, and a half widened again.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if constexpr (std::is_same<T, bf16_t>::value) return pack_bf16(a, b);
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

// a where bit v of `bits` is set, else b.
__device__ __forceinline__ float choose(uint32_t bits, int v, float a, float b) {
    const uint32_t all = (uint32_t)((int32_t)(bits << (31 - v)) >> 31);
    return __uint_as_float((__float_as_uint(a) & all) | (__float_as_uint(b) & ~all));
}

// The lowest k of 16 bits.
__device__ __forceinline__ uint32_t lowest(int k) { return (1u << min(max(k, 0), 16)) - 1u; }

template <int D, int MT> struct KeyRegs {
    using S = Shape8<D, MT>;
    u32x4 code[S::STEPS][S::NT][S::KL];
    __device__ __forceinline__ void load(const uint8_t* page, int col, int g, int step) {
        const int lane = MT == 16 ? 32 * D * (col >> 3) + 512 * g + 16 * (col & 7) : 512 * g + 16 * col;
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
#pragma unroll
            for (int i = 0; i < S::KL; ++i)
                code[step][t][i] =
                    *reinterpret_cast<const u32x4*>(page + lane + 512 * S::NG * i + (MT == 16 ? 128 * t : 32 * D * step));
    }
};

template <int D, int MT> struct ValueRegs {
    using S = Shape8<D, MT>;
    u32x4 code[S::STEPS][S::CT];
    __device__ __forceinline__ void load(const uint8_t* page, int col, int g, int step) {
        const int lane = Kv8<D>::kValue + 16 * D * g + 16 * col;
#pragma unroll
        for (int t = 0; t < S::CT; ++t)
            code[step][t] = *reinterpret_cast<const u32x4*>(page + lane + 32 * D * step + 16 * MT * t);
    }
};

// Which slots a row sees.
struct Sight {
    int n, filled;             // context; slots that hold anything
    int lim, lo;               // the row sees slots below lim,
    uint64_t bits;             // and those of the block whose bits are set, from lo on
    int sinks;                 // or below this
    __device__ uint32_t of_run(int j0) const {             // of slots j0 .. j0 + 15
        const int d = j0 - n;
        uint32_t by_bit = d >= 64 || d <= -16 ? 0u : (uint32_t)(d >= 0 ? bits >> d : bits << -d) & 0xffffu;
        by_bit &= lowest(filled - j0);
        return (lowest(lim - j0) | by_bit) & (~lowest(lo - j0) | lowest(sinks - j0));
    }
};

// A page as a wave meets it: what its two blocks say of themselves, and what of it is seen.
struct Page {
    int key[2], value[2];      // exponents; of a block that holds nothing the value's is 0
    uint32_t bad[2];
    int slot;                  // first of its slots
    bool none, masked, last;   // is no page; some row does not see all of it; slots behind the last hold nothing
    __device__ __forceinline__ Page(u32x4 head, int slot_, bool none_, bool masked_, int filled) : slot(slot_), none(none_) {
        last = none || slot + kCachePage > filled;
        masked = none || masked_;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int e = uniform((int)head[2 * u]);
            key[u] = min(max(e & 255, kKv8Low), kKv8High);
            value[u] = none || slot + 32 * u >= filled ? 0 : min(max(e >> 8 & 255, kKv8Low), kKv8High);
            bad[u] = none ? 0u : (uint32_t)uniform((int)head[2 * u + 1]);
        }
    }
};

// The rows' state of a wave, and one step's part in it.
template <typename T, int D, int MT> struct Rows8 {
    using S = Shape8<D, MT>;
    using F = typename Frag<T>::type;
    typename S::Acc o[S::CT];  // in units of 2^(vref - 134) times that of the weights
    float top, total;          // what weights are relative to (binary logarithm) and this lane's part of their sum
    int vref, vlow;            // exponent of values that the outputs are relative to; least of the blocks so far

    __device__ __forceinline__ void clear() {
        top = -__builtin_inff();
        total = 0.f;
        vref = 0;
        vlow = 255;
#pragma unroll
        for (int t = 0; t < S::CT; ++t)
#pragma unroll
            for (int i = 0; i < S::ACC; ++i) o[t][i] = 0.f;
    }

    __device__ __forceinline__ void rescale(float f) {
#pragma unroll
        for (int t = 0; t < S::CT; ++t)
#pragma unroll
            for (int i = 0; i < S::ACC; ++i) o[t][i] *= f;
    }

    // scores of a step; q(k): this lane's operand of the queries for step k of the contraction
    template <typename Q>
    __device__ __forceinline__ void scores(Q&& q, const u32x4 (&code)[S::NT][S::KL], typename S::Acc (&acc)[S::NT]) {
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
#pragma unroll
            for (int i = 0; i < S::ACC; ++i) acc[t][i] = 0.f;
        F next_q = q(0);
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
            const F qk = next_q;
            if (k + 1 < S::KS) next_q = q(k + 1);              // read a step ahead
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < S::NT; ++t)
                acc[t] = mma(widen8<T>(code[t][k / 2][2 * (k % 2)], code[t][k / 2][2 * (k % 2) + 1], 1.f), qk, acc[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    // Adds weights times values; x: scores, their binary logarithms are x * factor - ref.
    // P: type and number of parts of a weight.
    template <typename P, int PARTS>
    __device__ __forceinline__ void multiply(const float (&x)[16], float factor, float ref, const u32x4 (&code)[S::CT],
                                             float vscale) {
        using V = typename Frag<P>::type;
        // The weights of eight slots are made while those before multiply the values: between two
        // matrix instructions stand vector ones, in this order (the fences keep it), so that
        // neither waits for the other.
        u32x4 part[PARTS][2];
        float even = 0.f;
        auto make = [&](int u, int i) {
            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * u + i], factor, -ref));
            total += e;
            if (i % 2 == 0) {
                even = e;
            } else {
                const uint32_t h = pack2<P>(even, e);
                part[0][u][i / 2] = h;
                if constexpr (PARTS == 2)
                    part[1][u][i / 2] = pack2<P>(even - widen_raw<P>(h & 0xffffu), e - widen_raw<P>(h >> 16));
            }
        };
#pragma unroll
        for (int i = 0; i < 8; ++i) make(0, i);
        constexpr int kEach = 8 / S::CT;                       // weights for the next half by channel tile
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int t = 0; t < S::CT; ++t) {
                const V vf = widen8<P>(code[t][2 * u], code[t][2 * u + 1], vscale);
#pragma unroll
                for (int i = t * kEach; u == 0 && i < (t + 1) * kEach; ++i) make(1, i);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) o[t] = mma(vf, __builtin_bit_cast(V, part[p][u]), o[t]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    // Takes a page's scales in; whether its products can be of f16 numbers.
    __device__ __forceinline__ bool admit(const Page& page) {
        const int high = max(page.value[0], page.value[1]);
        if (high) vlow = min(vlow, page.value[1] ? min(page.value[0], page.value[1]) : page.value[0]);
        if (high > vref) {
            const int now = min(high + kHead, kKv8High);
            rescale(vref ? kv8_pow2(max(127 + vref - now, 0)) : 1.f);
            vref = now;
        }
        return vlow >= vref - kSpan;
    }

    // WIDE: the scales lie far apart; unit: binary logarithms per raw product
    template <bool WIDE>
    __device__ __forceinline__ void weigh(const typename S::Acc (&acc)[S::NT], const Page& page, int step, int g,
                                          u32x4 (&code)[S::CT], const Sight& sight, float unit) {
        const int slot = page.slot + S::run_slot(step, g);
        const bool second = MT == 16 ? g >= 2 : step == 1;     // of the page's blocks
        const int ke = second ? page.key[1] : page.key[0], ve = second ? page.value[1] : page.value[0];
        const float factor = fmaxf(unit * kv8_pow2(ke), 1e-37f);
        float x[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = acc[MT == 16 ? v / 4 % S::NT : 0][v % S::ACC];
        if (page.masked) {
            asm volatile("");                              // a branch, not selections on every page
            const uint32_t sees = page.none ? 0u : sight.of_run(slot);
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] = choose(sees, v, x[v], -__builtin_inff());
        }
        if (page.bad[0] | page.bad[1]) {
            asm volatile("");
            const uint32_t lost = (second ? page.bad[1] : page.bad[0]) >> (slot & 16) & sight.of_run(slot);
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] = choose(~lost, v, x[v], __builtin_nanf(""));
        }
        if (page.last) {
            asm volatile("");
            // behind the last slot anything may lie, and a weight of 0 does not make it 0
            const uint32_t keep = page.none ? 0u : lowest(sight.filled - slot);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                // bit i to byte i
                const uint32_t bytes = (((keep >> (4 * w) & 15u) * 0x00204081u) & 0x01010101u) * 255u;
#pragma unroll
                for (int t = 0; t < S::CT; ++t) code[t][w] &= bytes;
            }
        }
        float best = x[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) best = fmaxf(best, x[v]);
        best = max_over_groups<MT>(best * factor);
        if (__any(best > top)) {
            const float now = fmaxf(top, best + kLag), f = fade(top, now);
            top = now;
            total *= f;
            rescale(f);
        }
        const float ref = (top == -__builtin_inff() ? 0.f : top) - kLift;
        const float vscale = kv8_pow2(ve ? 134 + ve - vref : 127);
        if constexpr (WIDE) multiply<bf16_t, 2>(x, factor, ref, code, vscale);
        else multiply<f16_t, std::is_same<T, f16_t>::value ? 2 : 1>(x, factor, ref, code, vscale);
    }
};

// Four channels of a row's output.
template <typename T>
__device__ __forceinline__ void store4(const Kv8AttentionArgs& a, int b, const Row& row, int ch, const float* o, float inv) {
    if (!row.in_block) return;
    uint16_t* p = static_cast<uint16_t*>(a.out) + (int64_t)b * a.out_batch + (int64_t)row.t * a.out_token +
                  (int64_t)row.hq * a.out_head + ch;
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float x = row.valid ? o[2 * i] * inv : 0.f, y = row.valid ? o[2 * i + 1] * inv : 0.f;
        w[i] = (uint32_t)round_to<T>(x) | ((uint32_t)round_to<T>(y) << 16);
    }
    *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
}

// `ref`: binary logarithm of the unit that `total` counts in.  A sum of 0 is a row that saw
// nothing (the largest score's weight is at least 2^-kLag, or nearly).
__device__ __forceinline__ void store_lse8(const Kv8AttentionArgs& a, int b, const Row& row, float ref, float total) {
    if (!row.in_block) return;
    const float x = row.valid && total != 0.f ? (ref - kLift + __builtin_amdgcn_logf(total)) * 0.693147180559945309f
                                             : -__builtin_inff();
    a.lse[((int64_t)b * a.block.T + row.t) * a.q_heads + row.hq] = x;
}

// Floats of a piece's state in the workspace: outputs as the lanes hold them, then references and sums.
template <int D, int MT> constexpr int kStateFloats = MT * D + 2 * MT;

// The pages that the rows of a tile group see: [0, sinks) and [from, end) of the sequence's row.
struct Seen {
    int sinks, from, end;
    __device__ int count() const { return sinks + end - from; }
    __device__ int page(int i) const { return i < sinks ? i : i - sinks + from; }
};

// The sequences of a call, for the line of their pages: as many as any of their tile groups sees.
struct Kv8Seqs {
    const Kv8AttentionArgs& a;
    int batch, tokens;         // most tokens that the rows of a tile group lie in
    __device__ Kv8Seqs(const Kv8AttentionArgs& a_, int rows, int group)
        : a(a_), batch(a_.cache.batch), tokens(divide(rows - 1, group) + 2) {}
    __device__ int length(int b) const { return paged_length(a.block.lengths, b, a.cache.slots()); }
    __device__ int count(int b) const { return paged_count(a.block.counts, b, a.block.T); }
    __device__ int pages(int n, int count) const {
        const int all = seq_pages(seq_end(a.block, n, count, a.cache.slots()));
        if (!a.window) return all;
        const int64_t more = a.block.mode == DELS_KV4_CAUSAL ? min(tokens, count) : a.block.mode == DELS_KV4_NONE ? 0 : count;
        const int64_t span = (a.window + more + kCachePage - 2) / kCachePage + 1 + (a.sinks + kCachePage - 1) / kCachePage;
        return (int)min((int64_t)all, span);
    }
    // of rows first .. last of the block (tokens)
    __device__ Seen seen(int n, int count, int first, int last) const {
        int end = seq_end(a.block, n, count, a.cache.slots());
        if (a.block.mode == DELS_KV4_CAUSAL) end = (int)min((int64_t)end, (int64_t)n + last + 1);
        Seen s{0, 0, (end + kCachePage - 1) / kCachePage};
        if (a.window) {
            const int64_t start = max((int64_t)n + first - a.window + 1, (int64_t)0);
            s.from = (int)min(start / kCachePage, (int64_t)s.end);
            s.sinks = (int)min((a.sinks + kCachePage - 1) / kCachePage, (int64_t)s.from);
        }
        return s;
    }
};

// LDS of a workgroup.  Where TILES row tiles go over the same pages, each way keeps a ring of
// them there: the page as it lies in memory but for its head, of which every wave has its own.
template <typename T, int D, int MT, int TILES> struct Lds {
    using S = Shape8<D, MT>;
    static constexpr int kWays = kWaves / TILES;
    static constexpr int kRing = TILES == 1 ? 0 : kWays * D > 256 ? 2 : 3;
    static constexpr int kRound = 32;                       // output registers joined at a time
    union {
        uint8_t page[kWays][kRing ? kRing : 1][TILES == 1 ? 16 : Kv8<D>::kHead];
        float o[kWaves][kRound][64];
    };
    uint32_t head[kWaves][kRing ? kRing : 1][64];
    typename Frag<T>::type q[TILES][S::KS][64];             // the tiles' queries, in operand order
    float m[kWaves][MT], l[kWaves][MT];
    bool last;
};

// TILES of 8 waves share a way: row tiles over the same pages.  8 / TILES ways take every
// (8 / TILES)-th page each.
template <typename T, int D, int MT, int TILES>
__global__ __launch_bounds__(kThreads, 2) void kv8_attention_kernel(Kv8AttentionArgs a, Line line, float* states,
                                                                    unsigned int* counters) {
    using S = Shape8<D, MT>;
    using F = typename Frag<T>::type;
    using L = Lds<T, D, MT, TILES>;
    constexpr int WAYS = L::kWays, kTiles = TILES, kRound = L::kRound;
    constexpr int kRegs = S::CT * S::ACC;                   // output registers
    __shared__ __attribute__((aligned(128))) L lds;
    auto& s_o = lds.o;
    auto& s_m = lds.m;
    auto& s_l = lds.l;
    auto& s_last = lds.last;

    const PagedCache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane % MT, g = lane / MT, tile = wave / WAYS, way = wave % WAYS;
    const int slots = c.slots(), group = a.q_heads / c.heads;
    // pieces that follow each other on one XCD: they share pages where a head has several row tiles
    const int piece = (int)gridDim.x % 8 ? (int)blockIdx.x
                                         : (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
    const Kv8Seqs seqs(a, kTiles * MT, group);
    Scan<Kv8Seqs> scan(seqs, c.heads * line.tiles);
    const Cuts cuts(scan, line, kMostParts);
    Scan<Kv8Seqs>::Place at{};
    const int2 mine = cuts.piece(scan, piece, at);
    int u = mine.x;
    const int u_end = mine.y;
    if (u >= u_end) return;
    // scores in units of the maximum: |scale| and the query's sign
    const float mag = fabsf(a.scale);
    const float unit = (mag == 0.f ? 1.f : mag) * kLog2e;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, zero = mag == 0.f ? 0u : ~0u;

    while (u < u_end) {
        if (u >= at.start + at.pages * scan.per) at = scan.place(u);
        const int b = at.b;
        const int rel = u - at.start, ht = divide(rel, at.pages), first = rel - ht * at.pages;
        const int h = divide(ht, line.tiles), rt0 = (ht - h * line.tiles) * kTiles, rt = rt0 + tile;
        const int last = min(at.pages, first + (u_end - u));
        const int n = at.n, count = at.count, last_t = a.block.T - 1;
        // tokens of the tile group, and of this wave's tile
        const Seen seen = seqs.seen(n, count, divide(rt0 * MT, group), min(divide((rt0 + kTiles) * MT - 1, group), last_t));
        const int t_first = divide(rt * MT, group), t_last = min(divide(rt * MT + MT - 1, group), last_t);
        const int stop = min(last, seen.count());
        const bool past = rt * MT >= count * group;           // the tile has no valid row
        Sight sight;
        sight.n = n;
        sight.filled = seq_end(a.block, n, count, slots);     // slots past it may hold anything
        sight.sinks = a.window ? (int)min(a.sinks, (int64_t)slots) : slots;
        // slots from `clear` on are seen by no more rows than these bounds say: pages between need no mask
        const int clear_to = min(sight.filled, a.block.mode == DELS_KV4_CAUSAL ? n + t_first + 1
                                               : a.block.mode == DELS_KV4_FULL ? n + count : n);
        const int64_t clear_from = a.window ? (int64_t)n + t_last - a.window + 1 : 0;

        // the wave's pages
        const int32_t* ids = c.table + (int64_t)b * c.ld_table;
        const uint8_t* heads = c.data + (int64_t)h * Kv8<D>::kBytes;
        const int64_t page_stride = (int64_t)c.heads * Kv8<D>::kBytes;
        int p = first + way;
        // the numbers of the wave's next 64 pages, one a lane: a load per page would be
        // waited for with the first read of LDS
        int ids64, base;
        auto fetch_ids = [&](int from) {
            base = from;
            const int i = from + lane * WAYS;
            ids64 = i < stop ? ids[seen.page(i)] : -1;
        };
        auto id_at = [&](int i) {
            if (i - base >= 64 * WAYS) fetch_ids(i);
            return __builtin_amdgcn_readlane(ids64, (i - base) / WAYS);
        };
        fetch_ids(p);

        // the queries in operand order: step k of lane group g has channels
        // 16 (NG (k / 2) + g) + 8 (k % 2) .. + 7.  The waves of a tile share them out.
        constexpr int kQ = (S::KS + WAYS - 1) / WAYS;
        auto q_step = [&](int i) { return way + i * WAYS; };
        u32x4 qw[kQ];
        {
            const Row of = row_of(rt * MT + col, group, h, a.block.T, count);
            const uint16_t* from = static_cast<const uint16_t*>(a.q.p) + (int64_t)b * a.q.batch +
                                   (int64_t)of.t * a.q.token + (int64_t)of.hq * a.q.head;
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
                const int k = q_step(i);
                qw[i] = u32x4{0u, 0u, 0u, 0u};
                if (of.valid && k < S::KS)
                    qw[i] = *reinterpret_cast<const u32x4*>(from + 16 * (S::NG * (k / 2) + g) + 8 * (k % 2));
            }
        }
        const Row row = row_of(rt * MT + col, group, h, a.block.T, count);
        Rows8<T, D, MT> rows;
        sight.bits = 0;
        sight.lim = sight.lo = 0;
        if (row.valid) {
            sight.lim = a.block.mode == DELS_KV4_CAUSAL ? n + row.t + 1 : a.block.mode == DELS_KV4_FULL ? n + count : n;
            if (a.window) sight.lo = (int)max((int64_t)n + row.t - a.window + 1, (int64_t)0);
            if (a.block.mode == DELS_KV4_MASK)
                sight.bits = (uint64_t)a.block.mask[(int64_t)b * a.block.ld_mask + row.t] &
                             (count >= 64 ? ~0ull : (1ull << count) - 1);
        }
        sight.lim = min(sight.lim, sight.filled);
        rows.clear();

        // Pages p, p + WAYS, ... below `stop`; one that the table does not name is seen by no row.
        auto named = [&](int id) { return id >= 0 && id < c.num_pages; };
        auto address = [&](int id) { return heads + (named(id) ? id : 0) * page_stride; };
        auto put_queries = [&] {
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
#pragma unroll
                for (int x = 0; x < 4; ++x) qw[i][x] = (qw[i][x] ^ flip) & zero;
                if (q_step(i) < S::KS) lds.q[tile][q_step(i)][lane] = __builtin_bit_cast(F, qw[i]);
            }
        };
        auto query = [&](int k) { return lds.q[tile][k][lane]; };
        auto page_at = [&](int i, int id, u32x4 head) {
            const int slot = seen.page(i) * kCachePage;
            return Page(head, slot, !named(id),
                        slot + kCachePage > clear_to || (slot < clear_from && slot + kCachePage > sight.sinks), sight.filled);
        };
        using Narrow = std::false_type;
        using Wide = std::true_type;
        if constexpr (TILES == 1) {
            // Keys and values of the next page are loaded into their registers once a step's scores
            // or products are made, a page's work ahead of their use.  The loads are unconditional
            // (of page 0 where there is none to load) and in the order of their use, so that each
            // wait covers only what it needs.
            KeyRegs<D, MT> keys;
            ValueRegs<D, MT> values;
            u32x4 head;
            int id = id_at(p);
            auto load_head = [&](const uint8_t* page) { head = *reinterpret_cast<const u32x4*>(page + Kv8<D>::kHead); };
            if (p < stop) {
                load_head(address(id));
#pragma unroll
                for (int step = 0; step < S::STEPS; ++step) {
                    keys.load(address(id), col, g, step);
                    values.load(address(id), col, g, step);
                }
            }
            put_queries();
            lds_barrier();                                    // the loads stay in flight
            auto work = [&](auto wide, const Page& page) {
                const int next = id_at(p + WAYS);
                const uint8_t* next_page = address(next);
                load_head(next_page);
#pragma unroll
                for (int step = 0; step < S::STEPS; ++step) {
                    typename S::Acc acc[S::NT];
                    rows.scores(query, keys.code[step], acc);
                    keys.load(next_page, col, g, step);
                    asm volatile("" ::: "memory");
                    rows.template weigh<decltype(wide)::value>(acc, page, step, g, values.code[step], sight, unit);
                    values.load(next_page, col, g, step);
                    asm volatile("" ::: "memory");
                }
                id = next;
                p += WAYS;
            };
            while (p < stop) {
                const Page page = page_at(p, id, head);
                if (!rows.admit(page)) break;                 // and from there on
                work(Narrow{}, page);
            }
            while (p < stop) {
                const Page page = page_at(p, id, head);
                rows.admit(page);
                work(Wide{}, page);
            }
        } else {
            // The waves of a way copy a page into its ring, a share of 1 KiB pieces and the head each,
            // kRing - 1 pages ahead.  One barrier a page: past it, all shares of the page have
            // arrived and nobody reads the buffer that the next copy goes to.
            constexpr int kShare = Kv8<D>::kHead / 1024 / TILES, kPer = kShare + 1;
            const int pages = max(0, (stop - first + WAYS - 1) / WAYS);      // of the first way, which has most
            auto copy = [&](int i) {
                const int id = id_at(first + way + i * WAYS);
                const uint8_t* from = address(id);
                const int slot = i % L::kRing;
#pragma unroll
                for (int e = 0; e < kShare; ++e) {
                    const int at = 1024 * (tile * kShare + e);
                    dma16(from + at, 16 * lane, &lds.page[way][slot][at]);
                }
                dma4(from + Kv8<D>::kHead, 4 * (lane & 31), lds.head[wave][slot]);
                return id;
            };
            put_queries();
            int ids_ahead[L::kRing];                          // of pages i, i + 1, ..
#pragma unroll
            for (int i = 0; i < L::kRing - 1; ++i) ids_ahead[i + 1] = i < pages ? copy(i) : -1;
            auto arrive = [&](int i) {
                // what may still be on its way: the pages behind this one
                if (i + L::kRing - 2 < pages) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((L::kRing - 2) * kPer) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                lds_barrier();
                p = first + way + i * WAYS;
#pragma unroll
                for (int e = 0; e < L::kRing - 1; ++e) ids_ahead[e] = ids_ahead[e + 1];
                if (i + L::kRing - 1 < pages) ids_ahead[L::kRing - 1] = copy(i + L::kRing - 1);
                return !past && p < stop;
            };
            auto take = [&](int i) {
                return page_at(p, ids_ahead[0], *reinterpret_cast<const u32x4*>(lds.head[wave][i % L::kRing]));
            };
            auto work = [&](auto wide, int i, const Page& page) {
                const uint8_t* at = lds.page[way][i % L::kRing] + 16 * lane;
#pragma nounroll
                for (int step = 0; step < S::STEPS; ++step) {
                    u32x4 keys[S::NT][S::KL], values[S::CT];
#pragma unroll
                    for (int e = 0; e < S::KL; ++e)
                        keys[0][e] = *reinterpret_cast<const u32x4*>(at + 32 * D * step + 1024 * e);
#pragma unroll
                    for (int t = 0; t < S::CT; ++t)
                        values[t] = *reinterpret_cast<const u32x4*>(at + Kv8<D>::kValue + 32 * D * step +
                                                                    (16 * D - 512) * g + 512 * t);
                    typename S::Acc acc[S::NT];
                    rows.scores(query, keys, acc);
                    rows.template weigh<decltype(wide)::value>(acc, page, step, g, values, sight, unit);
                }
            };
            int i = 0;
            bool here = false;                                // page i has been met, but not worked on
            for (; i < pages; ++i) {
                if (!arrive(i)) continue;
                const Page page = take(i);
                here = !rows.admit(page);
                if (here) break;                              // and from there on
                work(Narrow{}, i, page);
            }
            for (; i < pages; ++i) {
                const bool mine = here || arrive(i);
                here = false;
                if (!mine) continue;
                const Page page = take(i);
                rows.admit(page);
                work(Wide{}, i, page);
            }
            __syncthreads();                                  // the ring's place is the join's
        }

        // ---- join the waves
        const float ref = rows.top;
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
        const float inv = l != 0.f ? 1.f / l : 0.f;
        const float f = fade(ref, m) * kv8_pow2(max(rows.vref - 7, 0));
#pragma unroll
        for (int r0 = 0; r0 < kRegs; r0 += kRound) {
#pragma unroll
            for (int j = 0; j < kRound && r0 + j < kRegs; ++j)
                s_o[wave][j][lane] = rows.o[(r0 + j) / S::ACC][(r0 + j) % S::ACC] * f;
            __syncthreads();
            for (int jq = way; 4 * jq < kRound && r0 + 4 * jq < kRegs; jq += WAYS) {
                float sum[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    sum[v] = 0.f;
#pragma unroll
                    for (int w = 0; w < WAYS; ++w) sum[v] += s_o[tile * WAYS + w][4 * jq + v][lane];
                }
                const int q = r0 / 4 + jq;                    // registers 4 q .. 4 q + 3
                if (whole) {
                    store4<T>(a, b, row, S::channel_of(q / (S::ACC / 4), q % (S::ACC / 4), g), sum, inv);
                } else {
                    auto* to = reinterpret_cast<unsigned long long*>(state + (q * 64 + lane) * 4);
#pragma unroll
                    for (int v = 0; v < 4; v += 2)
                        atomic_store_u64(to + v / 2, (unsigned long long)__float_as_uint(sum[v + 1]) << 32 |
                                                         __float_as_uint(sum[v]));
                }
            }
            __syncthreads();
        }
        if (way == 0 && g == 0) {
            if (whole) {
                store_lse8(a, b, row, m, l);
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
                constexpr int kMine = (kRegs / 4 + WAYS - 1) / WAYS;
                float sum[kMine][4];
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) sum[i][v] = 0.f;
                m = -__builtin_inff(), l = 0.f;
                constexpr int kFlight = WAYS;                 // states in flight: their loads go to memory
                for (int w0 = held.x; w0 < held.y; w0 += kFlight) {
                    float tops[kFlight], sums[kFlight];
                    unsigned long long two[kFlight][kMine][2];
#pragma unroll
                    for (int e = 0; e < kFlight; ++e) {
                        const int w = min(w0 + e, held.y - 1);
                        const float* st = state_of(w, w == held.x);
                        tops[e] = load(st + MT * D + col);
                        sums[e] = load(st + MT * D + MT + col);
#pragma unroll
                        for (int i = 0; i < kMine; ++i) {
                            const int q = min(way + i * WAYS, kRegs / 4 - 1);
                            auto* from = reinterpret_cast<unsigned long long*>(const_cast<float*>(st + (q * 64 + lane) * 4));
#pragma unroll
                            for (int v = 0; v < 2; ++v) two[e][i][v] = atomic_load_u64(from + v);
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
                            for (int v = 0; v < 4; ++v)
                                sum[i][v] = sum[i][v] * old +
                                            __uint_as_float((uint32_t)(two[e][i][v / 2] >> (32 * (v & 1)))) * f;
                    }
                }
                const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
                for (int i = 0; i < kMine; ++i) {
                    const int q = way + i * WAYS;
                    if (q < kRegs / 4)
                        store4<T>(a, b, row, S::channel_of(q / (S::ACC / 4), q % (S::ACC / 4), g), sum[i], inv);
                }
                if (way == 0 && g == 0) store_lse8(a, b, row, m, l);
            }
        }
        u += last - first;
    }
}

struct Plan { int rows, tiles; Line line; };

Plan plan(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t max_pages) {
    Plan p{};
    const int64_t rows = T * (q_heads / heads), cus = device_cu_count();
    p.rows = rows <= 16 ? 16 : 32;
    const int64_t tiles = (rows + p.rows - 1) / p.rows;
    // the widest workgroup that leaves the fewest waves without a tile
    p.tiles = 1;
    if (tiles > 1) {
        int64_t best = INT64_MAX;
        for (int wide : {8, 4, 2}) {
            const int64_t waves = (tiles + wide - 1) / wide * wide;
            if (waves < best) best = waves, p.tiles = wide;
        }
    }
    p.line.tiles = (int)((tiles + p.tiles - 1) / p.tiles);
    p.line.least = kMinPages;
    const int64_t units = batch * heads * p.line.tiles * std::max<int64_t>(max_pages, 1);
    p.line.pieces = (int)std::min<int64_t>({cus, kMaxCounters / kCounterWords,
                                            std::max(batch * heads * p.line.tiles, (units + kMinPages - 1) / kMinPages)});
    return p;
}

}  // namespace

size_t kv8_attention_data_bytes(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t head_dim,
                                int64_t max_pages) {
    // what any shorter block takes too, so that a workspace for the longest serves every one: up to
    // 8 tiles of 32 rows a piece, and no fewer pieces
    const int64_t rows = T * (q_heads / heads);
    const int64_t tiles = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
    const int64_t pieces = std::min<int64_t>(device_cu_count(), kMaxCounters / kCounterWords);
    (void)batch, (void)max_pages;
    return align256((size_t)pieces * 2 * tiles * sizeof(float) * (32 * head_dim + 2 * 32));
}

hipError_t launch_kv8_attention(const Kv8AttentionArgs& a, void* ws, size_t data_off, hipStream_t s) {
    const PagedCache& c = a.cache;
    const Plan p = plan(c.batch, a.block.T, a.q_heads, c.heads, c.max_pages);
    auto* states = reinterpret_cast<float*>(static_cast<char*>(ws) + data_off);
    auto* counters = reinterpret_cast<unsigned int*>(static_cast<char*>(ws) + kCountersOff);
    auto by_size = [&](auto tag, auto size) {
        using T = decltype(tag);
        constexpr int D = decltype(size)::value;
        auto go = [&](auto rows, auto tiles) {
            hipLaunchKernelGGL((kv8_attention_kernel<T, D, decltype(rows)::value, decltype(tiles)::value>),
                               dim3(p.line.pieces), dim3(kThreads), 0, s, a, p.line, states, counters);
        };
        using std::integral_constant;
        using I16 = integral_constant<int, 16>;
        using I32 = integral_constant<int, 32>;
        if (p.rows == 16) go(I16{}, integral_constant<int, 1>{});
        else if (p.tiles == 1) go(I32{}, integral_constant<int, 1>{});
        else if (p.tiles == 2) go(I32{}, integral_constant<int, 2>{});
        else if (p.tiles == 4) go(I32{}, integral_constant<int, 4>{});
        else go(I32{}, integral_constant<int, 8>{});
    };
    auto by_type = [&](auto tag) {
        if (c.head_dim == 64) by_size(tag, std::integral_constant<int, 64>{});
        else by_size(tag, std::integral_constant<int, 128>{});
    };
    if (a.dtype == DELS_DTYPE_BF16) by_type(bf16_t{});
    else by_type(f16_t{});
    return hipGetLastError();
}

}  // namespace dels
