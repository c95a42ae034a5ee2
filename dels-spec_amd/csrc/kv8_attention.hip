// Attention over the 8-bit key/value cache (format: kv8.h), whole or through a window.
//
//     x[t, j] = scale * q[t] . k[j]          j a slot that row t sees
//     lse[t]  = log sum_j exp(x[t, j])
//     o[t]    = sum_j exp(x[t, j] - lse[t]) v[j]
// A row that sees nothing has o = 0 and lse = -inf.  With a window, row t sees of those slots
// the ones from lengths + t - window + 1 on and the first `sinks`; where a tree's rows have positions,
// a row's own takes the place of lengths + t, and a slot of the block is where its row is.
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
// step of a bf16 output where values do not cancel), for f16 outputs in two parts, and for bf16 ones in two
// bf16 parts (2^-17) where the caller asks for it.  By norm, bf16 outputs of 2 x 512 rows over 3500 slots are
// 1.6713e-3 off the 64-bit ones, 1.6599e-3 with two parts or fp32 weights: the rounding of the output is
// what there is.  Two parts take 24 matrix instructions a step for 16: 8 x 16 rows 21 -> 24 us, 131k slots
// 60 -> 78, 2 x 512 rows 87 -> 124, 4093 rows through a window 114 -> 151, one row of 32 sequences
// 152 -> 155.  Scores, maxima, sums and outputs are fp32.
//
// What bounds it, at 32 query and 8 cache heads of 128 in bf16 (kernel times, medians under the profiler; the
// times above and beside the rules below are of calls without it):
//   32 sequences of up to 16300 slots, 1 token     153 us  memory: 955 MB at 6.2 TB/s
//   131k slots, 16 tokens                            61 us  memory and issue: 276 MB at 4.5 TB/s, matrix cores 23 %
//   4093 tokens through a window of 1024            130 us  issue: a step of 32 x 32 has 16 matrix
//                                                  (a call  instructions (512 cycles) and 140 vector ones, 64 of
//                                                  113 us)  them conversions; 0.57 PFLOP/s, those masked counted
//   8 sequences of up to 4000 slots, 16 tokens       21 us  latency: 2 us to know its pages, 13 for two or three
//                                                           pages a wave, 5 joining waves and parts
// Pages go straight from memory to registers, the next one's loads in flight behind a page's work; where
// eight row tiles share them, through LDS.
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

// 16 bytes of a page.  ONCE: one row tile is all there is, so each page is read once, and need not
// stay in the caches: 32 sequences of 16300 slots 171 -> 152 us for 16 rows, 175 -> 156 for 32.  Of two
// tiles the second finds the page there: 64 rows 287 us, 302 without.
template <bool ONCE> __device__ __forceinline__ u32x4 page_words(const uint8_t* p) {
    const auto* w = reinterpret_cast<const u32x4*>(p);
    if constexpr (ONCE) return __builtin_nontemporal_load(w);
    else return *w;
}

template <int D, int MT, bool ONCE> struct KeyRegs {
    using S = Shape8<D, MT>;
    u32x4 code[S::STEPS][S::NT][S::KL];
    __device__ __forceinline__ void load(const uint8_t* page, int col, int g, int step) {
        const int lane = MT == 16 ? 32 * D * (col >> 3) + 512 * g + 16 * (col & 7) : 512 * g + 16 * col;
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
#pragma unroll
            for (int i = 0; i < S::KL; ++i)
                code[step][t][i] =
                    page_words<ONCE>(page + lane + 512 * S::NG * i + (MT == 16 ? 128 * t : 32 * D * step));
    }
};

template <int D, int MT, bool ONCE> struct ValueRegs {
    using S = Shape8<D, MT>;
    u32x4 code[S::STEPS][S::CT];
    __device__ __forceinline__ void load(const uint8_t* page, int col, int g, int step) {
        const int lane = Kv8<D>::kValue + 16 * D * g + 16 * col;
#pragma unroll
        for (int t = 0; t < S::CT; ++t)
            code[step][t] = page_words<ONCE>(page + lane + 32 * D * step + 16 * MT * t);
    }
};

// A block mode of the kernel's own: a tree's rows have positions, and the mask has 64 words for each
// sequence with what the rows' windows leave of their bits, then 64 with where they begin to see.
constexpr int kTreeRows = 64, kTreeMode = DELS_KV4_MASK + 1;

// Which slots a row sees.
struct Sight {
    int n, filled;             // context; slots that hold anything
    int lim, lo;               // the row sees slots below lim, from lo on
    int sinks;                 // or below this,
    uint64_t bits;             // and those of the block whose bits are set
    __device__ uint32_t of_run(int j0) const {             // of slots j0 .. j0 + 15
        const int d = j0 - n;
        uint32_t by_bit = d >= 64 || d <= -16 ? 0u : (uint32_t)(d >= 0 ? bits >> d : bits << -d) & 0xffffu;
        by_bit &= lowest(filled - j0);
        return (lowest(lim - j0) & (~lowest(lo - j0) | lowest(sinks - j0))) | by_bit;
    }
};

// The lowest k of 64 bits.
__device__ __forceinline__ uint64_t lowest64(int64_t k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; }

// What a page's two blocks say of themselves, the same for the whole wave.
struct Page {
    uint32_t exponents[2], bad[2];
    __device__ Page() = default;
    __device__ __forceinline__ explicit Page(u32x4 head)
        : exponents{(uint32_t)uniform((int)head[0]), (uint32_t)uniform((int)head[2])},
          bad{(uint32_t)uniform((int)head[1]), (uint32_t)uniform((int)head[3])} {}
    __device__ int key(int u) const { return min(max((int)(exponents[u] & 255u), kKv8Low), kKv8High); }
    __device__ int value(int u) const { return min(max((int)(exponents[u] >> 8 & 255u), kKv8Low), kKv8High); }
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

    // Step k of the contraction of a step's scores; q: this lane's operand of the queries.
    static __device__ __forceinline__ void score(int k, const F& q, const u32x4 (&code)[S::NT][S::KL],
                                                 typename S::Acc (&acc)[S::NT]) {
        if (k == 0)
#pragma unroll
            for (int t = 0; t < S::NT; ++t)
#pragma unroll
                for (int i = 0; i < S::ACC; ++i) acc[t][i] = 0.f;
#pragma unroll
        for (int t = 0; t < S::NT; ++t)
            acc[t] = mma(widen8<T>(code[t][k / 2][2 * (k % 2)], code[t][k / 2][2 * (k % 2) + 1], 1.f), q, acc[t]);
    }

    // Adds weights times values; x: scores, their binary logarithms are x * factor - ref.
    // P: type and number of parts of a weight; next(k): step k of the next step's scores.
    template <typename P, int PARTS, typename Next>
    __device__ __forceinline__ void multiply(const float (&x)[16], float factor, float ref, const u32x4 (&code)[S::CT],
                                             float vscale, Next&& next) {
        using V = typename Frag<P>::type;
        // The weights are made while the next scores are: between two matrix instructions stand as
        // many cycles of vector ones, in this order (the fences keep it), so that neither waits for
        // the other.
        u32x4 part[PARTS][2];
        float even = 0.f;
        constexpr int kEach = 16 / S::KS;
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
            __builtin_amdgcn_sched_barrier(0);
            next(k);
#pragma unroll
            for (int i = k * kEach; i < (k + 1) * kEach; ++i) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], factor, -ref));
                total += e;
                if (i % 2 == 0) {
                    even = e;
                } else {
                    const uint32_t h = pack2<P>(even, e);
                    part[0][i / 8][i / 2 % 4] = h;
                    if constexpr (PARTS == 2)
                        part[1][i / 8][i / 2 % 4] =
                            pack2<P>(even - widen_raw<P>(h & 0xffffu), e - widen_raw<P>(h >> 16));
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int t = 0; t < S::CT; ++t) {
                __builtin_amdgcn_sched_barrier(0);
                const V vf = widen8<P>(code[t][2 * u], code[t][2 * u + 1], vscale);
#pragma unroll
                for (int p = 0; p < PARTS; ++p) o[t] = mma(vf, __builtin_bit_cast(V, part[p][u]), o[t]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    // Takes a page's scales in (of its first `blocks` blocks; the others hold nothing yet); whether
    // its products can be of f16 numbers, with weights in one part for bf16 outputs.
    __device__ __forceinline__ bool admit(const Page& page, int blocks) {
        if (!blocks) return vlow >= vref - kSpan;
        const int v0 = page.value(0), v1 = blocks > 1 ? page.value(1) : v0;
        vlow = min(vlow, min(v0, v1));
        if (__builtin_expect(max(v0, v1) > vref, 0)) {
            asm volatile("");
            const int now = min(max(v0, v1) + kHead, kKv8High);
            rescale(vref ? kv8_pow2(max(127 + vref - now, 0)) : 1.f);
            vref = now;
        }
        return vlow >= vref - kSpan;
    }

    // WIDE: the scales lie far apart.  MASKED: some row does not see all of the page, some slot holds
    // nothing or nothing finite, or the page is none.  unit: binary logarithms per raw product.
    // next: as multiply's.
    template <bool WIDE, bool MASKED, typename Next>
    __device__ __forceinline__ void weigh(const typename S::Acc (&acc)[S::NT], const Page& page, bool none, int slot,
                                          int step, int g, u32x4 (&code)[S::CT], const Sight& sight, float unit,
                                          Next&& next) {
        const bool second = MT == 16 ? g >= 2 : step == 1;     // of the page's blocks
        const float factor = fmaxf(unit * kv8_pow2(second ? page.key(1) : page.key(0)), 1e-37f);
        int ve = second ? page.value(1) : page.value(0);
        float x[16];
#pragma unroll
        for (int v = 0; v < 16; ++v) x[v] = acc[MT == 16 ? v / 4 % S::NT : 0][v % S::ACC];
        if constexpr (MASKED) {
            slot += S::run_slot(step, g);
            const uint32_t sees = none ? 0u : sight.of_run(slot);
#pragma unroll
            for (int v = 0; v < 16; ++v) x[v] = choose(sees, v, x[v], -__builtin_inff());
            const uint32_t lost = (second ? page.bad[1] : page.bad[0]) >> (slot & 16) & sees;
            if (__any(lost != 0u)) {
                asm volatile("");
#pragma unroll
                for (int v = 0; v < 16; ++v) x[v] = choose(~lost, v, x[v], __builtin_nanf(""));
            }
            // behind the last slot anything may lie, and a weight of 0 does not make it 0
            const uint32_t keep = none ? 0u : lowest(sight.filled - slot);
            if (__any(keep != 0xffffu)) {
                asm volatile("");
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    // bit i to byte i
                    const uint32_t bytes = (((keep >> (4 * w) & 15u) * 0x00204081u) & 0x01010101u) * 255u;
#pragma unroll
                    for (int t = 0; t < S::CT; ++t) code[t][w] &= bytes;
                }
            }
            if (!keep) ve = vref;                          // nor need its scale be one
        }
        float best = x[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) best = fmaxf(best, x[v]);
        best = max_over_groups<MT>(best * factor);
        if (__builtin_expect(__any(best > top), 0)) {
            asm volatile("");
            const float now = fmaxf(top, best + kLag), f = fade(top, now);
            top = now;
            total *= f;
            rescale(f);
        }
        const float ref = (top == -__builtin_inff() ? 0.f : top) - kLift;
        const float vscale = kv8_pow2(134 + ve - vref);
        if constexpr (WIDE) multiply<bf16_t, 2>(x, factor, ref, code, vscale, next);
        else multiply<f16_t, std::is_same<T, f16_t>::value ? 2 : 1>(x, factor, ref, code, vscale, next);
    }
};

// Four channels of a row's output.
template <typename T>
__device__ __forceinline__ void store4(const Kv8AttentionArgs& a, int b, const Row& row, int ch, const float* o,
                                       float inv) {
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
        const int64_t more = a.block.mode == DELS_KV4_CAUSAL ? min(tokens, count)
                             : a.block.mode == DELS_KV4_NONE ? 0
                                                             : count;
        const int64_t span = (a.window + more + kCachePage - 2) / kCachePage + 1;
        return (int)min((int64_t)all, span + (a.sinks + kCachePage - 1) / kCachePage);
    }
    // of rows first .. last of the block (tokens)
    __device__ Seen seen(int n, int count, int first, int last) const {
        int end = seq_end(a.block, n, count, a.cache.slots());
        if (a.block.mode == DELS_KV4_CAUSAL) end = (int)min((int64_t)end, (int64_t)n + last + 1);
        Seen s{0, 0, (end + kCachePage - 1) / kCachePage};
        if (a.window) {
            if (a.block.mode == kTreeMode) first = 0;         // any row may be where the first one is
            const int64_t start = max((int64_t)n + first - a.window + 1, (int64_t)0);
            s.from = (int)min(start / kCachePage, (int64_t)s.end);
            s.sinks = (int)min((a.sinks + kCachePage - 1) / kCachePage, (int64_t)s.from);
        }
        return s;
    }
};

// LDS of a workgroup.  Where TILES row tiles go over the same pages, each way keeps a ring of
// them there: the page as it lies in memory but for its head, of which every wave has its own.
template <typename T, int D, int MT, int TILES, bool RING> struct Lds {
    using S = Shape8<D, MT>;
    static constexpr int kWays = kWaves / TILES;
    static constexpr int kRing = !RING ? 0 : 4;
    // output registers joined at a time, in fours: all where LDS has room (131k slots 67 -> 63 us)
    static constexpr int kRound = TILES <= 2 ? 16 : 8;
    union {
        uint8_t page[kWays][kRing ? kRing : 1][RING ? Kv8<D>::kHead : 16];
        f32x4 o[kWaves][kRound][64];
    };
    uint32_t head[kWaves][kRing ? kRing : 1][64];
    typename Frag<T>::type q[TILES][S::KS][64];             // the tiles' queries, in operand order
    float m[kWaves][MT], l[kWaves][MT];
    bool last;
};

// The words of kTreeMode.  A launch of its own (3 us), as a loop over a tree's rows in the kernel below
// spills registers there (8 x 16 rows 20.8 -> 21.7 us, whatever their block).
__global__ __launch_bounds__(kTreeRows) void kv8_tree_rows_kernel(Kv8AttentionArgs a, int64_t* words) {
    const int b = blockIdx.x, t = threadIdx.x, last = a.block.T - 1;
    const int n = paged_length(a.block.lengths, b, a.cache.slots());
    const int64_t p = (int64_t)a.at[(int64_t)b * a.ld_at + min(t, last)] - n;
    const int depth = (int)min(max(p, (int64_t)0), (int64_t)last);
    uint64_t held = 0;
    for (int i = 0; i <= last; ++i) {
        const int other = __shfl(depth, i, 64);
        held |= (uint64_t)(other > depth - a.window || n + other < a.sinks) << i;
    }
    if (t > last) return;
    words += 2 * (int64_t)kTreeRows * b + t;
    words[0] = a.block.mask[(int64_t)b * a.block.ld_mask + t] & (int64_t)held;
    words[kTreeRows] = max((int64_t)n + depth - a.window + 1, (int64_t)0);
}
size_t tree_rows_bytes(int64_t batch) { return align256((size_t)batch * 2 * kTreeRows * sizeof(int64_t)); }

// TILES of 8 waves share a way: row tiles over the same pages.  8 / TILES ways take every
// (8 / TILES)-th page each.
template <typename T, int D, int MT, int TILES, bool RING, bool ONCE>
__global__ __launch_bounds__(kThreads, 2) void kv8_attention_kernel(Kv8AttentionArgs a, Line line, float* states,
                                                                    unsigned int* counters) {
    using S = Shape8<D, MT>;
    using F = typename Frag<T>::type;
    using L = Lds<T, D, MT, TILES, RING>;
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
        const Seen seen =
            seqs.seen(n, count, divide(rt0 * MT, group), min(divide((rt0 + kTiles) * MT - 1, group), last_t));
        const bool past = rt * MT >= count * group;           // the tile has no valid row
        const int stop = !RING && past ? 0 : min(last, seen.count());
        Sight sight;
        sight.n = n;
        sight.filled = seq_end(a.block, n, count, slots);     // slots past it may hold anything
        sight.sinks = a.window ? (int)min(a.sinks, (int64_t)slots) : slots;
        // entries of the list of pages that every row of the tile sees whole: there nothing is masked
        int plain, plain_end;
        {
            const int to = min(sight.filled, a.block.mode == DELS_KV4_CAUSAL ? n + divide(rt * MT, group) + 1
                                             : a.block.mode == DELS_KV4_FULL ? n + count : n);
            plain = seen.sinks;
            if (a.window) {
                const int last_row =
                    a.block.mode == kTreeMode ? last_t : min(divide(rt * MT + MT - 1, group), last_t);
                const int64_t from = max((int64_t)n + last_row - a.window + 1, (int64_t)0);
                plain += max(0, (int)min((from + kCachePage - 1) / kCachePage, (int64_t)seen.end) - seen.from);
            }
            plain_end = seen.sinks + to / kCachePage - seen.from;
        }

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
            if (a.block.mode >= DELS_KV4_MASK) {
                const int64_t* words = a.block.mask + (int64_t)b * a.block.ld_mask + row.t;
                sight.bits = (uint64_t)words[0] & lowest64(count);
                if (a.block.mode == kTreeMode) sight.lo = (int)words[kTreeRows];
                else if (a.window) sight.bits &= ~lowest64(row.t - a.window + 1) | lowest64((int64_t)sight.sinks - n);
            }
        }
        sight.lim = min(sight.lim, sight.filled);
        rows.clear();
        // two parts that the caller asks for are those of scales that lie far apart
        if (std::is_same<T, bf16_t>::value && a.split) rows.vlow = -256;

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
        using False = std::false_type;
        using True = std::true_type;
        // blocks of page i that hold anything, and whether it needs masks
        auto blocks_of = [&](int slot, int id) {
            return named(id) ? min(2, (sight.filled - slot + kKv8Block - 1) / kKv8Block) : 0;
        };
        auto is_plain = [&](int i, int id, const Page& page) {
            return i >= plain && i < plain_end && named(id) && !(page.bad[0] | page.bad[1]);
        };
        if constexpr (!RING) {
            // A step's scores are made during the step before.  Keys of a page are loaded into their
            // registers once the scores of the page before are made, values once the products are: a
            // page's work ahead of their use.  The loads are unconditional (of page 0 where there is
            // none to load) and in the order of their use, so that each wait covers only what it
            // needs.
            KeyRegs<D, MT, ONCE> keys;
            ValueRegs<D, MT, ONCE> values;
            u32x4 head;
            typename S::Acc acc[S::NT];
            auto load_head = [&](const uint8_t* page) { head = *reinterpret_cast<const u32x4*>(page + Kv8<D>::kHead); };
            int id = id_at(p), next_id = -1;                  // of pages p and p + WAYS
            if (p < stop) {
                next_id = id_at(p + WAYS);
                load_head(address(id));
#pragma unroll
                for (int step = 0; step < S::STEPS; ++step) {
                    keys.load(address(id), col, g, step);
                    values.load(address(id), col, g, step);
                }
            }
            put_queries();
            lds_barrier();                                    // the loads stay in flight
            if (p < stop) {
#pragma unroll
                for (int k = 0; k < S::KS; ++k) Rows8<T, D, MT>::score(k, query(k), keys.code[0], acc);
                keys.load(address(next_id), col, g, 0);
                asm volatile("" ::: "memory");
            }
            // Tiles over the same pages go through them in step, so that the second finds a page in the
            // caches: 64 rows over 32 sequences of 16300 slots 285 -> 224 us, of 2000 slots 38 -> 36; 128
            // rows 379 -> 352 and 56 -> 57.  All waves wait as often, those without pages too.
            int left = TILES == 1 ? 0 : max(0, (min(last, seen.count()) - first + WAYS - 1) / WAYS);
            auto keep_step = [&] {
                __builtin_amdgcn_s_barrier();
                --left;
            };
            auto work = [&](auto wide, auto masked, const Page& page, int slot) {
                if constexpr (TILES > 1) keep_step();
                const int after = id_at(p + 2 * WAYS);
                const bool none = !named(id);
                load_head(address(next_id));
#pragma unroll
                for (int step = 0; step < S::STEPS; ++step) {
                    constexpr int kLast = S::STEPS - 1;
                    typename S::Acc next[S::NT];
                    auto& code = keys.code[step == kLast ? 0 : step + 1];
                    rows.template weigh<decltype(wide)::value, decltype(masked)::value>(
                        acc, page, none, slot, step, g, values.code[step], sight, unit,
                        [&](int k) { Rows8<T, D, MT>::score(k, query(k), code, next); });
                    keys.load(address(step == kLast ? after : next_id), col, g, step == kLast ? 0 : step + 1);
                    values.load(address(next_id), col, g, step);
                    asm volatile("" ::: "memory");
#pragma unroll
                    for (int t = 0; t < S::NT; ++t) acc[t] = next[t];
                }
                id = next_id;
                next_id = after;
                p += WAYS;
            };
            // one loop for each kind of page: what they change stays in its registers
            Page page;
            int slot = 0;
            bool whole_page = false, narrow = true;
            auto meet = [&] {
                if (p >= stop) return;
                page = Page(head);
                slot = seen.page(p) * kCachePage;
                whole_page = is_plain(p, id, page);
                narrow = rows.admit(page, blocks_of(slot, id));
            };
            meet();
            while (p < stop && narrow) {
                while (p < stop && narrow && !whole_page) {
                    work(False{}, True{}, page, slot);
                    meet();
                }
                while (p < stop && narrow && whole_page) {
                    work(False{}, False{}, page, slot);
                    meet();
                }
            }
            while (p < stop) {
                work(True{}, True{}, page, slot);
                meet();
            }
            while (left > 0) keep_step();
        } else {
            // The waves of a way copy a page into its ring, a share of 1 KiB pieces and the head each,
            // kRing - 2 pages ahead of the one that arrives.  One barrier a page, at the start of the
            // work on the page before, which reads this one's keys ahead: past it, all shares of the
            // page have arrived and nobody reads the buffer that the next copy goes to, that of
            // two pages before.
            constexpr int kShare = Kv8<D>::kHead / 1024 / TILES, kPer = kShare + 1, kAhead = L::kRing - 2;
            const int pages = max(0, (stop - first + WAYS - 1) / WAYS);      // of the first way, which has most
            int ids_ahead[kAhead + 2];                        // of the page that is worked on, the next, ..
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
#pragma unroll
            for (int i = 0; i < kAhead; ++i) ids_ahead[i + 1] = i < pages ? copy(i) : -1;
            // waits for page i, past what may still be on its way: the pages behind it
            auto arrive = [&](int i) {
                if (i + kAhead <= pages) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((kAhead - 1) * kPer) : "memory");
                else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                lds_barrier();
                ids_ahead[kAhead + 1] = i + kAhead < pages ? copy(i + kAhead) : -1;
            };
            F qr[S::KS];                                      // the tile's queries
            // keys of the next two steps: those of the next one in keys[0] while the page's first step
            // is worked on, in keys[1] during its second
            u32x4 keys[2][1][S::KL];
            typename S::Acc acc[1];
            auto load_keys = [&](int i, int step) {
                const uint8_t* at = lds.page[way][i % L::kRing] + 16 * lane + 32 * D * step;
#pragma unroll
                for (int e = 0; e < S::KL; ++e) keys[1 - step][0][e] = *reinterpret_cast<const u32x4*>(at + 1024 * e);
            };
            auto score = [&](int k, const u32x4(&code)[1][S::KL], typename S::Acc(&to)[1]) {
                Rows8<T, D, MT>::score(k, qr[k], code, to);
            };
            int i = 0;
            Page page;
            int slot = 0;
            bool mine = false, whole_page = false, narrow = true;
            auto meet = [&] {                                 // page i, which has arrived
                if (i >= pages) return;
#pragma unroll
                for (int e = 0; e <= kAhead; ++e) ids_ahead[e] = ids_ahead[e + 1];
                p = first + way + i * WAYS;
                mine = !past && p < stop;
                whole_page = false;
                if (!mine) return;
                page = Page(*reinterpret_cast<const u32x4*>(lds.head[wave][i % L::kRing]));
                slot = seen.page(p) * kCachePage;
                whole_page = is_plain(p, ids_ahead[0], page);
                narrow = rows.admit(page, blocks_of(slot, ids_ahead[0]));
            };
            // page i, and the first scores of the one behind it
            auto work = [&](auto wide, auto masked) {
                const bool none = !named(ids_ahead[0]);
                const uint8_t* at = lds.page[way][i % L::kRing] + Kv8<D>::kValue + (16 * D - 512) * g + 16 * lane;
#pragma unroll
                for (int step = 0; step < S::STEPS; ++step) {
                    if (step == 0 && i + 1 < pages) arrive(i + 1);
                    load_keys(i + 1, step);                   // for the step after next
                    u32x4 values[S::CT];
#pragma unroll
                    for (int t = 0; t < S::CT; ++t)
                        values[t] = *reinterpret_cast<const u32x4*>(at + 32 * D * step + 512 * t);
                    typename S::Acc next[1];
                    rows.template weigh<decltype(wide)::value, decltype(masked)::value>(
                        acc, page, none, slot, step, g, values, sight, unit,
                        [&](int k) { score(k, keys[step], next); });
                    acc[0] = next[0];
                }
                ++i;
            };
            auto pass = [&] {                                 // a page that this wave has no part in
                if (i + 1 < pages) arrive(i + 1);
                ++i;
            };
            if (pages) {
                arrive(0);
#pragma unroll
                for (int k = 0; k < S::KS; ++k) qr[k] = query(k);
                load_keys(0, 0);
#pragma unroll
                for (int k = 0; k < S::KS; ++k) score(k, keys[S::STEPS - 1], acc);
                load_keys(0, 1);
            }
            // one loop for each kind of page: what they change stays in its registers
            meet();
            while (i < pages && narrow) {
                while (i < pages && narrow && !whole_page) {
                    if (mine) work(False{}, True{});
                    else pass();
                    meet();
                }
                while (i < pages && narrow && whole_page) {
                    work(False{}, False{});
                    meet();
                }
            }
            while (i < pages) {
                if (mine) work(True{}, True{});
                else pass();
                meet();
            }
            __syncthreads();                                  // the ring's place is the join's
        }

        // ---- join the waves
        const float total = sum_over_groups<MT>(rows.total);
        const bool whole = first == 0 && last == at.pages;
        // a piece has at most one state of rows that it begins and one of rows that it goes on with
        auto state_of = [&](int w, bool begins) {
            return states + ((int64_t)(2 * w + (begins ? 1 : 0)) * kTiles + tile) * kStateFloats<D, MT>;
        };
        float* state = state_of(piece, first == 0);
        float m = rows.top, l = total;
        // registers 4 q .. 4 q + 3 of the joined outputs
        auto put = [&](int q, const float* sum) {
            if (whole) {
                const int ch = S::channel_of(q / (S::ACC / 4), q % (S::ACC / 4), g);
                store4<T>(a, b, row, ch, sum, l != 0.f ? 1.f / l : 0.f);
            } else {
                store_state<4>(state, q, lane, sum);
            }
        };
        const float shift = kv8_pow2(max(rows.vref - 7, 0));
        if constexpr (WAYS == 1) {
#pragma unroll
            for (int q = 0; q < kRegs / 4; ++q) {
                float o[4];
#pragma unroll
                for (int v = 0; v < 4; ++v) o[v] = rows.o[(4 * q + v) / S::ACC][(4 * q + v) % S::ACC] * shift;
                put(q, o);
            }
        } else {
            if (g == 0) {
                s_m[wave][col] = rows.top;
                s_l[wave][col] = total;
            }
            __syncthreads();
            m = -__builtin_inff(), l = 0.f;
#pragma unroll
            for (int w = tile * WAYS; w < (tile + 1) * WAYS; ++w) m = fmaxf(m, s_m[w][col]);
#pragma unroll
            for (int w = tile * WAYS; w < (tile + 1) * WAYS; ++w) l += s_l[w][col] * fade(s_m[w][col], m);
            const float f = fade(rows.top, m) * shift;
#pragma unroll
            for (int r0 = 0; r0 < kRegs / 4; r0 += kRound) {
#pragma unroll
                for (int j = 0; j < kRound && r0 + j < kRegs / 4; ++j) {
                    f32x4 x;
#pragma unroll
                    for (int v = 0; v < 4; ++v) x[v] = rows.o[4 * (r0 + j) / S::ACC][(4 * (r0 + j) + v) % S::ACC] * f;
                    s_o[wave][j][lane] = x;
                }
                __syncthreads();
                for (int j = way; j < kRound && r0 + j < kRegs / 4; j += WAYS) {
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < WAYS; ++w) {
                        const f32x4 x = s_o[tile * WAYS + w][j][lane];
#pragma unroll
                        for (int v = 0; v < 4; ++v) sum[v] += x[v];
                    }
                    put(r0 + j, sum);
                }
                __syncthreads();
            }
        }
        if (way == 0 && g == 0) {
            if (whole) store_lse8(a, b, row, m, l);
            else store_state_row<D, MT>(state, col, m, l);
        }
        if (!whole) {
            const int lo = at.start + ht * at.pages;
            const int2 held = cuts.holders(scan, b, ht, lo, lo + at.pages);
            if (last_to_arrive(counters, held, s_last)) {
                constexpr int kMine = (kRegs / 4 + WAYS - 1) / WAYS;
                float sum[kMine][4];
#pragma unroll
                for (int i = 0; i < kMine; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) sum[i][v] = 0.f;
                m = -__builtin_inff(), l = 0.f;
                // no more states in flight than there are, in powers of two (8 x 16 rows 22.0 -> 20.7 us)
                auto add = [&](auto flight) {
                    constexpr int kFlight = decltype(flight)::value;
                    for (int w0 = held.x; w0 < held.y; w0 += kFlight) {
                        const LoadedStates<kFlight, D, MT, WAYS, kRegs / 4, 4> loaded(
                            w0, held, way, lane, col, [&](int w) { return state_of(w, w == held.x); });
#pragma unroll
                        for (int e = 0; e < kFlight; ++e) {
                            if (w0 + e >= held.y) break;
                            const float top = loaded.reference[e], now = fmaxf(m, top), old = fade(m, now),
                                        f = fade(top, now);
                            m = now;
                            l = __builtin_fmaf(l, old, loaded.sum[e] * f);
#pragma unroll
                            for (int i = 0; i < kMine; ++i)
#pragma unroll
                                for (int v = 0; v < 4; ++v)
                                    sum[i][v] = __builtin_fmaf(loaded.output(e, i, v), f, sum[i][v] * old);
                        }
                    }
                };
                const int many = held.y - held.x;
                if (WAYS > 4 && many > 4) add(std::integral_constant<int, WAYS>{});
                else if (WAYS > 2 && many > 2) add(std::integral_constant<int, std::min(WAYS, 4)>{});
                else add(std::integral_constant<int, std::min(WAYS, 2)>{});
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
    // Tiles of 16 rows where one takes all: 32 x 16 rows of 16300 slots 153 us, 157 as half a tile of 32;
    // 8 x 16 rows of 4000 slots 17.8 and 21.1.  Two of them take twice as long as one of 32 does where
    // memory bounds it (32 x 32 rows: 297 and 157 us), and 1.5 us less in short calls.
    p.rows = rows <= 16 ? 16 : 32;
    const int64_t tiles = (rows + p.rows - 1) / p.rows;
    // Tiles of a workgroup: the more, the fewer times a page is loaded and waves' states are joined,
    // as long as there is a workgroup for each CU; of those numbers the one that leaves the fewest
    // waves without a tile, and never half of them.  One otherwise: its pages are split over
    // eight waves, and over workgroups.  8 heads of 128, 4 rows a token: 32 sequences of 1000 slots, 8
    // tiles 108 us one by one, 56 in eights, 2 tiles 35 and 29 in twos; 2 of 16000, 8 tiles 50 us
    // one by one, 98 in eights; 4093 tokens through a window of 1024: 174, 155, 135 and 115 us by
    // ones, twos, fours and eights; 8 sequences of 4000 slots, 2 tiles: 21 by ones, 29 in twos.
    p.tiles = 1;
    int64_t fewest = 2 * tiles;
    for (int64_t wide : {8, 4, 2}) {
        const int64_t groups = (tiles + wide - 1) / wide;
        if (p.rows == 32 && batch * heads * groups >= cus && groups * wide < fewest)
            fewest = groups * wide, p.tiles = (int)wide;
    }
    p.line.tiles = (int)((tiles + p.tiles - 1) / p.tiles);
    p.line.least = kMinPages;
    const int64_t units = batch * heads * p.line.tiles * std::max<int64_t>(max_pages, 1);
    const int64_t most = std::max(batch * heads * p.line.tiles, (units + kMinPages - 1) / kMinPages);
    p.line.pieces = (int)std::min<int64_t>({cus, kMaxCounters / kCounterWords, most});
    return p;
}

}  // namespace

size_t kv8_attention_data_bytes(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t head_dim,
                                int64_t max_pages) {
    // what any shorter block takes too, so that a workspace for the longest serves every one: pieces
    // as if each tile were a group of its own, and as many tiles a piece as there are groups for
    const int64_t rows = T * (q_heads / heads), tile_rows = rows <= 16 ? 16 : 32, cus = device_cu_count();
    const int64_t tiles = (rows + tile_rows - 1) / tile_rows, groups = batch * heads * tiles;
    const int64_t units = groups * std::max<int64_t>(max_pages, 1);
    const int64_t pieces = std::min<int64_t>({cus, kMaxCounters / kCounterWords,
                                              std::max(groups, (units + kMinPages - 1) / kMinPages)});
    int64_t wide = 1;
    auto enough = [&](int64_t w) { return batch * heads * ((tiles + w - 1) / w) >= cus; };
    while (tile_rows == 32 && wide < 8 && wide < tiles && enough(2 * wide)) wide *= 2;
    return tree_rows_bytes(batch) +
           align256((size_t)pieces * 2 * wide * sizeof(float) * (tile_rows * head_dim + 2 * tile_rows));
}

hipError_t launch_kv8_attention(const Kv8AttentionArgs& given, void* ws, size_t data_off, hipStream_t s) {
    Kv8AttentionArgs a = given;
    const PagedCache& c = a.cache;
    const Plan p = plan(c.batch, a.block.T, a.q_heads, c.heads, c.max_pages);
    char* data = static_cast<char*>(ws) + data_off;
    if (a.at) {
        auto* words = reinterpret_cast<int64_t*>(data);
        hipLaunchKernelGGL(kv8_tree_rows_kernel, dim3(c.batch), dim3(kTreeRows), 0, s, a, words);
        a.block.mode = kTreeMode, a.block.mask = words, a.block.ld_mask = 2 * kTreeRows;
    }
    auto* states = reinterpret_cast<float*>(data + tree_rows_bytes(c.batch));
    auto* counters = reinterpret_cast<unsigned int*>(static_cast<char*>(ws) + kCountersOff);
    auto by_size = [&](auto tag, auto size) {
        using T = decltype(tag);
        constexpr int D = decltype(size)::value;
        auto go = [&](auto rows, auto tiles, auto ring, auto once) {
            constexpr int MT = decltype(rows)::value, TILES = decltype(tiles)::value;
            constexpr bool RING = decltype(ring)::value, ONCE = decltype(once)::value;
            hipLaunchKernelGGL((kv8_attention_kernel<T, D, MT, TILES, RING, ONCE>), dim3(p.line.pieces), dim3(kThreads),
                               0, s, a, p.line, states, counters);
        };
        using std::integral_constant;
        using I16 = integral_constant<int, 16>;
        using I32 = integral_constant<int, 32>;
        using Yes = std::true_type;
        using No = std::false_type;
        if (p.rows == 16) go(I16{}, integral_constant<int, 1>{}, No{}, Yes{});
        else if (p.tiles == 1 && p.line.tiles == 1) go(I32{}, integral_constant<int, 1>{}, No{}, Yes{});
        else if (p.tiles == 1) go(I32{}, integral_constant<int, 1>{}, No{}, No{});
        else if (p.tiles == 2) go(I32{}, integral_constant<int, 2>{}, No{}, No{});
        else if (p.tiles == 4) go(I32{}, integral_constant<int, 4>{}, No{}, No{});
        else go(I32{}, integral_constant<int, 8>{}, Yes{}, No{});
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
