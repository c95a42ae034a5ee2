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
// scale 1; the value scale of a slot multiplies its weight.  That product enters the
// matrix cores as two bf16 parts (2^-17 of each weight, whatever its size: one part
// alone would round every weight by 2^-8, as much as a bf16 output itself, and f16
// would lose the small ones).  Scores, maxima, sums and outputs are fp32.
//
// A wave takes a page of 64 slots at a time, 8 waves of a workgroup every eighth
// page; their states are joined through LDS.  The pages of all (sequence, head,
// rows) are numbered in one line, which is cut into equal pieces, one for each
// workgroup, whatever the lengths are: a piece that covers all pages of its rows
// writes their output, others write their state, which kv4_join_kernel joins.
#include <algorithm>

#include "../../include/dels.h"
#include "kv4.h"

namespace dels {

namespace {

constexpr int kAttnWaves = 8;
constexpr int kAttnThreads = 64 * kAttnWaves;
constexpr float kLog2e = 1.44269504088896340736f;
// A row's running maximum follows only when a score passes it by this many binary
// orders: until then the weights are at most 2^8, which costs fp32 nothing, and the
// outputs need no rescaling.
constexpr float kLag = 8.f;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Frag;
template <> struct Frag<bf16_t> { using type = bf16x8; };
template <> struct Frag<f16_t> { using type = f16x8; };

// Eight codes times a power of two.
template <typename T> __device__ __forceinline__ typename Frag<T>::type decode8(uint32_t w, float scale);
template <> __device__ __forceinline__ bf16x8 decode8<bf16_t>(uint32_t w, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <> __device__ __forceinline__ f16x8 decode8<f16_t>(uint32_t w, float scale) {
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3);
    return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Two numbers rounded to bf16, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// fp16 holds keys of up to 2^20 at a sixteenth of their size; the scale makes up for it.
template <typename T> constexpr int kKeyShift = 0;
template <> constexpr int kKeyShift<f16_t> = 4;

template <typename T>
__device__ __forceinline__ float key_scale(uint32_t word, int byte) {
    const int e = (int)((word >> (8 * byte)) & 255u);
    return __uint_as_float((uint32_t)max(e - kKeyShift<T>, 0) << 23);
}

// Shapes of a wave's work on MT rows: MT x MT tiles of the matrix instructions.
template <int D, int MT_> struct Shape {
    static constexpr int MT = MT_;
    static constexpr int NG = 64 / MT;              // lane groups: lane = MT * group + row
    static constexpr int DL = D / NG;               // channels of a key that a lane holds
    static constexpr int KS = DL / 8;               // steps of the first product
    static constexpr int KB = DL >= 32 ? DL / 32 : 1;   // key scales per lane
    static constexpr int KT = 32 / MT;              // key tiles of 32 slots
    static constexpr int ACC = MT == 16 ? 4 : 16;   // accumulator registers of a tile
    static constexpr int PF = 32 * MT / 64 / 8;     // weight operands (8 slots) per 32 slots
    static constexpr int CT = D / MT;               // channel tiles of the output
    static constexpr int VW = MT == 16 ? 4 : D / 32;    // consecutive channels of a lane: words of a load
    static constexpr int VL = CT / VW;              // loads of value words per operand
    using Acc = typename std::conditional<MT == 16, f32x4, f32x16>::type;
    // slot within 32 that row r of key tile a holds
    __device__ static int slot_of(int a, int r) {
        if constexpr (MT == 16) return 8 * (r >> 2) + 4 * a + (r & 3);
        return 16 * (r >> 4) + 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3);
    }
    // first of the VW channels that register i of a tile holds in channel block `vl`
    __device__ static int channel_of(int vl, int i, int g) {
        const int row = MT == 16 ? 4 * g + i : 8 * (i >> 2) + 4 * g + (i & 3);
        return vl * MT * VW + row * VW;
    }
};

// The line of pages: those of (b, h, row tile) one after the other, b first.  It is
// cut every `share` pages; a cut within `snap` pages of a row tile's end moves there,
// so that no piece holds a few pages of one tile and the rest of another's.
struct Line {
    int tiles;                 // row tiles per (b, h)
    int pieces;                // workgroups
    int min_pages;             // fewest pages of a piece
};
constexpr int kSnap = 8;       // one page for each wave

__device__ __forceinline__ int seq_end(const Kv4Block& k, int b, int slots) {
    const int n = kv4_length(k.lengths, b, slots);
    if (k.mode == DELS_KV4_NONE) return n;
    return (int)min((int64_t)slots, (int64_t)n + kv4_count(k.counts, b, k.T));
}
// Pages of sequence b (one at least: rows that see nothing are written too).
__device__ __forceinline__ int seq_pages(const Kv4Block& k, int b, int slots) {
    return max(1, (seq_end(k, b, slots) + kKv4Page - 1) / kKv4Page);
}

// What all lanes of a wave hold alike, kept in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Scan of the sequences' units by a wave, 64 at a time; up to 64 it is kept.
struct Scan {
    const Kv4Block& k;
    const Kv4Cache& c;
    int per;                   // row tiles of a sequence
    int own, cum;              // units of this lane's sequence, and of all up to it, in the 64 from b0
    int b0, before, total;

    __device__ Scan(const Kv4Block& k_, const Kv4Cache& c_, int per_) : k(k_), c(c_), per(per_) {
        seek(0, 0);
        total = __builtin_amdgcn_readlane(cum, 63);
        for (int b = 64 + (threadIdx.x & 63), rest = 0; c.batch > 64; b += 64) {
            rest += b < c.batch ? seq_pages(k, b, c.slots()) * per : 0;
            if ((b & ~63) + 64 >= c.batch) {
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) rest += __shfl_xor(rest, off, 64);
                total += uniform(rest);
                break;
            }
        }
    }
    __device__ void seek(int b0_, int before_) {
        const int lane = threadIdx.x & 63;
        b0 = b0_, before = before_;
        own = b0 + lane < c.batch ? seq_pages(k, b0 + lane, c.slots()) * per : 0;
        cum = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(cum, off, 64);
            cum += lane >= off ? o : 0;
        }
    }
    // Sequence of unit u < total, its first unit and its pages.
    struct Place { int b, start, pages; };
    __device__ Place place(int u) {
        if (u < before) seek(0, 0);
        for (;;) {
            const unsigned long long past = __ballot(before + cum > u);
            if (past) {
                const int l = __builtin_ctzll(past);
                return {b0 + l, __builtin_amdgcn_readlane(before + cum - own, l),
                        __builtin_amdgcn_readlane(own, l) / per};
            }
            const int all = __builtin_amdgcn_readlane(cum, 63);
            seek(b0 + 64, before + all);
        }
    }
    // Where the cut at unit u comes to lie.
    __device__ int cut(int u, int share) {
        if (u >= total) return total;
        const Place at = place(u);
        const int lo = at.start + (u - at.start) / at.pages * at.pages, hi = lo + at.pages;
        return snap(u, lo, hi, share);
    }
    __device__ static int snap(int u, int lo, int hi, int share) {
        const int reach = min(share / 2, kSnap);
        return u - lo <= reach ? lo : hi - u <= reach ? hi : u;
    }
};

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
    x.t = r / group;
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

// `ref`: binary logarithm of the unit that `total` counts in.
__device__ __forceinline__ void store_lse(const Kv4AttentionArgs& a, int b, const Row& row, float ref, float total) {
    if (!row.in_block) return;
    const float x = row.valid && total > 0.f ? (ref + __builtin_amdgcn_logf(total)) * 0.693147180559945309f
                                             : -__builtin_inff();
    a.lse[((int64_t)b * a.block.T + row.t) * a.q_heads + row.hq] = x;
}

// exp2(m - ref), 0 for m = -inf, whatever ref is.
__device__ __forceinline__ float fade(float m, float ref) {
    return m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - ref);
}

// Floats of a piece's state in the workspace: outputs as the lanes hold them, then references and sums.
template <int D, int MT> constexpr int kStateFloats = MT * D + 2 * MT;

// Byte offsets of a lane within a page; what differs between its loads is constant, so
// that a load is a page address, a lane offset and an immediate.
template <int D, int MT> struct LaneOffsets {
    uint32_t key, key_scale, half, value, value_scale;
    __device__ LaneOffsets(int col, int g) {
        using S = Shape<D, MT>;
        const int r = S::slot_of(0, col);
        key = r * Kv4<D>::kKeyRow + g * (S::DL / 2);
        key_scale = Kv4<D>::kKeyScale + 64 * (g * S::DL / 32) + 16 * ((r >> 3) & 3) + 4 * (r & 3);
        half = 8 * ((r >> 2) & 1);         // key tiles of 32 rows: their slot's byte within the scales
        value = Kv4<D>::kValue + 4 * (g * D + col * S::VW);
        value_scale = Kv4<D>::kValueScale + 16 * g;
    }
};
__device__ __forceinline__ const uint32_t* page_word(const uint8_t* page, uint32_t lane_off, int imm) {
    return reinterpret_cast<const uint32_t*>(page + lane_off + imm);
}

// What a wave loads of a page: keys, and values.
template <int D, int MT> struct KeyWords {
    using S = Shape<D, MT>;
    uint32_t code[2][S::KT][S::KS];
    uint32_t scale[S::KB];
    __device__ __forceinline__ void load(const uint8_t* page, const LaneOffsets<D, MT>& at) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int t = 0; t < S::KT; ++t)
#pragma unroll
                for (int k = 0; k < S::KS; ++k)
                    code[s][t][k] = page_word(page, at.key, (32 * s + 4 * t) * Kv4<D>::kKeyRow)[k];
#pragma unroll
        for (int i = 0; i < S::KB; ++i) scale[i] = *page_word(page, at.key_scale, 64 * i);
    }
};
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
    float top, total;          // running maximum (in raw products) and this lane's part of the sum
    int lim;                   // the row sees slots below it,
    uint64_t bits;             // and those of the block whose bits are set

    // n, filled: context, and the slots that hold anything; unit: binary logarithms per raw product
    // q: this lane's operands of the queries in LDS, 64 apart
    __device__ __forceinline__ void page(const F* q, const KeyWords<D, MT>& keys, ValueWords<D, MT>& values, uint32_t half,
                                         int first_slot, int n, int filled, int slots, int g, float unit) {
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
#pragma unroll
        for (int k = 0; k < S::KS; ++k) {
            const F qk = q[64 * k];
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
#pragma unroll
        for (int off = MT; off < 64; off <<= 1) best = fmaxf(best, __shfl_xor(best, off, 64));
        if (__any((best - top) * unit > kLag)) {
            const float now = fmaxf(top, best), f = fade(top * unit, now * unit);
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
                const bf16x8 vf = decode8<bf16_t>(values.code[u / S::PF][u % S::PF][t], 1.f);
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

// A page number, the same for all lanes: a scalar load, so that its arrival is not
// waited for together with the loads of a page.
__device__ __forceinline__ int page_id(const int32_t* row, int p) {
    return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(row + p);
}

#ifndef KV4_OCC
#define KV4_OCC 2
#endif
template <typename T, int D, int MT>
__global__ __launch_bounds__(kAttnThreads, MT == 16 ? KV4_OCC : 2) void kv4_attention_kernel(Kv4AttentionArgs a, Line line,
                                                                                float* __restrict__ states) {
    using S = Shape<D, MT>;
    constexpr int kRegs = S::CT * S::ACC;                   // output registers
    constexpr int kRound = 32;                              // registers joined at a time
    __shared__ float s_o[kAttnWaves][kRound][64];
    __shared__ float s_m[kAttnWaves][MT], s_l[kAttnWaves][MT];
    __shared__ typename Frag<T>::type s_q[S::KS][64];
    static_assert(S::KS <= kAttnWaves, "a wave per step of the first product loads the queries");

    const Kv4Cache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane % MT, g = lane / MT;
    const int slots = c.slots(), group = a.q_heads / c.heads;
    // pieces that follow each other on one XCD: they share pages where a head has several row tiles
    const int piece = (int)gridDim.x % 8 ? (int)blockIdx.x
                                         : (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
    const LaneOffsets<D, MT> at_lane(col, g);
    Scan scan(a.block, c, c.heads * line.tiles);
    const int share = max(line.min_pages, (scan.total + line.pieces - 1) / line.pieces);
    if ((int64_t)piece * share >= scan.total) return;
    int u = scan.cut(piece * share, share);
    const int u_end = scan.cut((int)min((int64_t)(piece + 1) * share, (int64_t)scan.total), share);
    if (u >= u_end) return;
    Scan::Place at = scan.place(u);
    // scores in units of the maximum: |scale| and the query's sign
    const float mag = fabsf(a.scale);
    const float unit = (mag == 0.f ? 1.f : mag) * kLog2e * (float)(1 << kKeyShift<T>);
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, zero = mag == 0.f ? 0u : ~0u;

    while (u < u_end) {
        if (u >= at.start + at.pages * scan.per) at = scan.place(u);
        const int b = at.b;
        const int rel = u - at.start, ht = rel / at.pages, first = rel - ht * at.pages;
        const int h = ht / line.tiles, rt = ht - h * line.tiles;
        const int last = min(at.pages, first + (u_end - u));
        const int n = uniform(kv4_length(a.block.lengths, b, slots));
        const int count = uniform(kv4_count(a.block.counts, b, a.block.T));
        const int filled = uniform(seq_end(a.block, b, slots));   // slots past it may hold anything
        int end = filled;
        if (a.block.mode == DELS_KV4_CAUSAL)                  // no row of the tile sees past its last token
            end = (int)min((int64_t)end, (int64_t)n + (rt * MT + MT - 1) / group + 1);
        const int stop = min(last, (end + kKv4Page - 1) / kKv4Page);

        // the wave's pages, the next one loaded while one is worked on
        const int32_t* ids = c.table + (int64_t)b * c.ld_table;
        const uint8_t* heads = c.data + (int64_t)h * Kv4<D>::kBytes;
        const int64_t page_stride = (int64_t)c.heads * Kv4<D>::kBytes;
        int p = first + wave;

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
        // the queries, in operand order: a wave loads what all of them read
        if (wave < S::KS) {
            u32x4 w = {0u, 0u, 0u, 0u};
            if (row.valid)
                w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q.p) + (int64_t)b * a.q.batch +
                                                    (int64_t)row.t * a.q.token + (int64_t)row.hq * a.q.head +
                                                    g * S::DL + 8 * wave);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (w[i] ^ flip) & zero;
            s_q[wave][lane] = __builtin_bit_cast(typename Frag<T>::type, w);
        }
        rows.top = -__builtin_inff();
        rows.total = 0.f;
#pragma unroll
        for (int t = 0; t < S::CT; ++t)
#pragma unroll
            for (int i = 0; i < S::ACC; ++i) rows.o[t][i] = 0.f;

        __syncthreads();
        auto named = [&](int id) { return id >= 0 && id < c.num_pages; };
        // Pages p, p + 8, ... below `stop`; one that the table does not name is passed over.
        // Keys are loaded a page ahead, values at the start of their page's work.  The
        // loads are unconditional (of page 0 where there is none to load) and in this
        // order, so that each wait covers only what it needs.  One copy of the work: two
        // that swap the keys' registers take longer to fetch than their moves.
        auto next_id = [&](int at_page) { return at_page < stop ? page_id(ids, at_page) : -1; };
        auto address = [&](int id) { return heads + (named(id) ? id : 0) * page_stride; };
        if (p < stop) {
            KeyWords<D, MT> keys, next_keys;
            ValueWords<D, MT> values;
            int id = next_id(p), next = next_id(p + kAttnWaves);
            keys.load(address(id), at_lane);
            for (; p < stop; p += kAttnWaves) {
                values.load(address(id), at_lane);
                asm volatile("" ::: "memory");
                next_keys.load(address(next), at_lane);
                asm volatile("" ::: "memory");
                const int after = next_id(p + 2 * kAttnWaves);
                if (named(id)) rows.page(&s_q[0][lane], keys, values, at_lane.half, p * kKv4Page, n, filled, slots, g, unit);
                keys = next_keys;
                id = next;
                next = after;
            }
        }

        // ---- join the waves
        const float ref = rows.top * unit;
        float total = rows.total;
#pragma unroll
        for (int off = MT; off < 64; off <<= 1) total += __shfl_xor(total, off, 64);
        if (g == 0) {
            s_m[wave][col] = ref;
            s_l[wave][col] = total;
        }
        __syncthreads();
        const bool whole = first == 0 && last == at.pages;
        float* state = states + (int64_t)(2 * piece + (first == 0 ? 1 : 0)) * kStateFloats<D, MT>;
        float m = -__builtin_inff(), l = 0.f;
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) m = fmaxf(m, s_m[w][col]);
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) l += s_l[w][col] * fade(s_m[w][col], m);
        const float f = fade(ref, m), inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
        for (int r0 = 0; r0 < kRegs; r0 += kRound) {
            // register (vl, i, v): channel block, row of the tile, channel of the VW
#pragma unroll
            for (int j = 0; j < kRound && r0 + j < kRegs; ++j) {
                const int r = r0 + j, v = r % S::VW, i = r / S::VW % S::ACC, vl = r / S::VW / S::ACC;
                s_o[wave][j][lane] = rows.o[vl * S::VW + v][i] * f;
            }
            __syncthreads();
            for (int jg = wave; jg * S::VW < kRound && r0 + jg * S::VW < kRegs; jg += kAttnWaves) {
                float sum[S::VW];
#pragma unroll
                for (int v = 0; v < S::VW; ++v) {
                    sum[v] = 0.f;
#pragma unroll
                    for (int w = 0; w < kAttnWaves; ++w) sum[v] += s_o[w][jg * S::VW + v][lane];
                }
                const int gi = r0 / S::VW + jg;
                if (whole) {
                    store_out<T, S::VW>(a, b, row, S::channel_of(gi / S::ACC, gi % S::ACC, g), sum, inv);
                } else {
                    float* to = state + (gi * 64 + lane) * S::VW;
#pragma unroll
                    for (int v = 0; v < S::VW; ++v) to[v] = sum[v];
                }
            }
            __syncthreads();
        }
        if (wave == 0 && g == 0) {
            if (whole) {
                store_lse(a, b, row, m, l);
            } else {
                state[MT * D + col] = m;
                state[MT * D + MT + col] = l;
            }
        }
        u += last - first;
    }
}

// Joins the states of the rows whose pages lie in several pieces.  Grid (sequence x
// head x row tile, quarter of the output registers), a wave per VW channels.
constexpr int kJoinWaves = 4;
template <typename T, int D, int MT>
__global__ __launch_bounds__(64 * kJoinWaves) void kv4_join_kernel(Kv4AttentionArgs a, Line line,
                                                                   const float* __restrict__ states) {
    using S = Shape<D, MT>;
    const Kv4Cache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % MT, g = lane / MT;
    const int per = c.heads * line.tiles, group = a.q_heads / c.heads;
    const int b = blockIdx.x / per, ht = blockIdx.x % per, h = ht / line.tiles, rt = ht % line.tiles;
    Scan scan(a.block, c, per);
    const int share = max(line.min_pages, (scan.total + line.pieces - 1) / line.pieces);
    int before = 0;                                         // pages of the sequences before b
    for (int i = lane; i < b; i += 64) before += seq_pages(a.block, i, c.slots());
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) before += __shfl_xor(before, off, 64);
    const int pages = seq_pages(a.block, b, c.slots());
    const int lo = before * per + ht * pages, hi = lo + pages;
    // cuts w0 .. w1 - 1 stay inside; the piece before the first has the tile's first pages
    int w0 = (lo + share - 1) / share, w1 = (hi - 1) / share + 1;
    while (w0 < w1 && Scan::snap(w0 * share, lo, hi, share) == lo) ++w0;
    while (w0 < w1 && Scan::snap((w1 - 1) * share, lo, hi, share) == hi) --w1;
    if (w0 >= w1) return;                                   // one piece covered them and wrote the output
    auto state_of = [&](int w) { return states + (int64_t)(2 * w + (w < w0 ? 1 : 0)) * kStateFloats<D, MT>; };
    float m = -__builtin_inff(), l = 0.f;
#pragma unroll 4
    for (int w = w0 - 1; w < w1; ++w) m = fmaxf(m, state_of(w)[MT * D + col]);
    const int gi = blockIdx.y * kJoinWaves + wave;
    float sum[S::VW];
#pragma unroll
    for (int v = 0; v < S::VW; ++v) sum[v] = 0.f;
#pragma unroll 4
    for (int w = w0 - 1; w < w1; ++w) {
        const float* st = state_of(w);
        const float f = fade(st[MT * D + col], m);
        l += st[MT * D + MT + col] * f;
        const float* from = st + (gi * 64 + lane) * S::VW;
#pragma unroll
        for (int v = 0; v < S::VW; ++v) sum[v] += from[v] * f;
    }
    const Row row = row_of(rt * MT + col, group, h, a.block.T, kv4_count(a.block.counts, b, a.block.T));
    store_out<T, S::VW>(a, b, row, S::channel_of(gi / S::ACC, gi % S::ACC, g), sum, l > 0.f ? 1.f / l : 0.f);
    if (gi == 0 && g == 0) store_lse(a, b, row, m, l);
}

struct Plan { int rows; Line line; };

Plan plan(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t max_pages) {
    Plan p{};
    const int64_t rows = T * (q_heads / heads);
    p.rows = rows <= 16 ? 16 : 32;
    p.line.tiles = (int)((rows + p.rows - 1) / p.rows);
    p.line.min_pages = kAttnWaves;
    const int64_t units = batch * heads * p.line.tiles * std::max<int64_t>(max_pages, 1);
    const int64_t resident = (int64_t)device_cu_count() * (p.rows == 16 ? KV4_OCC / 2 : 1);
    p.line.pieces = (int)std::min<int64_t>(resident, (units + p.line.min_pages - 1) / p.line.min_pages);
    return p;
}

template <typename F> hipError_t by_type(int dtype, int head_dim, int rows, F&& f) {
    auto by_rows = [&](auto tag, auto size) {
        if (rows == 16) f(tag, size, std::integral_constant<int, 16>{});
        else f(tag, size, std::integral_constant<int, 32>{});
    };
    auto by_size = [&](auto tag) {
        if (head_dim == 64) by_rows(tag, std::integral_constant<int, 64>{});
        else by_rows(tag, std::integral_constant<int, 128>{});
    };
    if (dtype == DELS_DTYPE_BF16) by_size(bf16_t{});
    else by_size(f16_t{});
    return hipGetLastError();
}

}  // namespace

size_t kv4_attention_data_bytes(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t head_dim,
                                int64_t max_pages) {
    const Plan p = plan(batch, T, q_heads, heads, max_pages);
    return align256((size_t)p.line.pieces * 2 * sizeof(float) * (p.rows * head_dim + 2 * p.rows));
}

hipError_t launch_kv4_attention(const Kv4AttentionArgs& a, void* ws, size_t data_off, hipStream_t s) {
    const Kv4Cache& c = a.cache;
    const Plan p = plan(c.batch, a.block.T, a.q_heads, c.heads, c.max_pages);
    auto* states = reinterpret_cast<float*>(static_cast<char*>(ws) + data_off);
    return by_type(a.dtype, c.head_dim, p.rows, [&](auto tag, auto size, auto rows) {
        using T = decltype(tag);
        constexpr int D = decltype(size)::value, MT = decltype(rows)::value;
        using S = Shape<D, MT>;
        static_assert(S::CT * S::ACC / S::VW % kJoinWaves == 0, "a wave of the join per VW channels");
        hipLaunchKernelGGL((kv4_attention_kernel<T, D, MT>), dim3(p.line.pieces), dim3(kAttnThreads), 0, s, a, p.line,
                           states);
        hipLaunchKernelGGL((kv4_join_kernel<T, D, MT>),
                           dim3((unsigned)c.batch * c.heads * p.line.tiles, S::CT * S::ACC / S::VW / kJoinWaves),
                           dim3(64 * kJoinWaves), 0, s, a, p.line, states);
    });
}

}  // namespace dels
