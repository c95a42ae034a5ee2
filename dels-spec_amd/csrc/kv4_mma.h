// What the matrix-core kernels over the 4-bit key/value cache share: operands made of
// codes, the shapes of a wave's work, a page's key words, and the line of pages that
// is cut over the workgroups.
#pragma once

#include "../../include/dels.h"
#include "kv4.h"

namespace dels {

constexpr int kKv4Waves = 8;                     // waves of a workgroup
constexpr int kKv4Threads = 64 * kKv4Waves;
constexpr float kLog2e = 1.44269504088896340736f;

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

// A row's number over the lane groups of MT lanes: the largest, and the sum.
template <int MT, typename F> __device__ __forceinline__ float over_groups(float x, F&& join) {
    const uint32_t b = __float_as_uint(x);
    const auto far = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    x = join(__uint_as_float(far[0]), __uint_as_float(far[1]));
    if constexpr (MT == 16) {
        const uint32_t c = __float_as_uint(x);
        const auto near = __builtin_amdgcn_permlane16_swap(c, c, false, false);
        x = join(__uint_as_float(near[0]), __uint_as_float(near[1]));
    }
    return x;
}
template <int MT> __device__ __forceinline__ float max_over_groups(float x) {
    return over_groups<MT>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int MT> __device__ __forceinline__ float sum_over_groups(float x) {
    return over_groups<MT>(x, [](float a, float b) { return a + b; });
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
template <typename T> constexpr int kKeyShift = std::is_same<T, f16_t>::value ? 4 : 0;

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

// Where a sequence's slots that hold anything end, and its pages (one at least: rows that
// see nothing are written too).
__device__ __forceinline__ int seq_end(const Kv4Block& k, int n, int count, int slots) {
    return k.mode == DELS_KV4_NONE ? n : (int)min((int64_t)slots, (int64_t)n + count);
}
__device__ __forceinline__ int seq_pages(int end) { return max(1, (end + kKv4Page - 1) / kKv4Page); }
__device__ __forceinline__ int seq_pages(const Kv4Block& k, int b, int slots) {
    return seq_pages(seq_end(k, kv4_length(k.lengths, b, slots), kv4_count(k.counts, b, k.T), slots));
}

// What all lanes of a wave hold alike, kept in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Quotient of numbers that are not negative, two thirds of the signed one's instructions.
__device__ __forceinline__ int divide(int x, int y) { return (int)((unsigned)x / (unsigned)y); }

// Scan of the sequences' units by a wave, 64 at a time; up to 64 it is kept, with what
// was loaded for it.
struct Scan {
    const Kv4Block& k;
    const Kv4Cache& c;
    int per;                   // row tiles of a sequence
    int n, count, pages;       // context, valid rows and pages of this lane's sequence
    int cum;                   // units of all up to it, in the 64 from b0
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
        const int lane = threadIdx.x & 63, slots = c.slots();
        b0 = b0_, before = before_;
        n = count = pages = 0;
        if (b0 + lane < c.batch) {
            n = kv4_length(k.lengths, b0 + lane, slots);
            count = kv4_count(k.counts, b0 + lane, k.T);
            pages = seq_pages(seq_end(k, n, count, slots));
        }
        cum = sum_upto(pages * per);
    }
    // Sequence of unit u < total, its first unit, its pages, context and valid rows.
    struct Place { int b, start, pages, n, count; };
    __device__ Place of_lane(int l) const {
        const int p = __builtin_amdgcn_readlane(pages, l);
        return {b0 + l, before + __builtin_amdgcn_readlane(cum, l) - p * per, p, __builtin_amdgcn_readlane(n, l),
                __builtin_amdgcn_readlane(count, l)};
    }
    __device__ Place place(int u) {
        if (u < before) seek(0, 0);
        for (;;) {
            const unsigned long long past = __ballot(before + cum > u);
            if (past) {
                return of_lane(__builtin_ctzll(past));
            }
            const int all = __builtin_amdgcn_readlane(cum, 63);
            seek(b0 + 64, before + all);
        }
    }
};

// The line of pages: those of (b, h, tiles of a workgroup) one after the other, b first.
struct Line {
    int tiles;                 // groups of 8 / WAYS row tiles per (b, h)
    int pieces;                // workgroups
    int least;                 // fewest pages of a part of a tile group's pages
};

// How the line is cut into at most `pieces` pieces.
//  * Where it is not much less even, every tile group into parts of its own, as many as
//    its pages call for (at most `most`), a workgroup each: the smallest part for which
//    there are workgroups enough, up to a quarter (and a page a wave) over an even share.
//  * Else every `share` pages; a cut within kSnap pages of where the next tiles begin moves
//    there, so that no piece holds a few pages of some and the rest of others.  A piece
//    over several tile groups begins and joins its waves for each (about 8 us).  So are
//    batches of more than 64 sequences cut, whatever their lengths, and `most` does not
//    hold there: a long sequence among many short ones may lie in as many pieces as its
//    share of the line.
// Attention of 8 x 16 rows over up to 4000 slots: 35 us with even cuts alone, 27 with parts.
struct Cuts {
    static constexpr int kSnap = 8;
    int share;
    int parts, upto;           // of this lane's sequence: parts per tile group; pieces of all up to it
    bool own_parts;

    __device__ Cuts(const Scan& s, const Line& line, int most) {
        // `least` keeps tiles of few pages whole; it gathers no more of them than an even share
        const int groups = s.c.batch * s.per;
        share = max(min(line.least, divide(s.total + groups - 1, groups)), divide(s.total + line.pieces - 1, line.pieces));
        own_parts = false;
        parts = upto = 0;
        if (s.c.batch > 64) return;
        const int step = kKv4Waves * max(1, share / 64);
        for (int part = (share + 7) / 8 * 8; part <= share + share / 4 + kKv4Waves; part += step) {
            parts = min(divide(s.pages + part - 1, part), most);
            upto = sum_upto(parts * s.per);
            own_parts = __builtin_amdgcn_readlane(upto, 63) <= line.pieces;
            if (own_parts) return;
        }
    }
    // Units of a piece: first, past the last; and the place of the first, where it is known.
    __device__ int2 piece(Scan& s, int w, Scan::Place& first) const {
        if (own_parts) {
            const unsigned long long past = __ballot(upto > w);
            if (!past) return {0, 0};
            const int l = __builtin_ctzll(past), n = __builtin_amdgcn_readlane(parts, l);
            const int pages = __builtin_amdgcn_readlane(s.pages, l);
            const int i = w - (__builtin_amdgcn_readlane(upto, l) - n * s.per), ht = divide(i, n), k = i - ht * n;
            first = s.of_lane(l);
            const int at = first.start + ht * pages;
            const int q = divide(pages, n), r = pages - q * n;   // k * pages / n, without its overflow
            return {at + k * q + divide(k * r, n), at + (k + 1) * q + divide((k + 1) * r, n)};
        }
        if ((int64_t)w * share >= s.total) return {0, 0};
        int2 r = {0, 0};
#pragma nounroll
        for (int e = 0; e < 2; ++e) {
            r.x = r.y;
            const int u = (int)min((int64_t)(w + e) * share, (int64_t)s.total);
            r.y = u;
            if (u < s.total) {
                const Scan::Place at = s.place(u);
                const int lo = at.start + divide(u - at.start, at.pages) * at.pages;
                r.y = snap(u, lo, lo + at.pages);
            }
        }
        return r;
    }
    // Pieces that hold the pages lo .. hi - 1 of tile group ht of sequence b: first, past the last.
    __device__ int2 holders(const Scan& s, int b, int ht, int lo, int hi) const {
        if (own_parts) {
            const int n = __builtin_amdgcn_readlane(parts, b);
            const int w = __builtin_amdgcn_readlane(upto, b) - n * s.per + ht * n;
            return {w, w + n};
        }
        // cuts w0 .. w1 - 1 stay inside; the piece before the first has the first pages
        int w0 = (lo + share - 1) / share, w1 = (hi - 1) / share + 1;
        while (w0 < w1 && snap(w0 * share, lo, hi) == lo) ++w0;
        while (w0 < w1 && snap((w1 - 1) * share, lo, hi) == hi) --w1;
        return {w0 - 1, w1};
    }
    // Where the cut at unit u comes to lie; lo, hi: the ends of the tiles that hold it.
    __device__ int snap(int u, int lo, int hi) const {
        const int reach = min(share / 2, kSnap);
        return u - lo <= reach ? lo : hi - u <= reach ? hi : u;
    }
};

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

// f(query type, head size) as types.
template <typename F> hipError_t kv4_by_type(int dtype, int head_dim, F&& f) {
    auto by_size = [&](auto tag) {
        if (head_dim == 64) f(tag, std::integral_constant<int, 64>{});
        else f(tag, std::integral_constant<int, 128>{});
    };
    if (dtype == DELS_DTYPE_BF16) by_size(bf16_t{});
    else by_size(f16_t{});
    return hipGetLastError();
}

}  // namespace dels
