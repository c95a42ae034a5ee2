// What the matrix-core kernels over a paged key/value cache share, whatever a page holds:
// operand types and products, rows of a block, and the line of all sequences' pages that
// is cut into pieces, one a workgroup.
#pragma once

#include "../../include/dels.h"
#include "dels_device.h"
#include "dels_internal.h"

namespace dels {

constexpr int kLineWaves = 8;          // waves of a workgroup
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kCounterWords = 16;      // words from one arrival counter to the next

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Frag;
template <> struct Frag<bf16_t> { using type = bf16x8; };
template <> struct Frag<f16_t> { using type = f16x8; };

// What all lanes of a wave hold alike, kept in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Quotient of numbers that are not negative, two thirds of the signed one's instructions.
__device__ __forceinline__ int divide(int x, int y) { return (int)((unsigned)x / (unsigned)y); }

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

// Two numbers rounded to bf16, the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

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

// exp2(m - ref), 0 for m = -inf, whatever ref is.
__device__ __forceinline__ float fade(float m, float ref) {
    return m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - ref);
}

// Context length and valid block rows of sequence b, within the table's slots.
__device__ __forceinline__ int paged_length(const int32_t* lengths, int b, int slots) {
    return min(max(lengths[b], 0), slots);
}
__device__ __forceinline__ int paged_count(const int32_t* counts, int b, int T) {
    return counts ? min(max(counts[b], 0), T) : T;
}

// Sum over the lanes up to this one: within rows of 16 lanes, then from row to row.
__device__ __forceinline__ int sum_upto(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);     // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // row_bcast:31 into rows 2 and 3
    return x;
}

// Where a sequence's slots that hold anything end, and its pages (one at least: rows that
// see nothing are written too).
__device__ __forceinline__ int seq_end(const PagedBlock& k, int n, int count, int slots) {
    return k.mode == DELS_KV4_NONE ? n : (int)min((int64_t)slots, (int64_t)n + count);
}
__device__ __forceinline__ int seq_pages(int end) { return max(1, (end + kCachePage - 1) / kCachePage); }
__device__ __forceinline__ int seq_pages(const PagedBlock& k, int b, int slots) {
    return seq_pages(seq_end(k, paged_length(k.lengths, b, slots), paged_count(k.counts, b, k.T), slots));
}

// The sequences of a call whose rows see all slots, for the line of their pages.
struct PagedSeqs {
    const PagedBlock& k;
    const PagedCache& c;
    int batch;
    __device__ PagedSeqs(const PagedBlock& k_, const PagedCache& c_) : k(k_), c(c_), batch(c_.batch) {}
    __device__ int length(int b) const { return paged_length(k.lengths, b, c.slots()); }
    __device__ int count(int b) const { return paged_count(k.counts, b, k.T); }
    __device__ int pages(int n, int count) const { return seq_pages(seq_end(k, n, count, c.slots())); }
};

// Scan of the sequences' units by a wave, 64 at a time; up to 64 it is kept, with what
// was loaded for it.  Seqs says how many sequences there are (batch), and of each its
// context, valid rows and pages: length(b), count(b), pages(n, count).
template <typename Seqs> struct Scan {
    const Seqs& seqs;
    int per;                   // row tiles of a sequence
    int n, count, pages;       // context, valid rows and pages of this lane's sequence
    int cum;                   // units of all up to it, in the 64 from b0
    int b0, before, total;

    __device__ Scan(const Seqs& seqs_, int per_) : seqs(seqs_), per(per_) {
        seek(0, 0);
        total = __builtin_amdgcn_readlane(cum, 63);
        for (int b = 64 + (threadIdx.x & 63), rest = 0; seqs.batch > 64; b += 64) {
            rest += b < seqs.batch ? seqs.pages(seqs.length(b), seqs.count(b)) * per : 0;
            if ((b & ~63) + 64 >= seqs.batch) {
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
        n = count = pages = 0;
        if (b0 + lane < seqs.batch) {
            n = seqs.length(b0 + lane);
            count = seqs.count(b0 + lane);
            pages = seqs.pages(n, count);
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

    template <typename Seqs> __device__ Cuts(const Scan<Seqs>& s, const Line& line, int most) {
        // `least` keeps tiles of few pages whole; it gathers no more of them than an even share
        const int groups = s.seqs.batch * s.per;
        share = max(min(line.least, divide(s.total + groups - 1, groups)),
                    divide(s.total + line.pieces - 1, line.pieces));
        own_parts = false;
        parts = upto = 0;
        if (s.seqs.batch > 64) return;
        const int step = kLineWaves * max(1, share / 64);
        for (int part = (share + 7) / 8 * 8; part <= share + share / 4 + kLineWaves; part += step) {
            parts = min(divide(s.pages + part - 1, part), most);
            upto = sum_upto(parts * s.per);
            own_parts = __builtin_amdgcn_readlane(upto, 63) <= line.pieces;
            if (own_parts) return;
        }
    }
    // Units of a piece: first, past the last; and the place of the first, where it is known.
    template <typename Seqs> __device__ int2 piece(Scan<Seqs>& s, int w, typename Scan<Seqs>::Place& first) const {
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
                const auto at = s.place(u);
                const int lo = at.start + divide(u - at.start, at.pages) * at.pages;
                r.y = snap(u, lo, lo + at.pages);
            }
        }
        return r;
    }
    // Pieces that hold the pages lo .. hi - 1 of tile group ht of sequence b: first, past the last.
    template <typename Seqs> __device__ int2 holders(const Scan<Seqs>& s, int b, int ht, int lo, int hi) const {
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

// ---- states of parts, and who joins them ------------------------------------------
//
// A part of a tile group's pages leaves the state of its MT rows in the workspace: their outputs of D
// channels as the lanes hold them, then each row's reference (a binary logarithm) and sum.  States are
// written and read with device-coherent stores and loads, and every store is waited for before the
// arrival is counted: no cache fences.  The last part to arrive joins all of them in their order, so that
// results do not depend on who that is.

// Floats of a state.
template <int D, int MT> constexpr int kStateFloats = MT * D + 2 * MT;

// N outputs of a lane, its i-th ones.
template <int N> __device__ __forceinline__ void store_state(float* state, int i, int lane, const float* x) {
    auto* to = reinterpret_cast<unsigned long long*>(state + (i * 64 + lane) * N);
#pragma unroll
    for (int v = 0; v < N; v += 2)
        atomic_store_u64(to + v / 2, (unsigned long long)__float_as_uint(x[v + 1]) << 32 | __float_as_uint(x[v]));
}
template <int D, int MT>
__device__ __forceinline__ void store_state_row(float* state, int row, float reference, float sum) {
    auto* to = reinterpret_cast<unsigned int*>(state + MT * D + row);
    atomic_store_u32(to, __float_as_uint(reference));
    atomic_store_u32(to + MT, __float_as_uint(sum));
}

// Counts the arrival of this workgroup, which has one of the parts held.x .. held.y - 1 and has stored its
// state; whether it is the last of them, which leaves the counter at 0.  `flag`: a word of LDS.
__device__ __forceinline__ bool last_to_arrive(unsigned int* counters, int2 held, bool& flag) {
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned int* counter = counters + held.x * kCounterWords;
        const unsigned prev = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        flag = prev == (unsigned)(held.y - held.x) - 1u;
        if (flag) __hip_atomic_exchange(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return flag;
}

// FLIGHT states of parts w0 .. loaded at once, as their loads go to memory: a row's references and sums,
// and of this lane's GROUPS outputs of N each the groups way, way + WAYS, ..
template <int FLIGHT, int D, int MT, int WAYS, int GROUPS, int N> struct LoadedStates {
    static constexpr int kMine = (GROUPS + WAYS - 1) / WAYS;
    float reference[FLIGHT], sum[FLIGHT];
    unsigned long long two[FLIGHT][kMine][N / 2];

    // state_of(w): that of part w; parts past the last one are that again.
    template <typename F>
    __device__ __forceinline__ LoadedStates(int w0, int2 held, int way, int lane, int row, F&& state_of) {
        auto load = [](const float* p) {
            return __uint_as_float(__hip_atomic_load(reinterpret_cast<const unsigned int*>(p), __ATOMIC_RELAXED,
                                                     __HIP_MEMORY_SCOPE_AGENT));
        };
#pragma unroll
        for (int e = 0; e < FLIGHT; ++e) {
            float* state = state_of(min(w0 + e, held.y - 1));
            reference[e] = load(state + MT * D + row);
            sum[e] = load(state + MT * D + MT + row);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                auto* from = reinterpret_cast<unsigned long long*>(
                    state + (min(way + i * WAYS, GROUPS - 1) * 64 + lane) * N);
#pragma unroll
                for (int v = 0; v < N / 2; ++v) two[e][i][v] = atomic_load_u64(from + v);
            }
        }
    }
    __device__ __forceinline__ float output(int e, int i, int v) const {
        return __uint_as_float((uint32_t)(two[e][i][v / 2] >> (32 * (v & 1))));
    }
};

}  // namespace dels
