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

// Shapes of a wave's work on RT rows: MT x MT tiles of the matrix instructions.
template <int D, int RT> struct Shape {
    static constexpr int MT = RT == 16 ? 16 : 32;
    static constexpr int NR = RT / MT;              // tiles of rows
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
    static constexpr int STEP = RT == 64 ? 1 : 2;   // 32-slot halves per softmax step
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

// The line of pages: pages of (b, h, row tile) one after the other, b first.
struct Line {
    int tiles;                 // row tiles per (b, h)
    int pieces;                // workgroups
    int min_pages;             // fewest pages of a piece
};

__device__ __forceinline__ int seq_end(const Kv4Block& k, int b, int slots) {
    const int n = kv4_length(k.lengths, b, slots);
    if (k.mode == DELS_KV4_NONE) return n;
    return (int)min((int64_t)slots, (int64_t)n + kv4_count(k.counts, b, k.T));
}
// Pages of sequence b (one at least: rows that see nothing are written too).
__device__ __forceinline__ int seq_pages(const Kv4Block& k, int b, int slots) {
    return max(1, (seq_end(k, b, slots) + kKv4Page - 1) / kKv4Page);
}

// Where unit `u` of the line lies, by all lanes of a wave.
struct Place { int b, start, pages; };          // `start`: first unit of sequence b
__device__ __forceinline__ int line_units(const Kv4Block& k, const Kv4Cache& c, int per) {
    const int lane = threadIdx.x & 63;
    int sum = 0;
    for (int b = lane; b < c.batch; b += 64) sum += seq_pages(k, b, c.slots());
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
    return sum * per;
}
__device__ __forceinline__ Place line_place(const Kv4Block& k, const Kv4Cache& c, int per, int u) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int b0 = 0;; b0 += 64) {
        const int own = b0 + lane < c.batch ? seq_pages(k, b0 + lane, c.slots()) * per : 0;
        int cum = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int o = __shfl_up(cum, off, 64);
            cum += lane >= off ? o : 0;
        }
        const int all = __shfl(cum, 63, 64);
        if (u < before + all || b0 + 64 >= c.batch) {
            const unsigned long long past = __ballot(before + cum > u);
            const int l = past ? __builtin_ctzll(past) : 63;
            return {b0 + l, before + __shfl(cum - own, l, 64), __shfl(own, l, 64) / per};
        }
        before += all;
    }
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
template <int D, int RT> constexpr int kStateFloats = RT * D + 2 * RT;

template <typename T, int D, int RT>
__global__ __launch_bounds__(kAttnThreads, RT == 16 ? 4 : 2) void kv4_attention_kernel(Kv4AttentionArgs a, Line line,
                                                                                      float* __restrict__ states) {
    using S = Shape<D, RT>;
    using F = typename Frag<T>::type;
    constexpr int MT = S::MT, NR = S::NR;
    constexpr int kRegs = S::CT * S::ACC;                   // output registers of a row tile
    constexpr int kRound = 32;                              // registers joined at a time
    __shared__ float s_o[kAttnWaves][kRound][64];
    __shared__ float s_m[kAttnWaves][RT], s_l[kAttnWaves][RT];
    __shared__ F s_q[RT == 64 ? NR * S::KS * 64 : 1];       // queries in operand order (64 rows; else registers)

    const Kv4Cache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane % MT, g = lane / MT;
    const int slots = c.slots(), group = a.q_heads / c.heads, per = c.heads * line.tiles;
    // pieces that follow each other on one XCD: they share pages where a head has several row tiles
    const int piece = (int)gridDim.x % 8 ? (int)blockIdx.x
                                         : (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
    const int units = line_units(a.block, c, per);
    const int share = max(line.min_pages, (units + line.pieces - 1) / line.pieces);
    int u = piece * share;
    const int u_end = min(units, u + share);
    if (u >= u_end) return;
    Place at = line_place(a.block, c, per, u);
    // scores in units of the maximum: |scale| and the query's sign
    const float mag = fabsf(a.scale);
    const float unit = (mag == 0.f ? 1.f : mag) * kLog2e * (float)(1 << kKeyShift<T>);
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, zero = mag == 0.f ? 0u : ~0u;

    while (u < u_end) {
        if (u >= at.start + at.pages * per) at = line_place(a.block, c, per, u);
        const int b = __builtin_amdgcn_readfirstlane(at.b);
        const int rel = u - at.start, ht = rel / at.pages, first = rel - ht * at.pages;
        const int h = ht / line.tiles, rt = ht - h * line.tiles;
        const int last = min(at.pages, first + (u_end - u));
        const int n = kv4_length(a.block.lengths, b, slots), count = kv4_count(a.block.counts, b, a.block.T);
        const int filled = seq_end(a.block, b, slots);       // slots past it may hold anything
        int end = filled;
        if (a.block.mode == DELS_KV4_CAUSAL)                  // no row of the tile sees past its last token
            end = (int)min((int64_t)end, (int64_t)n + (rt * RT + RT - 1) / group + 1);
        const int stop = min(last, (end + kKv4Page - 1) / kKv4Page);

        // rows of this lane: the slots below `lim`, and by mask
        int lim[NR];
        uint64_t bits[NR];
        F q[RT == 64 ? 1 : NR * S::KS];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            const Row row = row_of(rt * RT + nr * MT + col, group, h, a.block.T, count);
            bits[nr] = 0;
            lim[nr] = 0;
            if (row.valid) {
                lim[nr] = a.block.mode == DELS_KV4_CAUSAL ? n + row.t + 1 : a.block.mode == DELS_KV4_FULL ? n + count : n;
                if (a.block.mode == DELS_KV4_MASK)
                    bits[nr] = (uint64_t)a.block.mask[(int64_t)b * a.block.ld_mask + row.t] &
                               (count >= 64 ? ~0ull : (1ull << count) - 1);
            }
            lim[nr] = min(lim[nr], slots);
            const uint16_t* qp = static_cast<const uint16_t*>(a.q.p) + (int64_t)b * a.q.batch +
                                 (int64_t)row.t * a.q.token + (int64_t)row.hq * a.q.head + g * S::DL;
#pragma unroll
            for (int k = 0; k < S::KS; ++k) {
                if (RT == 64 && k % kAttnWaves != wave) continue;
                u32x4 w = {0u, 0u, 0u, 0u};
                if (row.valid) w = *reinterpret_cast<const u32x4*>(qp + 8 * k);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (w[i] ^ flip) & zero;
                if constexpr (RT == 64) s_q[(nr * S::KS + k) * 64 + lane] = __builtin_bit_cast(F, w);
                else q[nr * S::KS + k] = __builtin_bit_cast(F, w);
            }
        }
        if constexpr (RT == 64) __syncthreads();

        typename S::Acc o[NR][S::CT];
        float top[NR], total[NR];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            top[nr] = -__builtin_inff();
            total[nr] = 0.f;
#pragma unroll
            for (int t = 0; t < S::CT; ++t)
#pragma unroll
                for (int i = 0; i < S::ACC; ++i) o[nr][t][i] = 0.f;
        }

        for (int p = first + wave; p < stop; p += kAttnWaves) {
            const uint8_t* page = kv4_page(c, b, h, p, Kv4<D>::kBytes);
            const bool bad = page == nullptr;
            if (bad) continue;
            // ---- loads of the page
            uint32_t kw[2][S::KT][S::KS];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int t = 0; t < S::KT; ++t) {
                    const uint32_t* kp = reinterpret_cast<const uint32_t*>(
                        page + (32 * s + S::slot_of(t, col)) * Kv4<D>::kKeyRow + g * (S::DL / 2));
#pragma unroll
                    for (int k = 0; k < S::KS; ++k) kw[s][t][k] = kp[k];
                }
            uint32_t ks[S::KB];
            {
                const int blk = g * S::DL / 32;
                const int r = S::slot_of(0, col);             // its byte position holds for all tiles but the half
#pragma unroll
                for (int i = 0; i < S::KB; ++i)
                    ks[i] = *reinterpret_cast<const uint32_t*>(page + Kv4<D>::kKeyScale + 64 * (blk + i) +
                                                               16 * ((r >> 3) & 3) + 4 * (r & 3)) >>
                            (8 * ((r >> 2) & 1));
            }
            uint32_t vw[2][S::PF][S::CT];
            u32x4 vs[2][S::PF];
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int f = 0; f < S::PF; ++f) {
                    const int kg = 4 * s + (MT == 16 ? g : 2 * f + g);
                    const uint32_t* vp = reinterpret_cast<const uint32_t*>(page + Kv4<D>::kValue) + kg * D;
#pragma unroll
                    for (int l = 0; l < S::VL; ++l)
#pragma unroll
                        for (int i = 0; i < S::VW; ++i) vw[s][f][l * S::VW + i] = vp[l * MT * S::VW + col * S::VW + i];
                    vs[s][f] = *reinterpret_cast<const u32x4*>(page + Kv4<D>::kValueScale + 16 * kg);
                }
            const bool masked = (p + 1) * kKv4Page > n;
            if (masked) {
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int f = 0; f < S::PF; ++f) {
                        const int j = p * kKv4Page + 32 * s + 8 * (MT == 16 ? g : 2 * f + g);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            vs[s][f][i] &= (j + 2 * i < filled ? 0xffffu : 0u) | (j + 2 * i + 1 < filled ? 0xffff0000u : 0u);
                    }
            }

#pragma unroll
            for (int s0 = 0; s0 < 2; s0 += S::STEP) {
                float x[NR][S::STEP][S::PF][8];
#pragma unroll
                for (int s = 0; s < S::STEP; ++s) {
                    typename S::Acc acc[NR][S::KT];
#pragma unroll
                    for (int t = 0; t < S::KT; ++t) {
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                            for (int i = 0; i < S::ACC; ++i) acc[nr][t][i] = 0.f;
#pragma unroll
                        for (int k = 0; k < S::KS; ++k) {
                            const float sc = key_scale<T>(ks[k * 8 / 32 % S::KB], 2 * (s0 + s) + (MT == 16 ? t : 0));
                            const F kf = decode8<T>(kw[s0 + s][t][k], sc);
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) {
                                if constexpr (RT == 64) acc[nr][t] = mma(kf, s_q[(nr * S::KS + k) * 64 + lane], acc[nr][t]);
                                else acc[nr][t] = mma(kf, q[nr * S::KS + k], acc[nr][t]);
                            }
                        }
                    }
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                        for (int f = 0; f < S::PF; ++f)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                x[nr][s][f][i] = MT == 16 ? acc[nr][i >> 2 & (S::KT - 1)][i & 3]
                                                          : acc[nr][0][(8 * f + i) % S::ACC];
                }
                // slot of x[.][s][f][i]: 64 p + 32 (s0 + s) + 8 kg' + i
                if (masked) {
#pragma unroll
                    for (int nr = 0; nr < NR; ++nr)
#pragma unroll
                        for (int s = 0; s < S::STEP; ++s)
#pragma unroll
                            for (int f = 0; f < S::PF; ++f)
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const int j = p * kKv4Page + 32 * (s0 + s) + 8 * (MT == 16 ? g : 2 * f + g) + i;
                                    const int d = j - n;
                                    const bool by_bit = d >= 0 && d < 64 && ((bits[nr] >> (d & 63)) & 1) && j < slots;
                                    if (!(j < lim[nr] || by_bit)) x[nr][s][f][i] = -__builtin_inff();
                                }
                }
#pragma unroll
                for (int nr = 0; nr < NR; ++nr) {
                    float best = x[nr][0][0][0];
#pragma unroll
                    for (int s = 0; s < S::STEP; ++s)
#pragma unroll
                        for (int f = 0; f < S::PF; ++f)
#pragma unroll
                            for (int i = 0; i < 8; ++i) best = fmaxf(best, x[nr][s][f][i]);
#pragma unroll
                    for (int off = MT; off < 64; off <<= 1) best = fmaxf(best, __shfl_xor(best, off, 64));
                    if (__any((best - top[nr]) * unit > kLag)) {
                        const float now = fmaxf(top[nr], best), f = fade(top[nr] * unit, now * unit);
                        top[nr] = now;
                        total[nr] *= f;
#pragma unroll
                        for (int t = 0; t < S::CT; ++t)
#pragma unroll
                            for (int i = 0; i < S::ACC; ++i) o[nr][t][i] *= f;
                    }
                }
                float ref[NR];
#pragma unroll
                for (int nr = 0; nr < NR; ++nr)
                    ref[nr] = top[nr] == -__builtin_inff() ? 0.f : top[nr] * unit;
#pragma unroll
                for (int s = 0; s < S::STEP; ++s)
#pragma unroll
                    for (int f = 0; f < S::PF; ++f) {
                        bf16x8 hi[NR], lo[NR];
#pragma unroll
                        for (int nr = 0; nr < NR; ++nr) {
                            float sum = 0.f;
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[nr][s][f][i], unit, -ref[nr]));
                                sum += e;
                                const uint32_t w = vs[s0 + s][f][i / 2];
                                const float v = e * __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
                                hi[nr][i] = (__bf16)v;
                                lo[nr][i] = (__bf16)(v - (float)hi[nr][i]);
                            }
                            total[nr] += sum;
                        }
#pragma unroll
                        for (int t = 0; t < S::CT; ++t) {
                            const bf16x8 vf = decode8<bf16_t>(vw[s0 + s][f][t], 1.f);
#pragma unroll
                            for (int nr = 0; nr < NR; ++nr) {
                                o[nr][t] = mma(vf, hi[nr], o[nr][t]);
                                o[nr][t] = mma(vf, lo[nr], o[nr][t]);
                            }
                        }
                    }
            }
        }

        // ---- join the waves
        float ref[NR];
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            ref[nr] = top[nr] * unit;
#pragma unroll
            for (int off = MT; off < 64; off <<= 1) total[nr] += __shfl_xor(total[nr], off, 64);
            if (g == 0) {
                s_m[wave][nr * MT + col] = ref[nr];
                s_l[wave][nr * MT + col] = total[nr];
            }
        }
        __syncthreads();
        const bool whole = first == 0 && last == at.pages;
        float* state = states + (int64_t)(2 * piece + (first == 0 ? 1 : 0)) * kStateFloats<D, RT>;
#pragma unroll
        for (int nr = 0; nr < NR; ++nr) {
            float m = -__builtin_inff(), l = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) m = fmaxf(m, s_m[w][nr * MT + col]);
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) l += s_l[w][nr * MT + col] * fade(s_m[w][nr * MT + col], m);
            const float f = fade(ref[nr], m), inv = l > 0.f ? 1.f / l : 0.f;
            const Row row = row_of(rt * RT + nr * MT + col, group, h, a.block.T, count);
#pragma unroll
            for (int r0 = 0; r0 < kRegs; r0 += kRound) {
                // register (vl, i, v) of the tile: channel block, row of the tile, channel of the VW
#pragma unroll
                for (int j = 0; j < kRound && r0 + j < kRegs; ++j) {
                    const int r = r0 + j, v = r % S::VW, i = r / S::VW % S::ACC, vl = r / S::VW / S::ACC;
                    s_o[wave][j][lane] = o[nr][vl * S::VW + v][i] * f;
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
                    const int gi = r0 / S::VW + jg, i = gi % S::ACC, vl = gi / S::ACC;
                    if (whole) {
                        store_out<T, S::VW>(a, b, row, S::channel_of(vl, i, g), sum, inv);
                    } else {
                        float* to = state + ((nr * (kRegs / S::VW) + gi) * 64 + lane) * S::VW;
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
                    state[RT * D + nr * MT + col] = m;
                    state[RT * D + RT + nr * MT + col] = l;
                }
            }
        }
        __syncthreads();
        u += last - first;
    }
}

// Joins the states of the rows whose pages lie in several pieces: one workgroup
// per (sequence, head, row tile), lanes as in the kernel above.
template <typename T, int D, int RT>
__global__ __launch_bounds__(kAttnThreads) void kv4_join_kernel(Kv4AttentionArgs a, Line line,
                                                                const float* __restrict__ states) {
    using S = Shape<D, RT>;
    constexpr int MT = S::MT, NR = S::NR, kRegs = S::CT * S::ACC;
    const Kv4Cache& c = a.cache;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane % MT, g = lane / MT;
    const int per = c.heads * line.tiles, group = a.q_heads / c.heads;
    const int b = blockIdx.x / per, ht = blockIdx.x % per, h = ht / line.tiles, rt = ht % line.tiles;
    const int units = line_units(a.block, c, per);
    const int share = max(line.min_pages, (units + line.pieces - 1) / line.pieces);
    // units before sequence b
    int before = 0;
    for (int i = lane; i < b; i += 64) before += seq_pages(a.block, i, c.slots());
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) before += __shfl_xor(before, off, 64);
    const int pages = seq_pages(a.block, b, c.slots());
    const int u0 = before * per + ht * pages, u1 = u0 + pages;
    const int w0 = u0 / share, w1 = (u1 - 1) / share;
    if (w0 == w1) return;                                   // one piece covered them and wrote the output
    const int count = kv4_count(a.block.counts, b, a.block.T);
    auto state_of = [&](int w) {
        return states + (int64_t)(2 * w + (w * share <= u0 ? 1 : 0)) * kStateFloats<D, RT>;
    };
#pragma unroll
    for (int nr = 0; nr < NR; ++nr) {
        const int r = nr * MT + col;
        float m = -__builtin_inff(), l = 0.f;
        for (int w = w0; w <= w1; ++w) m = fmaxf(m, state_of(w)[RT * D + r]);
        for (int w = w0; w <= w1; ++w) {
            const float* st = state_of(w);
            l += st[RT * D + RT + r] * fade(st[RT * D + r], m);
        }
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const Row row = row_of(rt * RT + r, group, h, a.block.T, count);
        for (int gi = wave; gi < kRegs / S::VW; gi += kAttnWaves) {
            float sum[S::VW];
#pragma unroll
            for (int v = 0; v < S::VW; ++v) sum[v] = 0.f;
            for (int w = w0; w <= w1; ++w) {
                const float* st = state_of(w);
                const float f = fade(st[RT * D + r], m);
                const float* from = st + ((nr * (kRegs / S::VW) + gi) * 64 + lane) * S::VW;
#pragma unroll
                for (int v = 0; v < S::VW; ++v) sum[v] += from[v] * f;
            }
            store_out<T, S::VW>(a, b, row, S::channel_of(gi / S::ACC, gi % S::ACC, g), sum, inv);
        }
        if (wave == 0 && g == 0) store_lse(a, b, row, m, l);
    }
}

int rows_of(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

struct Plan { int rt; Line line; bool split; };

Plan plan(int64_t batch, int64_t T, int64_t q_heads, int64_t heads, int64_t max_pages) {
    Plan p{};
    const int64_t rows = T * (q_heads / heads);
    p.rt = rows_of(rows);
    p.line.tiles = (int)((rows + p.rt - 1) / p.rt);
    p.line.min_pages = kAttnWaves;
    const int64_t units = batch * heads * p.line.tiles * std::max<int64_t>(max_pages, 1);
    const int64_t slots = (int64_t)device_cu_count() * (p.rt == 16 ? 2 : 1);
    p.line.pieces = (int)std::min<int64_t>(slots, (units + p.line.min_pages - 1) / p.line.min_pages);
    p.split = true;
    return p;
}

template <int RT> size_t state_bytes(int64_t D) { return sizeof(float) * (RT * D + 2 * RT); }

template <typename F> hipError_t by_type(int dtype, int head_dim, int rt, F&& f) {
    auto by_rows = [&](auto tag, auto size) {
        if (rt == 16) f(tag, size, std::integral_constant<int, 16>{});
        else if (rt == 32) f(tag, size, std::integral_constant<int, 32>{});
        else f(tag, size, std::integral_constant<int, 64>{});
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
    return align256((size_t)p.line.pieces * 2 * sizeof(float) * (p.rt * head_dim + 2 * p.rt));
}

hipError_t launch_kv4_attention(const Kv4AttentionArgs& a, void* ws, size_t data_off, hipStream_t s) {
    const Kv4Cache& c = a.cache;
    const Plan p = plan(c.batch, a.block.T, a.q_heads, c.heads, c.max_pages);
    auto* states = reinterpret_cast<float*>(static_cast<char*>(ws) + data_off);
    return by_type(a.dtype, c.head_dim, p.rt, [&](auto tag, auto size, auto rows) {
        using T = decltype(tag);
        constexpr int D = decltype(size)::value, RT = decltype(rows)::value;
        hipLaunchKernelGGL((kv4_attention_kernel<T, D, RT>), dim3(p.line.pieces), dim3(kAttnThreads), 0, s, a, p.line,
                           states);
        hipLaunchKernelGGL((kv4_join_kernel<T, D, RT>), dim3((unsigned)c.batch * c.heads * p.line.tiles),
                           dim3(kAttnThreads), 0, s, a, p.line, states);
    });
}

}  // namespace dels
