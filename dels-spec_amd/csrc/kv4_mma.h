// What the matrix-core kernels over the 4-bit key/value cache share: operands made of
// codes, the shapes of a wave's work, and a page's key words.
#pragma once

#include "../../include/dels.h"
#include "kv4.h"

namespace dels {

constexpr int kKv4Waves = kLineWaves;            // waves of a workgroup
constexpr int kKv4Threads = 64 * kKv4Waves;

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
