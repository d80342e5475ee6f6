// Rows on their way into the key/value cache and back: what append, read and the pass from the qkv projection share.
#pragma once

#include "qlin_kv.hpp"
#include "qlin_rows.hpp"

namespace qlin {

// Largest of a value over the 2, 4 .. N lanes of a group.
template <int N>
__device__ __forceinline__ uint32_t lanes_max(uint32_t m, int from = 1) {
#pragma unroll
    for (int o = 1; o < N; o <<= 1)
        if (o >= from) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    return m;
}

// Quantizes columns d0 .. d0 + 7 of a row, x (zeros past the head), of which DP / 8 lanes hold the rest, and stores
// codes, units and scale of the key (VALUE: the value) of token `off` of the block where `store` says so.  All lanes of
// the row have to call it.  False: the row holds Inf or NaN; its codes are 0 and its scale is NaN.
//   8 bits: s = max(top * (1/127), 2^-64), code = clamp(round(x * (1/s)), -127, 127)
//   4 bits: s = max(top * (1/1785), 2^-64), u = clamp(ceil(a * (1/s) * (1/7)), 1, 255) with a the largest of 32 columns,
//           code = clamp(round(x * (1/(u s))), -7, 7)
// every operation one f32 rounding.  u is rounded up, so that no code passes 7 by more than the roundings.
template <int DP, int BITS, bool VALUE>
__device__ __forceinline__ bool quantize_row(const KvBlock<DP, BITS>& blk, int off, int d0, const float x[8], bool rne, bool store) {
    uint32_t m = 0;  // largest bit pattern of |x|: for non-negative floats their order, Inf and NaN on top
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    uint32_t a = 0;
    if constexpr (BITS == 4) {
        a = lanes_max<kKvGroup / 8>(m);
        m = lanes_max<DP / 8>(a, kKvGroup / 8);
    } else {
        m = lanes_max<DP / 8>(m);
    }
    const bool fin = m < 0x7f800000u;
    float s = fin ? fmaxf(__uint_as_float(m) * (BITS == 8 ? 1.0f / 127.0f : 1.0f / 1785.0f), kKvScaleMin) : __uint_as_float(0x7fc00000u);
    float inv = fin ? 1.0f / s : 0.0f, u = 1.0f;
    if constexpr (BITS == 4) {
        if (fin) {
            u = fminf(fmaxf(ceilf((__uint_as_float(a) * inv) * (1.0f / 7.0f)), 1.0f), 255.0f);
            inv = 1.0f / (u * s);
        }
    }
    uint32_t w[BITS / 4] = {};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = fin ? x[i] : 0.0f;
        const int c = rne ? quant_finite<true>(v, inv) : quant_finite<false>(v, inv);
        if constexpr (BITS == 8) w[i / 4] |= (uint32_t)(c + 128) << (8 * (i % 4));
        else w[0] |= (uint32_t)(c + 8) << (4 * i);
    }
    if (store) {
        uint8_t* row = VALUE ? blk.v(off) : blk.k(off);
        if constexpr (BITS == 8) {
            *reinterpret_cast<uint2*>(row + d0) = make_uint2(w[0], w[1]);
        } else {
            if constexpr (VALUE) {
                uint16_t* v = blk.v4(d0 / 4, off);
                v[0] = (uint16_t)w[0];
                v[2] = (uint16_t)(w[0] >> 16);
            } else {
                *reinterpret_cast<uint32_t*>(row + d0 / 2) = w[0];
            }
            if (d0 % kKvGroup == 0) *(VALUE ? blk.vu(d0 / kKvGroup, off) : blk.ku(d0 / kKvGroup, off)) = (uint8_t)u;
        }
        if (d0 == 0) *(VALUE ? blk.vs(off) : blk.ks(off)) = s;
    }
    return fin;
}

}  // namespace qlin
