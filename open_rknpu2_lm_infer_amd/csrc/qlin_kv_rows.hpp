// Rows on their way into the key/value cache and back: what append, read and the pass from the qkv projection share.
#pragma once

#include <type_traits>

#include "qlin_kv.hpp"
#include "qlin_rows.hpp"

namespace qlin {

// f over the N lanes of a group (2 .. 64, aligned), each step joining halves of twice the lanes: exchanges within four lanes, mirrors of
// eight and of sixteen, then swaps of rows and halves of the wave.  FROM: lanes that agree already.
template <int N, int FROM = 1, typename F>
__device__ __forceinline__ uint32_t over_lanes(uint32_t x, F f) {
    auto dpp = [&](auto ctrl) { return f(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true)); };
    if constexpr (N > 1 && FROM <= 1) x = dpp(std::integral_constant<int, 0xb1>{});   // quad_perm 1 0 3 2
    if constexpr (N > 2 && FROM <= 2) x = dpp(std::integral_constant<int, 0x4e>{});   // quad_perm 2 3 0 1
    if constexpr (N > 4 && FROM <= 4) x = dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
    if constexpr (N > 8 && FROM <= 8) x = dpp(std::integral_constant<int, 0x140>{});  // row_mirror
    typedef unsigned int pair __attribute__((ext_vector_type(2)));
    if constexpr (N > 16 && FROM <= 16) {
        const pair r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(x, x, false, false));
        x = f(r[0], r[1]);
    }
    if constexpr (N > 32 && FROM <= 32) {
        const pair r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(x, x, false, false));
        x = f(r[0], r[1]);
    }
    return x;
}
template <int N, int FROM = 1>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    return over_lanes<N, FROM>(x, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int N>
__device__ __forceinline__ float lanes_sum(float x) {
    return __uint_as_float(over_lanes<N>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

// Quantizes columns d0 .. d0 + 7 of a row, x (zeros past the head), of which DP / 8 lanes hold the rest, and stores
// codes, units and scale of the key (VALUE: the value) of token `off` of the block where `store` says so.  All lanes of
// the row have to call it.  False: the row holds Inf or NaN; its codes are 0 and its scale is NaN.
//   8 bits: s = max(top * (1/127), 2^-64), code = round(x * (1/s))
//   4 bits: s = max(top * (1/1785), 2^-64), u = clamp(ceil(a * (1/s) * (1/7)), 1, 255) with a the largest of 32 columns,
//           code = round(x * (1/(u s)))
// every operation one f32 rounding.  Codes need no clamp to -127 .. 127 and -7 .. 7: |x| <= top (a), and s (u, which is rounded up,
// times s) is at least a 127th (a 7th) of it but for some roundings of 2^-24, so what is rounded passes 127 (7) by 2^-15 at
// most.  (4096 tokens of 8
// heads of 128 in 4 bits: 9.0 us, 23 MB; lane exchanges through the LDS took 0.7 longer.)
template <int DP, int BITS, bool VALUE>
__device__ __forceinline__ bool quantize_row(const KvBlock<DP, BITS>& blk, int off, int d0, const float x[8], bool rne, bool store) {
    uint32_t m = 0;  // largest bit pattern of |x|: for non-negative floats their order, Inf and NaN on top
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    uint32_t a = 0;
    if constexpr (BITS == 4) {
        a = lanes_max<kKvGroup / 8>(m);
        m = lanes_max<DP / 8, kKvGroup / 8>(a);
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
    // codes side by side, sums of shifted ones: each is above zero with what is added to all of them
    uint32_t w[BITS / 4];
#pragma unroll
    for (int i = 0; i < BITS / 4; ++i) w[i] = BITS == 8 ? 0x80808080u : 0x88888888u;
    auto pack = [&](auto even) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = quant_finite<decltype(even)::value>(fin ? x[i] : 0.0f, inv);
            w[BITS == 8 ? i / 4 : 0] += (uint32_t)c << (BITS * (BITS == 8 ? i % 4 : i));
        }
    };
    if (rne) pack(std::true_type{});
    else pack(std::false_type{});
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
