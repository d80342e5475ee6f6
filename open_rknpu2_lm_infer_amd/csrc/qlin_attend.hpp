// Parts that the attention kernels share: exact fp16 codes from the cache's bytes or nibbles, query rows, output rows.
#pragma once

#include "qlin_kv.hpp"
#include "qlin_rows.hpp"

namespace qlin {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr float kNan = __builtin_nanf("");
constexpr float kNegInf = -__builtin_inff();

// P is scaled by 2^kPShift before it is rounded to fp16 (11 bits), so that it stays normal down to
// 2^-22 and non-zero down to 2^-32 of the largest; the factor is in the sum too and cancels.
constexpr float kPShift = 8.0f;

// Two fp16 codes times 2^-9 from bytes i and j of the cache (code + 128) that sel picks from
// (hi, lo): the permuted pair is (b_i, b_j) * 2^-24, both exact; * 2^15 - 128 * 2^-9 is exact.
__device__ __forceinline__ uint32_t codes2(uint32_t hi, uint32_t lo, uint32_t sel) {
    const half2v b = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(hi, lo, sel));
    const half2v m = {(_Float16)32768.0f, (_Float16)32768.0f}, a = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, m, a));
}
// What codes are worth in the matrix core's operands: 2^-9 in 8 bits, and 2^-16 for a code times its unit in 4.
template <int BITS>
constexpr float kCodeUnit = BITS == 8 ? 512.0f : 65536.0f;

// Eight codes of consecutive columns, bytes of (w0, w1).
__device__ __forceinline__ half8v codes8(uint32_t w0, uint32_t w1) {
    const uint4v r = {codes2(w0, w0, 0x0c010c00u), codes2(w0, w0, 0x0c030c02u), codes2(w1, w1, 0x0c010c00u),
                      codes2(w1, w1, 0x0c030c02u)};
    return __builtin_bit_cast(half8v, r);
}

// 4 bits: a nibble (code + 8) in the lowest bits of a half is n * 2^-24, in the next four n * 2^-20.  Times unit * 2^8 or
// unit * 2^4, less unit * 2^-13, either is code * unit * 2^-16: factors and result (up to 7 * 255, 11 bits) are exact in fp16, small
// results as subnormals, which the matrix core takes as they are.  So a unit costs nothing but its factors, and two of the
// four nibbles of a half no shift.
struct Unit2 {
    half2v lo, hi, less;
};
// Units of bytes i and j of w: 0x6400 | u is 1024 + u.
__device__ __forceinline__ Unit2 units2(uint32_t w, int i, int j) {
    const half2v k = {(_Float16)1024.0f, (_Float16)1024.0f}, lo = {(_Float16)256.0f, (_Float16)256.0f},
                 hi = {(_Float16)16.0f, (_Float16)16.0f}, less = {(_Float16)-0x1p-13f, (_Float16)-0x1p-13f};
    const half2v u = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04000400u | (uint32_t)j << 16 | (uint32_t)i)) - k;
    return {u * lo, u * hi, u * less};
}
// Nibbles x of both halves of w.
__device__ __forceinline__ uint32_t nibbles2(uint32_t w, int x, const Unit2& u) {
    const uint32_t y = x < 2 ? w : w >> 8;
    return __builtin_bit_cast(uint32_t, x % 2 ? __builtin_elementwise_fma(__builtin_bit_cast(half2v, y & 0x00f000f0u), u.hi, u.less)
                                              : __builtin_elementwise_fma(__builtin_bit_cast(half2v, y & 0x000f000fu), u.lo, u.less));
}
// Eight codes of consecutive columns of a key, in the order that the halves of a word give them: columns 0 4 1 5 2 6 3 7.
// Queries are laid out alike (operand_column).
__device__ __forceinline__ half8v nibbles8(uint32_t w, const Unit2& u) {
    const uint4v r = {nibbles2(w, 0, u), nibbles2(w, 1, u), nibbles2(w, 2, u), nibbles2(w, 3, u)};
    return __builtin_bit_cast(half8v, r);
}
// Which of eight consecutive columns is element i of a key's operand.
template <int BITS>
__host__ __device__ constexpr int operand_column(int i) {
    return BITS == 8 ? i : i % 2 * 4 + i / 2;
}

// The running maximum of a vector is raised only when a token passes it by more than this (bits): most
// steps leave the output as it is.  P stays at or below 2^(kPShift + kSlack), inside fp16.
constexpr float kSlack = 5.0f;
static_assert(kPShift + kSlack < 16.0f, "P has to stay below fp16's 65504");

// fp16 high part, and with two limbs the rest (exact in fp16 unless it underflows).
template <int LIMBS>
__device__ __forceinline__ void split_f16(float x, _Float16 out[LIMBS]) {
    out[0] = (_Float16)x;
    if constexpr (LIMBS == 2) out[1] = (_Float16)(x - (float)out[0]);
}

// Columns of a query row on their way to the matrix core: KS groups of eight as they lie in memory, RUN of them side by
// side (one load of a key's bytes) at column first and every STEP columns; columns past the
// head's are zeros.  All loads are issued before any is used.
template <int KS, bool Q16>
struct QueryRow {
    uint4v w[KS][Q16 ? 1 : 2];
};
template <int KS, int STEP, int RUN, bool Q16>
__device__ __forceinline__ void load_query(const AttendParams& p, QueryRow<KS, Q16>& r, int64_t at, int first) {
    constexpr int W = Q16 ? 1 : 2;
    auto column = [](int k) { return k / RUN * STEP + k % RUN * 8; };
    if (p.q_vec) {  // heads of whole groups of 8, 16-byte aligned
        const uint8_t* q = reinterpret_cast<const uint8_t*>(p.q) + (at + first) * (2 * W);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const bool in = first + column(k) < p.c.dim;
#pragma unroll
            for (int i = 0; i < W; ++i) r.w[k][i] = *reinterpret_cast<const uint4v*>(q + (in ? column(k) * 2 * W : -first * 2 * W) + 16 * i);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < W; ++i) r.w[k][i] = first + column(k) < p.c.dim ? r.w[k][i] : uint4v{0, 0, 0, 0};
    } else {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4 * W; ++i) {
                const int d = first + column(k) + (Q16 ? 2 * i : i), last = p.c.dim - 1;
                uint32_t x;
                if constexpr (Q16) {
                    const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q) + at;
                    x = (d <= last ? (uint32_t)q[min(d, last)] : 0) | (d < last ? (uint32_t)q[min(d + 1, last)] : 0) << 16;
                } else {
                    x = d <= last ? reinterpret_cast<const uint32_t*>(p.q)[at + d] : 0;
                }
                r.w[k][i / 4][i % 4] = x;
            }
    }
}
// Element i of group k.
template <int KS, bool Q16>
__device__ __forceinline__ float query_at(const QueryRow<KS, Q16>& r, int k, int i) {
    if constexpr (Q16) return (float)__builtin_bit_cast(half8v, r.w[k][0])[i];
    else return __uint_as_float(r.w[k][i / 4][i % 4]);
}

// N consecutive columns of an output row.
template <int N>
__device__ __forceinline__ void store_out(const AttendParams& p, int64_t at, int d0, const float* y) {
    if (p.o_vec && N % 4 == 0) {  // 16-byte aligned heads of whole groups of 8
        if (d0 >= p.c.dim) return;
#pragma unroll
        for (int i = 0; i + 4 <= N; i += 4) {
            if (p.o_f16) {
                typedef _Float16 half4v __attribute__((ext_vector_type(4)));
                const half4v h = {(_Float16)y[i], (_Float16)y[i + 1], (_Float16)y[i + 2], (_Float16)y[i + 3]};
                *reinterpret_cast<half4v*>(reinterpret_cast<_Float16*>(p.o) + at + d0 + i) = h;
            } else {
                *reinterpret_cast<float4v*>(reinterpret_cast<float*>(p.o) + at + d0 + i) = float4v{y[i], y[i + 1], y[i + 2], y[i + 3]};
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (d0 + i >= p.c.dim) continue;
        if (p.o_f16) reinterpret_cast<_Float16*>(p.o)[at + d0 + i] = (_Float16)y[i];
        else reinterpret_cast<float*>(p.o)[at + d0 + i] = y[i];
    }
}

template <int N>
struct Bytes {
    uint32_t w[N / 4];
};

typedef const __attribute__((address_space(4))) int32_t* const_ids;
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

// Where a wave finds 16 tokens: the block of their page and head as a buffer, and the offsets of their keys,
// values, scales and, in 4 bits, of the units of their columns' first group (the next one's are a page's tokens
// further).  An id outside the cache leads to page 0 (bad); a group that is not there is a
// buffer of no bytes, which reads without an access.
template <int DP, int BITS>
struct Half16 {
    __amdgpu_buffer_rsrc_t block;
    int k, v, ks, vs, ku, vu;
    bool bad;
};
template <int DP, int BITS>
__device__ __forceinline__ Half16<DP, BITS> find_half(const KvCache& c, int id, int head, int off, bool there) {
    constexpr int ROW = DP * BITS / 8;
    Half16<DP, BITS> x;
    x.bad = false;
    const int page = kv_page(id, c.pages, &x.bad), values = ROW << c.shift, bytes = (int)kv_block_bytes(BITS, DP, c.shift);
    x.block = __builtin_amdgcn_make_buffer_rsrc(c.data + ((int64_t)page * c.heads + head) * bytes, (short)0,
                                                there ? bytes : 0, 0x00027000);  // raw, 32-bit elements
    x.k = off * ROW;
    x.v = values + off * ROW;
    x.ks = 2 * values + 4 * off;
    x.vs = x.ks + (4 << c.shift);
    x.ku = 2 * values + (8 << c.shift) + off;
    x.vu = x.ku + (DP / kKvGroup << c.shift);
    return x;
}

// N bytes of a buffer, at a lane's offset from `from` on: up to 16 of them, or 16 every STEP.
template <int N, int STEP>
__device__ __forceinline__ void load_bytes(Bytes<N>& r, __amdgpu_buffer_rsrc_t b, int at, int from) {
    if constexpr (N == 4) r.w[0] = __builtin_amdgcn_raw_buffer_load_b32(b, at, from, 0);
    else if constexpr (N == 8) {
        const uint2v x = __builtin_bit_cast(uint2v, __builtin_amdgcn_raw_buffer_load_b64(b, at, from, 0));
        r.w[0] = x[0];
        r.w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            const uint4v x = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(b, at + STEP * i, from, 0));
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * i + j] = x[j];
        }
    }
}

// Sum and maximum over the four lanes n, n + 16, n + 32, n + 48.
template <bool MAX>
__device__ __forceinline__ float over_groups(float x) {
    typedef unsigned int pair __attribute__((ext_vector_type(2)));
    pair r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = MAX ? fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) : __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return MAX ? fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) : __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// What the waves of a workgroup join in: 16 vectors a tile.
template <int DP, int R>
struct AttendLds {
    alignas(16) float o[2][16 * R][DP + 4];  // rows padded: 16 lanes' rows start in different banks
    float m[4][16 * R], l[4][16 * R];
    int seen[16 * R], most;  // SHARED: tokens that each vector sees, the most of them
};
}  // namespace qlin
