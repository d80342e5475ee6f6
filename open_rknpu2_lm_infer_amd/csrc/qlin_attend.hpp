// Parts that the attention kernels share: exact fp16 codes from the cache's bytes, query rows, output rows.
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
constexpr float kCodeUnit = 512.0f;  // 1 / 2^-9

// Eight codes of consecutive columns, bytes of (w0, w1).
__device__ __forceinline__ half8v codes8(uint32_t w0, uint32_t w1) {
    const uint4v r = {codes2(w0, w0, 0x0c010c00u), codes2(w0, w0, 0x0c030c02u), codes2(w1, w1, 0x0c010c00u),
                      codes2(w1, w1, 0x0c030c02u)};
    return __builtin_bit_cast(half8v, r);
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

// Columns of a query row on their way to the matrix core: KS groups of eight as they lie in memory, two
// (PAIR: one 16-byte chunk of a key's bytes) or one at column first and every STEP columns; columns past the
// head's are zeros.  All loads are issued before any is used.
template <int KS, bool Q16>
struct QueryRow {
    uint4v w[KS][Q16 ? 1 : 2];
};
template <int KS, int STEP, bool PAIR, bool Q16>
__device__ __forceinline__ void load_query(const AttendParams& p, QueryRow<KS, Q16>& r, int64_t at, int first) {
    constexpr int W = Q16 ? 1 : 2;
    auto column = [](int k) { return PAIR ? k / 2 * STEP + k % 2 * 8 : k * STEP; };
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
// values and scales.  An id outside the cache leads to page 0 (bad); a group that is not there is a
// buffer of no bytes, which reads without an access.
template <int DP>
struct Half16 {
    __amdgpu_buffer_rsrc_t block;
    int k, v, ks, vs;
    bool bad;
};
template <int DP>
__device__ __forceinline__ Half16<DP> find_half(const KvCache& c, int id, int head, int off, bool there) {
    Half16<DP> x;
    x.bad = false;
    const int page = kv_page(id, c.pages, &x.bad), values = DP << c.shift, bytes = (2 * DP + 8) << c.shift;
    x.block = __builtin_amdgcn_make_buffer_rsrc(c.data + ((int64_t)page * c.heads + head) * bytes, (short)0,
                                                there ? bytes : 0, 0x00027000);  // raw, 32-bit elements
    x.k = off * DP;
    x.v = values + off * DP;
    x.ks = 2 * values + 4 * off;
    x.vs = x.ks + (4 << c.shift);
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

}  // namespace qlin
