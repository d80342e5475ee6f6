// Key/value cache in 8 and 4 bits: new rows quantized into their pages, and read back.
//
// A row is the key (or value) of one token and one head, dim values x; the rules are at quantize_row.  In 8 bits it is
//   s = max(absmax |x| * (1/127), 2^-64),  code = round(x * (1/s)),
// every operation one f32 rounding, 1/127 the f32 nearest to it.  That is the rule of the per-token
// activation quantization but for its division by 127, whose place a multiplication takes: the
// scales agree to one step of f32.  A row that holds
// Inf or NaN gets codes 0 and the scale NaN: whoever reads it gets NaN, and the error word says so.
//
// Both kernels move their bytes once and do a few operations a value, so memory bounds them (and
// the launch, for a few tokens).  A group of dim_padded / 8 lanes holds a row, 8 values a lane: 16 bytes of
// fp16 in, 8 bytes of codes out, and the absmax is a few lane exchanges.  One row a group and many
// workgroups: two or four rows a group, their loads in flight together, are slower (both kernels over
// 4096 tokens of 8 heads of 128: 15.9 us with one, 16.3 with two, 19.2 with four).  At that size the
// append moves 25 MB in 8.8 us (2.9 TB/s) and the read as much in 6.7 (3.8 TB/s); one token takes them
// 3.1 and 2.6 us, most of it the dependent loads of its place in the batch and in the page table.
#include "qlin_kv_rows.hpp"

namespace qlin {
namespace {

// Unit of work u of a sequence: head h of new row t, its key and its value.
struct Unit {
    KvSeq s;
    int i, t, h;
    bool ok;  // there is such a row
    bool bad;
    bool none;  // no unit of the workgroup has a row
};

template <int LPU>
__device__ __forceinline__ Unit find_unit(const KvRows& p) {
    constexpr int UPB = 256 / LPU;
    Unit r;
    r.i = p.by_blocks.div(blockIdx.x);
    const int first = p.by_blocks.mod(blockIdx.x) * UPB, u = first + threadIdx.x / LPU;
    r.s = kv_seq(p.b.row_start, p.b.length, r.i, p.b.rows, p.b.max_new, p.b.max_len);
    r.t = p.by_heads.div(u);
    r.h = p.by_heads.mod(u);
    r.ok = r.t < r.s.rows;
    r.bad = r.s.bad;
    r.none = first >= r.s.rows * p.c.heads;
    return r;
}

// A workgroup without a row, as a sequence of fewer than max_new rows has them, ends here: of a prompt of 512 tokens among 63
// decoded tokens 98 of 100 are such.  The rows' addresses wait for what decides it as they are.  (That batch, 8 heads of 128: stored
// in 9.7 us, and in 23.4 where they load and quantize a row to no purpose; read in 8.9 and 9.8.)
__device__ __forceinline__ bool leave(const KvRows& p, const Unit& u) {
    if (!u.none) return false;
    if (u.bad && threadIdx.x == 0) atomicOr(p.err + kErrBatch, 1u);
    return true;
}

// The table's entry for a unit's token (of none: some entry, or a length where the table may have none).
__device__ __forceinline__ int load_id(const KvRows& p, const Unit& u) {
    const int pos = kv_clamp(u.s.len - u.s.rows + u.t, 0, max(p.b.max_len - 1, 0));
    const int32_t* at = p.b.max_len > 0 ? p.b.table + (u.i * p.b.table_ld + (pos >> p.c.shift)) : p.b.length;
    return *at;
}
// The slot of a unit's token: its page (-1: no such token, or a page outside the cache) and place in it.
__device__ __forceinline__ int find_page(const KvRows& p, Unit& u, int id, int* off) {
    const int pos = u.s.len - u.s.rows + u.t;
    *off = pos & ((1 << p.c.shift) - 1);
    if (!u.ok || pos < 0) return -1;
    bool bad = false;
    const int page = kv_page(id, p.c.pages, &bad);
    u.bad |= bad;
    return bad ? -1 : page;
}

// Columns d0 .. d0 + 7 of a row as they lie in memory (past the head: of its last columns).
template <typename T, bool VEC>
struct RawRow {
    uint4 w[sizeof(T) / 2];  // VEC
    uint32_t x[VEC ? 1 : 8];
};
template <typename T, bool VEC>
__device__ __forceinline__ void load_raw(RawRow<T, VEC>& r, const T* row, int d0, int dim) {
    if constexpr (VEC) {
        const uint4* at = reinterpret_cast<const uint4*>(row + (d0 < dim ? d0 : 0));
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = at[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = min(d0 + i, dim - 1);
            if constexpr (sizeof(T) == 2) r.x[i] = reinterpret_cast<const uint16_t*>(row)[d];
            else r.x[i] = reinterpret_cast<const uint32_t*>(row)[d];
        }
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ float raw_value(const RawRow<T, VEC>& r, int i) {
    if constexpr (!VEC) {
        if constexpr (sizeof(T) == 2) return f32_of_f16_bits(r.x[i]);
        else return __uint_as_float(r.x[i]);
    } else {
        const uint4& w = r.w[sizeof(T) == 2 ? 0 : i / 4];
        const int word = sizeof(T) == 2 ? i / 2 : i % 4;
        const uint32_t y = word == 0 ? w.x : word == 1 ? w.y : word == 2 ? w.z : w.w;
        if constexpr (sizeof(T) == 2) return f32_of_f16_bits(y >> (16 * (i % 2)));
        else return __uint_as_float(y);
    }
}

template <int DP, int BITS, typename T, bool VEC>
__global__ __launch_bounds__(256) void kv_append_kernel(KvRows p) {
    constexpr int LPU = DP / 8;
    Unit u = find_unit<LPU>(p);
    if (leave(p, u)) return;
    const int d0 = (threadIdx.x % LPU) * 8;
    // the page's id, the key and the value are on their way together: no branch of a part of the lanes before any is there.
    // (One after the other 4096 tokens of 8 heads of 128 took 9.6 us in 4 bits.)
    const int id = load_id(p, u);
    const int64_t row = u.ok ? u.s.row0 + u.t : 0, col = (int64_t)u.h * p.c.dim;
    RawRow<T, VEC> raw[2];
    load_raw<T, VEC>(raw[0], reinterpret_cast<const T*>(p.k) + row * p.ldk + col, d0, p.c.dim);
    load_raw<T, VEC>(raw[1], reinterpret_cast<const T*>(p.v) + row * p.ldv + col, d0, p.c.dim);
    float x[2][8];
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[y][i] = u.ok && d0 + i < p.c.dim ? raw_value<T, VEC>(raw[y], i) : 0.0f;
    // the positions of a sequence whose row starts or length are out of bounds are clamped ones, other tokens' slots
    // on pages that other sequences may read: nothing of it is stored
    int off = 0;
    const int page = u.bad ? -1 : find_page(p, u, id, &off);
    const KvBlock<DP, BITS> blk(p.c, max(page, 0), u.h);
    const bool k = quantize_row<DP, BITS, false>(blk, off, d0, x[0], p.rne, page >= 0);
    const bool v = quantize_row<DP, BITS, true>(blk, off, d0, x[1], p.rne, page >= 0);
    const bool finite = page < 0 || (k && v);
    if (u.bad) atomicOr(p.err + kErrBatch, 1u);
    if (!finite) atomicOr(p.err + kErrNonfinite, 1u);
}

template <int DP, int BITS, typename T, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRows p) {
    constexpr int LPU = DP / 8;
    Unit u = find_unit<LPU>(p);
    if (leave(p, u)) return;
    const int d0 = (threadIdx.x % LPU) * 8;
    int off;
    const int page = find_page(p, u, load_id(p, u), &off);
    if (u.bad) atomicOr(p.err + kErrBatch, 1u);
    if (!u.ok) return;
    const KvBlock<DP, BITS> blk(p.c, max(page, 0), u.h);
    constexpr uint32_t zero = BITS == 8 ? 0x80808080u : 0x88888888u;
    uint2 w[2] = {make_uint2(zero, zero), make_uint2(zero, zero)};
    // no such token: zeros; a page outside the cache: NaN
    const float none = u.s.len - u.s.rows + u.t < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
    float s[2] = {none, none};
    int unit[2] = {1, 1};
    if (page >= 0) {
        if constexpr (BITS == 8) {
            w[0] = *reinterpret_cast<const uint2*>(blk.k(off) + d0);
            w[1] = *reinterpret_cast<const uint2*>(blk.v(off) + d0);
        } else {
            w[0].x = *reinterpret_cast<const uint32_t*>(blk.k(off) + d0 / 2);
            const uint16_t* v = blk.v4(d0 / 4, off);
            w[1].x = v[0] | (uint32_t)v[2] << 16;
            unit[0] = *blk.ku(d0 / kKvGroup, off);
            unit[1] = *blk.vu(d0 / kKvGroup, off);
        }
        s[0] = *blk.ks(off);
        s[1] = *blk.vs(off);
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        T* dst = reinterpret_cast<T*>(z ? p.v : p.k) + (u.s.row0 + u.t) * (z ? p.ldv : p.ldk) + (int64_t)u.h * p.c.dim;
        alignas(16) T y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int c;
            if constexpr (BITS == 8) c = (int)(((i < 4 ? w[z].x : w[z].y) >> (8 * (i % 4))) & 0xffu) - 128;
            else c = ((int)((w[z].x >> (4 * i)) & 0xfu) - 8) * unit[z];
            const float x = (float)c * s[z];
            if constexpr (sizeof(T) == 2) y[i] = __builtin_bit_cast(T, f16_of_f32(x));
            else y[i] = x;
        }
        if constexpr (VEC) {
            if (d0 < p.c.dim) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                    reinterpret_cast<uint4*>(dst + d0)[i] = reinterpret_cast<const uint4*>(y)[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d0 + i < p.c.dim) dst[d0 + i] = y[i];
        }
    }
}

// Words of a block: codes, then scales, then (4 bits) units.
__global__ __launch_bounds__(256) void kv_clear_kernel(uint32_t* data, int64_t words, int64_t block_words, int64_t code_words,
                                                       int64_t scale_words, uint32_t zero) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256) {
        const int64_t at = i % block_words;
        data[i] = at < code_words ? zero : at < code_words + scale_words ? __float_as_uint(kKvScaleMin) : 0x01010101u;
    }
}

template <int DP, int BITS, typename T, bool VEC>
hipError_t launch_rows(KvRows p, bool append, hipStream_t st) {
    const int64_t per_seq = (int64_t)p.b.max_new * p.c.heads, upb = 256 / (DP / 8);
    p.by_blocks = fast_div((int)((per_seq + upb - 1) / upb));
    p.by_heads = fast_div(p.c.heads);
    const dim3 grid((uint32_t)(p.by_blocks.d * (int64_t)p.b.seqs));
    if (append) kv_append_kernel<DP, BITS, T, VEC><<<grid, 256, 0, st>>>(p);
    else kv_read_kernel<DP, BITS, T, VEC><<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

template <int DP, int BITS>
hipError_t launch_dp(const KvRows& p, bool append, hipStream_t st) {
    // 16-byte accesses: every row and head 16-byte aligned, heads of whole groups of 8
    const int per16 = p.f16 ? 8 : 4;
    const bool vec = p.c.dim % 8 == 0 && p.ldk % per16 == 0 && p.ldv % per16 == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0;
    if (p.f16) {
        return vec ? launch_rows<DP, BITS, __half, true>(p, append, st) : launch_rows<DP, BITS, __half, false>(p, append, st);
    }
    return vec ? launch_rows<DP, BITS, float, true>(p, append, st) : launch_rows<DP, BITS, float, false>(p, append, st);
}

template <int BITS>
hipError_t launch_bits(const KvRows& p, bool append, hipStream_t st) {
    switch (p.c.dim_padded) {
        case 64: return launch_dp<64, BITS>(p, append, st);
        case 128: return launch_dp<128, BITS>(p, append, st);
        default: return launch_dp<256, BITS>(p, append, st);
    }
}

hipError_t launch_any(const KvRows& p, bool append, hipStream_t st) {
    return p.c.bits == 4 ? launch_bits<4>(p, append, st) : launch_bits<8>(p, append, st);
}

}  // namespace

hipError_t launch_kv_clear(const KvCache& c, hipStream_t st) {
    const int64_t block = kv_block_bytes(c.bits, c.dim_padded, c.shift) / 4;
    kv_clear_kernel<<<dim3(4096), 256, 0, st>>>(reinterpret_cast<uint32_t*>(c.data), block * c.heads * c.pages, block,
                                                ((int64_t)c.dim_padded * c.bits << c.shift) / 16, (int64_t)2 << c.shift,
                                                c.bits == 4 ? 0x88888888u : 0x80808080u);
    return hipGetLastError();
}
hipError_t launch_kv_append(const KvRows& p, hipStream_t st) { return launch_any(p, true, st); }
hipError_t launch_kv_read(const KvRows& p, hipStream_t st) { return launch_any(p, false, st); }

}  // namespace qlin
