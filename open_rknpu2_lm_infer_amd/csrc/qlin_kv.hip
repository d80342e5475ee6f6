// Key/value cache in 8 bits: new rows quantized into their pages, and read back.
//
// A row is the key (or value) of one token and one head, dim values x:
//   s = max(absmax |x| * (1/127), 2^-64),  code = clamp(round(x * (1/s)), -127, 127),
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
// append moves 25 MB in 9.3 us (2.7 TB/s) and the read as much in 6.7 (3.8 TB/s); one token takes them
// 3.1 and 2.6 us, most of it the dependent loads of its place in the batch and in the page table.
#include "qlin_kv.hpp"
#include "qlin_rows.hpp"

namespace qlin {
namespace {

// Unit of work u of a sequence: head h of new row t, its key and its value.
struct Unit {
    KvSeq s;
    int i, t, h;
    bool ok;  // there is such a row
    bool bad;
};

template <int LPU>
__device__ __forceinline__ Unit find_unit(const KvRows& p) {
    constexpr int UPB = 256 / LPU;
    Unit r;
    r.i = p.by_blocks.div(blockIdx.x);
    const int u = p.by_blocks.mod(blockIdx.x) * UPB + threadIdx.x / LPU;
    r.s = kv_seq(p.b.row_start, p.b.length, r.i, p.b.rows, p.b.max_new, p.b.max_len);
    r.t = p.by_heads.div(u);
    r.h = p.by_heads.mod(u);
    r.ok = r.t < r.s.rows;
    r.bad = r.s.bad;
    return r;
}

// The slot of a unit's token: its page (-1: no such token, or a page outside the cache) and place in it.
__device__ __forceinline__ int find_page(const KvRows& p, Unit& u, int* off) {
    const int pos = u.s.len - u.s.rows + u.t;
    *off = pos & ((1 << p.c.shift) - 1);
    if (!u.ok || pos < 0) return -1;
    bool bad = false;
    const int page = kv_page(p.b.table[u.i * p.b.table_ld + (pos >> p.c.shift)], p.c.pages, &bad);
    u.bad |= bad;
    return bad ? -1 : page;
}

template <int DP, typename T, bool VEC>
__global__ __launch_bounds__(256) void kv_append_kernel(KvRows p) {
    constexpr int LPU = DP / 8;
    Unit u = find_unit<LPU>(p);
    const int d0 = (threadIdx.x % LPU) * 8;
    // the rows' loads do not wait for the page's
    float x[2][8] = {};
    if (u.ok) {
        const int64_t row = u.s.row0 + u.t, col = (int64_t)u.h * p.c.dim;
        load8<T, VEC>(reinterpret_cast<const T*>(p.k) + row * p.ldk + col, d0, p.c.dim, x[0]);
        load8<T, VEC>(reinterpret_cast<const T*>(p.v) + row * p.ldv + col, d0, p.c.dim, x[1]);
    }
    // the positions of a sequence whose row starts or length are out of bounds are clamped ones, other tokens' slots
    // on pages that other sequences may read: nothing of it is stored
    int off = 0;
    const int page = u.bad ? -1 : find_page(p, u, &off);
    const KvBlock<DP> blk(p.c, max(page, 0), u.h);
    bool finite = true;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        uint32_t m = 0;  // largest bit pattern of |x|: for non-negative floats their order, Inf and NaN on top
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[y][i]) & 0x7fffffffu);
#pragma unroll
        for (int o = LPU / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
        const bool fin = m < 0x7f800000u;
        const float s = fin ? fmaxf(__uint_as_float(m) * (1.0f / 127.0f), kKvScaleMin) : __uint_as_float(0x7fc00000u);
        const float inv = fin ? 1.0f / s : 0.0f;
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = fin ? x[y][i] : 0.0f;
            const int c = p.rne ? quant_finite<true>(v, inv) : quant_finite<false>(v, inv);
            w[i / 4] |= (uint32_t)(c + 128) << (8 * (i % 4));
        }
        if (page >= 0) {
            *reinterpret_cast<uint2*>((y ? blk.v(off) : blk.k(off)) + d0) = make_uint2(w[0], w[1]);
            if (d0 == 0) *(y ? blk.vs(off) : blk.ks(off)) = s;
            finite &= fin;
        }
    }
    if (u.bad) atomicOr(p.err + kErrBatch, 1u);
    if (!finite) atomicOr(p.err + kErrNonfinite, 1u);
}

template <int DP, typename T, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRows p) {
    constexpr int LPU = DP / 8;
    Unit u = find_unit<LPU>(p);
    const int d0 = (threadIdx.x % LPU) * 8;
    int off;
    const int page = find_page(p, u, &off);
    if (u.bad) atomicOr(p.err + kErrBatch, 1u);
    if (!u.ok) return;
    const KvBlock<DP> blk(p.c, max(page, 0), u.h);
    uint2 w[2] = {make_uint2(0x80808080u, 0x80808080u), make_uint2(0x80808080u, 0x80808080u)};
    // no such token: zeros; a page outside the cache: NaN
    const float none = u.s.len - u.s.rows + u.t < 0 ? 0.0f : __uint_as_float(0x7fc00000u);
    float s[2] = {none, none};
    if (page >= 0) {
        w[0] = *reinterpret_cast<const uint2*>(blk.k(off) + d0);
        w[1] = *reinterpret_cast<const uint2*>(blk.v(off) + d0);
        s[0] = *blk.ks(off);
        s[1] = *blk.vs(off);
    }
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        T* dst = reinterpret_cast<T*>(z ? p.v : p.k) + (u.s.row0 + u.t) * (z ? p.ldv : p.ldk) + (int64_t)u.h * p.c.dim;
        alignas(16) T y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float x = (float)((int)(((i < 4 ? w[z].x : w[z].y) >> (8 * (i % 4))) & 0xffu) - 128) * s[z];
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

__global__ __launch_bounds__(256) void kv_clear_kernel(uint32_t* data, int64_t words, int64_t block_words, int64_t code_words) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += (int64_t)gridDim.x * 256)
        data[i] = i % block_words < code_words ? 0x80808080u : __float_as_uint(kKvScaleMin);
}

template <int DP, typename T, bool VEC>
hipError_t launch_rows(KvRows p, bool append, hipStream_t st) {
    const int64_t per_seq = (int64_t)p.b.max_new * p.c.heads, upb = 256 / (DP / 8);
    p.by_blocks = fast_div((int)((per_seq + upb - 1) / upb));
    p.by_heads = fast_div(p.c.heads);
    const dim3 grid((uint32_t)(p.by_blocks.d * (int64_t)p.b.seqs));
    if (append) kv_append_kernel<DP, T, VEC><<<grid, 256, 0, st>>>(p);
    else kv_read_kernel<DP, T, VEC><<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

template <int DP>
hipError_t launch_dp(const KvRows& p, bool append, hipStream_t st) {
    // 16-byte accesses: every row and head 16-byte aligned, heads of whole groups of 8
    const int per16 = p.f16 ? 8 : 4;
    const bool vec = p.c.dim % 8 == 0 && p.ldk % per16 == 0 && p.ldv % per16 == 0 &&
                     ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0;
    if (p.f16) {
        return vec ? launch_rows<DP, __half, true>(p, append, st) : launch_rows<DP, __half, false>(p, append, st);
    }
    return vec ? launch_rows<DP, float, true>(p, append, st) : launch_rows<DP, float, false>(p, append, st);
}

hipError_t launch_any(const KvRows& p, bool append, hipStream_t st) {
    switch (p.c.dim_padded) {
        case 64: return launch_dp<64>(p, append, st);
        case 128: return launch_dp<128>(p, append, st);
        default: return launch_dp<256>(p, append, st);
    }
}

}  // namespace

hipError_t launch_kv_clear(const KvCache& c, hipStream_t st) {
    const int64_t block = kv_block_bytes(c.dim_padded, c.shift) / 4;
    kv_clear_kernel<<<dim3(4096), 256, 0, st>>>(reinterpret_cast<uint32_t*>(c.data), block * c.heads * c.pages, block,
                                                 ((int64_t)c.dim_padded << c.shift) / 2);
    return hipGetLastError();
}
hipError_t launch_kv_append(const KvRows& p, hipStream_t st) { return launch_any(p, true, st); }
hipError_t launch_kv_read(const KvRows& p, hipStream_t st) { return launch_any(p, false, st); }

}  // namespace qlin
