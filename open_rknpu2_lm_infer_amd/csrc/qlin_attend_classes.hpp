// Attention of very few vectors over the 4-bit key/value cache: up to 16 / C of a KV head (a decoded token's query heads).
//
// The matrix core works on 16 columns whatever there is to work on; qlin_attend_kern.hpp gives each vector one of them, and
// where there are 4 vectors three quarters of its exponents are those of columns that are none.  Here the 16 columns are 16 / C
// vectors times C classes of tokens: column n is vector n % (16 / C), and of the C tiles of 16 tokens that a step
// has, it takes tile n / (16 / C).  The logits of all tiles are computed for all columns and each lane keeps its own
// tile's; a column has a running maximum, sum and output over its tokens, P of a column is zero for the others' tokens, and
// classes are joined as waves are.  Two thirds of what is left for the vector units is making fp16 of the nibbles.
//
// A step's tokens lie in one page (pages of at least 16 C tokens): one id, one buffer, and a lane's scales in one load.
//
// What bounds it, 8 KV heads of 128, 4 query heads each (us, as graph nodes): HBM where there is much to read, 64 sequences of
// 4096 tokens, 302 MB, 62, 4.9 TB/s; below that some 6 a workgroup that are no work of a step but the chain of loads
// before the first (length, page id, bytes) and the join behind the last, and 1.4 a step and wave (one token over 300 tokens 6.7, over
// 32768 in 256 workgroups 12.6 and 3.9 for the join's launch).  64 sequences of up to 4096 tokens 48 where all
// columns' exponents are computed took 61.  Workgroups of 8 waves take 9% longer over 54 batches of 1 to 64 sequences of
// 300 to 32768 tokens, and twice the parts 6%.
#pragma once

#include "qlin_attend.hpp"

namespace qlin {
namespace {

// What a wave loads for a step: lanes as in StepData, for C tiles; scales of a lane's own tile.
template <int DP, int C>
struct ClassStep {
    static constexpr int KB = DP / 8, VB = DP / 16;  // bytes of a key, of two tokens' values
    static constexpr int RUN = KB < 16 ? 2 : 4;      // groups of eight columns side by side
    static constexpr int KU = DP == 256 ? 2 : 1;     // groups of 32 columns of a key's
    Bytes<KB> k[C];
    Bytes<VB> v[C][2];
    float4v ks, vs;
    uint32_t ku[C][KU], vu[C];
};

// x of the lane's own class.
template <int C>
__device__ __forceinline__ float4v own_class(const float4v (&x)[C], int cls) {
    float4v y = x[0];
#pragma unroll
    for (int c = 1; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = cls == c ? x[c][i] : y[i];
    return y;
}

// Largest (sum) over the lanes of a vector's classes: rotations of a row of 16 lanes by 8, then by 4.
template <int C, bool MAX>
__device__ __forceinline__ float over_classes(float x) {
    const float y = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xf, 0xf, true));  // row_ror:8
    x = MAX ? fmaxf(x, y) : x + y;
    if constexpr (C == 4) {
        const float z = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xf, 0xf, true));  // row_ror:4
        x = MAX ? fmaxf(x, z) : x + z;
    }
    return x;
}

// What the waves of a workgroup join in.
template <int DP, int C>
struct ClassLds {
    alignas(16) float o[4][16 / C][DP + 4];
    float m[4][16 / C], l[4][16 / C];
};
template <int DP, int C, bool Q16>
__device__ __forceinline__ void attend_classes(const AttendParams& p, int block, ClassLds<DP, C>& lds) {
    using Step = ClassStep<DP, C>;
    constexpr int ROW = DP / 2, KS = DP / 32, DT = DP / 16, V = 16 / C, TOKENS = 16 * C, QL = Q16 ? 1 : 2, PL = 2;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4, cls = n / V;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // heads fastest, parts slowest (see attend_part), the last ones first: those of long sequences do not come to an end
    // after all others, and those that are empty end at once; one tile of vectors
    const int h = p.by_heads.mod(block);
    const int b = p.by_heads.div(block);
    const int seq = p.by_seqs.mod(b), part = p.parts - p.prefix_parts - 1 - p.by_seqs.div(b);
    const int group = p.group.d;

    const int j0 = p.own_from + part * p.chunk;
    // page ids through the scalar cache: nothing writes them while the kernel runs.  The first step's, where the table has a
    // column for it, does not wait for the sequence's length
    const const_ids table = (const_ids)(uintptr_t)(p.b.table + seq * p.b.table_ld);
    const const_ids prefix = (const_ids)(uintptr_t)p.prefix_pages;
    const int first = j0 + TOKENS * wave;
    const int first_id = first < p.b.max_len ? (first < p.prefix ? prefix : table)[first >> p.c.shift] : 0;
    const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
    if (s.bad && tid == 0) atomicOr(p.err + kErrBatch, 1u);
    const int vectors = s.rows * group;
    if (vectors == 0) return;
    if (part > 0 && j0 >= s.len) return;  // the join knows how many parts there are
    const int cap = min(s.len, j0 + p.chunk);
    const int end = __builtin_amdgcn_readfirstlane(min(cap, kv_visible(s, p.group.div(min(V, vectors) - 1))));
    const int v = n % V, seen = v < vectors ? kv_visible(s, p.group.div(v)) : -1;

    // queries first (columns without a vector take the first row's)
    const int64_t out_row = s.row0 + p.group.div(seen >= 0 ? v : 0);
    const int head = h * group + p.group.mod(seen >= 0 ? v : 0);
    QueryRow<KS, Q16> qr;
    load_query<KS, 32 * Step::RUN, Step::RUN, Q16>(p, qr, out_row * p.ldq + (int64_t)head * p.c.dim, 8 * Step::RUN * g);

    const int off_mask = (1 << p.c.shift) - 1;
    bool bad_page = false, bad = false;  // who sees none of a bad step's tokens keeps its result
    Step d;
    Half16<DP, 4> next;
    auto page_of = [&](int j) {  // end > 0
        const int jj = min(j, end - 1);
        return (jj < p.prefix ? prefix : table)[jj >> p.c.shift];
    };
    auto find_step = [&](int j, int id) {
        next = find_half<DP, 4>(p.c, id, h, j & off_mask, j < end);
        next.bad = next.bad && j < end;
        bad_page |= next.bad;
    };
    auto load_k = [&] {
#pragma unroll
        for (int t = 0; t < C; ++t) {
            load_bytes<Step::KB, 64>(d.k[t], next.block, n * ROW + (Step::KB < 16 ? Step::KB : 16) * g, next.k + 16 * t * ROW);
#pragma unroll
            for (int c = 0; c < Step::KU; ++c)
                d.ku[t][c] = __builtin_amdgcn_raw_buffer_load_b8(next.block, n + (((DP == 64 ? g / 2 : g) + 4 * c) << p.c.shift), next.ku + 16 * t, 0);
        }
    };
    auto load_scales = [&] {
        bad = next.bad;
        const int at = 64 * cls + 16 * g;
        d.ks = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(next.block, at, next.ks, 0));
        d.vs = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(next.block, at, next.vs, 0));
    };
    auto load_v = [&] {
#pragma unroll
        for (int t = 0; t < C; ++t) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                load_bytes<Step::VB, 16>(d.v[t][i], next.block, (4 * g + 2 * i) * ROW + n * Step::VB, next.v + 16 * t * ROW);
            d.vu[t] = __builtin_amdgcn_raw_buffer_load_b32(next.block, 4 * g + (n * DT / kKvGroup << p.c.shift), next.vu + 16 * t, 0);
        }
    };
    int j = first;
    if (end > 0) {
        find_step(j, first_id);
        load_k();
        load_scales();
        load_v();
    }

    // queries, as the B operand: lane (n, g) holds the columns of its vector that it holds of a key
    half8v qf[KS][QL];
    float unit = p.scale2 * kCodeUnit<4>;  // what the f16 operands were divided by, times scale2
    {
        float x[DP / 4], up = 1.0f;
#pragma unroll
        for (int i = 0; i < DP / 4; ++i) x[i] = query_at<KS, Q16>(qr, i / 8, i % 8);
        if constexpr (QL == 2) {
            // the row's largest value goes to [2^13, 2^14): the low parts stay normal, f32 rows of any size fit
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 4; ++i) m = fmaxf(m, fabsf(x[i]));
            m = over_groups<true>(m);
            const int e = kv_clamp((int)((__float_as_uint(m) >> 23) & 0xff) - 127, -100, 126);
            up = __uint_as_float((uint32_t)(13 - e + 127) << 23);  // 2^(13 - e)
            unit *= __uint_as_float((uint32_t)(e - 13 + 127) << 23);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 y[QL];
                split_f16<QL>(x[8 * k + operand_column<4>(i)] * up, y);
#pragma unroll
                for (int q = 0; q < QL; ++q) qf[k][q][i] = y[q];
            }
    }

    float m = kNegInf, l = 0.0f;
    float4v o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};

    // The next step's bytes are loaded over this one's as those are used (see attend_part).
    for (; j < end; j += 4 * TOKENS) {
        find_step(j + 4 * TOKENS, page_of(j + 4 * TOKENS));
        float4v sc[C];
#pragma unroll
        for (int t = 0; t < C; ++t) {
            sc[t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const half8v a = nibbles8(d.k[t].w[k], units2(d.ku[t][k / 4], 0, 0));
#pragma unroll
                for (int q = 0; q < QL; ++q) sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[k][q], sc[t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k();
        // tokens 16 cls + 4 g + i
        const float4v x0 = own_class<C>(sc, cls);
        const int left = min(seen, cap) - j - 16 * cls - 4 * g;
        float x[4], iv[4], top = kNegInf;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float lv = bad ? kNan : __builtin_amdgcn_logf(d.vs[i]);
            iv[i] = __builtin_amdgcn_rcpf(d.vs[i]);
            const float y = __builtin_fmaf(x0[i] * unit, d.ks[i], lv);
            // masked tokens are chosen away, whatever their scales hold
            x[i] = i < left ? y : kNegInf;
            top = fmaxf(top, x[i]);
        }
        top = over_groups<true>(top);
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {
            const float m_new = fmaxf(m, top);
            const float fade = m == m_new ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= fade;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= fade;
        }
        const float base = m == kNegInf ? 0.0f : m - kPShift;
        uint32_t pw[PL][2];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const float2v e = {__builtin_amdgcn_exp2f(x[i] - base), __builtin_amdgcn_exp2f(x[i + 1] - base)};
#pragma unroll
            for (int c = 0; c < 2; ++c) l = i + c < left ? __builtin_fmaf(e[c], iv[i + c], l) : l;
            const half2v y = __builtin_convertvector(e, half2v);
            const half2v z = __builtin_convertvector(e - __builtin_convertvector(y, float2v), half2v);
            pw[0][i / 2] = __builtin_bit_cast(uint32_t, y);
            pw[1][i / 2] = __builtin_bit_cast(uint32_t, z);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_scales();
        // O^T: columns n * DT + t (row n of the operand) over tokens 4 g + i of two tiles; P of the lane's own tile alone
#pragma unroll
        for (int pair = 0; pair < C / 2; ++pair) {
            half8v pf[PL];
#pragma unroll
            for (int q = 0; q < PL; ++q) {
                uint4v w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = cls == 2 * pair + i / 2 ? pw[q][i % 2] : 0;
                pf[q] = __builtin_bit_cast(half8v, w);
            }
            Unit2 vu[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) vu[i] = units2(d.vu[2 * pair + i / 2], i % 2 * 2, i % 2 * 2 + 1);
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                uint4v w;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = nibbles2(d.v[2 * pair + i / 2][i % 2].w[t / 4], t % 4, vu[i]);
                const half8v a = __builtin_bit_cast(half8v, w);
#pragma unroll
                for (int q = 0; q < PL; ++q) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf[q], o[t], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v();
    }
    if (bad_page && lane == 0) atomicOr(p.err + kErrBatch, 1u);

    // Join: the classes in the lanes of a row of 16, then the waves in the LDS, where a thread takes NC columns of a vector.
    l = over_groups<false>(l);
    const float m_wave = over_classes<C, true>(m);
    const float fade = m_wave == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - m_wave);
    l = over_classes<C, false>(l * fade);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = over_classes<C, false>(o[t][i] * fade);
    if (cls == 0) {
        // columns (4 g + i) * DT + t of a vector
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < DT; u += 4)
                *reinterpret_cast<float4v*>(&lds.o[wave][v][(4 * g + i) * DT + u]) = float4v{o[u][i], o[u + 1][i], o[u + 2][i], o[u + 3][i]};
        if (g == 0) {
            lds.m[wave][v] = m_wave;
            lds.l[wave][v] = l;
        }
    }
    __syncthreads();
    constexpr int NC = V * DP / 256;
    const int vec = tid / (DP / NC), d0 = tid % (DP / NC) * NC;
    if (vec >= vectors) return;
    float w[4], m_all = kNegInf, l_all = 0.0f, y[NC] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) m_all = fmaxf(m_all, lds.m[i][vec]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = m_all == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(lds.m[i][vec] - m_all);
        l_all = __builtin_fmaf(w[i], lds.l[i][vec], l_all);
#pragma unroll
        for (int c = 0; c < NC; ++c) y[c] = __builtin_fmaf(w[i], lds.o[i][vec][d0 + c], y[c]);
    }
    const int64_t row = s.row0 + p.group.div(vec);
    const int at = h * group + p.group.mod(vec);
    if (p.parts == 1) {
        const float f = l_all == 0.0f ? 0.0f : kCodeUnit<4> / l_all;
#pragma unroll
        for (int c = 0; c < NC; ++c) y[c] *= f;
        store_out<NC>(p, row * p.ldo + (int64_t)at * p.c.dim, d0, y);
    } else {
        const int64_t slot = (row * p.q_heads + at) * p.parts + p.prefix_parts + part;
#pragma unroll
        for (int c = 0; c < NC; ++c) p.part_o[slot * DP + d0 + c] = y[c];
        if (d0 == 0) {
            p.part_ml[2 * slot] = m_all;
            p.part_ml[2 * slot + 1] = l_all;
        }
    }
}

// A launch of them without a prefix.
template <int DP, int C, bool Q16>
__global__ __launch_bounds__(256) void attend_classes_kernel(AttendParams p) {
    __shared__ ClassLds<DP, C> lds;
    attend_classes<DP, C, Q16>(p, blockIdx.x, lds);
}

}  // namespace
}  // namespace qlin
