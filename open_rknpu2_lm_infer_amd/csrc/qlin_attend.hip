// Attention of new rows over the 8-bit key/value cache.
//
//   l_j = scale * s^K_j * (q . k_j)          j = the tokens a row sees (itself and before)
//   o   = sum_j e^(l_j) s^V_j v_j / sum_j e^(l_j),   no token: 0
//
// in one pass over the tokens with a running maximum.  Codes are exact in fp16, so q . k_j runs on
// the matrix cores (f32 sums) without any rounding of the keys, and the value scale goes into the
// probabilities: with l'_j = l_j log2 e + log2 s^V_j and m the running maximum of l',
// P_j = 2^(l'_j - m) multiplies the codes v_j, and the sum of e^(l_j) is sum_j P_j / s^V_j.
// Taking the maximum over l' and not l keeps P inside fp16's range whatever the scales are: m lags the largest l' by
// at most kSlack, so P_j <= 2^kSlack, and 2^(kPShift + kSlack) as the matrix core gets it.
//
// A query row and head is a "vector"; the q_heads / kv_heads vectors of each row that share a KV
// head, and the rows of a sequence, are worked on together, 16 to a tile.  Products are computed
// transposed, S^T = K Q^T and O^T = V^T P^T: then the matrix core's result layout (a lane holds
// four consecutive tokens of one vector) is the operand layout of the second product with its k
// axis permuted, and P never leaves its lane.
//
// What bounds it, 8 KV heads of 128, 4 query heads each: with few rows a token's bytes, 2 * 128 + 8 a head (64
// sequences of up to 4096 tokens, 263 MB: 65 us, 4.1 TB/s; one of 32768, 69 MB in 32 parts of 1024, 256 workgroups: 13.9
// us, 5 TB/s, and 4.6 us for the join), with one short sequence the chain of dependent loads, steps and the
// waves' join (300 tokens: 7.8 us).  A prefix of 8192 tokens for 32 rows, 128 vectors a KV head in tiles of 32, takes 21.7 us
// with the rows' own tokens: the vector units' exponents and byte permutes (31% of their time) and waits (42%), with
// one wave a SIMD.
#include "qlin_attend.hpp"

namespace qlin {
namespace {

// What a wave loads for one step of 32 tokens: two tiles of 16.  Lane l (n = l % 16, g = l / 16)
// holds, as the matrix core's A operand, columns 64 c + 16 g .. + 15 of key n of each tile (a load covers 64
// bytes of each of 16 keys), and columns n * DP/16 .. + DP/16 - 1 of values 4g .. 4g + 3 of each tile.
template <int DP>
struct StepData {
    Bytes<DP / 4> k[2];
    Bytes<DP / 16> v[8];
    float4v ks[2], vs[2];  // scales of tokens 4g .. 4g + 3
};

// Sum and maximum over the four lanes n, n + 16, n + 32, n + 48.
template <bool MAX>
__device__ __forceinline__ float over_groups(float x) {
    typedef unsigned int pair __attribute__((ext_vector_type(2)));
    pair r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    x = MAX ? fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) : __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return MAX ? fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) : __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Workgroup: 4 waves, R tiles of 16 vectors of one KV head, one part of the tokens.  The waves take
// steps of 32 tokens in turn, each with a running maximum, sum and output of its own, and join
// them at the end: nothing is shared before that.
// P goes to the matrix core as a sum of two fp16 values, 22 bits, so that an fp16 output is off by its own rounding
// alone, 2.1e-4 of it (2.6e-4 and 2.8e-4 with P rounded to one fp16 value, in 7.2, 56.4 and 24.4 us for one token at 300, 64
// sequences of up to 4096 and a prefix of 8192 for 32 rows, against 7.4, 56.8 and 26.0).  f32 queries are such sums
// too; fp16 ones are exact.
// SHARED: the part of the prefix, for the rows of all sequences at once.
template <int DP, int R>
struct AttendLds {
    alignas(16) float o[2][16 * R][DP + 4];  // rows padded: 16 lanes' rows start in different banks
    float m[4][16 * R], l[4][16 * R];
    int seen[16 * R], most;  // SHARED: tokens that each vector sees, the most of them
};
template <int DP, int R, bool Q16, bool SHARED>
__device__ __forceinline__ void attend_part(const AttendParams& p, int block, AttendLds<DP, R>& lds) {
    constexpr int KS = DP / 32;   // matrix steps of a q . k
    constexpr int DT = DP / 16;   // tiles of 16 output columns
    constexpr int VT = 16 * R;    // vectors of the workgroup
    constexpr int QL = Q16 ? 1 : 2, PL = 2;  // fp16 values of a query and of a P

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunk = SHARED ? p.prefix_chunk : p.chunk;
    // heads fastest, parts slowest: workgroups go to the 8 XCDs in turn, and the later parts of ragged
    // sequences are empty.  (With the parts fastest, 64 sequences of 1024 tokens in a batch cut for
    // 4096 in four parts ran on two XCDs: 68 us against 26.)
    int b = block;
    const int h = p.by_heads.mod(b);
    b = p.by_heads.div(b);
    const int tile = (SHARED ? p.by_prefix_tiles : p.by_tiles).mod(b);
    b = (SHARED ? p.by_prefix_tiles : p.by_tiles).div(b);
    const int seq = SHARED ? 0 : p.by_seqs.mod(b), part = SHARED ? b : p.by_seqs.div(b), v0 = tile * VT;
    const int group = p.group.d;

    // the vectors: (row, head) pairs from first_row on, and how many tokens each sees (-1: no vector)
    int first_row, cap, end;
    const int j0 = (SHARED ? 0 : p.own_from) + part * chunk;
    int seen[R];
    if constexpr (SHARED) {
        first_row = 0;
        cap = min(p.prefix, j0 + chunk);
        if (tid == 0) lds.most = 0;
        if (tid < VT) lds.seen[tid] = -1;
        __syncthreads();
        const int r_lo = p.group.div(v0), r_hi = min(p.group.div(v0 + VT - 1) + 1, p.b.rows);
        for (int i = tid; i < p.b.seqs; i += 256) {
            const KvSeq q = kv_seq(p.b.row_start, p.b.length, i, p.b.rows, p.b.max_new, p.b.max_len);
            for (int r = max(q.row0, r_lo); r < min(q.row0 + q.rows, r_hi); ++r) {
                const int y = kv_visible(q, r - q.row0);
                for (int x = max(r * group, v0); x < min((r + 1) * group, v0 + VT); ++x) lds.seen[x - v0] = y;
                atomicMax(&lds.most, y);
            }
        }
        __syncthreads();
        end = min(cap, lds.most);
#pragma unroll
        for (int r = 0; r < R; ++r) seen[r] = lds.seen[16 * r + n];
    } else {
        const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
        if (s.bad && tid == 0) atomicOr(p.err + kErrBatch, 1u);
        if (v0 >= s.rows * group) return;
        if (part > 0 && j0 >= s.len) return;  // the join knows how many parts there are
        first_row = s.row0;
        cap = min(s.len, j0 + chunk);
        end = min(cap, kv_visible(s, p.group.div(min(v0 + VT - 1, s.rows * group - 1))));  // its last row sees most
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int v = v0 + 16 * r + n;
            seen[r] = v < s.rows * group ? kv_visible(s, p.group.div(v)) : -1;
        }
    }
    end = __builtin_amdgcn_readfirstlane(end);

    // the queries' loads first: they do not wait for page ids (vectors that are none take the first row's)
    QueryRow<KS, Q16> qr[R];
    int64_t out_row[R];
    int head[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int v = seen[r] >= 0 ? v0 + 16 * r + n : 0;
        out_row[r] = first_row + p.group.div(v);
        head[r] = h * group + p.group.mod(v);
        load_query<KS, 64, true, Q16>(p, qr[r], out_row[r] * p.ldq + (int64_t)head[r] * p.c.dim, 16 * g);
    }

    // page ids through the scalar cache: nothing writes them while the kernel runs
    const const_ids table = (const_ids)(uintptr_t)(p.b.table + seq * p.b.table_ld);
    const const_ids prefix = (const_ids)(uintptr_t)p.prefix_pages;
    const int off_mask = (1 << p.c.shift) - 1;
    bool bad_page = false, bad[2] = {false, false};  // of a tile: who sees none of its tokens keeps its result
    StepData<DP> d;
    Half16<DP> next[2];
    auto find_step = [&](int j) {  // end > 0
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int jt = j + 16 * t, jj = min(jt, end - 1);
            const int id = (SHARED || jj < p.prefix ? prefix : table)[jj >> p.c.shift];
            next[t] = find_half<DP>(p.c, id, h, jt & off_mask, jt < end);
            next[t].bad = next[t].bad && jt < end;
            bad_page |= next[t].bad;
        }
    };
    auto load_k = [&] {
#pragma unroll
        for (int t = 0; t < 2; ++t) load_bytes<DP / 4, 64>(d.k[t], next[t].block, n * DP + 16 * g, next[t].k);
    };
    auto load_scales = [&] {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            bad[t] = next[t].bad;
            d.ks[t] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(next[t].block, 16 * g, next[t].ks, 0));
            d.vs[t] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(next[t].block, 16 * g, next[t].vs, 0));
        }
    };
    auto load_v = [&] {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_bytes<DP / 16, 16>(d.v[i], next[i / 4].block, (4 * g + i % 4) * DP + n * (DP / 16), next[i / 4].v);
    };
    int j = j0 + 32 * wave;
    if (end > 0) {
        find_step(j);
        load_k();
        load_scales();
        load_v();
    }

    // queries, as the B operand: lane (n, g) holds columns 64 c + 16 g .. + 15 of vector n, two matrix steps each
    half8v qf[R][KS][QL];
    float unit[R];  // what the f16 operands were divided by, times scale2
#pragma unroll
    for (int r = 0; r < R; ++r) {
        unit[r] = p.scale2 * kCodeUnit;
        float x[DP / 4];
#pragma unroll
        for (int i = 0; i < DP / 4; ++i) x[i] = query_at<KS, Q16>(qr[r], i / 8, i % 8);
        if constexpr (QL == 2) {
            // the row's largest value goes to [2^13, 2^14): the low parts stay normal, f32 rows of any size fit
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 4; ++i) m = fmaxf(m, fabsf(x[i]));
            m = over_groups<true>(m);
            const int e = kv_clamp((int)((__float_as_uint(m) >> 23) & 0xff) - 127, -100, 126);
            const float up = __uint_as_float((uint32_t)(13 - e + 127) << 23);  // 2^(13 - e)
            unit[r] *= __uint_as_float((uint32_t)(e - 13 + 127) << 23);
#pragma unroll
            for (int i = 0; i < DP / 4; ++i) x[i] *= up;
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 y[QL];
                split_f16<QL>(x[8 * k + i], y);
#pragma unroll
                for (int q = 0; q < QL; ++q) qf[r][k][q][i] = y[q];
            }
    }

    float m[R], l[R];
    float4v o[R][DT];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = kNegInf;
        l[r] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[r][t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // The next step's keys are loaded over this one's when those are used, then its scales, then its values:
    // one set of registers, and some loads are in flight at any time.
    for (; j < end; j += kAttendStep) {
        find_step(j + kAttendStep);
        // S^T: tokens 16 t + 4 g + i of vector n
        float4v sc[2][R];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < R; ++r) sc[t][r] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const half8v a = codes8(d.k[t].w[2 * k], d.k[t].w[2 * k + 1]);
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int q = 0; q < QL; ++q)
                        sc[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[r][k][q], sc[t][r], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k();
        float lv[8], iv[8];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lv[4 * t + i] = bad[t] ? kNan : __builtin_amdgcn_logf(d.vs[t][i]);
                iv[4 * t + i] = __builtin_amdgcn_rcpf(d.vs[t][i]);
            }
        half8v pf[R][PL];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int left = min(seen[r], cap) - j - 4 * g;
            float x[8];
            float top = kNegInf;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = __builtin_fmaf(sc[t][r][i] * unit[r], d.ks[t][i], lv[4 * t + i]);
                    // masked tokens are chosen away, whatever their scales hold
                    x[4 * t + i] = 16 * t + i < left ? y : kNegInf;
                    top = fmaxf(top, x[4 * t + i]);
                }
            top = over_groups<true>(top);
            if (__builtin_amdgcn_ballot_w64(top > m[r] + kSlack)) {
                const float m_new = fmaxf(m[r], top);
                const float fade = m[r] == m_new ? 1.0f : __builtin_amdgcn_exp2f(m[r] - m_new);
                m[r] = m_new;
                l[r] *= fade;
#pragma unroll
                for (int t = 0; t < DT; ++t) o[r][t] *= fade;
            }
            const float base = m[r] == kNegInf ? 0.0f : m[r] - kPShift;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2v e = {__builtin_amdgcn_exp2f(x[i] - base), __builtin_amdgcn_exp2f(x[i + 1] - base)};
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    l[r] = 16 * (i / 4) + (i + c) % 4 < left ? __builtin_fmaf(e[c], iv[i + c], l[r]) : l[r];
                const half2v y = __builtin_convertvector(e, half2v);
                const half2v z = __builtin_convertvector(e - __builtin_convertvector(y, float2v), half2v);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    pf[r][0][i + c] = y[c];
                    pf[r][1][i + c] = z[c];
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_scales();
        // O^T: columns n * DP/16 + t (row n of the operand) over tokens 4g + i of both tiles
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const uint32_t lo = t & 3, sel = 0x0c000c00u | (4 + lo) << 16 | lo;
            const uint4v w = {codes2(d.v[1].w[t / 4], d.v[0].w[t / 4], sel), codes2(d.v[3].w[t / 4], d.v[2].w[t / 4], sel),
                              codes2(d.v[5].w[t / 4], d.v[4].w[t / 4], sel), codes2(d.v[7].w[t / 4], d.v[6].w[t / 4], sel)};
            const half8v a = __builtin_bit_cast(half8v, w);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int q = 0; q < PL; ++q)
                    o[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf[r][q], o[r][t], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v();
    }
    if (bad_page && lane == 0) atomicOr(p.err + kErrBatch, 1u);

    // join the waves: a common maximum, then 3 -> 1 and 2 -> 0, then 1 -> 0
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] = over_groups<false>(l[r]);
        if (g == 0) {
            lds.m[wave][16 * r + n] = m[r];
            lds.l[wave][16 * r + n] = l[r];
        }
    }
    __syncthreads();
    float m_all[R], l_all[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int v = 16 * r + n;
        m_all[r] = fmaxf(fmaxf(lds.m[0][v], lds.m[1][v]), fmaxf(lds.m[2][v], lds.m[3][v]));
        const float base = m_all[r] == kNegInf ? 0.0f : m_all[r];
        l_all[r] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l_all[r] += lds.l[w][v] * __builtin_amdgcn_exp2f(lds.m[w][v] - base);
        const float fade = __builtin_amdgcn_exp2f(m[r] - base);
#pragma unroll
        for (int t = 0; t < DT; ++t) o[r][t] *= fade;
    }
    // columns (4 g + i) * DT + t of a vector, t = 4 u .. 4 u + 3
    auto four = [&](int r, int i, int u) -> float4v {
        return {o[r][4 * u][i], o[r][4 * u + 1][i], o[r][4 * u + 2][i], o[r][4 * u + 3][i]};
    };
    auto put = [&](int slot) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < DT / 4; ++u)
                    *reinterpret_cast<float4v*>(&lds.o[slot][16 * r + n][(4 * g + i) * DT + 4 * u]) = four(r, i, u);
    };
    auto add = [&](int slot) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < DT / 4; ++u) {
                    const float4v y = *reinterpret_cast<const float4v*>(&lds.o[slot][16 * r + n][(4 * g + i) * DT + 4 * u]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[r][4 * u + c][i] += y[c];
                }
    };
    if (wave >= 2) put(wave - 2);
    __syncthreads();
    if (wave < 2) add(wave);
    __syncthreads();
    if (wave == 1) put(0);
    __syncthreads();
    if (wave != 0) return;
    add(0);

#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (seen[r] < 0) continue;
        if (p.parts == 1) {
            const float f = l_all[r] == 0.0f ? 0.0f : kCodeUnit / l_all[r];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < DT / 4; ++u) {
                    const float4v y = four(r, i, u) * f;
                    const float z[4] = {y[0], y[1], y[2], y[3]};
                    store_out<4>(p, out_row[r] * p.ldo + (int64_t)head[r] * p.c.dim, (4 * g + i) * DT + 4 * u, z);
                }
        } else {
            const int64_t slot = (out_row[r] * p.q_heads + head[r]) * p.parts + (SHARED ? 0 : p.prefix_parts) + part;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < DT / 4; ++u)
                    *reinterpret_cast<float4v*>(p.part_o + slot * DP + (4 * g + i) * DT + 4 * u) = four(r, i, u);
            if (g == 0) {
                p.part_ml[2 * slot] = m_all[r];
                p.part_ml[2 * slot + 1] = l_all[r];
            }
        }
    }
}

// A launch: the first `shared` workgroups work on the prefix with RS tiles (0: there is none), the others on the
// sequences' own tokens with RO.
template <int DP, int RS, int RO, bool Q16>
__global__ __launch_bounds__(256, DP * (RS > RO ? RS : RO) * (Q16 ? 1 : 2) <= 64 ? 4 : DP * (RS > RO ? RS : RO) * (Q16 ? 1 : 2) <= 128 ? 3 : 1)
void attend_kernel(AttendParams p, int shared) {
    __shared__ union {
        AttendLds<DP, (RS > 0 ? RS : RO)> prefix;
        AttendLds<DP, RO> own;
    } lds;
    if constexpr (RS > 0) {
        if ((int)blockIdx.x < shared) {
            attend_part<DP, RS, Q16, true>(p, blockIdx.x, lds.prefix);
            return;
        }
    }
    attend_part<DP, RO, Q16, false>(p, blockIdx.x - shared, lds.own);
}

// Joins the parts of vectors: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  DP / 4 lanes hold a vector's
// columns, four each.  MANY parts: a workgroup per vector, its groups of lanes take the parts in turn
// and are joined in the LDS.  Few: a group per vector.  Maxima and outputs of four parts are loaded together
// and the maximum runs along: what is short here is the chain of loads (sequence, parts), not their bytes.
template <int DP, bool MANY>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p) {
    constexpr int LPV = DP / 4, GROUPS = 256 / LPV, STEP = MANY ? GROUPS : 1;
    __shared__ __align__(16) float lds_o[MANY ? GROUPS : 1][DP];
    __shared__ float lds_m[GROUPS], lds_l[GROUPS];
    const int seq = p.by_join.div(blockIdx.x);
    const int group = threadIdx.x / LPV, d = (threadIdx.x % LPV) * 4;
    const int x = MANY ? p.by_join.mod(blockIdx.x) : p.by_join.mod(blockIdx.x) * GROUPS + group;
    const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
    const int t = p.by_q_heads.div(x), head = p.by_q_heads.mod(x);
    if (t >= s.rows) return;
    const int parts = p.prefix_parts + kv_parts(s.len - p.own_from, p.chunk);
    const int64_t row = s.row0 + t, slot = (row * p.q_heads + head) * p.parts;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + slot;
    float m = kNegInf, l = 0.0f;
    float4v o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = MANY ? group : 0; i < parts; i += 4 * STEP) {
        float2 y[4];
        float4v z[4];
        float top = m;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int at = min(i + k * STEP, parts - 1);
            y[k] = ml[at];
            z[k] = *reinterpret_cast<const float4v*>(p.part_o + (slot + at) * DP + d);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * STEP < parts) top = fmaxf(top, y[k].x);
        const float base = top == kNegInf ? 0.0f : top, fade = __builtin_amdgcn_exp2f(m - base);
        m = top;
        l *= fade;
        o *= fade;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k * STEP >= parts) continue;
            const float f = __builtin_amdgcn_exp2f(y[k].x - base);
            l = __builtin_fmaf(f, y[k].y, l);
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = __builtin_fmaf(f, z[k][c], o[c]);
        }
    }
    if constexpr (MANY) {
        *reinterpret_cast<float4v*>(&lds_o[group][d]) = o;
        if (d == 0) {
            lds_m[group] = m;
            lds_l[group] = l;
        }
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) m = fmaxf(m, lds_m[i]);
        const float base = m == kNegInf ? 0.0f : m;
        l = 0.0f;
        o = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            const float f = __builtin_amdgcn_exp2f(lds_m[i] - base);
            l = __builtin_fmaf(f, lds_l[i], l);
            const float4v z = *reinterpret_cast<const float4v*>(&lds_o[i][d]);
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = __builtin_fmaf(f, z[c], o[c]);
        }
    }
    const float f = l == 0.0f ? 0.0f : kCodeUnit / l;
    const float y[4] = {o[0] * f, o[1] * f, o[2] * f, o[3] * f};
    store_out<4>(p, row * p.ldo + (int64_t)head * p.c.dim, d, y);
}

// Vectors of a workgroup, given how many share its tokens: one or two tiles here (two of 256 columns would
// not fit the registers), or the wide kernel's.  That one reads a token's bytes once for 128 vectors but
// waits at a barrier for every 32 tokens: with up to 256 vectors (512 where rows are f32 in or out) more workgroups of
// this one are faster.  One sequence, 4096 tokens, 8 KV heads, us here and there:
//   vectors           256          384          512          768         1024
//   fp16, 64       17.0 / 23.5  25.5 / 24.3  24.4 / 27.9  33.6 / 32.1  34.4 / 32.9
//   fp16, 128      21.6 / 32.3  34.1 / 34.7  30.9 / 37.8  45.7 / 46.9  48.4 / 46.5
//   fp16, 256      30.6 / 43.8  51.5 / 60.3  53.2 / 68.6  75.5 / 80.4  96.2 / 93.1
//   f32, 128       23.9 / 38.3  38.5 / 42.0  33.8 / 46.7  50.9 / 57.9  53.9 / 62.2
//   prefix, fp16   24.9 / 35.7  36.3 / 41.2  35.4 / 47.6  48.4 / 54.5  57.3 / 65.1   (128 columns)
//   prefix, f32    26.4 / 43.5  40.4 / 54.2  39.0 / 58.6  54.6 / 75.9  64.1 / 87.3
// What a batch holds beside that moves the crossing, and the limit on vectors alone is a middle: of 257 to 512 fp16 vectors
// in 36 random batches of 1 to 16 sequences this kernel takes 0.83 of the other's time on average, half of it for one
// sequence of a few hundred tokens, 1.35 of it for one of 15000 tokens and up to 1.85 for 16 sequences.
int tile_of(const AttendParams& p, int64_t vectors) {
    if (vectors > (p.q_f16 && p.o_f16 ? 256 : 512)) return kAttendWide;
    return vectors <= 16 || p.c.dim_padded > 128 ? 16 : 32;
}

template <int DP, bool Q16>
hipError_t launch_typed(const AttendParams& p, hipStream_t st) {
    const int own = attend_tile(p), shared = p.prefix_parts ? attend_tile_prefix(p) : 0;
    const uint32_t own_blocks = (uint32_t)((p.parts - p.prefix_parts) * (int64_t)p.b.seqs * p.c.heads * p.by_tiles.d);
    const uint32_t shared_blocks = (uint32_t)(p.prefix_parts * (int64_t)p.c.heads * p.by_prefix_tiles.d);
    if (shared >= kAttendWide)
        if (hipError_t e = launch_attend_wide(p, true, st)) return e;
    if (own >= kAttendWide) return launch_attend_wide(p, false, st);
    const uint32_t first = shared >= kAttendWide ? 0 : shared_blocks;
    const dim3 grid(first + own_blocks);
    if (first == 0) {
        if constexpr (DP <= 128)
            if (own == 32) {
                attend_kernel<DP, 0, 2, Q16><<<grid, 256, 0, st>>>(p, 0);
                return hipGetLastError();
            }
        attend_kernel<DP, 0, 1, Q16><<<grid, 256, 0, st>>>(p, 0);
        return hipGetLastError();
    }
    if constexpr (DP <= 128) {  // the prefix's rows are those of all sequences: at least as many
        if (own == 32) attend_kernel<DP, 2, 2, Q16><<<grid, 256, 0, st>>>(p, first);
        else if (shared == 32) attend_kernel<DP, 2, 1, Q16><<<grid, 256, 0, st>>>(p, first);
        else attend_kernel<DP, 1, 1, Q16><<<grid, 256, 0, st>>>(p, first);
    } else {
        attend_kernel<DP, 1, 1, Q16><<<grid, 256, 0, st>>>(p, first);
    }
    return hipGetLastError();
}

template <int DP>
hipError_t launch_dp(const AttendParams& p, hipStream_t st) {
    const hipError_t e = p.q_f16 ? launch_typed<DP, true>(p, st) : launch_typed<DP, false>(p, st);
    if (e != hipSuccess || p.parts == 1) return e;
    // few parts: fewer than the groups of lanes a workgroup has for them
    AttendParams j = p;
    const int64_t vectors = (int64_t)p.b.max_new * p.q_heads, groups = 256 / (DP / 4);
    const bool many = p.parts >= groups;
    const int64_t blocks = many ? vectors : (vectors + groups - 1) / groups;
    j.by_join = fast_div((int)blocks);
    if (many) attend_join_kernel<DP, true><<<dim3((uint32_t)(blocks * p.b.seqs)), 256, 0, st>>>(j);
    else attend_join_kernel<DP, false><<<dim3((uint32_t)(blocks * p.b.seqs)), 256, 0, st>>>(j);
    return hipGetLastError();
}

}  // namespace

int attend_tile(const AttendParams& p) { return tile_of(p, (int64_t)p.b.max_new * p.group.d); }
int attend_tile_prefix(const AttendParams& p) { return tile_of(p, (int64_t)p.b.rows * p.group.d); }

hipError_t launch_attend(const AttendParams& p, hipStream_t st) {
    switch (p.c.dim_padded) {
        case 64: return launch_dp<64>(p, st);
        case 128: return launch_dp<128>(p, st);
        default: return launch_dp<256>(p, st);
    }
}

}  // namespace qlin
