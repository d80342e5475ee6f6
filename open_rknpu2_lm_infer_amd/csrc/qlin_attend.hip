// Attention of new rows over the 8-bit key/value cache.
//
//   l_j = scale * s^K_j * (q . k_j)          j = the tokens a row sees (itself and before)
//   o   = sum_j e^(l_j) s^V_j v_j / sum_j e^(l_j),   no token: 0
//
// in one pass over the tokens with a running maximum.  Codes are exact in fp16, so q . k_j runs on
// the matrix cores (f32 sums) without any rounding of the keys, and the value scale goes into the
// probabilities: with l'_j = l_j log2 e + log2 s^V_j and m the running maximum of l',
// P_j = 2^(l'_j - m) <= 1 multiplies the codes v_j, and the sum of e^(l_j) is sum_j P_j / s^V_j.
// Taking the maximum over l' and not l keeps P inside fp16's range whatever the scales are.
//
// A query row and head is a "vector"; the q_heads / kv_heads vectors of each row that share a KV
// head, and the rows of a sequence, are worked on together, 16 to a tile.  Products are computed
// transposed, S^T = K Q^T and O^T = V^T P^T: then the matrix core's result layout (a lane holds
// four consecutive tokens of one vector) is the operand layout of the second product with its k
// axis permuted, and P never leaves its lane.
#include "qlin_kv.hpp"
#include "qlin_rows.hpp"

namespace qlin {
namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr float kNan = __builtin_nanf("");

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

template <int N>
struct Bytes {
    uint32_t w[N / 4];
};

// N consecutive bytes, N-byte aligned (16-byte aligned beyond 16).
template <int N>
__device__ __forceinline__ void load_bytes(Bytes<N>& r, const uint8_t* p) {
    if constexpr (N == 4) r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        r.w[0] = x.x;
        r.w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 16; ++i) {
            const uint4 x = reinterpret_cast<const uint4*>(p)[i];
            r.w[4 * i] = x.x;
            r.w[4 * i + 1] = x.y;
            r.w[4 * i + 2] = x.z;
            r.w[4 * i + 3] = x.w;
        }
    }
}

// What a wave loads for one step of 32 tokens: two tiles of 16.  Lane l (n = l % 16, g = l / 16)
// holds, as the matrix core's A operand, columns g * DP/4 .. + DP/4 - 1 of key n of each tile, and
// columns n * DP/16 .. + DP/16 - 1 of values 4g .. 4g + 3 of each tile.
template <int DP>
struct StepData {
    Bytes<DP / 4> k[2];
    Bytes<DP / 16> v[8];
    float4 ks[2], vs[2];  // scales of tokens 4g .. 4g + 3
};

template <int DP>
__device__ __forceinline__ void load_step(StepData<DP>& r, const KvCache& c, int64_t row0, int64_t row1, int n, int g) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int64_t row = t ? row1 : row0;
        load_bytes<DP / 4>(r.k[t], c.k + (row + n) * DP + g * (DP / 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) load_bytes<DP / 16>(r.v[4 * t + i], c.v + (row + 4 * g + i) * DP + n * (DP / 16));
        r.ks[t] = *reinterpret_cast<const float4*>(c.ks + row + 4 * g);
        r.vs[t] = *reinterpret_cast<const float4*>(c.vs + row + 4 * g);
    }
}

// fp16 high part, and the rest (exact in fp16 unless it underflows) where f32 is asked for.
template <int LIMBS>
__device__ __forceinline__ void split_f16(float x, _Float16 out[LIMBS]) {
    out[0] = (_Float16)x;
    if constexpr (LIMBS == 2) out[1] = (_Float16)(x - (float)out[0]);
}

// Workgroup: 4 waves, R tiles of 16 vectors of one KV head, one part of the tokens.  The waves take
// steps of 32 tokens in turn, each with a running maximum, sum and output of its own, and join
// them at the end.  LIMBS = 2 (f32 rows in or out): queries and P as a sum of two fp16 values,
// 22 bits; fp16 queries are exact with one, and P rounded to 11 bits is off by as much as an fp16 output.
template <int DP, int R, int LIMBS>
__global__ __launch_bounds__(256) void attend_kernel(AttendParams p, int prefix_blocks) {
    constexpr int KS = DP / 32;   // matrix steps of a q . k
    constexpr int DT = DP / 16;   // tiles of 16 output columns
    constexpr int VT = 16 * R;    // vectors of the workgroup
    __shared__ float lds_o[2][VT][DP];
    __shared__ float lds_m[4][VT], lds_l[4][VT];
    __shared__ int lds_seen[VT];  // tokens that each vector sees
    __shared__ int lds_range;     // the most of them

    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool shared_part = (int)blockIdx.x < prefix_blocks;
    int b = shared_part ? blockIdx.x : blockIdx.x - prefix_blocks;
    const int parts = shared_part ? p.prefix_parts : p.parts - p.prefix_parts;
    const int part = b % parts;
    b /= parts;
    const int h = b % p.c.heads;
    b /= p.c.heads;

    // the vectors: (row, head) pairs from first_row on
    int first_row, rows_left, seq = 0;
    KvSeq s{};
    if (shared_part) {
        first_row = 0;
        rows_left = p.b.rows;
    } else {
        const int tiles = (p.b.max_new * p.group + VT - 1) / VT;
        seq = b / tiles;
        b -= seq * tiles;
        s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
        if (s.bad && tid == 0) atomicOr(p.err, kErrBatch);
        first_row = s.row0;
        rows_left = s.rows;
    }
    const int v0 = b * VT;
    if (v0 >= rows_left * p.group) return;
    const int j0 = (shared_part ? 0 : p.own_from) + part * (shared_part ? p.prefix_chunk : p.chunk);
    if (!shared_part && part > 0 && j0 >= s.len) return;  // the join knows how many parts there are
    const int cap = shared_part ? min(p.prefix, j0 + p.prefix_chunk) : min(s.len, j0 + p.chunk);

    // tokens that each vector sees
    if (tid == 0) lds_range = 0;
    if (tid < VT) lds_seen[tid] = -1;
    __syncthreads();
    if (shared_part) {
        const int r_lo = v0 / p.group, r_hi = min((v0 + VT - 1) / p.group + 1, p.b.rows);
        for (int i = tid; i < p.b.seqs; i += 256) {
            const KvSeq q = kv_seq(p.b.row_start, p.b.length, i, p.b.rows, p.b.max_new, p.b.max_len);
            for (int r = max(q.row0, r_lo); r < min(q.row0 + q.rows, r_hi); ++r) {
                const int seen = kv_visible(q, r - q.row0);
                for (int x = max(r * p.group, v0); x < min((r + 1) * p.group, v0 + VT); ++x) lds_seen[x - v0] = seen;
            }
        }
    } else if (tid < VT && v0 + tid < rows_left * p.group) {
        lds_seen[tid] = kv_visible(s, (v0 + tid) / p.group);
    }
    __syncthreads();
    if (tid < VT && lds_seen[tid] >= 0) atomicMax(&lds_range, lds_seen[tid]);
    __syncthreads();
    const int end = __builtin_amdgcn_readfirstlane(min(cap, lds_range));  // no vector sees more

    // queries, as the B operand: lane (n, g) holds columns g * DP/4 + 8 s .. + 7 of vector n
    half8v qf[R][KS][LIMBS];
    float unit[R];  // what the f16 operands were divided by, times scale2
    int seen[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int v = v0 + 16 * r + n;
        seen[r] = lds_seen[16 * r + n];
        const bool ok = seen[r] >= 0;
        const int row = first_row + (ok ? v / p.group : 0), head = h * p.group + (ok ? v % p.group : 0);
        const int64_t at = (int64_t)row * p.ldq + (int64_t)head * p.c.dim;
        unit[r] = p.scale2 * kCodeUnit;
        float x[DP / 4];
#pragma unroll
        for (int i = 0; i < DP / 4; ++i) {
            const int d = g * (DP / 4) + i;
            x[i] = !ok || d >= p.c.dim ? 0.0f
                   : p.q_f16           ? (float)reinterpret_cast<const _Float16*>(p.q)[at + d]
                                       : reinterpret_cast<const float*>(p.q)[at + d];
        }
        if constexpr (LIMBS == 2) {
            // the row's largest value goes to [2^13, 2^14): the low parts stay normal, f32 rows of any size fit
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < DP / 4; ++i) m = fmaxf(m, fabsf(x[i]));
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
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
                _Float16 y[LIMBS];
                split_f16<LIMBS>(x[8 * k + i], y);
#pragma unroll
                for (int q = 0; q < LIMBS; ++q) qf[r][k][q][i] = y[q];
            }
    }

    float m[R], l[R];
    float4v o[R][DT];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -__builtin_inff();
        l[r] = 0.0f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[r][t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int32_t* table = p.b.table + seq * p.b.table_ld;
    const int off_mask = (1 << p.c.shift) - 1;
    bool bad_page = false;
    // tokens of a tile past the end are read from the last page (never past the cache) and masked
    auto tile_row = [&](int j, bool* bad) {
        const int jj = min(j, end - 1);
        const int page = kv_page((jj < p.prefix ? p.prefix_pages : table)[jj >> p.c.shift], p.c.pages, bad);
        return kv_row(page, p.c.heads, h, p.c.shift, j & off_mask);
    };
    for (int j = j0 + 32 * wave; j < end; j += kAttendStep) {
        bool bad = false;
        StepData<DP> d;
        const int64_t row0 = tile_row(j, &bad), row1 = tile_row(j + 16, &bad);
        load_step<DP>(d, p.c, row0, row1, n, g);
        bad_page |= bad;
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
                    for (int q = 0; q < LIMBS; ++q)
                        sc[t][r] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[r][k][q], sc[t][r], 0, 0, 0);
            }
        }
        half8v pf[R][LIMBS];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float x[8], inv[8];
            float top = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float ks[4] = {d.ks[t].x, d.ks[t].y, d.ks[t].z, d.ks[t].w};
                const float vs[4] = {d.vs[t].x, d.vs[t].y, d.vs[t].z, d.vs[t].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = __builtin_fmaf(sc[t][r][i] * unit[r], bad ? kNan : ks[i], __builtin_amdgcn_logf(vs[i]));
                    const bool in = j + 16 * t + 4 * g + i < min(seen[r], cap);
                    // masked tokens are chosen away, whatever their scales hold
                    x[4 * t + i] = in ? y : -__builtin_inff();
                    inv[4 * t + i] = in ? __builtin_amdgcn_rcpf(vs[i]) : 0.0f;
                    top = fmaxf(top, x[4 * t + i]);
                }
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float m_new = fmaxf(m[r], top);
            const float base = m_new == -__builtin_inff() ? 0.0f : m_new;
            const float fade = __builtin_amdgcn_exp2f(m[r] - base);
            m[r] = m_new;
            l[r] *= fade;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[r][t] *= fade;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = __builtin_amdgcn_exp2f(x[i] - base + kPShift);
                l[r] = __builtin_fmaf(e, inv[i], l[r]);
                _Float16 y[LIMBS];
                split_f16<LIMBS>(e, y);
#pragma unroll
                for (int q = 0; q < LIMBS; ++q) pf[r][q][i] = y[q];
            }
        }
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
                for (int q = 0; q < LIMBS; ++q)
                    o[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pf[r][q], o[r][t], 0, 0, 0);
        }
    }
    if (bad_page && lane == 0) atomicOr(p.err, kErrBatch);

    // join the waves: a common maximum, then 3 -> 1 and 2 -> 0, then 1 -> 0
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l[r] += __shfl_xor(l[r], 16, 64);
        l[r] += __shfl_xor(l[r], 32, 64);
        if (g == 0) {
            lds_m[wave][16 * r + n] = m[r];
            lds_l[wave][16 * r + n] = l[r];
        }
    }
    __syncthreads();
    float m_all[R], l_all[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int v = 16 * r + n;
        m_all[r] = fmaxf(fmaxf(lds_m[0][v], lds_m[1][v]), fmaxf(lds_m[2][v], lds_m[3][v]));
        const float base = m_all[r] == -__builtin_inff() ? 0.0f : m_all[r];
        l_all[r] = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) l_all[r] += lds_l[w][v] * __builtin_amdgcn_exp2f(lds_m[w][v] - base);
        const float fade = __builtin_amdgcn_exp2f(m[r] - base);
#pragma unroll
        for (int t = 0; t < DT; ++t) o[r][t] *= fade;
    }
    auto put = [&](int slot) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) lds_o[slot][16 * r + n][(4 * g + i) * DT + t] = o[r][t][i];
    };
    auto add = [&](int slot) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[r][t][i] += lds_o[slot][16 * r + n][(4 * g + i) * DT + t];
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
        const int v = v0 + 16 * r + n;
        const int64_t row = first_row + v / p.group;
        const int head = h * p.group + v % p.group;
        if (p.parts == 1) {
            const float f = l_all[r] == 0.0f ? 0.0f : kCodeUnit / l_all[r];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const int d = (4 * g + i) * DT + t;
                    if (d >= p.c.dim) continue;
                    const float y = o[r][t][i] * f;
                    const int64_t at = row * p.ldo + (int64_t)head * p.c.dim + d;
                    if (p.o_f16) reinterpret_cast<_Float16*>(p.o)[at] = (_Float16)y;
                    else reinterpret_cast<float*>(p.o)[at] = y;
                }
        } else {
            const int64_t slot = (row * p.q_heads + head) * p.parts + (shared_part ? 0 : p.prefix_parts) + part;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < DT; ++t) p.part_o[slot * DP + (4 * g + i) * DT + t] = o[r][t][i];
            if (g == 0) {
                p.part_ml[2 * slot] = m_all[r];
                p.part_ml[2 * slot + 1] = l_all[r];
            }
        }
    }
}

// Joins the parts of every vector: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  DP / 4 lanes a
// vector, four columns each.
template <int DP>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendParams p) {
    constexpr int LPV = DP / 4, VPB = 256 / LPV;
    const int per_seq = (p.b.max_new * p.q_heads + VPB - 1) / VPB;
    const int seq = blockIdx.x / per_seq;
    const int x = (blockIdx.x - seq * per_seq) * VPB + threadIdx.x / LPV;
    const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
    const int t = x / p.q_heads, head = x % p.q_heads;
    if (t >= s.rows) return;
    const int parts = p.prefix_parts + kv_parts(s.len - p.own_from, p.chunk);
    const int d = (threadIdx.x % LPV) * 4;
    const int64_t row = s.row0 + t, slot = (row * p.q_heads + head) * p.parts;
    float m = -__builtin_inff();
    for (int i = 0; i < parts; ++i) m = fmaxf(m, p.part_ml[2 * (slot + i)]);
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < parts; ++i) {
        const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * (slot + i)] - base);
        const float4 y = *reinterpret_cast<const float4*>(p.part_o + (slot + i) * DP + d);
        l = __builtin_fmaf(f, p.part_ml[2 * (slot + i) + 1], l);
        o.x = __builtin_fmaf(f, y.x, o.x);
        o.y = __builtin_fmaf(f, y.y, o.y);
        o.z = __builtin_fmaf(f, y.z, o.z);
        o.w = __builtin_fmaf(f, y.w, o.w);
    }
    const float f = l == 0.0f ? 0.0f : kCodeUnit / l;
    const float y[4] = {o.x * f, o.y * f, o.z * f, o.w * f};
    const int64_t at = row * p.ldo + (int64_t)head * p.c.dim + d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (d + i >= p.c.dim) continue;
        if (p.o_f16) reinterpret_cast<_Float16*>(p.o)[at + i] = (_Float16)y[i];
        else reinterpret_cast<float*>(p.o)[at + i] = y[i];
    }
}

template <int DP, int LIMBS>
hipError_t launch_dp(const AttendParams& p, hipStream_t st) {
    constexpr int R = 1;
    const int64_t tiles = ((int64_t)p.b.max_new * p.group + 16 * R - 1) / (16 * R);
    const int64_t own = (int64_t)(p.parts - p.prefix_parts) * p.c.heads * tiles * p.b.seqs;
    const int64_t shared = p.prefix_parts * (int64_t)p.c.heads * (((int64_t)p.b.rows * p.group + 16 * R - 1) / (16 * R));
    attend_kernel<DP, R, LIMBS><<<dim3((uint32_t)(own + shared)), 256, 0, st>>>(p, (int)shared);
    if (hipError_t e = hipGetLastError()) return e;
    if (p.parts == 1) return hipSuccess;
    constexpr int VPB = 256 / (DP / 4);
    const int64_t per_seq = ((int64_t)p.b.max_new * p.q_heads + VPB - 1) / VPB;
    attend_join_kernel<DP><<<dim3((uint32_t)(per_seq * p.b.seqs)), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace

int attend_tile(const AttendParams&) { return 16; }

hipError_t launch_attend(const AttendParams& p, hipStream_t st) {
    const bool two = !p.q_f16 || !p.o_f16;
    switch (p.c.dim_padded) {
        case 64: return two ? launch_dp<64, 2>(p, st) : launch_dp<64, 1>(p, st);
        case 128: return two ? launch_dp<128, 2>(p, st) : launch_dp<128, 1>(p, st);
        default: return two ? launch_dp<256, 2>(p, st) : launch_dp<256, 1>(p, st);
    }
}

}  // namespace qlin
