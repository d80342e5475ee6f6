// Attention of many rows over the 8-bit key/value cache: prompts, chunks of prompts, and the shared
// prefix of a batch.  The formulas are those of qlin_attend.hip.
//
// A workgroup holds 128 vectors, 32 a wave, and walks over its tokens 32 at a time.  The
// bytes of a tile are loaded two tiles ahead, made into fp16 codes once for the four waves and laid down
// in the LDS: keys as they are, values transposed.  The matrix core's result layout of S^T = K Q^T (a
// lane holds four tokens of every eight of one vector) is the operand layout of O^T = V^T P^T with its
// k axis permuted, so the values' tokens are written in that order and P never leaves its lane.
//
// The products of one tile run beside the exponentials of another: S of tile u + 1 while P of tile u is
// made, then O of tile u while the maximum of tile u + 1 is found.  Three tiles lie in the LDS: the values of u,
// the keys of u + 1, and u + 2 on its way in.
//
// What bounds it (a prompt of 4096 tokens, 32 query and 8 KV heads of 128, 137 GFLOP: 167 to 178 us a call, 770 to 820 TFLOP/s):
// the LDS, busy 51% of the time, the vector units, 50%, and the matrix cores, 36%, each of which the two waves of a SIMD
// leave idle in turn.  For 16 matrix instructions of 32 x 32 x 16 a wave reads 16 KB of operands and 12 KB of scale
// factors; the matrix instructions, their operands' reads and the barriers alone take 124 us.  64 vectors a wave would halve the reads, but their
// registers leave one wave a SIMD (198 to 247 us).  Heads of 64 take 141 us, of 256 412 (one wave a SIMD).  f32 queries of
// 128 columns are two values of fp16 each and spill 23 to 25 registers: 305 us (f32 outputs of fp16 queries 224, no spill).
#include <atomic>
#include <type_traits>

#include "qlin_attend.hpp"

namespace qlin {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kTokens = 32;  // of a tile
constexpr int kThreads = 256;

// LDS of one tile.  Rows are padded by 16 bytes: eight lanes' 16-byte accesses to eight rows then
// fall into different banks.
template <int DP>
struct TileLds {
    static constexpr int KROW = 2 * DP + 16, VROW = 2 * kTokens + 16;
    static constexpr int V = kTokens * KROW, S = V + DP * VROW, BYTES = S + 3 * kTokens * 4;
};

// A thread's share of a tile on its way from the cache to the LDS: 16 bytes of a key, and four columns
// of four tokens' values; SUBS of each.  A wave's share i lies in one 16-token half of the tile.
template <int DP>
struct Share {
    static constexpr int SUBS = DP == 256 ? 2 : 1;
    static constexpr int KCOLS = DP / 16, VCOLS = DP / 4;  // lanes across a row
    uint4v k[SUBS];
    uint32_t v[SUBS][4];
    float ks[SUBS], vs[SUBS];
    bool bad[SUBS];
};

// LIMBS fp16 values make a probability.  Two where rows are f32 in or out: 22 bits.  One where both are fp16: its
// rounding to 11 bits adds to the output's own (2.6e-4 of the output against 64 bits, 2.1e-4 with two), and the second
// value would cost half as many matrix instructions again (the prompt of 4096 tokens 177 us with one, 222 with two, a chunk
// of 512 over 8192 102 and 122).  Queries of f32 are two values, those of fp16 one, exact.
template <int DP, int LIMBS, bool Q16, bool SHARED>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void attend_wide_kernel(AttendParams p) {
    using L = TileLds<DP>;
    using Sh = Share<DP>;
    constexpr int KS = DP / 16, ND = DP / 32, VT = kAttendWide, QL = Q16 ? 1 : 2;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, hi = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = p.group.d;
    const int chunk = SHARED ? p.prefix_chunk : p.chunk;
    // heads fastest: with 8 of them, neighbours in the launch order (8 XCDs in turn) read the same head's
    // tokens from the same XCD's L2; then the vectors, those that see most first; parts slowest, as the
    // later ones of ragged sequences are empty
    int b = blockIdx.x;
    const int h = p.by_heads.mod(b);
    b = p.by_heads.div(b);
    const FastDiv& by_tiles = SHARED ? p.by_prefix_tiles : p.by_tiles;
    const int v0 = ((int)by_tiles.d - 1 - by_tiles.mod(b)) * VT;
    b = by_tiles.div(b);
    const int seq = SHARED ? 0 : p.by_seqs.mod(b), part = SHARED ? b : p.by_seqs.div(b);

    // how many tokens each vector sees (-1: no vector); vector v0 + 32 wave + n
    int first_row = 0, cap, end, least;  // no vector sees end or more; all see the first `least`
    int seen;
    const int j0 = (SHARED ? 0 : p.own_from) + part * chunk;
    const int v = v0 + 32 * wave + n;
    if constexpr (SHARED) {
        int* lds_seen = reinterpret_cast<int*>(lds);  // before the first tile
        cap = min(p.prefix, j0 + chunk);
        if (tid < VT) lds_seen[tid] = -1;
        __syncthreads();
        const int r_lo = p.group.div(v0), r_hi = min(p.group.div(v0 + VT - 1) + 1, p.b.rows);
        for (int i = tid; i < p.b.seqs; i += kThreads) {
            const KvSeq q = kv_seq(p.b.row_start, p.b.length, i, p.b.rows, p.b.max_new, p.b.max_len);
            for (int r = max(q.row0, r_lo); r < min(q.row0 + q.rows, r_hi); ++r) {
                const int y = kv_visible(q, r - q.row0);
                for (int x = max(r * group, v0); x < min((r + 1) * group, v0 + VT); ++x) lds_seen[x - v0] = y;
            }
        }
        __syncthreads();
        end = 0;
        least = cap;
#pragma unroll
        for (int i = 0; i < VT; i += 64) {
            const int x = lds_seen[i + lane];
            end = max(end, x);
            least = x < 0 ? least : min(least, x);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            end = max(end, __shfl_xor(end, o, 64));
            least = min(least, __shfl_xor(least, o, 64));
        }
        end = min(cap, end);
        seen = lds_seen[32 * wave + n];
        __syncthreads();
    } else {
        const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
        if (s.bad && tid == 0) atomicOr(p.err + kErrBatch, 1u);
        const int vectors = s.rows * group;
        if (v0 >= vectors) return;
        if (part > 0 && j0 >= s.len) return;  // the join knows how many parts there are
        first_row = s.row0;
        cap = min(s.len, j0 + chunk);
        end = min(cap, kv_visible(s, p.group.div(min(v0 + VT, vectors) - 1)));
        least = min(cap, kv_visible(s, p.group.div(v0)));
        seen = v < vectors ? kv_visible(s, p.group.div(v)) : -1;
    }
    end = __builtin_amdgcn_readfirstlane(end);
    least = __builtin_amdgcn_readfirstlane(least);

    // queries, as the B operand: lane (n, hi) holds columns 16 s + 8 hi .. + 7 of its vector (vectors that
    // are none take the first row's)
    half8v qf[KS][QL];
    float unit = 1.0f;
    const int64_t row = first_row + p.group.div(seen >= 0 ? v : 0);
    const int head = h * group + p.group.mod(seen >= 0 ? v : 0);
    auto load_queries = [&] {
        QueryRow<KS, Q16> qr;
        load_query<KS, 16, false, Q16>(p, qr, row * p.ldq + (int64_t)head * p.c.dim, 8 * hi);
        float up = 1.0f;
        if constexpr (QL == 2) {
            // the row's largest value goes to [2^13, 2^14): the low parts stay normal, f32 rows of any size fit
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(query_at<KS, Q16>(qr, k, i)));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const int e = kv_clamp((int)((__float_as_uint(top) >> 23) & 0xff) - 127, -100, 126);
            up = __uint_as_float((uint32_t)(13 - e + 127) << 23);  // 2^(13 - e)
            unit = p.scale2 * kCodeUnit * __uint_as_float((uint32_t)(e - 13 + 127) << 23);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 z[QL];
                split_f16<QL>(query_at<KS, Q16>(qr, k, i) * up, z);
#pragma unroll
                for (int q = 0; q < QL; ++q) qf[k][q][i] = z[q];
            }
    };

    // a wave's shares lie in 16-token half `half(i)` of a tile; 64 columns take two waves only
    auto half = [&](int i) { return DP == 256 ? i : DP == 128 ? wave >> 1 : wave & 1; };
    const bool helps = DP > 64 || wave < 2;
    const bool scales = DP == 256 ? wave == 0 : DP == 128 ? (wave & 1) == 0 : wave < 2;  // these waves bring the scales
    const const_ids table = (const_ids)(uintptr_t)(p.b.table + seq * p.b.table_ld);
    const const_ids prefix = (const_ids)(uintptr_t)p.prefix_pages;
    const int off_mask = (1 << p.c.shift) - 1;
    bool bad_page = false;
    const int k_row = DP == 256 ? tid / 16 : tid % 128 / Sh::KCOLS % 16, k_at = k_row * DP + tid % Sh::KCOLS * 16;
    const int v_quad = DP == 256 ? wave : tid / Sh::VCOLS % 4, v_at = 4 * v_quad * DP + tid % Sh::VCOLS * 4;
    // A tile on its way: the page ids (loaded a step ahead of their use), the buffers, the bytes.
    int ids[Sh::SUBS];
    auto load_ids = [&](int j) {
#pragma unroll
        for (int i = 0; i < Sh::SUBS; ++i) {
            const int jt = min(j + 16 * half(i), end - 1);
            ids[i] = (SHARED || jt < p.prefix ? prefix : table)[jt >> p.c.shift];
        }
    };
    // Past the end the last page is read again, an id outside the cache reads page 0: all of that is masked or
    // made NaN.
    Half16<DP> at[Sh::SUBS];
    auto find = [&](int j) {
#pragma unroll
        for (int i = 0; i < Sh::SUBS; ++i) {
            const int jt = j + 16 * half(i);
            at[i] = find_half<DP>(p.c, ids[i], h, jt & off_mask, true);
            at[i].bad = at[i].bad && jt < end;
            bad_page |= at[i].bad;
        }
    };
    auto load_share = [&](Sh& sh) {
        if (DP == 64 && !helps) return;
#pragma unroll
        for (int i = 0; i < Sh::SUBS; ++i) {
            sh.bad[i] = at[i].bad;
            sh.k[i] = __builtin_bit_cast(uint4v, __builtin_amdgcn_raw_buffer_load_b128(at[i].block, k_at, at[i].k, 0));
#pragma unroll
            for (int x = 0; x < 4; ++x)
                sh.v[i][x] = __builtin_amdgcn_raw_buffer_load_b32(at[i].block, v_at + x * DP, at[i].v, 0);
            const int s = 4 * (lane & 15);
            sh.ks[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(at[i].block, s, at[i].ks, 0));
            sh.vs[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(at[i].block, s, at[i].vs, 0));
        }
    };
    const float key_unit = QL == 2 ? 1.0f : p.scale2 * kCodeUnit;
    // a share's way into the LDS, in pieces: 16 bytes of keys are two, four columns of values one each, then the scales
    constexpr int PIECES = 6 * Sh::SUBS;
    auto store_piece = [&](const Sh& sh, uint8_t* buf, int piece) {
        if (DP == 64 && !helps) return;
        const int i = piece / 6, x = piece % 6 - 2;
        if (x < 0) {
            uint8_t* to = buf + (16 * half(i) + k_row) * L::KROW + tid % Sh::KCOLS * 32 + 16 * (x + 2);
            *reinterpret_cast<half8v*>(to) = codes8(sh.k[i][2 * (x + 2)], sh.k[i][2 * (x + 2) + 1]);
        } else {
            // tokens 4 quad + 0..3 of the half: quad 2 b + h goes to place 8 h + 4 b of 16
            const int place = 16 * half(i) + 8 * (v_quad & 1) + 4 * (v_quad >> 1);
            const uint32_t sel = 0x0c000c00u | (4 + x) << 16 | x;
            const uint2v w = {codes2(sh.v[i][1], sh.v[i][0], sel), codes2(sh.v[i][3], sh.v[i][2], sel)};
            // column d is row d / ND of tile d % ND: a lane's columns of all tiles are neighbours
            const int d = tid % Sh::VCOLS * 4 + x;
            *reinterpret_cast<uint2v*>(buf + L::V + (d % ND * 32 + d / ND) * L::VROW + 2 * place) = w;
        }
    };
    auto store_scales = [&](const Sh& sh, uint8_t* buf) {
        if (!scales || lane >= 16) return;
#pragma unroll
        for (int i = 0; i < Sh::SUBS; ++i) {
            float* s = reinterpret_cast<float*>(buf + L::S) + 16 * half(i) + lane;
            const float inv = __builtin_amdgcn_rcpf(sh.vs[i]);
            s[0] = sh.bad[i] ? kNan : sh.ks[i] * key_unit;
            s[kTokens] = __builtin_amdgcn_logf(sh.vs[i]);
            s[2 * kTokens] = inv < __builtin_inff() ? inv : 0.0f;  // a token that is none adds 0 * 0, not 0 * inf
        }
    };

    float m = kNegInf, l = 0.0f, top = kNegInf;
    float16v x, o[ND];  // exponents of a tile: tokens 8 c + 4 hi + i of vector n; outputs
    half8v pf[2][LIMBS];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

    // The two phases of a step are written in the order that the instructions are to be issued in, held by
    // scheduling barriers: LDS reads early, and after each matrix instruction the vector work that runs beside it.
    auto pin = [] { __builtin_amdgcn_sched_barrier(0); };
    // P of elements 2 i and 2 i + 1 of x
    auto exponents = [&](int i, float base, const float4v* iv) {
        const float2v e = {__builtin_amdgcn_exp2f(x[2 * i] - base), __builtin_amdgcn_exp2f(x[2 * i + 1] - base)};
        l = __builtin_fmaf(e[0], iv[i / 2][2 * i % 4], l);
        l = __builtin_fmaf(e[1], iv[i / 2][2 * i % 4 + 1], l);
        const half2v z = __builtin_convertvector(e, half2v);
        pf[i / 4][0][2 * i % 8] = z[0];
        pf[i / 4][0][2 * i % 8 + 1] = z[1];
        if constexpr (LIMBS == 2) {
            const half2v w = __builtin_convertvector(e - __builtin_convertvector(z, float2v), half2v);
            pf[i / 4][1][2 * i % 8] = w[0];
            pf[i / 4][1][2 * i % 8 + 1] = w[1];
        }
    };
    // exponents from products, elements 2 i and 2 i + 1; MASK where some vector does not see all of the tile
    auto scale = [&](const float16v& s, int i, int left, const float4v* ks, const float4v* lv, auto mask) {
#pragma unroll
        for (int e = 2 * i; e < 2 * i + 2; ++e) {
            float z = s[e];
            if constexpr (QL == 2) z *= unit;
            z = __builtin_fmaf(z, ks[e / 4][e % 4], lv[e / 4][e % 4]);
            // masked tokens are chosen away, whatever their scales hold
            if constexpr (decltype(mask)::value) z = 8 * (e / 4) + e % 4 < left ? z : kNegInf;
            x[e] = z;
        }
        // the exponents are computed here, not where they are used next
        float t = top, a = x[2 * i], b = x[2 * i + 1];
        asm volatile("v_max3_f32 %0, %1, %2, %0" : "+v"(t), "+v"(a), "+v"(b));
        top = t;
        x[2 * i] = a;
        x[2 * i + 1] = b;
    };
    auto key = [&](const uint8_t* buf, int k) { return *reinterpret_cast<const half8v*>(buf + n * L::KROW + 16 * hi + 32 * k); };
    auto value = [&](const uint8_t* buf, int c, int t) {
        return *reinterpret_cast<const half8v*>(buf + L::V + (32 * t + n) * L::VROW + 16 * hi + 32 * c);
    };
    // scale factors of tokens 8 c + 4 hi + 0..3: 0 of the keys, 1 logarithms of the values', 2 their inverses
    auto factor = [&](const uint8_t* buf, int which, int c) {
        return *reinterpret_cast<const float4v*>(reinterpret_cast<const float*>(buf + L::S) + which * kTokens + 8 * c + 4 * hi);
    };
    // First P of tile u (its values lie in bu) beside the products of tile u + 1 (NEXT: its keys in bk). Then
    // the outputs of tile u beside the exponents of tile u + 1, at token j, and the way of tile u + 2 into bn.
    // The wave in the second goes first where both of a SIMD could issue, so that they do not run the same phase side
    // by side (the prompt of 4096 tokens 193 -> 178 us; in the first instead 182, in both 184).
    auto advance = [&](const uint8_t* bu, const uint8_t* bk, uint8_t* bn, Sh& sh, int j, auto next, auto mask) {
        constexpr bool NEXT = decltype(next)::value;
        constexpr int SV = 2 * ND;                                  // matrix steps of O
        constexpr int EP = (8 + KS - 1) / KS;                       // pairs of exponents beside a matrix step of S
        constexpr int FROM = SV >= 8 ? 1 : 0;                       // the products are on their way until then
        constexpr int SP = (8 + SV - FROM - 1) / (SV - FROM);       // pairs beside a matrix step of O
        constexpr int PP = (PIECES + SV - 1) / SV;
        constexpr int AHEAD = KS / 2 < ND ? KS / 2 : ND;            // operands on their way
        float4v iv[5], ks[5], lv[5];
        half8v kf[KS], vf[SV];
        float16v s;
        if constexpr (NEXT) {
#pragma unroll
            for (int k = 0; k < AHEAD; ++k) kf[k] = key(bk, k);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
        }
        iv[0] = factor(bu, 2, 0);
        pin();
        // the first pairs run while the keys are on their way
        const float base = m == kNegInf ? 0.0f : m - kPShift;
        exponents(0, base, iv);
        pin();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
#pragma unroll
            for (int i = k * EP; i < (k + 1) * EP; ++i)
                if (i < 8 && i % 2 == 0 && i / 2 < 3) iv[i / 2 + 1] = factor(bu, 2, i / 2 + 1);  // two pairs ahead
            if (NEXT && k + AHEAD < KS) kf[k + AHEAD] = key(bk, k + AHEAD);
            if (k >= KS - AHEAD) vf[k - (KS - AHEAD)] = value(bu, (k - (KS - AHEAD)) / ND, (k - (KS - AHEAD)) % ND);
            if (NEXT && k == KS - 1) {
                ks[0] = factor(bk, 0, 0);
                lv[0] = factor(bk, 1, 0);
            }
            if constexpr (NEXT)
#pragma unroll
                for (int q = 0; q < QL; ++q) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k], qf[k][q], s, 0, 0, 0);
#pragma unroll
            for (int i = k * EP + 1; i < (k + 1) * EP + 1; ++i)
                if (i < 8) exponents(i, base, iv);
            pin();
        }
        __builtin_amdgcn_s_setprio(1);
        if constexpr (NEXT) find(j + 2 * kTokens);
        top = kNegInf;
        const int left = min(seen, cap) - j - 4 * hi;
#pragma unroll
        for (int t = 0; t < SV; ++t) {
            if (t + AHEAD < SV) vf[t + AHEAD] = value(bu, (t + AHEAD) / ND, (t + AHEAD) % ND);
            if constexpr (NEXT) {
#pragma unroll
                for (int i = (t - FROM) * SP; i < (t - FROM + 1) * SP; ++i)
                    if (i >= 0 && i < 8 && i % 2 == 0 && i / 2 < 3) {
                        ks[i / 2 + 1] = factor(bk, 0, i / 2 + 1);
                        lv[i / 2 + 1] = factor(bk, 1, i / 2 + 1);
                    }
            }
#pragma unroll
            for (int q = 0; q < LIMBS; ++q) o[t % ND] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[t], pf[t / ND][q], o[t % ND], 0, 0, 0);
            if constexpr (NEXT) {
#pragma unroll
                for (int i = (t - FROM) * SP; i < (t - FROM + 1) * SP; ++i)
                    if (i >= 0 && i < 8) scale(s, i, left, ks, lv, mask);
#pragma unroll
                for (int i = t * PP; i < (t + 1) * PP; ++i)
                    if (i < PIECES) store_piece(sh, bn, i);
            }
            pin();
        }
        if constexpr (NEXT) store_scales(sh, bn);
        __builtin_amdgcn_s_setprio(0);
    };
    auto passed = [&] {  // some vector's maximum is to be raised
        typedef unsigned int pair __attribute__((ext_vector_type(2)));
        const pair r = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false));
        top = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        return __builtin_amdgcn_ballot_w64(top > m + kSlack) != 0;
    };
    auto raise = [&] {
        const float m_new = fmaxf(m, top);
        const float fade = m == m_new ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= fade;
#pragma unroll
        for (int t = 0; t < ND; ++t) o[t] *= fade;
    };

    if (j0 < end) {
        // the first three tiles' bytes are asked for together
        Sh sh, sh0, sh1;
        load_ids(j0);
        find(j0);
        load_share(sh0);
        load_ids(j0 + kTokens);
        find(j0 + kTokens);
        load_share(sh1);
        load_ids(j0 + 2 * kTokens);
        find(j0 + 2 * kTokens);
        load_share(sh);
        load_ids(j0 + 3 * kTokens);
        load_queries();
        auto store_share = [&](const Sh& sh, uint8_t* buf) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) store_piece(sh, buf, i);
            store_scales(sh, buf);
        };
        store_share(sh0, lds);
        store_share(sh1, lds + L::BYTES);
        __syncthreads();
        {
            float4v ks[4], lv[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                ks[c] = factor(lds, 0, c);
                lv[c] = factor(lds, 1, c);
            }
            float16v s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int q = 0; q < QL; ++q) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(key(lds, k), qf[k][q], s, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i) scale(s, i, min(seen, cap) - j0 - 4 * hi, ks, lv, std::true_type{});
        }
        if (passed()) raise();
        // tile u's values, tile u + 1's keys, tile u + 2's place
        int bu = 0, bk = L::BYTES, bn = 2 * L::BYTES;
        int j = j0;
        auto step = [&](auto mask) {
            advance(lds + bu, lds + bk, lds + bn, sh, j + kTokens, std::true_type{}, mask);
            load_share(sh);
            load_ids(j + 4 * kTokens);
            lds_barrier();  // the bytes of later tiles stay on their way
            const int t = bu;
            bu = bk;
            bk = bn;
            bn = t;
            j += kTokens;
        };
        // raising a maximum is rare and kept out of the loop, which leaves the outputs to the matrix core
        auto walk = [&](int stop, auto mask) {
            while (j < stop) {
                bool up;
                do {
                    step(mask);
                    up = passed();
                } while (!up && j < stop);
                if (up) raise();
            }
        };
        walk(least - 2 * kTokens + 1, std::false_type{});
        walk(end - kTokens, std::true_type{});
        advance(lds + bu, nullptr, nullptr, sh, 0, std::false_type{}, std::false_type{});
    }
    if (bad_page && lane == 0) atomicOr(p.err + kErrBatch, 1u);

    l += __shfl_xor(l, 32, 64);
    if (seen < 0) return;
    if (p.parts == 1) {
        const float f = l == 0.0f ? 0.0f : kCodeUnit / l;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float z[ND];
#pragma unroll
            for (int t = 0; t < ND; ++t) z[t] = o[t][i] * f;
            store_out<ND>(p, row * p.ldo + (int64_t)head * p.c.dim, (8 * (i / 4) + 4 * hi + i % 4) * ND, z);
        }
    } else {
        const int64_t slot = (row * p.q_heads + head) * p.parts + (SHARED ? 0 : p.prefix_parts) + part;
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int t = 0; t < ND; ++t) p.part_o[slot * DP + (8 * (i / 4) + 4 * hi + i % 4) * ND + t] = o[t][i];
        if (hi == 0) {
            p.part_ml[2 * slot] = m;
            p.part_ml[2 * slot + 1] = l;
        }
    }
}

template <int DP, int LIMBS, bool Q16, bool SHARED>
hipError_t launch_one(const AttendParams& p, hipStream_t st) {
    constexpr int bytes = 3 * TileLds<DP>::BYTES;
    // the LDS is asked for once on each device (those past 63: on every call), and again after a failure
    static std::atomic<uint64_t> asked{0};
    int device;
    if (const hipError_t e = hipGetDevice(&device)) return e;
    const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
    if (!(asked.load(std::memory_order_relaxed) & bit)) {
        if (const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&attend_wide_kernel<DP, LIMBS, Q16, SHARED>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, bytes))
            return e;
        asked.fetch_or(bit, std::memory_order_relaxed);
    }
    const int64_t tiles = SHARED ? p.by_prefix_tiles.d : p.by_tiles.d;
    const int64_t blocks = tiles * p.c.heads * (SHARED ? p.prefix_parts : (p.parts - p.prefix_parts) * (int64_t)p.b.seqs);
    attend_wide_kernel<DP, LIMBS, Q16, SHARED><<<dim3((uint32_t)blocks), kThreads, bytes, st>>>(p);
    return hipGetLastError();
}

template <int DP, bool SHARED>
hipError_t launch_typed(const AttendParams& p, hipStream_t st) {
    if (!p.q_f16) return launch_one<DP, 2, false, SHARED>(p, st);
    return p.o_f16 ? launch_one<DP, 1, true, SHARED>(p, st) : launch_one<DP, 2, true, SHARED>(p, st);
}

template <int DP>
hipError_t launch_dp(const AttendParams& p, bool prefix, hipStream_t st) {
    return prefix ? launch_typed<DP, true>(p, st) : launch_typed<DP, false>(p, st);
}

}  // namespace

hipError_t launch_attend_wide(const AttendParams& p, bool prefix, hipStream_t st) {
    switch (p.c.dim_padded) {
        case 64: return launch_dp<64>(p, prefix, st);
        case 128: return launch_dp<128>(p, prefix, st);
        default: return launch_dp<256>(p, prefix, st);
    }
}

}  // namespace qlin
