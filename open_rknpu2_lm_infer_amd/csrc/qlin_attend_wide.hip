// Attention of many rows over the 8-bit key/value cache: prompts, chunks of prompts, and the shared
// prefix of a batch.  The formulas are those of qlin_attend.hip.
//
// A workgroup holds 128 vectors, 32 a wave, and walks over its tokens 64 at a time.  The bytes of a
// tile are loaded a tile ahead, made into fp16 codes once for the four waves and laid down in the LDS:
// keys as they are, values transposed.  The matrix core's result layout of S^T = K Q^T (a lane holds
// four tokens of every eight of one vector) is the operand layout of O^T = V^T P^T with its k axis
// permuted, so the values' tokens are written in that order and P never leaves its lane.
#include "qlin_attend.hpp"

#include <type_traits>

namespace qlin {
namespace {

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr int kTokens = 64;   // of a tile
constexpr int kThreads = 256;

// LDS of one tile.  Rows are padded by 16 bytes: eight lanes' 16-byte accesses to eight rows then
// fall into different banks.
template <int DP>
struct TileLds {
    static constexpr int KROW = 2 * DP + 16, VROW = 2 * kTokens + 16;
    static constexpr int V = kTokens * KROW, S = V + DP * VROW, BYTES = S + 3 * kTokens * 4;
};

// A thread's share of a tile on its way from the cache to the LDS.
template <int DP>
struct Share {
    static constexpr int KP = kTokens * DP / 16 / kThreads > 0 ? kTokens * DP / 16 / kThreads : 1;  // 16 bytes of a key each
    static constexpr int VT = 8 * (DP / 4);                                                      // 8 tokens x 4 columns each
    static constexpr int VP = VT / kThreads > 0 ? VT / kThreads : 1;
    uint4v k[KP];
    uint32_t v[VP][8];
    float ks, vs;
    bool bad;
};

// Rows of the tile that a thread's shares lie in.
template <int DP>
__device__ __forceinline__ int key_row(int i) { return (threadIdx.x + i * kThreads) / (DP / 16); }
template <int DP>
__device__ __forceinline__ int value_group(int i) { return (threadIdx.x + i * kThreads) / (DP / 4); }  // 2 c + h

template <int DP, int LIMBS, bool Q16, bool SHARED>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void attend_wide_kernel(AttendParams p) {
    using L = TileLds<DP>;
    using Sh = Share<DP>;
    constexpr int KS = DP / 16, ND = DP / 32;
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
    const int v0 = ((int)by_tiles.d - 1 - by_tiles.mod(b)) * kAttendWide;
    b = by_tiles.div(b);
    const int seq = SHARED ? 0 : p.by_seqs.mod(b), part = SHARED ? b : p.by_seqs.div(b);

    // how many tokens each vector sees (-1: no vector)
    int first_row = 0, cap, end, seen;
    const int j0 = (SHARED ? 0 : p.own_from) + part * chunk;
    const int v = v0 + 32 * wave + n;
    if constexpr (SHARED) {
        int* lds_seen = reinterpret_cast<int*>(lds);  // before the first tile
        cap = min(p.prefix, j0 + chunk);
        if (tid < kAttendWide) lds_seen[tid] = -1;
        __syncthreads();
        const int r_lo = p.group.div(v0), r_hi = min(p.group.div(v0 + kAttendWide - 1) + 1, p.b.rows);
        for (int i = tid; i < p.b.seqs; i += kThreads) {
            const KvSeq q = kv_seq(p.b.row_start, p.b.length, i, p.b.rows, p.b.max_new, p.b.max_len);
            for (int r = max(q.row0, r_lo); r < min(q.row0 + q.rows, r_hi); ++r) {
                const int y = kv_visible(q, r - q.row0);
                for (int x = max(r * group, v0); x < min((r + 1) * group, v0 + kAttendWide); ++x) lds_seen[x - v0] = y;
            }
        }
        __syncthreads();
        seen = lds_seen[32 * wave + n];
        end = max(lds_seen[lane], lds_seen[lane + 64]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) end = max(end, __shfl_xor(end, o, 64));
        end = min(cap, end);
        __syncthreads();
    } else {
        const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
        if (s.bad && tid == 0) atomicOr(p.err, kErrBatch);
        if (v0 >= s.rows * group) return;
        if (part > 0 && j0 >= s.len) return;  // the join knows how many parts there are
        first_row = s.row0;
        cap = min(s.len, j0 + chunk);
        end = min(cap, kv_visible(s, p.group.div(min(v0 + kAttendWide - 1, s.rows * group - 1))));
        seen = v < s.rows * group ? kv_visible(s, p.group.div(v)) : -1;
    }
    end = __builtin_amdgcn_readfirstlane(end);
    int most = seen, least = seen < 0 ? 0x7fffffff : seen;  // over the wave's vectors
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        most = max(most, __shfl_xor(most, o, 64));
        least = min(least, __shfl_xor(least, o, 64));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(min(least, cap));

    // page ids of the tile at token j, then its bytes; tokens past the end repeat the last one
    const int32_t* table = p.b.table + seq * p.b.table_ld;
    const int off_mask = (1 << p.c.shift) - 1;
    auto id_of = [&](int tok) {
        return (SHARED || tok < p.prefix ? p.prefix_pages : table)[tok >> p.c.shift];
    };
    auto token = [&](int j, int row) { return min(j + row, end - 1); };
    int id_k[Sh::KP], id_v[Sh::VP], id_s;
    auto load_ids = [&](int j) {
#pragma unroll
        for (int i = 0; i < Sh::KP; ++i) id_k[i] = id_of(token(j, key_row<DP>(i) % kTokens));
#pragma unroll
        for (int i = 0; i < Sh::VP; ++i) id_v[i] = id_of(token(j, value_group<DP>(i) % 8 / 2 * 16));
        id_s = id_of(token(j, lane));
    };
    bool bad_page = false;
    Sh sh;
    auto load_share = [&](int j) {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < Sh::KP; ++i) {
            const KvBlock<DP> blk(p.c, kv_page(id_k[i], p.c.pages, &bad), h);
            const int tok = token(j, key_row<DP>(i) % kTokens);
            sh.k[i] = *reinterpret_cast<const uint4v*>(blk.k(tok & off_mask) + (tid + i * kThreads) % (DP / 16) * 16);
        }
#pragma unroll
        for (int i = 0; i < Sh::VP; ++i) {
            const KvBlock<DP> blk(p.c, kv_page(id_v[i], p.c.pages, &bad), h);
            // tokens 16 c + 4 h + {0..3} and 8 more; a 16-token group lies in one page, those past
            // the end in its last rows or in the last token's page
            const int g = value_group<DP>(i) % 8, t0 = j + g / 2 * 16;
            const int off = (t0 < end ? t0 : (end - 1) & ~15) & off_mask;
#pragma unroll
            for (int x = 0; x < 8; ++x)
                sh.v[i][x] = *reinterpret_cast<const uint32_t*>(blk.v(off + 4 * (g & 1) + x + (x & 4)) + (tid + i * kThreads) % (DP / 4) * 4);
        }
        sh.bad = false;
        const KvBlock<DP> blk(p.c, kv_page(id_s, p.c.pages, &sh.bad), h);
        const int tok = token(j, lane) & off_mask;
        sh.ks = *blk.ks(tok);
        sh.vs = *blk.vs(tok);
        bad_page |= sh.bad;
    };
    const float key_unit = LIMBS == 2 ? 1.0f : p.scale2 * kCodeUnit;
    auto store_share = [&](uint8_t* buf) {
#pragma unroll
        for (int i = 0; i < Sh::KP; ++i) {
            if (kTokens * DP / 16 < kThreads && tid >= kTokens * DP / 16) break;
            uint8_t* at = buf + key_row<DP>(i) * L::KROW + (tid + i * kThreads) % (DP / 16) * 32;
            *reinterpret_cast<half8v*>(at) = codes8(sh.k[i][0], sh.k[i][1]);
            *reinterpret_cast<half8v*>(at + 16) = codes8(sh.k[i][2], sh.k[i][3]);
        }
#pragma unroll
        for (int i = 0; i < Sh::VP; ++i) {
            if (Sh::VT < kThreads && tid >= Sh::VT) break;
            const int g = value_group<DP>(i), c0 = (tid + i * kThreads) % (DP / 4) * 4;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t sel = 0x0c000c00u | (4 + x) << 16 | x;
                const uint4v w = {codes2(sh.v[i][1], sh.v[i][0], sel), codes2(sh.v[i][3], sh.v[i][2], sel),
                                  codes2(sh.v[i][5], sh.v[i][4], sel), codes2(sh.v[i][7], sh.v[i][6], sel)};
                // column d is row d / ND of tile d % ND: a lane's columns of all tiles are neighbours
                const int d = c0 + x;
                *reinterpret_cast<uint4v*>(buf + L::V + (d % ND * 32 + d / ND) * L::VROW + g * 16) = w;
            }
        }
        if (tid < kTokens) {
            float* s = reinterpret_cast<float*>(buf + L::S);
            s[tid] = sh.bad ? kNan : sh.ks * key_unit;
            s[kTokens + tid] = __builtin_amdgcn_logf(sh.vs);
            s[2 * kTokens + tid] = __builtin_amdgcn_rcpf(sh.vs);
        }
    };

    // queries, as the B operand: lane (n, hi) holds columns 16 s + 8 hi .. + 7 of vector n (vectors that are
    // none take the first row's)
    half8v qf[KS][LIMBS];
    float unit = 1.0f;
    const bool ok = seen >= 0;
    const int64_t row = first_row + p.group.div(ok ? v : 0);
    const int head = h * group + p.group.mod(ok ? v : 0);
    {
        QueryRow<KS, Q16> qr;
        load_query<KS, 16, Q16>(p, qr, row * p.ldq + (int64_t)head * p.c.dim, 8 * hi);
        float up = 1.0f;
        if constexpr (LIMBS == 2) {
            // the row's largest value goes to [2^13, 2^14): the low parts stay normal, f32 rows of any size fit
            float m = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(query_at<KS, Q16>(qr, k, i)));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const int e = kv_clamp((int)((__float_as_uint(m) >> 23) & 0xff) - 127, -100, 126);
            up = __uint_as_float((uint32_t)(13 - e + 127) << 23);  // 2^(13 - e)
            unit = p.scale2 * kCodeUnit * __uint_as_float((uint32_t)(e - 13 + 127) << 23);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                _Float16 y[LIMBS];
                split_f16<LIMBS>(query_at<KS, Q16>(qr, k, i) * up, y);
#pragma unroll
                for (int q = 0; q < LIMBS; ++q) qf[k][q][i] = y[q];
            }
    }

    float m = kNegInf, l = 0.0f;
    float16v o[ND];
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

    // 32 tokens of a tile, at + 0 ..: MASK where some vector does not see all of them.
    auto work = [&](const uint8_t* buf, int at, int j, auto mask) {
        constexpr bool MASK = decltype(mask)::value;
        const int left = min(seen, cap) - j - 4 * hi;  // MASK: of the lane's tokens, 8 c + i each
        const uint8_t* kb = buf + (at + n) * L::KROW + 16 * hi;
        const uint8_t* vb = buf + L::V + n * L::VROW + 2 * at + 16 * hi;
        const float* sc = reinterpret_cast<const float*>(buf + L::S) + at + 4 * hi;
        float16v s;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const half8v a = *reinterpret_cast<const half8v*>(kb + 32 * k);
#pragma unroll
            for (int q = 0; q < LIMBS; ++q) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qf[k][q], s, 0, 0, 0);
        }
        float top = kNegInf;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float4v ks = *reinterpret_cast<const float4v*>(sc + 8 * c), lv = *reinterpret_cast<const float4v*>(sc + kTokens + 8 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x = s[4 * c + i];
                if constexpr (LIMBS == 2) x *= unit;
                x = __builtin_fmaf(x, ks[i], lv[i]);
                // masked tokens are chosen away, whatever their scales hold
                if constexpr (MASK) x = 8 * c + i < left ? x : kNegInf;
                s[4 * c + i] = x;
                top = fmaxf(top, x);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {
            const float m_new = fmaxf(m, top);
            const float fade = m == m_new ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            m = m_new;
            l *= fade;
#pragma unroll
            for (int t = 0; t < ND; ++t) o[t] *= fade;
        }
        const float base = m == kNegInf ? 0.0f : m - kPShift;
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // 16 tokens
            half8v pf[LIMBS];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const float4v iv = *reinterpret_cast<const float4v*>(sc + 2 * kTokens + 16 * c + 8 * y);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[8 * c + 4 * y + i] - base);
                    if constexpr (MASK) l = 16 * c + 8 * y + i < left ? __builtin_fmaf(e, iv[i], l) : l;
                    else l = __builtin_fmaf(e, iv[i], l);
                    _Float16 z[LIMBS];
                    split_f16<LIMBS>(e, z);
#pragma unroll
                    for (int q = 0; q < LIMBS; ++q) pf[q][4 * y + i] = z[q];
                }
            }
#pragma unroll
            for (int t = 0; t < ND; ++t) {
                const half8v a = *reinterpret_cast<const half8v*>(vb + 32 * t * L::VROW + 32 * c);
#pragma unroll
                for (int q = 0; q < LIMBS; ++q) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pf[q], o[t], 0, 0, 0);
            }
        }
    };

    if (j0 < end) {
        load_ids(j0);
        load_share(j0);
        load_ids(j0 + kTokens);
        store_share(lds);
        __syncthreads();
        int buf = 0;
        for (int j = j0; j < end; j += kTokens) {
            const bool more = j + kTokens < end;
            if (more) {
                load_share(j + kTokens);
                load_ids(j + 2 * kTokens);
            }
#pragma unroll 1
            for (int t = 0; t < kTokens && j + t < most; t += 32) {
                if (j + t + 32 <= least) work(lds + buf, t, j + t, std::false_type{});
                else work(lds + buf, t, j + t, std::true_type{});
            }
            buf ^= L::BYTES;
            if (more) store_share(lds + buf);
            __syncthreads();
        }
    }
    if (bad_page && tid < kTokens) atomicOr(p.err, kErrBatch);

    l += __shfl_xor(l, 32, 64);
    if (!ok) return;
    if (p.parts == 1) {
        const float f = l == 0.0f ? 0.0f : kCodeUnit / l;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float y[ND];
#pragma unroll
            for (int t = 0; t < ND; ++t) y[t] = o[t][i] * f;
            store_out<ND>(p, row * p.ldo + (int64_t)head * p.c.dim, (8 * (i / 4) + 4 * hi + i % 4) * ND, y);
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
    constexpr int bytes = 2 * TileLds<DP>::BYTES;
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&attend_wide_kernel<DP, LIMBS, Q16, SHARED>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (attr != hipSuccess) return attr;
    const int64_t tiles = ((int64_t)(SHARED ? p.b.rows : p.b.max_new) * p.group.d + kAttendWide - 1) / kAttendWide;
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
