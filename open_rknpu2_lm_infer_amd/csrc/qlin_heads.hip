// Heads of query and key rows normalized and turned by their positions, and the same on the way into the cache.
//
//   n = x / sqrt(mean x^2 + eps) * gamma        a head's columns; without gamma n = x
//   y_l = a (n_l cos t - n_r sin t),  y_r = a (n_r cos t + n_l sin t)      t = position * w_i for pair i = (l, r)
//
// The angle is position * w_i quarter turns in 64 bits less the nearest whole number: what is left, at most half a
// quarter turn, is rounded to f32, off by 2^-26 of a quarter, and by position * 2^-51 more for the roundings of w_i and of the
// product in 64 bits, which pass the former from position 2^25 on (near 2^31 they are 2^-20).  The whole number's last two
// bits say which of (c, s), (-s, c), (-c, -s), (s, -c) it is.  sin and cos of up to an eighth of a turn are their
// series to the 9th and 10th power, the next terms being 2e-9 and 5e-10.  No table of positions is read: a workgroup
// computes its rows' factors, one a thread, into the LDS, from where the lanes of all their heads have them.
//
// A group of dim_padded / 8 lanes holds a head, 8 values a lane: four pairs, or eight of the columns that are not
// turned.  Every value is read by the lane that writes it, so rows may be worked on in place.  Keys on their way into
// the cache are laid down in the LDS and taken up again in the order of their columns, 8 a lane, which is what
// quantize_row wants.
//
// What bounds it (us, heads of 128, as graph nodes): memory for many f32 rows, 8192 of 40 heads, 336 MB, 63.6, 5.3 TB/s, what a
// copy reaches; as many fp16 rows take 38, 4.4 TB/s, their accesses being 8 bytes a lane; 4096 fp16 rows of 32 + 8 + 8 heads
// into the cache 20.4, 93 MB, with vector instructions issuing half of that time.  One row is latency: 2.8, and 3.8 into the
// cache (lengths, page id, values, angles one after the other).
#include "qlin_kv_rows.hpp"
#include "qlin_rope.hpp"

namespace qlin {
namespace {

typedef _Float16 half4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void turn(double quarters, float& c, float& s) {
    const double whole = __builtin_rint(quarters);
    const float f = (float)(quarters - whole), z = f * f;
    const int k = (int)whole;  // positions below 2^31 and at most a radian each: below 2^31
    // (pi/2)^n / n! with alternating signs
    float a = __builtin_fmaf(z, 1.6044118478735982e-4f, -4.681754135318687e-3f);
    a = __builtin_fmaf(z, a, 7.969262624616704e-2f);
    a = __builtin_fmaf(z, a, -6.4596409750624626e-1f);
    a = __builtin_fmaf(z, a, 1.5707963267948966f) * f;
    float b = __builtin_fmaf(z, -2.5202042373060605e-5f, 9.192602748394264e-4f);
    b = __builtin_fmaf(z, b, -2.0863480763352961e-2f);
    b = __builtin_fmaf(z, b, 2.5366950790104803e-1f);
    b = __builtin_fmaf(z, b, -1.2337005501361697f);
    b = __builtin_fmaf(z, b, 1.0f);
    c = k & 1 ? a : b;
    s = k & 1 ? b : a;
    c = (k + 1) & 2 ? -c : c;
    s = k & 2 ? -s : s;
}

// Columns of a lane's eight values: blocks of four at a and b.
struct Blocks {
    int a, b;
    bool has_a, has_b;
};

// A lane's eight values on their way, as they lie in memory: what converts them waits for them.
template <typename T, bool VEC>
struct Raw {
    uint32_t w[VEC ? 2 * sizeof(T) : 8];
};
template <typename T, bool VEC>
__device__ __forceinline__ float raw_at(const Raw<T, VEC>& r, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[j]);
    else if constexpr (VEC) return f32_of_f16_bits(r.w[j / 2] >> (16 * (j % 2)));
    else return f32_of_f16_bits(r.w[j]);
}

// BITS 0: rows with positions.  8, 4: rows of a batch, into a cache of that width.  VEC: blocks of four columns are whole
// and aligned.  WIDE: twice the lanes a head.
template <int DP, bool WIDE, typename T, bool VEC, int BITS>
__global__ __launch_bounds__(256) void heads_kernel(HeadsParams p) {
    constexpr int LPH = DP / 8 * (WIDE ? 2 : 1), GROUPS = 256 / LPH;
    constexpr int AHEAD = VEC ? 2 : 1;  // heads of a group that are on their way
    __shared__ __align__(16) float angles[4][DP];  // cosine and sine of the pairs of a row
    __shared__ __align__(16) float keys[BITS ? GROUPS : 1][BITS ? DP + 4 : 4];
    const int lane = threadIdx.x % LPH, group = threadIdx.x / LPH;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // rows row0 .. row0 + rows - 1, at positions pos0 .. (batch)
    int block = blockIdx.x;
    if constexpr (BITS != 0) {
        // workgroups go to the 8 XCDs in turn: those of neighbouring rows to one of them, in whose L2 the scales of a page's
        // tokens come together
        const int xcd = block % 8, all = gridDim.x;
        block = xcd * (all / 8) + min(xcd, all % 8) + block / 8;
    }
    const int unit = p.by_splits.div(block), split = p.by_splits.mod(block);
    int64_t row0;
    int rows, pos0 = 0, seq = 0;
    bool bad = false;
    if constexpr (BITS == 0) {
        row0 = (int64_t)unit * p.block_rows;
        rows = (int)min((int64_t)p.block_rows, p.rows - row0);
    } else {
        seq = p.by_new.div(unit);
        const int t = p.by_new.mod(unit) * p.block_rows;
        const KvSeq s = kv_seq(p.b.row_start, p.b.length, seq, p.b.rows, p.b.max_new, p.b.max_len);
        bad = s.bad;
        if (t >= s.rows) {
            if (bad && threadIdx.x == 0) atomicOr(p.err + kErrBatch, 1u);
            return;
        }
        row0 = s.row0 + t;
        rows = min(p.block_rows, s.rows - t);
        pos0 = s.len - s.rows + t;
    }
    const bool by_wave = p.block_rows > 1;
    const int r = by_wave ? wave : 0;  // this group's row
    const bool works = r < rows;
    const int64_t row = row0 + r;

    // the columns of queries and keys: pairs first, then those that are not turned
    const int pairs = p.rope.rotary / 2, first = p.rope.first;
    const int turned = (pairs + 3) / 4;
    const bool turns = lane < turned;
    const int e0 = 8 * (lane - turned), rest = p.dim - p.rope.rotary;
    auto column = [&](int j) {  // of value j, -1: none
        if (turns) {
            if (p.rope.interleaved) return 8 * lane + j < p.rope.rotary ? first + 8 * lane + j : -1;
            const int i = 4 * lane + j % 4;
            return i < pairs ? first + i + (j < 4 ? 0 : pairs) : -1;
        }
        const int e = e0 + j;
        return e < rest ? (e < first ? e : e + p.rope.rotary) : -1;
    };
    const Blocks straight = {8 * lane, 8 * lane + 4, 8 * lane < p.dim, 8 * lane + 4 < p.dim};
    const Blocks qk = VEC ? Blocks{max(column(0), 0), max(column(4), 0), column(0) >= 0, column(4) >= 0} : straight;

    constexpr int PER_WAVE = 64 / LPH;
    const int heads = p.q_heads + (BITS ? 2 : 1) * p.k_heads;
    const int step = p.splits * (by_wave ? PER_WAVE : GROUPS);
    // Without a branch, of a head and columns that are there: no load waits for another.
    const int64_t from = (row0 + min(r, rows - 1)) * p.ldx;
    auto load = [&](int h, Raw<T, VEC>& x) {
        h = min(h, heads - 1);
        const T* at = reinterpret_cast<const T*>(p.x) + from + (int64_t)h * p.dim;
        const bool value = BITS && h >= p.q_heads + p.k_heads;
        if constexpr (VEC) {
            constexpr int N = sizeof(T);  // words of a block
            typedef uint32_t block_t __attribute__((ext_vector_type(N)));
            const Blocks b = value ? straight : qk;
            const block_t y = *reinterpret_cast<const block_t*>(at + (b.has_a ? b.a : 0));
            const block_t z = *reinterpret_cast<const block_t*>(at + (b.has_b ? b.b : 0));
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x.w[i] = y[i];
                x.w[N + i] = z[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = value ? min(8 * lane + j, p.dim - 1) : max(column(j), 0);
                if constexpr (sizeof(T) == 2) x.w[j] = reinterpret_cast<const uint16_t*>(at)[c];
                else x.w[j] = reinterpret_cast<const uint32_t*>(at)[c];
            }
        }
    };

    // the first heads' values and the norms' factors do not wait for the angles
    int h = by_wave ? split * PER_WAVE + group % PER_WAVE : split * GROUPS + group;
    Raw<T, VEC> raw[AHEAD + 1];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(h + i * step, raw[i]);
    float g[2][8] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float* gamma = k ? p.k_gamma : p.q_gamma;
        if (!gamma) continue;
        if constexpr (VEC) {
            const float4v y = *reinterpret_cast<const float4v*>(gamma + qk.a), z = *reinterpret_cast<const float4v*>(gamma + qk.b);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                g[k][j] = y[j];
                g[k][4 + j] = z[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) g[k][j] = gamma[max(column(j), 0)];
        }
    }
    for (int k = threadIdx.x; k < rows * pairs; k += 256) {
        const int y = p.by_pairs.div(k), i = p.by_pairs.mod(k);
        int pos = pos0 + y;
        if constexpr (BITS == 0) pos = p.positions[row0 + y];
        float c, s;
        turn(pos * p.rope.quarters[i], c, s);
        angles[y][2 * i] = c * p.rope.amplitude;
        angles[y][2 * i + 1] = s * (p.inverse ? -p.rope.amplitude : p.rope.amplitude);
    }
    int off = 0, page = -1;
    if constexpr (BITS != 0) {
        const int pos = pos0 + r;
        off = pos & ((1 << p.c.shift) - 1);
        // nothing is stored of a sequence whose row starts or length are at fault
        if (!bad && works && pos >= 0) {
            const int id = kv_page(p.b.table[seq * p.b.table_ld + (pos >> p.c.shift)], p.c.pages, &bad);
            page = bad ? -1 : id;
        }
    }
    __syncthreads();
    float co[4] = {}, si[4] = {};
    if (turns && works) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = 2 * (VEC ? 4 * lane + i : min(4 * lane + i, pairs - 1));
            co[i] = angles[r][at];
            si[i] = angles[r][at + 1];
        }
    }

    bool finite = true;
    for (int done = 0; done < heads; done += step) {
        // (past the end the last head again: a branch here makes every load be waited for at once, the prompt's pass 37 us and
        // not 32; single columns, which are eight loads, have it)
        if (VEC || done + AHEAD * step < heads) load(h + AHEAD * step, raw[AHEAD]);
        const bool query = h < p.q_heads, value = BITS && h >= p.q_heads + p.k_heads;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            bool there;
            if constexpr (VEC) there = value ? (j < 4 ? straight.has_a : straight.has_b) : (j < 4 ? qk.has_a : qk.has_b);
            else there = value ? 8 * lane + j < p.dim : column(j) >= 0;
            x[j] = there ? raw_at<T, VEC>(raw[0], j) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) raw[i] = raw[i + 1];
        const int head = h;
        h += step;
        if (!works || head >= heads) continue;
        if (!value) {
            if (query ? p.q_gamma != nullptr : p.k_gamma != nullptr) {
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], x[j], sum);
                sum = lanes_sum<LPH>(sum);
                // at least the smallest normal number: what v_rsq_f32 gives for less is no number to scale zeros by.  (A
                // NaN stays one.)
                const float m = __builtin_fmaf(sum, p.inv_dim, p.eps), f = __builtin_amdgcn_rsqf(m < 0x1p-126f ? 0x1p-126f : m);
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = (x[j] * f) * (query ? g[0][j] : g[1][j]);
            }
            if (turns) {
                auto rotate = [&](float& l, float& r, int i) {
                    const float y = __builtin_fmaf(l, co[i], -(r * si[i]));
                    r = __builtin_fmaf(r, co[i], l * si[i]);
                    l = y;
                };
                if (p.rope.interleaved) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) rotate(x[2 * i], x[2 * i + 1], i);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) rotate(x[i], x[4 + i], i);
                }
            }
        }
        if (BITS == 0 || query) {
            const int64_t at = row * p.ldy + (int64_t)head * p.dim;
            if constexpr (VEC) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (!(k ? qk.has_b : qk.has_a)) continue;
                    const int64_t c = at + (k ? qk.b : qk.a);
                    const float* y = x + 4 * k;
                    if (p.y_f16)
                        *reinterpret_cast<half4v*>(reinterpret_cast<_Float16*>(p.y) + c) =
                            half4v{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
                    else
                        *reinterpret_cast<float4v*>(reinterpret_cast<float*>(p.y) + c) = float4v{y[0], y[1], y[2], y[3]};
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = column(j);
                    if (c < 0) continue;
                    if (p.y_f16) reinterpret_cast<_Float16*>(p.y)[at + c] = (_Float16)x[j];
                    else reinterpret_cast<float*>(p.y)[at + c] = x[j];
                }
            }
        } else if constexpr (BITS != 0) {
            const KvBlock<DP, BITS> blk(p.c, max(page, 0), head - p.q_heads - (value ? p.k_heads : 0));
            const int d0 = 8 * lane;
            if (!value) {
                // a head's lanes are of one wave, whose accesses to the LDS are done in their order
                float* to = keys[group];
                if constexpr (VEC) {
                    if (qk.has_a) *reinterpret_cast<float4v*>(to + qk.a) = float4v{x[0], x[1], x[2], x[3]};
                    if (qk.has_b) *reinterpret_cast<float4v*>(to + qk.b) = float4v{x[4], x[5], x[6], x[7]};
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (const int c = column(j); c >= 0) to[c] = x[j];
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                if constexpr (VEC) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float4v y = *reinterpret_cast<const float4v*>(to + d0 + 4 * k);
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[4 * k + j] = d0 + 4 * k < p.dim ? y[j] : 0.0f;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = d0 + j < p.dim ? to[min(d0 + j, DP - 1)] : 0.0f;
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
            if (d0 < DP) {
                const bool fin = value ? quantize_row<DP, BITS, true>(blk, off, d0, x, p.rne, page >= 0)
                                       : quantize_row<DP, BITS, false>(blk, off, d0, x, p.rne, page >= 0);
                finite &= fin || page < 0;
            }
        }
    }
    if constexpr (BITS != 0) {
        if (bad && threadIdx.x % 64 == 0) atomicOr(p.err + kErrBatch, 1u);
        if (!finite) atomicOr(p.err + kErrNonfinite, 1u);
    }
}

template <int DP, int BITS, typename T>
hipError_t launch_typed(const HeadsParams& p, dim3 grid, hipStream_t st) {
    if (heads_vec(p)) heads_kernel<DP, false, T, true, BITS><<<grid, 256, 0, st>>>(p);
    else if (heads_wide(p)) heads_kernel<DP, true, T, false, BITS><<<grid, 256, 0, st>>>(p);
    else heads_kernel<DP, false, T, false, BITS><<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

template <int BITS>
hipError_t launch_bits(const HeadsParams& p, dim3 grid, hipStream_t st) {
    switch (p.dim <= 64 ? 64 : p.dim <= 128 ? 128 : 256) {
        case 64: return p.x_f16 ? launch_typed<64, BITS, __half>(p, grid, st) : launch_typed<64, BITS, float>(p, grid, st);
        case 128: return p.x_f16 ? launch_typed<128, BITS, __half>(p, grid, st) : launch_typed<128, BITS, float>(p, grid, st);
        default: return p.x_f16 ? launch_typed<256, BITS, __half>(p, grid, st) : launch_typed<256, BITS, float>(p, grid, st);
    }
}

int lanes(const HeadsParams& p) { return p.dim <= 64 ? 8 : p.dim <= 128 ? 16 : 32; }

}  // namespace

bool heads_vec(const HeadsParams& p) { return p.vec && p.dim % 4 == 0 && p.rope.rotary % 8 == 0 && p.rope.first % 4 == 0; }
bool heads_wide(const HeadsParams& p) {
    return (p.rope.rotary / 2 + 3) / 4 + (p.dim - p.rope.rotary + 7) / 8 > lanes(p);
}
int heads_at_once(const HeadsParams& p) { return 64 / (lanes(p) * (heads_wide(p) ? 2 : 1)); }

hipError_t launch_heads(const HeadsParams& p, hipStream_t st) {
    return launch_bits<0>(p, dim3((uint32_t)(((int64_t)p.rows + p.block_rows - 1) / p.block_rows * p.splits)), st);
}
hipError_t launch_heads_append(const HeadsParams& p, hipStream_t st) {
    const dim3 grid((uint32_t)((int64_t)p.b.seqs * p.by_new.d * p.splits));
    return p.c.bits == 4 ? launch_bits<4>(p, grid, st) : launch_bits<8>(p, grid, st);
}

}  // namespace qlin
