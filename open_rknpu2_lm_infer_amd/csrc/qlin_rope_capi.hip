// C ABI of rotary positions: the handle with its frequencies, and the calls on plain rows.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <new>

#include "../../include/qlinear.h"
#include "qlin_rope_handle.hpp"

using namespace qlin;

namespace {

constexpr double kTwoPi = 6.283185307179586;

// Radians a position adds to pair i of n / 2.
double frequency(const qlin_rope_config& g, int i) {
    const double n = g.rotary_dim;
    double base = g.base;
    if (g.scaling == QLIN_ROPE_BASE && g.rotary_dim > 2) base *= std::pow(g.factor, n / (n - 2));
    const double w = std::pow(base, -2.0 * i / n);
    double kept = 1.0;  // how much of the frequency is not divided by the factor
    if (g.scaling == QLIN_ROPE_LINEAR) {
        kept = 0.0;
    } else if (g.scaling == QLIN_ROPE_BANDS) {
        kept = std::clamp((g.original_len * w / kTwoPi - g.low) / (g.high - g.low), 0.0, 1.0);
    } else if (g.scaling == QLIN_ROPE_RAMP) {
        const auto pair = [&](double turns) { return n * std::log(g.original_len / (turns * kTwoPi)) / (2 * std::log(base)); };
        const double lo = std::max(std::floor(pair(g.high)), 0.0), hi = std::min(std::ceil(pair(g.low)), n - 1);
        kept = 1.0 - std::clamp((i - lo) / std::max(hi - lo, 0.001), 0.0, 1.0);
    }
    if (g.scaling == QLIN_ROPE_PLAIN || g.scaling == QLIN_ROPE_BASE) return w;
    return w * (kept + (1.0 - kept) / g.factor);
}

bool good(const qlin_rope_config& g) {
    if (g.head_dim <= 0 || g.rotary_dim <= 0 || g.rotary_dim % 2 || g.first < 0 || g.first > g.head_dim - g.rotary_dim ||
        (g.layout != QLIN_ROPE_HALF && g.layout != QLIN_ROPE_INTERLEAVED) || g.scaling < QLIN_ROPE_PLAIN ||
        g.scaling > QLIN_ROPE_RAMP || !std::isfinite(g.base) || !(g.base > 1.0) || !(g.amplitude >= 0.0) ||
        g.amplitude > (double)std::numeric_limits<float>::max())
        return false;
    if (g.scaling == QLIN_ROPE_PLAIN) return true;
    if (!std::isfinite(g.factor) || !(g.factor >= 1.0)) return false;
    if (g.scaling != QLIN_ROPE_BANDS && g.scaling != QLIN_ROPE_RAMP) return true;
    return std::isfinite(g.original_len) && g.original_len > 0.0 && std::isfinite(g.low) && std::isfinite(g.high) && g.low > 0.0 &&
           g.high > g.low;
}

bool is_dtype(int32_t t) { return t == QLIN_F32 || t == QLIN_F16; }

int run(const qlin_rope* rope, int32_t rows, int32_t dim, int32_t q_heads, int32_t k_heads, const float* q_gamma, const float* k_gamma,
        float eps, const void* X, int32_t x_dtype, int64_t ldx, const int32_t* positions, void* Y, int32_t y_dtype, int64_t ldy,
        uint32_t flags, void* stream) {
    const int64_t heads = (int64_t)q_heads + k_heads, cols = heads * dim;
    if (rows < 0 || dim <= 0 || q_heads < 0 || k_heads < 0 || heads <= 0 || !is_dtype(x_dtype) || !is_dtype(y_dtype) || ldx < cols ||
        ldy < cols || (flags & ~QLIN_ROPE_INVERSE) || (rows > 0 && (!X || !Y || (rope && !positions))) || (rope && rope->dim != dim))
        return QLIN_ERR_PARAM;
    if ((q_gamma || k_gamma) && !(eps > 0.0f && std::isfinite(eps))) return QLIN_ERR_PARAM;
    if (dim > kKvMaxDim || heads > kKvMaxHeads || rows > kKvMaxGrid) return QLIN_ERR_UNSUPPORTED;
    int device;
    if (hipGetDevice(&device) != hipSuccess) return QLIN_ERR_NODEVICE;
    if (rope && rope->device != device) return QLIN_ERR_PARAM;
    if (rows == 0) return QLIN_OK;
    HeadsParams p{};
    heads_common(&p, rope, dim, q_heads, k_heads, q_gamma, k_gamma, eps, X, x_dtype == QLIN_F16, ldx, Y, y_dtype == QLIN_F16, ldy);
    p.inverse = (flags & QLIN_ROPE_INVERSE) != 0;
    p.rows = rows;
    p.positions = positions;
    heads_split(&p, 1, rows, (int)heads);
    return launch_heads(p, (hipStream_t)stream) == hipSuccess ? QLIN_OK : QLIN_ERR_DEVICE;
}

}  // namespace

namespace qlin {

void heads_common(HeadsParams* p, const qlin_rope* rope, int dim, int q_heads, int k_heads, const float* q_gamma, const float* k_gamma,
                  float eps, const void* x, bool x_f16, int64_t ldx, void* y, bool y_f16, int64_t ldy) {
    // blocks of four columns: rows and their start are aligned to one
    const auto aligned = [](const void* at, bool f16, int64_t ld) {
        return ld % 4 == 0 && reinterpret_cast<uintptr_t>(at) % (f16 ? 8 : 16) == 0;
    };
    if (rope) p->rope = rope->table;
    p->x = x;
    p->ldx = ldx;
    p->x_f16 = x_f16;
    p->dim = dim;
    p->q_heads = q_heads;
    p->k_heads = k_heads;
    p->q_gamma = q_gamma;
    p->k_gamma = k_gamma;
    p->vec = aligned(x, x_f16, ldx) && aligned(y, y_f16, ldy) &&
             (reinterpret_cast<uintptr_t>(q_gamma) | reinterpret_cast<uintptr_t>(k_gamma)) % 16 == 0;
    p->eps = eps;
    p->inv_dim = 1.0f / (float)dim;
    p->y = y;
    p->ldy = ldy;
    p->y_f16 = y_f16;
}

void heads_split(HeadsParams* p, int64_t seqs, int64_t rows, int heads) {
    const int64_t all = seqs * rows, wave = heads_at_once(*p);
    const bool streamed = !p->x_f16 && heads_vec(*p) && heads >= 4 * wave && all * heads * p->dim >= 40000000;
    p->block_rows = rows > 2 && all >= (heads <= 2 * wave ? 1024 : 2048) && !streamed ? 4 : 1;
    const int64_t once = wave * (4 / p->block_rows), passes = (heads + once - 1) / once;
    const int64_t blocks = (rows + p->block_rows - 1) / p->block_rows;
    p->splits = (int)std::clamp<int64_t>(1024 / std::max<int64_t>(seqs * blocks, 1), 1, passes);
    p->by_splits = fast_div(p->splits);
    p->by_new = fast_div((int)blocks);
    p->by_pairs = fast_div(std::max(p->rope.rotary / 2, 1));
}

}  // namespace qlin

extern "C" {

int qlin_rope_create(const qlin_rope_config* config, qlin_rope** out) {
    if (!out) return QLIN_ERR_PARAM;
    *out = nullptr;
    if (!config || !good(*config)) return QLIN_ERR_PARAM;
    if (config->head_dim > kKvMaxDim) return QLIN_ERR_UNSUPPORTED;
    int device;
    if (hipGetDevice(&device) != hipSuccess) return QLIN_ERR_NODEVICE;
    auto* r = new (std::nothrow) qlin_rope();
    if (!r) return QLIN_ERR_NOMEM;
    const int pairs = config->rotary_dim / 2;
    r->dim = config->head_dim;
    r->device = device;
    r->amplitude = config->amplitude > 0.0                  ? config->amplitude
                   : config->scaling == QLIN_ROPE_RAMP ? 0.1 * std::log(config->factor) + 1.0
                                                            : 1.0;
    double quarters[kKvMaxDim / 2];
    for (int i = 0; i < pairs; ++i) {
        r->radians[i] = frequency(*config, i);
        quarters[i] = r->radians[i] * (4.0 / kTwoPi);
    }
    r->table = {nullptr, (float)r->amplitude, config->rotary_dim, config->first, config->layout == QLIN_ROPE_INTERLEAVED};
    void* data;
    if (hipMalloc(&data, pairs * sizeof(double)) != hipSuccess) {
        (void)hipGetLastError();
        delete r;
        return QLIN_ERR_NOMEM;
    }
    r->table.quarters = static_cast<const double*>(data);
    if (hipMemcpy(data, quarters, pairs * sizeof(double), hipMemcpyHostToDevice) != hipSuccess) {
        qlin_rope_free(r);
        return QLIN_ERR_DEVICE;
    }
    *out = r;
    return QLIN_OK;
}

void qlin_rope_free(qlin_rope* r) {
    if (!r) return;
    (void)hipFree(const_cast<double*>(r->table.quarters));
    delete r;
}

int qlin_rope_query(const qlin_rope* r, double* radians, double* amplitude) {
    if (!r || !radians || !amplitude) return QLIN_ERR_PARAM;
    std::copy_n(r->radians, r->table.rotary / 2, radians);
    *amplitude = r->amplitude;
    return QLIN_OK;
}

int qlin_rope_run(const qlin_rope* rope, int32_t rows, int32_t heads, const void* X, int32_t x_dtype, int64_t ldx,
                  const int32_t* positions, void* Y, int32_t y_dtype, int64_t ldy, uint32_t flags, void* stream) {
    if (!rope) return QLIN_ERR_PARAM;
    return run(rope, rows, rope->dim, heads, 0, nullptr, nullptr, 0.0f, X, x_dtype, ldx, positions, Y, y_dtype, ldy, flags, stream);
}

int qlin_rope_run_norm(const qlin_rope* rope, int32_t rows, int32_t head_dim, int32_t q_heads, int32_t k_heads, const float* q_gamma,
                       const float* k_gamma, float eps, const void* X, int32_t x_dtype, int64_t ldx, const int32_t* positions,
                       void* Y, int32_t y_dtype, int64_t ldy, uint32_t flags, void* stream) {
    return run(rope, rows, head_dim, q_heads, k_heads, q_gamma, k_gamma, eps, X, x_dtype, ldx, positions, Y, y_dtype, ldy, flags,
               stream);
}

}  // extern "C"
