// What the C entry points know of a rotary-position handle, and how they fill the kernels' parameters.
#pragma once

#include "qlin_rope.hpp"

struct qlin_rope {
    qlin::RopeTable table;
    int dim, device;
    double amplitude;
    double radians[qlin::kKvMaxDim / 2];  // a position
};

namespace qlin {

// Rows, norms and output of a call; what is left are its rows or its batch, and heads_split.
void heads_common(HeadsParams* p, const qlin_rope* rope, int dim, int q_heads, int k_heads, const float* q_gamma, const float* k_gamma,
                  float eps, const void* x, bool x_f16, int64_t ldx, void* y, bool y_f16, int64_t ldy);
// How rows are shared out: one a workgroup and, while they are few, its heads over several workgroups; of many fp16 rows four
// a workgroup, one a wave, which then shares what is computed once among 12 heads instead of 3 (40 heads of 128 and
// their cache's 8 values, us with one and four rows: 1024 rows 10.9 and 11.0, 2048 18.8 and 15.6, 4096 32.5 and 24.8; f32 rows, which memory
// bounds, 19.0 and 17.9 at 2048, 40.3 and 40.6 at 4096, 8192 rows turned alone 67.0 and 73.3).
void heads_split(HeadsParams* p, int64_t seqs, int64_t rows, int heads);

}  // namespace qlin
