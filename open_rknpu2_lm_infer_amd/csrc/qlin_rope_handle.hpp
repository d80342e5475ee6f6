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
// Workgroups a row: as many as its heads fill while there are few rows, else fewer, since each computes the row's angles.
void heads_split(HeadsParams* p, int64_t rows, int heads);

}  // namespace qlin
