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
// How rows are shared out: one a workgroup and, while they are few, its heads over several workgroups; of many rows four a
// workgroup, one a wave, which then shares what is computed once among more heads, and has no wave without one.  Many are
// 2048, and 1024 where a row's heads are work for two waves at most.  f32 rows in blocks of four columns that fill a
// workgroup stay alone from 160 MB on, which memory takes better in long pieces, and so do sequences of one or two rows, whose
// blocks of four would be empty.  With one and four rows a workgroup, us as graph nodes:
//   heads of 128, f32, turned: 6 heads, 1024 rows 3.9 and 3.6, 8192 rows 16.1 and 11.2, 65536 rows 129 and 75; 16 heads, 1024 rows
//     4.7 and 5.0, 8192 rows 22.2 and 21.6; 40 heads, 1024 rows 9.0 and 9.0, 2048 15.0 and 14.1, 6000 (122 MB) 42.1 and 42.5,
//     8192 (168 MB) 63.4 and 68.5; 24 heads, 16384 rows (201 MB) 74 and 79
//   fp16: 40 heads, 1024 rows 6.5 and 6.7, 2048 10.7 and 9.7, 30000 117 and 118, normalized too 127 and 117
//   40 heads and the cache's 8 values: fp16, 1024 rows 9.3 and 9.6, 2048 14.4 and 13.5, 16384 96 and 91; f32, 2048 19.3
//     and 18.0, 6144 (151 MB) 53 and 50, 16384 135 and 147
//     of fp16 sequences of few rows: 2048 of 1 row 14.6 and 22.3, of 2 23.6 and 26.4, 1024 of 3 18.9 and 17.9, 512 of 8 23.4 and 20.5
//   20 heads of 84, normalized: fp16, 1024 rows 9.2 and 10.1, 2048 15.2 and 12.4, f32, 30000 rows (201 MB) 241 and 176
void heads_split(HeadsParams* p, int64_t seqs, int64_t rows, int heads);

}  // namespace qlin
