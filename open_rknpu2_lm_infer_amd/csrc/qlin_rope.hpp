// Rotary positions and head norms: what the C entry points hand to the kernels of qlin_heads.hip.
#pragma once

#include "qlin_kv.hpp"

namespace qlin {

// Pairs of columns that a position turns: pair i of `rotary` / 2 is columns first + i and first + rotary / 2 + i, or
// (interleaved) first + 2 i and first + 2 i + 1.
struct RopeTable {
    const double* quarters;  // [rotary / 2] quarter turns a position
    float amplitude;
    int rotary, first, interleaved;
};

struct HeadsParams {
    RopeTable rope;  // rotary 0: nothing is turned
    int inverse;
    const void* x;  // [rows, ldx]: q_heads heads of dim columns, then k_heads, then (cache) as many values
    int64_t ldx;
    int x_f16;
    int dim, q_heads, k_heads;
    int vec;  // rows, their starts and the norms' factors are aligned to four columns
    const float *q_gamma, *k_gamma;  // null: not normalized
    float eps, inv_dim;
    void* y;  // [rows, ldy]: queries and keys, or (cache) queries alone
    int64_t ldy;
    int y_f16;
    int block_rows;  // rows of a workgroup: 1, or 4, one a wave
    int splits;      // workgroups that share them
    FastDiv by_splits, by_pairs;
    // rows with positions
    int rows;
    const int32_t* positions;
    // rows of a batch, whose keys and values go into the cache
    KvCache c;
    KvBatch b;
    FastDiv by_new;  // by a sequence's blocks of rows
    int rne;
    uint32_t* err;
};
// Four columns side by side: pairs and the others are groups of eight, heads and rows of four.
bool heads_vec(const HeadsParams& p);
// Lanes a head takes beside its columns' eighth: twice as many where the pairs and the other columns are no groups of eight.
bool heads_wide(const HeadsParams& p);
int heads_at_once(const HeadsParams& p);  // of a wave
hipError_t launch_heads(const HeadsParams& p, hipStream_t stream);          // rows
hipError_t launch_heads_append(const HeadsParams& p, hipStream_t stream);   // batch

}  // namespace qlin
