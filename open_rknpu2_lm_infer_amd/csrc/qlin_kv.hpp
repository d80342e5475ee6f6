// Key/value cache: what the C entry points hand to the kernels of qlin_kv.hip and qlin_attend.hip.
#pragma once

#include "qlin_internal.hpp"
#include "qlin_kv_index.hpp"

namespace qlin {

// Smallest scale of a cache row.  A row whose largest value is below 127 * 2^-64 keeps this scale
// (a zero row among them: its codes are zero), so that 1 / scale and sums of it stay inside f32.
constexpr float kKvScaleMin = 0x1p-64f;
constexpr int kKvMaxDim = 256;
constexpr int kKvMinPage = 16, kKvMaxPage = 4096;  // tokens, powers of two
constexpr int kKvMaxHeads = 1024;
constexpr int kKvMaxSeqs = 1 << 20, kKvMaxRows = 1 << 24, kKvMaxLen = 1 << 30;
constexpr int64_t kKvMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads of one launch

// The cache in device memory.  Codes are stored as code + 128, one byte each: a byte b between two
// zero bytes is the fp16 subnormal b * 2^-24, so one byte permute and one packed FMA make two exact
// fp16 codes of four bytes.  Columns dim .. dim_padded - 1 hold code 0.
struct KvCache {
    uint8_t *k, *v;  // [pages][heads][page tokens][dim_padded]
    float *ks, *vs;  // [pages][heads][page tokens]
    int pages, heads, dim, dim_padded, shift;  // 1 << shift tokens a page
};

struct KvBatch {
    int seqs, rows, max_new, max_len;
    const int32_t* row_start;  // [seqs + 1]
    const int32_t* length;     // [seqs]
    const int32_t* table;      // [seqs, table_ld]
    int64_t table_ld;
};

struct KvRows {
    KvCache c;
    KvBatch b;
    void *k, *v;  // [rows, ld]: head h in columns h * dim .. h * dim + dim - 1
    int64_t ldk, ldv;
    int f16;
    int rne;
    uint32_t* err;
};
hipError_t launch_kv_append(const KvRows& p, hipStream_t stream);
hipError_t launch_kv_read(const KvRows& p, hipStream_t stream);

struct AttendParams {
    KvCache c;
    KvBatch b;
    const void* q;  // [rows, ldq]
    int64_t ldq;
    int q_f16;
    int q_heads, group;  // group = q_heads / kv heads
    float scale2;        // scale * log2 e
    void* o;             // [rows, ldo]
    int64_t ldo;
    int o_f16;
    int prefix;                   // tokens of the shared prefix, a multiple of the page; 0: none
    const int32_t* prefix_pages;  // its pages
    int own_from;                 // first token that a sequence's own parts cover: prefix, or 0 (no parts of the prefix)
    // Partial results (parts > 1), one slot per (row, query head, part): dim_padded unnormalized
    // outputs each, then (running maximum, sum) pairs.
    int parts, prefix_parts;  // in all; of the prefix (they come first)
    int chunk, prefix_chunk;  // tokens a part
    float* part_o;
    float* part_ml;
    uint32_t* err;
};
// Tokens worked on at once by a workgroup of the attention kernel: chunks are multiples of it.
constexpr int kAttendStep = 128;
int attend_tile(const AttendParams& p);  // vectors of a workgroup
hipError_t launch_attend(const AttendParams& p, hipStream_t stream);

}  // namespace qlin
