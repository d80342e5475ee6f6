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
// Of the softmax's scale.  The kernels multiply it, log2 e and 2^9 by a row's power of two (f32 rows) before they
// multiply by a key's scale: finite up to here for queries below 2^47, so that a key of zeros has the exponent 0 and not 0 * inf.
constexpr float kKvMaxScale = 0x1p64f;
constexpr int kKvMaxSeqs = 1 << 20, kKvMaxRows = 1 << 24, kKvMaxLen = 1 << 30;
constexpr int64_t kKvMaxGrid = (1 << 24) - 1;  // workgroups of 256 threads of one launch

// The cache in device memory.  Codes are stored as code + 128, one byte each: a byte b between two
// zero bytes is the fp16 subnormal b * 2^-24, so one byte permute and one packed FMA make two exact
// fp16 codes of two bytes.  Columns dim .. dim_padded - 1 hold code 0.
//
// A block of a page and head is contiguous: keys [page tokens][dim_padded], values alike, then the
// key scales f32 [page tokens] and the value scales.  One address leads to all of it.
struct KvCache {
    uint8_t* data;  // [pages][heads] blocks
    int pages, heads, dim, dim_padded, shift;  // 1 << shift tokens a page
};
__host__ __device__ __forceinline__ int64_t kv_block_bytes(int dim_padded, int shift) {
    return (int64_t)(2 * dim_padded + 8) << shift;
}
template <int DP>
struct KvBlock {
    uint8_t* base;
    int shift;
    __device__ KvBlock(const KvCache& c, int page, int head)
        : base(c.data + ((int64_t)page * c.heads + head) * kv_block_bytes(DP, c.shift)), shift(c.shift) {}
    __device__ uint8_t* k(int off) const { return base + off * DP; }
    __device__ uint8_t* v(int off) const { return base + (((int64_t)DP << shift) + off * DP); }
    __device__ float* ks(int off) const { return reinterpret_cast<float*>(base + ((int64_t)(2 * DP) << shift)) + off; }
    __device__ float* vs(int off) const { return ks(off + (1 << shift)); }
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
    uint32_t* err;  // [kErrWords]
    FastDiv by_blocks, by_heads;  // of workgroup and unit indexes
};
hipError_t launch_kv_append(const KvRows& p, hipStream_t stream);
hipError_t launch_kv_read(const KvRows& p, hipStream_t stream);
hipError_t launch_kv_clear(const KvCache& c, hipStream_t stream);  // every row: code 0, the smallest scale

struct AttendParams {
    KvCache c;
    KvBatch b;
    const void* q;  // [rows, ldq]
    int64_t ldq;
    int q_f16, q_vec;    // q_vec, o_vec: heads of whole groups of 8, 16-byte aligned
    int q_heads;
    FastDiv group;       // by q_heads / kv heads
    float scale2;        // scale * log2 e
    void* o;             // [rows, ldo]
    int64_t ldo;
    int o_f16, o_vec;
    int prefix;                   // tokens of the shared prefix, a multiple of the page; 0: none
    const int32_t* prefix_pages;  // its pages
    int own_from;                 // first token that a sequence's own parts cover: prefix, or 0 (no parts of the prefix)
    // Partial results (parts > 1), one slot per (row, query head, part): dim_padded unnormalized
    // outputs each, then (running maximum, sum) pairs.
    int parts, prefix_parts;  // in all; of the prefix (they come first)
    int chunk, prefix_chunk;  // tokens a part
    FastDiv by_heads, by_seqs, by_tiles, by_prefix_tiles;  // of workgroup indexes; tiles of vectors
    FastDiv by_q_heads, by_join;                           // of the join's
    float* part_o;
    float* part_ml;
    uint32_t* err;  // [kErrWords]
};
// Tokens worked on at once by a workgroup of the attention kernel: chunks are multiples of it.
constexpr int kAttendStep = 128;
// Vectors of a workgroup: over a sequence's own tokens, over the prefix.
int attend_tile(const AttendParams& p);
int attend_tile_prefix(const AttendParams& p);
constexpr int kAttendWide = 128;  // of the kernel for many vectors
hipError_t launch_attend(const AttendParams& p, hipStream_t stream);
hipError_t launch_attend_wide(const AttendParams& p, bool prefix, hipStream_t stream);

}  // namespace qlin
