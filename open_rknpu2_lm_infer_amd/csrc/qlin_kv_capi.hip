// C ABI of the key/value cache: its handle, the argument checks, and how an attention call is cut
// into parts.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>

#include "../../include/qlinear.h"
#include "qlin_kv.hpp"

using namespace qlin;

struct qlin_kv_cache {
    KvCache c;
    int device;
    uint64_t device_bytes;
};

namespace {

bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Checks a batch against its cache, the workspace and the current device, and begins a run on the workspace.
int begin(qlin_workspace* ws, const qlin_kv_cache* cache, const qlin_kv_batch* b, void* stream, KvBatch* out,
          WorkspaceParts* parts) {
    if (!ws || !cache || !b || b->seqs <= 0 || b->rows < 0 || b->max_new < 0 || b->max_len < 0 || !b->row_start ||
        !b->length || (b->max_len > 0 && !b->page_table) || b->max_new > b->rows ||
        b->page_ld < ceil_div(b->max_len, (int64_t)1 << cache->c.shift) || b->page_ld < 0)
        return QLIN_ERR_PARAM;
    if (b->seqs > kKvMaxSeqs || b->rows > kKvMaxRows || b->max_len > kKvMaxLen) return QLIN_ERR_UNSUPPORTED;
    if (workspace_device(ws) != cache->device) return QLIN_ERR_PARAM;
    int dev;
    if (hipGetDevice(&dev) != hipSuccess) return QLIN_ERR_NODEVICE;
    if (dev != cache->device) return QLIN_ERR_PARAM;
    *out = KvBatch{b->seqs, b->rows, b->max_new, b->max_len, b->row_start, b->length, b->page_table, b->page_ld};
    *parts = workspace_begin(ws, (hipStream_t)stream);
    return QLIN_OK;
}

// Rows whose heads are whole groups of 8 columns, each 16-byte aligned.
bool aligned(const void* p, int64_t ld, int dtype, int dim) {
    return dim % 8 == 0 && ld % (dtype == QLIN_F16 ? 8 : 4) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

bool is_dtype(int32_t t) { return t == QLIN_F32 || t == QLIN_F16; }

int rows_call(qlin_workspace* ws, const qlin_kv_cache* cache, const qlin_kv_batch* batch, void* K, int64_t ldk, void* V,
              int64_t ldv, int32_t dtype, uint32_t flags, void* stream, bool append) {
    if (!cache || !batch || (batch->rows > 0 && (!K || !V)) || !is_dtype(dtype) || (flags & ~QLIN_ROUND_HALF_EVEN)) return QLIN_ERR_PARAM;
    const int64_t cols = (int64_t)cache->c.heads * cache->c.dim;
    if (ldk < cols || ldv < cols) return QLIN_ERR_PARAM;
    KvRows p{};
    WorkspaceParts parts;
    if (int rc = begin(ws, cache, batch, stream, &p.b, &parts)) return rc;
    if (p.b.max_new == 0) return QLIN_OK;
    // a row and head takes dim_padded / 8 lanes of 256-thread workgroups
    const int64_t lanes = (int64_t)p.b.max_new * cache->c.heads * cache->c.dim_padded / 8;
    if (lanes > (int64_t)1 << 30 || ceil_div(lanes, 256) * p.b.seqs > kKvMaxGrid)
        return QLIN_ERR_UNSUPPORTED;
    p.c = cache->c;
    p.k = K;
    p.v = V;
    p.ldk = ldk;
    p.ldv = ldv;
    p.f16 = dtype == QLIN_F16;
    p.rne = (flags & QLIN_ROUND_HALF_EVEN) != 0;
    p.err = parts.err;
    const hipError_t e = append ? launch_kv_append(p, (hipStream_t)stream) : launch_kv_read(p, (hipStream_t)stream);
    return e == hipSuccess ? QLIN_OK : QLIN_ERR_DEVICE;
}

// Tokens a part and the parts of `tokens` tokens, for `blocks` workgroups a part: `cover` workgroups for
// every CU, at least one step of a workgroup each, at most `cap` parts of at most `most` tokens.  A context of
// up to kOnePart tokens is not cut: a workgroup takes 1.1 us for a step of 128, the join 2.7 us and its launch.
// (One token, 8 KV heads of 128: 300 tokens 7.9 against 8.7 us in two parts and more, 512 8.8 against 8.3, 768
// 10.6 against 9.1.)
constexpr int kOnePart = 512;
void cut(int64_t tokens, int64_t blocks, int cover, int most, int64_t cap, int* parts, int* chunk) {
    const int64_t steps = std::max<int64_t>(1, ceil_div(tokens, kAttendStep));
    int64_t want = std::max(ceil_div(cover, blocks), ceil_div(tokens, most));
    want = tokens <= kOnePart ? 1 : std::max<int64_t>(1, std::min({steps, want, cap}));
    const int64_t per = ceil_div(steps, want);
    *chunk = (int)(per * kAttendStep);
    *parts = (int)ceil_div(steps, per);
}

int attention(qlin_workspace* ws, const qlin_kv_cache* cache, const qlin_kv_batch* batch, int32_t prefix,
              const int32_t* prefix_pages, int32_t q_heads, const void* Q, int32_t q_dtype, int64_t ldq, float scale,
              void* O, int32_t o_dtype, int64_t ldo, void* stream) {
    if (!cache || !batch || (batch->rows > 0 && (!Q || !O)) || !is_dtype(q_dtype) || !is_dtype(o_dtype) || !std::isfinite(scale) ||
        q_heads <= 0 || q_heads % cache->c.heads != 0 || prefix < 0 || (prefix > 0 && !prefix_pages))
        return QLIN_ERR_PARAM;
    if (prefix & ((1 << cache->c.shift) - 1)) return QLIN_ERR_PARAM;
    const int64_t cols = (int64_t)q_heads * cache->c.dim;
    if (ldq < cols || ldo < cols) return QLIN_ERR_PARAM;
    AttendParams p{};
    WorkspaceParts wp;
    if (q_heads > kKvMaxHeads || std::fabs(scale) > kKvMaxScale || prefix > kKvMaxLen || (int64_t)batch->rows * q_heads > 1 << 30) return QLIN_ERR_UNSUPPORTED;
    if (int rc = begin(ws, cache, batch, stream, &p.b, &wp)) return rc;
    if (p.b.max_new == 0) return QLIN_OK;
    p.c = cache->c;
    p.q = Q;
    p.ldq = ldq;
    p.q_vec = aligned(Q, ldq, q_dtype, cache->c.dim);
    p.q_f16 = q_dtype == QLIN_F16;
    p.q_heads = q_heads;
    const int group = q_heads / cache->c.heads;
    p.group = fast_div(group);
    p.scale2 = scale * 1.44269504f;
    p.o = O;
    p.ldo = ldo;
    p.o_vec = aligned(O, ldo, o_dtype, cache->c.dim);
    p.o_f16 = o_dtype == QLIN_F16;
    p.prefix = prefix;
    p.prefix_pages = prefix_pages;
    p.err = wp.err;
    const int64_t tiles = ceil_div((int64_t)p.b.max_new * group, attend_tile(p));
    const int64_t prefix_tiles = ceil_div((int64_t)p.b.rows * group, attend_tile_prefix(p));
    const int64_t own_blocks = (int64_t)p.b.seqs * cache->c.heads * tiles, prefix_blocks = cache->c.heads * prefix_tiles;
    if (own_blocks > kKvMaxGrid) return QLIN_ERR_UNSUPPORTED;
    // Parts that the workspace's scratch holds results of, that one launch covers, and that one can join (a
    // workgroup for each vector of a batch of which all sequences had max_new rows).
    const int64_t vectors = (int64_t)p.b.rows * q_heads;
    const bool joins = (int64_t)p.b.max_new * q_heads * p.b.seqs <= kKvMaxGrid;
    const int64_t cap = joins ? std::min(wp.part_floats / (vectors * (cache->c.dim_padded + 2)),
                                         kKvMaxGrid / (own_blocks + prefix_blocks)) : 1;
    // The prefix gets parts of its own where the scratch can hold its results; else every sequence reads it itself.
    const bool apart = prefix > 0 && cap >= 2;
    p.own_from = apart ? prefix : 0;
    // The kernel for few vectors runs best with one workgroup a CU (64 sequences of up to 4096 tokens: 73 us
    // uncut, 76 and 80 us in parts of 1024 and 512); parts of 2048 tokens bound what a single long sequence of a
    // ragged batch costs.  The one for many vectors has two workgroups a CU, of which the second hides the first's
    // waits; the prefix, whose results are all joined, one.
    const bool few = attend_tile(p) < kAttendWide;
    int parts = 1;
    cut(std::max(p.b.max_len - p.own_from, 0), own_blocks, few ? wp.cu_count : 2 * wp.cu_count, few ? 2048 : kKvMaxLen,
        apart ? cap / 2 : cap, &parts, &p.chunk);
    if (apart) cut(prefix, prefix_blocks, wp.cu_count, kKvMaxLen, cap - parts, &p.prefix_parts, &p.prefix_chunk);
    p.parts = parts + p.prefix_parts;
    p.by_seqs = fast_div(p.b.seqs);
    p.by_q_heads = fast_div(q_heads);
    p.by_heads = fast_div(cache->c.heads);
    p.by_tiles = fast_div((int)tiles);
    p.by_prefix_tiles = fast_div((int)prefix_tiles);
    p.part_o = wp.part;
    p.part_ml = wp.part + vectors * p.parts * cache->c.dim_padded;
    return launch_attend(p, (hipStream_t)stream) == hipSuccess ? QLIN_OK : QLIN_ERR_DEVICE;
}

}  // namespace

extern "C" {

int qlin_kv_create(const qlin_kv_config* config, qlin_kv_cache** out) {
    if (!out) return QLIN_ERR_PARAM;
    *out = nullptr;
    if (!config || config->kv_heads <= 0 || config->head_dim <= 0 || config->pages <= 0 ||
        !power_of_two(config->page_tokens))
        return QLIN_ERR_PARAM;
    if (config->head_dim > kKvMaxDim || config->kv_heads > kKvMaxHeads || config->page_tokens < kKvMinPage ||
        config->page_tokens > kKvMaxPage)
        return QLIN_ERR_UNSUPPORTED;
    int dev;
    if (hipGetDevice(&dev) != hipSuccess) return QLIN_ERR_NODEVICE;
    auto* x = new (std::nothrow) qlin_kv_cache();
    if (!x) return QLIN_ERR_NOMEM;
    KvCache& c = x->c;
    c.pages = config->pages;
    c.heads = config->kv_heads;
    c.dim = config->head_dim;
    c.dim_padded = c.dim <= 64 ? 64 : c.dim <= 128 ? 128 : 256;
    while ((1 << c.shift) < config->page_tokens) ++c.shift;
    x->device = dev;
    x->device_bytes = (uint64_t)c.pages * c.heads * kv_block_bytes(c.dim_padded, c.shift);
    if (hipMalloc(&c.data, x->device_bytes) != hipSuccess) {
        (void)hipGetLastError();
        delete x;
        return QLIN_ERR_NOMEM;
    }
    if (launch_kv_clear(c, nullptr) != hipSuccess || hipDeviceSynchronize() != hipSuccess) {
        qlin_kv_free(x);
        return QLIN_ERR_DEVICE;
    }
    *out = x;
    return QLIN_OK;
}

void qlin_kv_free(qlin_kv_cache* x) {
    if (!x) return;
    (void)hipFree(x->c.data);
    delete x;
}

int qlin_kv_query(const qlin_kv_cache* x, qlin_kv_info* out) {
    if (!x || !out) return QLIN_ERR_PARAM;
    out->kv_heads = x->c.heads;
    out->head_dim = x->c.dim;
    out->page_tokens = 1 << x->c.shift;
    out->pages = x->c.pages;
    out->head_dim_padded = x->c.dim_padded;
    out->device = x->device;
    out->device_bytes = x->device_bytes;
    return QLIN_OK;
}

int qlin_kv_append(qlin_workspace* ws, qlin_kv_cache* cache, const qlin_kv_batch* batch, const void* K, int64_t ldk,
                   const void* V, int64_t ldv, int32_t dtype, uint32_t flags, void* stream) {
    return rows_call(ws, cache, batch, const_cast<void*>(K), ldk, const_cast<void*>(V), ldv, dtype, flags, stream, true);
}

int qlin_kv_read(qlin_workspace* ws, const qlin_kv_cache* cache, const qlin_kv_batch* batch, void* K, int64_t ldk, void* V,
                 int64_t ldv, int32_t dtype, void* stream) {
    return rows_call(ws, cache, batch, K, ldk, V, ldv, dtype, 0, stream, false);
}

int qlin_kv_attention(qlin_workspace* ws, const qlin_kv_cache* cache, const qlin_kv_batch* batch, int32_t q_heads,
                      const void* Q, int32_t q_dtype, int64_t ldq, float scale, void* O, int32_t o_dtype, int64_t ldo,
                      void* stream) {
    return attention(ws, cache, batch, 0, nullptr, q_heads, Q, q_dtype, ldq, scale, O, o_dtype, ldo, stream);
}

int qlin_kv_attention_prefix(qlin_workspace* ws, const qlin_kv_cache* cache, const qlin_kv_batch* batch,
                             int32_t prefix_tokens, const int32_t* prefix_pages, int32_t q_heads, const void* Q,
                             int32_t q_dtype, int64_t ldq, float scale, void* O, int32_t o_dtype, int64_t ldo,
                             void* stream) {
    return attention(ws, cache, batch, prefix_tokens, prefix_pages, q_heads, Q, q_dtype, ldq, scale, O, o_dtype, ldo,
                     stream);
}

}  // extern "C"
