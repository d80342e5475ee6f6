// Where the rows and tokens of a key/value cache batch lie: plain integer functions, the same on
// the device and in host tests.  Everything a kernel reads from the caller's device arrays (row
// starts, lengths, page ids) goes through here, so that no value of them leads outside a buffer.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define QLIN_HD __host__ __device__ __forceinline__
#else
#define QLIN_HD inline
#endif

namespace qlin {

// n / d and n % d for 0 <= n < 2^31 with one multiplication: with 2^(L-1) < d <= 2^L and
// mul = floor(2^(31+L) / d) + 1, the product n * mul / 2^(31+L) exceeds n / d by less than 1 / d.
struct FastDiv {
    uint32_t mul, d;
    int shift;
    QLIN_HD int div(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift); }
    QLIN_HD int mod(int n) const { return n - div(n) * static_cast<int>(d); }
};
inline FastDiv fast_div(int d) {
    int l = 0;
    while ((static_cast<int64_t>(1) << l) < d) ++l;
    return {static_cast<uint32_t>((static_cast<uint64_t>(1) << (31 + l)) / d + 1), static_cast<uint32_t>(d), 31 + l};
}

// One sequence of a batch: its new rows are row0 .. row0 + rows - 1 of the row tensors, and the
// t-th of them is position len - rows + t of the sequence (negative: no such token).
struct KvSeq {
    int row0, rows, len;
    bool bad;  // the arrays held something outside the batch's limits
};

QLIN_HD int kv_clamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

QLIN_HD KvSeq kv_seq(const int32_t* row_start, const int32_t* length, int i, int rows, int max_new, int max_len) {
    const int a = row_start[i], b = row_start[i + 1], n = length[i];
    KvSeq s;
    s.bad = a < 0 || b < a || b > rows || n < 0 || n > max_len;
    s.row0 = kv_clamp(a, 0, rows);
    s.rows = kv_clamp(b, s.row0, rows) - s.row0;
    s.len = kv_clamp(n, 0, max_len);
    if (s.rows > max_new) {
        s.rows = max_new;  // the grid covers no more
        s.bad = true;
    }
    return s;
}

// Tokens that new row t of a sequence sees: its own position and everything before it.
QLIN_HD int kv_visible(const KvSeq& s, int t) { return kv_clamp(s.len - s.rows + t + 1, 0, s.len); }

// The page id, or 0 with *bad set for an id outside the cache.
QLIN_HD int kv_page(int id, int pages, bool* bad) {
    if (static_cast<uint32_t>(id) < static_cast<uint32_t>(pages)) return id;
    *bad = true;
    return 0;
}

// Parts of `chunk` tokens that a sequence of `tokens` tokens is worked on in (one at least).
QLIN_HD int kv_parts(int tokens, int chunk) { return tokens <= chunk ? 1 : (tokens - 1) / chunk + 1; }

}  // namespace qlin
