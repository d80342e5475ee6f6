// Tables of a serving step: what the C entry point hands to the kernels of qlin_kv_step.hip, and the rules for one slot,
// plain integer functions, the same on the device and in host tests.
#pragma once

#include "qlin_kv_index.hpp"

namespace qlin {

// What one slot asks for.  Its own pages are the columns from `shared` (those of the prefix) on.
struct StepSlot {
    int len;   // tokens after what it gives back, before what it is given
    int from;  // first column that is given back (back > 0) or given
    int back;  // pages given back
    int want;  // tokens asked for; 0 where they are more than can ever be granted
    int need;  // pages for them
    bool asks, shrinks, bad;
};

// Columns that n tokens take, those of the prefix among them in any case.  n is 0 .. 2^30.
QLIN_HD int step_columns(int n, int shift, int shared) {
    const int c = (n + (1 << shift) - 1) >> shift;
    return c > shared ? c : shared;
}

QLIN_HD StepSlot step_slot(int n, int change, int shift, int shared, int rows, int max_new, int max_len) {
    StepSlot s{n, 0, 0, 0, 0, change > 0, change < 0, n < 0 || n > max_len};
    if (s.bad || change == 0) return s;
    const int held = step_columns(n, shift, shared);
    if (change < 0) {
        s.len = change < -n ? 0 : n + change;
        s.from = step_columns(s.len, shift, shared);
        s.back = held - s.from;
        return s;
    }
    if (change > max_new || change > rows || change > max_len - n) return s;
    s.want = change;
    s.from = held;
    s.need = step_columns(n + change, shift, shared) - held;
    return s;
}

// Last i of start[0 .. n] (not decreasing, start[0] = 0) with start[i] <= k, for U values of k below start[n]: whose the
// k-th things are.  The searches go step by step beside each other.
template <int U, typename P>
QLIN_HD void step_owners(P start, int n, const int (&k)[U], int (&i)[U]) {
    for (int u = 0; u < U; ++u) i[u] = 0;
    for (int left = n; left > 1;) {
        const int half = left >> 1;
        for (int u = 0; u < U; ++u) i[u] += start[i[u] + half] <= k[u] ? half : 0;
        left -= half;
    }
}
template <typename P>
QLIN_HD int step_owner(P start, int n, int k) {
    const int one[1] = {k};
    int i[1];
    step_owners<1>(start, n, one, i);
    return i[0];
}

// Sums that stay at kStepMost once they reach it: above everything that can be granted.
constexpr int kStepMost = 1 << 30;
QLIN_HD int step_add(int a, int b) {
    const uint32_t c = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
    return c > static_cast<uint32_t>(kStepMost) ? kStepMost : static_cast<int>(c);
}

// Slot of the token at place pos, whose page is `id`.  Of a page of the slot's own outside the cache (bad): -1, so that whoever
// stores by slots is led nowhere.  A prefix's pages are not the tables' business: their ids are taken as they are.
QLIN_HD int64_t step_place(int id, int pos, int shift, int shared, int pages, bool* bad) {
    bool outside = false;
    kv_page(id, pages, &outside);
    outside = outside && (pos >> shift) >= shared;
    *bad |= outside;
    return outside ? -1 : static_cast<int64_t>(id) * (1 << shift) + (pos & ((1 << shift) - 1));
}

// Scratch of a call, int32: totals, then [seqs + 1] first pages given and given back.
constexpr int kStepTotals = 4;
constexpr int64_t kv_step_scratch(int seqs) { return kStepTotals + 2 * (static_cast<int64_t>(seqs) + 1); }

struct StepParams {
    int seqs, rows, max_new, max_len, shared, pages, shift;
    const int32_t* change;
    int32_t* length;
    int32_t* table;
    int64_t table_ld;
    int32_t* free_pages;
    int32_t* free_count;
    int32_t* row_start;
    int32_t* row_seq;
    int32_t* positions;
    int64_t* slots;
    int32_t* refused;
    int32_t* totals;  // scratch
    int32_t *need_start, *back_start;
    uint32_t* err;
};

}  // namespace qlin
