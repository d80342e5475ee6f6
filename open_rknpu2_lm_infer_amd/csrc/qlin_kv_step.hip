// Tables of a serving step from the requests' lengths: rows, pages and slots of the key/value cache.
//
// Slot i holds n_i tokens and asks for c_i more, or gives -c_i back.  Pages given back go on top of the free list in the
// order of the slots, then those asked for are taken from its top in the same order:
//   wanted   w_i = c_i where c_i <= max_new, c_i <= rows and n_i + c_i <= max_len, else 0;  then sum_{j <= i} w_j <= rows
//   granted  p_i = pages that n_i + w_i tokens take beyond those of n_i;  p_i = 0 or sum_{j <= i} p_j <= free pages
// Every sum is a scan, so that nothing depends on the order in which threads run.  Sums grow along the slots: who comes too
// late for rows (or pages) is followed by none that is granted rows (pages), and what the granted take is the sum itself.  Who is
// too large to be served at all is in no sum.
//
// One workgroup scans, up to 4096 slots at a time, and gives pages back; whose the k-th row, page taken or page given back is,
// is found by a binary search in the scanned starts, which lie in the LDS up to 4096 slots.  With few rows the same
// workgroup takes pages and writes the rows' maps too: one launch.  With more a second launch does, the first having laid
// down its starts.
//
// What bounds it: the chain of loads, scans and stores of one workgroup, 4.7 us for 64 slots of which 60 get up to 4 rows
// each (2 of them the launch), as much to take the rows back; 3000 slots that are granted 14000 pages and 230000 rows 8.4 us
// and 7.6 for the second launch's searches, and 12.9 to give those pages back, whose table entries one CU reads and writes
// one by one.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "qlin_kv.hpp"
#include "qlin_kv_step.hpp"

namespace qlin {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
enum : int { kAvail = 0, kNeed = 1, kRows = 2 };  // of the scratch's totals

// Sum over the lanes up to this one of its wave, or of its row of 16.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_from(int x) {
    return step_add(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, ROWS == 0xf));
}
__device__ __forceinline__ int row_scan(int x) {
    x = add_from<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
    x = add_from<0x112, 0xf>(x);
    x = add_from<0x114, 0xf>(x);
    return add_from<0x118, 0xf>(x);
}
__device__ __forceinline__ int wave_scan(int x) {
    x = row_scan(x);
    x = add_from<0x142, 0xa>(x);     // the last lane of rows 0 and 2 to rows 1 and 3
    return add_from<0x143, 0xc>(x);  // lane 31 to the upper half
}

// Inclusive sums of N values over the workgroup, and their totals.
template <int N>
struct Scan {
    int at[N], total[N];
};
template <int N>
__device__ __forceinline__ Scan<N> scan(const int (&v)[N], int (*lds)[kWaves]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Scan<N> s;
#pragma unroll
    for (int k = 0; k < N; ++k) s.at[k] = wave_scan(v[k]);
    __syncthreads();  // who still reads an earlier scan's
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < N; ++k) lds[k][wave] = s.at[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int all = row_scan(lds[k][lane % kWaves]);
        s.total[k] = __builtin_amdgcn_readlane(all, kWaves - 1);
        s.at[k] = step_add(s.at[k], wave == 0 ? 0 : __builtin_amdgcn_readlane(all, max(wave - 1, 0)));
    }
    return s;
}

// Pages given back: from the table to the free list, from thread `first` on every `stride`, U at a time.  from: the first
// column that a slot gives back.
template <int U, typename P, typename F>
__device__ __forceinline__ void give_back(const StepParams& p, P back_start, F from, int count, int total, int first, int stride) {
    for (int k0 = first; k0 < total; k0 += U * stride) {
        int k[U], i[U], id[U];
        int32_t* at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) k[u] = min(k0 + u * stride, total - 1);  // the last one again, which is stored once
        step_owners<U>(back_start, p.seqs, k, i);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            at[u] = p.table + i[u] * p.table_ld + from(i[u]) + k[u] - back_start[i[u]];
            id[u] = *at[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u * stride >= total) continue;
            *at[u] = -1;
            bool bad = count + k[u] >= p.pages;  // more pages than there are: some were in the list already
            if (!bad) p.free_pages[count + k[u]] = id[u];
            kv_page(id[u], p.pages, &bad);
            if (bad) atomicOr(p.err + kErrBatch, 1u);
        }
    }
}

// Pages taken and the rows' maps, U at a time.  What the list holds is not written here, and of the table only what a slot is given.
template <int U, typename P>
__device__ __forceinline__ void take(const StepParams& p, P need_start, P row_start, int avail, int need, int rows, int first, int stride) {
    const int items = p.row_seq || p.positions || p.slots ? rows : 0;
    for (int k0 = first; k0 < max(need, items); k0 += U * stride) {
        int k[U], i[U], old[U];
        if (k0 < need) {
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = min(k0 + u * stride, need - 1);
            step_owners<U>(need_start, p.seqs, k, i);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 + u * stride >= need) continue;
                old[u] = p.length[i[u]] - (row_start[i[u] + 1] - row_start[i[u]]);
                const int id = p.free_pages[avail - 1 - k[u]];
                p.table[i[u] * p.table_ld + step_columns(old[u], p.shift, p.shared) + k[u] - need_start[i[u]]] = id;
                bool bad = false;
                kv_page(id, p.pages, &bad);
                if (bad) atomicOr(p.err + kErrBatch, 1u);
            }
        }
        if (k0 < items) {
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = min(k0 + u * stride, items - 1);
            step_owners<U>(row_start, p.seqs, k, i);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 + u * stride >= items) continue;
                const int r = k[u], begin = row_start[i[u]], next = row_start[i[u] + 1];
                old[u] = p.length[i[u]] - (next - begin);
                const int pos = old[u] + r - begin;
                if (p.row_seq) p.row_seq[r] = i[u];
                if (p.positions) p.positions[r] = pos;
                if (p.slots) {
                    // a page taken in this step comes from the list, as its table entry is being written
                    const int column = pos >> p.shift, fresh = column - step_columns(old[u], p.shift, p.shared);
                    const int id = fresh >= 0 ? p.free_pages[avail - 1 - (need_start[i[u]] + fresh)] : p.table[i[u] * p.table_ld + column];
                    bool bad = false;
                    p.slots[r] = step_place(id, pos, p.shift, p.shared, p.pages, &bad);
                    if (bad) atomicOr(p.err + kErrBatch, 1u);
                }
            }
        }
    }
}

// A thread has ITEMS slots of each 1024 * ITEMS.  ONE: there are no more, and their starts lie in the LDS.  rows_too: pages
// are taken and the rows' maps written here, not by the second launch.
template <int ITEMS, bool ONE>
__global__ __launch_bounds__(kThreads) void kv_step_kernel(StepParams p, int rows_too) {
    constexpr int CAP = kThreads * ITEMS;
    __shared__ int sums[3][kWaves];
    // of pages given back and taken; of rows, or (not rows_too) the first columns given back
    __shared__ int starts[ONE ? 3 : 1][ONE ? CAP + 1 : 1];
    const int tid = threadIdx.x;
    int count = *p.free_count;
    bool bad = false;
    StepSlot s[ITEMS];
    auto load = [&](int i0) {  // slots i0 + ITEMS tid ..
        int n[ITEMS], c[ITEMS];
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = min(i0 + ITEMS * tid + k, p.seqs - 1);
            n[k] = p.length[i];
            c[k] = p.change[i];
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            s[k] = i0 + ITEMS * tid + k < p.seqs ? step_slot(n[k], c[k], p.shift, p.shared, p.rows, p.max_new, p.max_len) : StepSlot{};
            bad |= s[k].bad;
        }
    };
    auto sum = [&](auto member) {
        int x = 0;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) x = step_add(x, s[k].*member);
        return x;
    };
    // pages given back by all slots, before any is granted some
    int back = 0;
    if constexpr (!ONE) {
        for (int i0 = 0; i0 < p.seqs; i0 += CAP) {
            load(i0);
            const int v[1] = {sum(&StepSlot::back)};
            const Scan<1> t = scan<1>(v, sums);
            int at = back + t.at[0] - v[0];
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                if (i0 + ITEMS * tid + k < p.seqs) p.back_start[i0 + ITEMS * tid + k] = at;
                at += s[k].back;
            }
            back += t.total[0];
        }
        if (tid == 0) p.back_start[p.seqs] = back;
    }
    bad |= count < 0 || count > p.pages;
    count = kv_clamp(count, 0, p.pages);
    int rows_sum = 0, need_sum = 0, rows = 0, need = 0, refused = 0, avail = 0;
    for (int i0 = 0; i0 < p.seqs; i0 += CAP) {
        load(i0);
        const int all[3] = {sum(&StepSlot::want), sum(&StepSlot::need), ONE ? sum(&StepSlot::back) : 0};
        const Scan<3> t = scan<3>(all, sums);
        if constexpr (ONE) back = t.total[2];
        avail = min(count + back, p.pages);
        int row_at = t.at[0] - all[0], need_at = t.at[1] - all[1], back_at = t.at[2] - all[2];  // before this thread's slots
        int row_total = t.total[0], need_total = t.total[1];
        if (step_add(rows_sum, row_total) <= p.rows && step_add(need_sum, need_total) <= avail) {
            rows_sum += row_total;
            need_sum += need_total;
        } else {
            // some are refused: rows first, then pages, then what is left
            int upto = step_add(rows_sum, row_at);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                upto = step_add(upto, s[k].want);
                if (upto > p.rows) s[k].want = s[k].need = 0;
            }
            rows_sum = step_add(rows_sum, row_total);
            const int v[1] = {sum(&StepSlot::need)};
            const Scan<1> u = scan<1>(v, sums);
            upto = step_add(need_sum, u.at[0] - v[0]);
#pragma unroll
            for (int k = 0; k < ITEMS; ++k) {
                upto = step_add(upto, s[k].need);
                if (s[k].need > 0 && upto > avail) s[k].want = s[k].need = 0;
            }
            need_sum = step_add(need_sum, u.total[0]);
            const int w[2] = {sum(&StepSlot::want), sum(&StepSlot::need)};
            const Scan<2> x = scan<2>(w, sums);
            row_at = x.at[0] - w[0];
            need_at = x.at[1] - w[1];
            row_total = x.total[0];
            need_total = x.total[1];
        }
        row_at += rows;
        need_at += need;
        int none = 0;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = i0 + ITEMS * tid + k;
            if (i >= p.seqs) continue;
            p.row_start[i] = row_at;
            if constexpr (ONE) {
                starts[0][i] = back_at;
                starts[1][i] = need_at;
                starts[2][i] = rows_too ? row_at : s[k].from;
            }
            if (!ONE || !rows_too) p.need_start[i] = need_at;
            if (s[k].asks || s[k].back > 0 || s[k].shrinks) p.length[i] = s[k].len + s[k].want;
            row_at += s[k].want;
            need_at += s[k].need;
            back_at += s[k].back;
            none += s[k].asks && s[k].want == 0;
        }
        rows += row_total;
        need += need_total;
        if (p.refused) {
            const int v[1] = {none};
            refused += scan<1>(v, sums).total[0];
        }
    }
    if (count + back > p.pages) bad = true;  // more pages than there are: some were in the list already
    if (bad) atomicOr(p.err + kErrBatch, 1u);
    if (tid == 0) {
        p.row_start[p.seqs] = rows;
        *p.free_count = avail - need;
        if (p.refused) *p.refused = refused;
        if constexpr (ONE) {
            starts[0][p.seqs] = back;
            starts[1][p.seqs] = need;
            starts[2][p.seqs] = rows;
        }
        if (!ONE || !rows_too) {
            p.need_start[p.seqs] = need;
            p.totals[kAvail] = avail;
            p.totals[kNeed] = need;
            p.totals[kRows] = rows;
        }
    }
    __syncthreads();  // lengths and starts
    auto from_length = [&](int i) { return step_columns(p.length[i], p.shift, p.shared); };
    if constexpr (ONE) {
        if (!rows_too) {
            give_back<4>(p, starts[0], [&](int i) { return starts[2][i]; }, count, back, tid, kThreads);
            return;
        }
        give_back<2>(p, starts[0], from_length, count, back, tid, kThreads);
        __syncthreads();
        take<2>(p, starts[1], starts[2], avail, need, rows, tid, kThreads);
    } else {
        give_back<4>(p, p.back_start, from_length, count, back, tid, kThreads);
    }
}

__global__ __launch_bounds__(256) void kv_step_take_kernel(StepParams p) {
    take<1>(p, p.need_start, p.row_start, p.totals[kAvail], p.totals[kNeed], p.totals[kRows], blockIdx.x * 256 + threadIdx.x,
         gridDim.x * 256);
}

// Rows up to which one workgroup does it all (us a step there and in two launches, half the steps taking as much back:
// 256 rows 3.5 and 4.9, 4096 4.6 and 5.7, 8192 5.3 and 5.4, 16384 8.1 and 5.6).
constexpr int kOneRows = 8192;

}  // namespace

hipError_t launch_kv_step(StepParams p, int32_t* scratch, hipStream_t st) {
    p.totals = scratch;
    p.need_start = scratch + kStepTotals;
    p.back_start = p.need_start + p.seqs + 1;
    const bool rows_too = p.seqs <= 4 * kThreads && p.rows <= kOneRows;
    if (p.seqs <= kThreads) kv_step_kernel<1, true><<<1, kThreads, 0, st>>>(p, rows_too);
    else if (p.seqs <= 4 * kThreads) kv_step_kernel<4, true><<<1, kThreads, 0, st>>>(p, rows_too);
    else kv_step_kernel<4, false><<<1, kThreads, 0, st>>>(p, 0);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || rows_too) return e;
    const int blocks = (p.rows + 255) / 256;
    kv_step_take_kernel<<<std::clamp(blocks, 128, 2048), 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace qlin
