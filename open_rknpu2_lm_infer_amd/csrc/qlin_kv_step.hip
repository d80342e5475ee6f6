// Tables of a serving step from the requests' lengths: rows, pages and slots of the key/value cache.
//
// Slot i holds n_i tokens and asks for c_i more, or gives -c_i back.  Pages given back go on top of the free list in the
// order of the slots, then those asked for are taken from its top in the same order:
//   wanted   w_i = c_i where the slot's own limits allow it,  and sum_{j <= i} w_j <= rows
//   granted  p_i = pages that n_i + w_i tokens take beyond those of n_i;  p_i = 0 or sum_{j <= i} p_j <= free pages
// Every sum is a scan, so that nothing depends on the order in which threads run.  Sums grow along the slots: who is
// refused for want of rows (or pages) is followed by none that is granted some, and what the granted take is the sum itself.
//
// One workgroup scans, 1024 slots at a time.  Whose the k-th row, page taken or page given back is, is found by a binary
// search in the scanned starts.  With few rows the same workgroup does that too, with the starts in the LDS: one launch;
// with more, two more launches do: the pages given back have to lie in the list before any is taken.
#include <hip/hip_runtime.h>

#include "qlin_kv.hpp"
#include "qlin_kv_step.hpp"

namespace qlin {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
enum : int { kCount = 0, kAvail = 1, kNeed = 2, kBack = 3, kRows = 4, kTotals = 8 };

// Inclusive sums of N values over the workgroup, and their totals.
template <int N>
struct Scan {
    int at[N], total[N];
};
template <int N>
__device__ __forceinline__ Scan<N> scan(const int (&v)[N], int (*lds)[kWaves]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Scan<N> s;
#pragma unroll
    for (int k = 0; k < N; ++k) s.at[k] = v[k];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int y = __shfl_up(s.at[k], o, 64);
            s.at[k] = step_add(s.at[k], lane >= o ? y : 0);
        }
    __syncthreads();  // who still reads an earlier scan's
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < N; ++k) lds[k][wave] = s.at[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const int x = lds[k][w];
            before = w < wave ? step_add(before, x) : before;
            all = step_add(all, x);
        }
        s.at[k] = step_add(s.at[k], before);
        s.total[k] = all;
    }
    return s;
}

// Pages given back: from the table to the free list, from thread `first` on every `stride`.
template <typename P>
__device__ __forceinline__ void give_back(const StepParams& p, P back_start, int count, int total, int first, int stride) {
    for (int k = first; k < total; k += stride) {
        const int i = step_owner(back_start, p.seqs, k);
        const int column = step_columns(p.length[i], p.shift, p.shared) + k - back_start[i];
        int32_t* at = p.table + i * p.table_ld + column;
        const int id = *at;
        *at = -1;
        bool bad = count + k >= p.pages;  // more pages than there are: some were in the list already
        if (!bad) p.free_pages[count + k] = id;
        kv_page(id, p.pages, &bad);
        if (bad) atomicOr(p.err + kErrBatch, 1u);
    }
}

// Pages taken and the rows' maps.  What the list holds is not written here, and of the table only what a slot is given.
template <typename P>
__device__ __forceinline__ void take(const StepParams& p, P need_start, P row_start, int avail, int need, int rows, int first, int stride) {
    for (int k = first; k < need; k += stride) {
        const int i = step_owner(need_start, p.seqs, k);
        const int old = p.length[i] - (row_start[i + 1] - row_start[i]);
        const int id = p.free_pages[avail - 1 - k];
        p.table[i * p.table_ld + step_columns(old, p.shift, p.shared) + k - need_start[i]] = id;
        bool bad = false;
        kv_page(id, p.pages, &bad);
        if (bad) atomicOr(p.err + kErrBatch, 1u);
    }
    if (!p.row_seq && !p.positions && !p.slots) return;
    for (int r = first; r < rows; r += stride) {
        const int i = step_owner(row_start, p.seqs, r);
        const int begin = row_start[i], old = p.length[i] - (row_start[i + 1] - begin), pos = old + r - begin;
        if (p.row_seq) p.row_seq[r] = i;
        if (p.positions) p.positions[r] = pos;
        if (p.slots) {
            // a page taken in this step comes from the list, as its table entry is being written
            const int column = pos >> p.shift, fresh = column - step_columns(old, p.shift, p.shared);
            const int id = fresh >= 0 ? p.free_pages[avail - 1 - (need_start[i] + fresh)] : p.table[i * p.table_ld + column];
            p.slots[r] = ((int64_t)id << p.shift) + (pos & ((1 << p.shift) - 1));
        }
    }
}

// ALL: up to 1024 slots, and the rows and pages too.
template <bool ALL>
__global__ __launch_bounds__(kThreads) void kv_step_kernel(StepParams p) {
    __shared__ int sums[3][kWaves];
    __shared__ int lds[ALL ? 3 : 1][ALL ? kThreads + 1 : 1];
    const int tid = threadIdx.x;
    int count = *p.free_count;
    bool bad = count < 0 || count > p.pages;
    count = kv_clamp(count, 0, p.pages);
    auto slot = [&](int i) {
        StepSlot s{};
        if (i < p.seqs) s = step_slot(p.length[i], p.change[i], p.shift, p.shared, p.rows, p.max_new, p.max_len);
        bad |= s.bad;
        return s;
    };
    int back = 0;
    if constexpr (!ALL) {
        for (int i0 = 0; i0 < p.seqs; i0 += kThreads) {
            const int v[1] = {slot(i0 + tid).back};
            const Scan<1> s = scan<1>(v, sums);
            if (i0 + tid < p.seqs) p.back_start[i0 + tid] = back + s.at[0] - v[0];
            back += s.total[0];
        }
        if (tid == 0) p.back_start[p.seqs] = back;
    }
    int rows_sum = 0, need_sum = 0, rows = 0, need = 0, refused = 0, avail = 0;
    for (int i0 = 0; i0 < p.seqs; i0 += kThreads) {
        const int i = i0 + tid;
        StepSlot s = slot(i);
        const int all[3] = {s.want, s.need, ALL ? s.back : 0};
        const Scan<3> t = scan<3>(all, sums);
        if constexpr (ALL) back = t.total[2];
        avail = min(count + back, p.pages);
        int row_at = rows + t.at[0], need_at = need + t.at[1], row_total = t.total[0], need_total = t.total[1];
        const bool short_of = step_add(rows_sum, t.total[0]) > p.rows || step_add(need_sum, t.total[1]) > avail;
        if (!short_of) {
            rows_sum += t.total[0];
            need_sum += t.total[1];
        } else {
            // some are refused: rows first, then pages, then what is left
            if (step_add(rows_sum, t.at[0]) > p.rows) s.want = s.need = 0;
            rows_sum = step_add(rows_sum, t.total[0]);
            const int v[1] = {s.need};
            const Scan<1> u = scan<1>(v, sums);
            if (s.need > 0 && step_add(need_sum, u.at[0]) > avail) s.want = s.need = 0;
            need_sum = step_add(need_sum, u.total[0]);
            const int w[2] = {s.want, s.need};
            const Scan<2> x = scan<2>(w, sums);
            row_at = rows + x.at[0];
            need_at = need + x.at[1];
            row_total = x.total[0];
            need_total = x.total[1];
        }
        if (i < p.seqs) {
            p.row_start[i] = row_at - s.want;
            if (s.len + s.want != p.length[i]) p.length[i] = s.len + s.want;
            if constexpr (ALL) {
                lds[0][i] = row_at - s.want;
                lds[1][i] = need_at - s.need;
                lds[2][i] = t.at[2] - s.back;
            } else {
                p.need_start[i] = need_at - s.need;
            }
        }
        rows += row_total;
        need += need_total;
        refused += __syncthreads_count(s.asks && s.want == 0);
    }
    if (bad) atomicOr(p.err + kErrBatch, 1u);
    if (tid == 0) {
        p.row_start[p.seqs] = rows;
        *p.free_count = avail - need;
        if (p.refused) *p.refused = refused;
        if (count + back > p.pages) atomicOr(p.err + kErrBatch, 1u);
        if constexpr (ALL) {
            lds[0][p.seqs] = rows;
            lds[1][p.seqs] = need;
            lds[2][p.seqs] = back;
        } else {
            p.need_start[p.seqs] = need;
            p.totals[kCount] = count;
            p.totals[kAvail] = avail;
            p.totals[kNeed] = need;
            p.totals[kBack] = back;
            p.totals[kRows] = rows;
        }
    }
    if constexpr (ALL) {
        __syncthreads();  // lengths and starts
        give_back(p, lds[2], count, back, tid, kThreads);
        __syncthreads();
        take(p, lds[1], lds[0], avail, need, rows, tid, kThreads);
    }
}

__global__ __launch_bounds__(256) void kv_step_back_kernel(StepParams p) {
    give_back(p, p.back_start, p.totals[kCount], p.totals[kBack], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}
__global__ __launch_bounds__(256) void kv_step_take_kernel(StepParams p) {
    take(p, p.need_start, p.row_start, p.totals[kAvail], p.totals[kNeed], p.totals[kRows], blockIdx.x * 256 + threadIdx.x,
         gridDim.x * 256);
}

// Rows up to which one workgroup does it all.
constexpr int kOneRows = 4096;

}  // namespace

int64_t kv_step_scratch(int seqs) { return kTotals + 2 * ((int64_t)seqs + 1); }

hipError_t launch_kv_step(StepParams p, int32_t* scratch, hipStream_t st) {
    p.totals = scratch;
    p.need_start = scratch + kTotals;
    p.back_start = p.need_start + p.seqs + 1;
    if (p.seqs <= kThreads && p.rows <= kOneRows) {
        kv_step_kernel<true><<<1, kThreads, 0, st>>>(p);
        return hipGetLastError();
    }
    kv_step_kernel<false><<<1, kThreads, 0, st>>>(p);
    if (const hipError_t e = hipGetLastError()) return e;
    kv_step_back_kernel<<<256, 256, 0, st>>>(p);
    if (const hipError_t e = hipGetLastError()) return e;
    const int64_t items = p.rows;
    const int grid = (int)((items + 255) / 256 < 128 ? 128 : (items + 255) / 256 > 2048 ? 2048 : (items + 255) / 256);
    kv_step_take_kernel<<<grid, 256, 0, st>>>(p);
    return hipGetLastError();
}

}  // namespace qlin
