// Rotary positions, the pass from the qkv projection and the tables of a serving step without a GPU: the integer rules of the
// tables, and what the entry points refuse.  The HIP calls of libqlinear.so bind to the definitions below (device memory is
// host memory, kernels do not run).
//
//   step_calls_test rules     the rules of a slot against a plain account, searches in starts, sums that stay in bounds
//   step_calls_test tables    whole steps made of those rules, page by page, with every kind of bad number in the arrays
//   step_calls_test refusals  arguments outside the documented limits are refused before any launch
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <limits>
#include <vector>

#include <hip/hip_runtime_api.h>

#include "../../include/qlinear.h"
#include "../../open_rknpu2_lm_infer_amd/csrc/qlin_kv_step.hpp"

namespace {
int g_launches = 0, g_device = 0, g_fail = 0;
uint64_t g_threads = 0;  // of the largest launch
hipError_t alloc(void** p, size_t n) {
    if (g_fail > 0 && --g_fail == 0) return hipErrorOutOfMemory;
    *p = std::calloc(1, n ? n : 1);
    return *p ? hipSuccess : hipErrorOutOfMemory;
}
dim3 g_grid, g_block;
}  // namespace

extern "C" {
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = g_device, hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { return alloc(p, n); }
hipError_t hipFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipMemset(void* p, int v, size_t n) { return std::memset(p, v, n), hipSuccess; }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { return std::memcpy(d, s, n), hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
    void* p;
    const hipError_t e = alloc(&p, 1);
    *s = static_cast<hipStream_t>(p);
    return e;
}
hipError_t hipStreamDestroy(hipStream_t s) { return std::free(s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode*) { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t, hipStream_t) { return g_grid = g, g_block = b, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* st) {
    *g = g_grid;
    *b = g_block;
    *lds = 0;
    *st = nullptr;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 g, dim3 b, void**, size_t, hipStream_t) {
    g_threads = std::max(g_threads, (uint64_t)g.x * g.y * g.z * b.x * b.y * b.z);
    return ++g_launches, hipSuccess;
}
}

namespace {

int g_bad = 0;
void expect(bool ok, const char* what) {
    if (!ok) {
        std::printf("FAILED: %s\n", what);
        ++g_bad;
    }
}

constexpr int kBig = std::numeric_limits<int>::max(), kLow = std::numeric_limits<int>::min();

int columns(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

void rules() {
    const int vals[] = {kLow, kLow + 1, -4097, -64, -1, 0, 1, 15, 16, 17, 40, 64, 65, 4096, 1 << 30, kBig};
    for (int n : vals)
        for (int c : vals)
            for (int shift : {4, 6})
                for (int shared : {0, 1, 3})
                    for (int rows : {0, 40, 1 << 24})
                        for (int max_new : {0, 17, 1 << 24})
                            for (int max_len : {64, 1 << 30}) {
                                if (shared << shift > max_len) continue;
                                const qlin::StepSlot s = qlin::step_slot(n, c, shift, shared, rows, max_new, max_len);
                                const bool bad = n < 0 || n > max_len;
                                expect(s.bad == bad && s.asks == (c > 0), "what is wrong is said");
                                if (bad) {
                                    expect(s.len == n && !s.back && !s.want && !s.need, "a slot at fault is left alone");
                                    continue;
                                }
                                const int page = 1 << shift, held = std::max(columns(n, page), shared);
                                if (c <= 0) {
                                    const int len = (int)std::max<int64_t>((int64_t)n + c, 0);
                                    expect(s.len == len && s.want == 0 && s.need == 0, "tokens taken back");
                                    expect(s.back == (c < 0 ? held - std::max(columns(len, page), shared) : 0), "pages given back");
                                    expect(s.back == 0 || (s.from >= shared && s.from + s.back == held), "the last of its own columns");
                                } else {
                                    const bool fits = c <= max_new && c <= rows && (int64_t)n + c <= max_len;
                                    expect(s.len == n && s.back == 0 && s.want == (fits ? c : 0), "tokens asked for");
                                    expect(s.need == (fits ? std::max(columns((int64_t)n + c, page), shared) - held : 0), "pages for them");
                                }
                            }
    for (int a : {0, 1, 5, 1 << 24, (1 << 30) - 1, 1 << 30})
        for (int b : {0, 1, 5, 1 << 24, (1 << 30) - 1, 1 << 30})
            expect(qlin::step_add(a, b) == std::min<int64_t>((int64_t)a + b, 1 << 30), "sums");
    std::srand(1);
    for (int round = 0; round < 200; ++round) {
        const int n = 1 + std::rand() % 40;
        std::vector<int> start(n + 1, 0), whose;
        for (int i = 0; i < n; ++i) {
            const int m = std::rand() % 3 ? 0 : std::rand() % 5;
            start[i + 1] = start[i] + m;
            whose.insert(whose.end(), m, i);
        }
        for (int k = 0; k < (int)whose.size(); ++k) expect(qlin::step_owner(start.data(), n, k) == whose[k], "whose a thing is");
    }
}

// The kernels' accesses to the table and the list for scanned starts of any slots, checked against their bounds.
void tables() {
    std::srand(2);
    for (int round = 0; round < 3000; ++round) {
        const int shift = 4, page = 16, seqs = 1 + std::rand() % 12, cols = 1 + std::rand() % 6, max_len = cols * page - std::rand() % page;
        const int shared = std::rand() % (max_len / page + 1) / 2, rows = std::rand() % 60, max_new = std::rand() % 50, pages = std::rand() % 40;
        int count = std::rand() % 4 ? std::rand() % (pages + 1) : std::rand() % 200 - 100;
        count = qlin::kv_clamp(count, 0, pages);
        std::vector<qlin::StepSlot> s(seqs);
        std::vector<int> length(seqs), back{0}, need{0}, row{0};
        for (int i = 0; i < seqs; ++i) {
            const int n = std::rand() % 8 ? std::rand() % (max_len + 1) : std::rand() % 400 - 200;
            const int c = std::rand() % 6 ? std::rand() % 70 - 30 : (std::rand() % 2 ? kLow : kBig);
            s[i] = qlin::step_slot(n, c, shift, shared, rows, max_new, max_len);
            back.push_back(back.back() + s[i].back);
        }
        const int avail = std::min(count + back.back(), pages);
        int64_t row_sum = 0, need_sum = 0;
        for (int i = 0; i < seqs; ++i) {
            row_sum += s[i].want;
            if (row_sum > rows) s[i].want = s[i].need = 0;
            need_sum += s[i].need;
            if (s[i].need > 0 && need_sum > avail) s[i].want = s[i].need = 0;
            length[i] = s[i].len + s[i].want;
            need.push_back(need.back() + s[i].need);
            row.push_back(row.back() + s[i].want);
        }
        expect(need.back() <= avail && row.back() <= rows, "no more than there is");
        for (int k = 0; k < back.back(); ++k) {
            const int i = qlin::step_owner(back.data(), seqs, k), c = qlin::step_columns(length[i], shift, shared) + k - back[i];
            expect(c >= shared && c < cols, "a column given back");
        }
        for (int k = 0; k < need.back(); ++k) {
            const int i = qlin::step_owner(need.data(), seqs, k), old = length[i] - (row[i + 1] - row[i]);
            const int c = qlin::step_columns(old, shift, shared) + k - need[i];
            expect(c >= shared && c < cols && avail - 1 - k >= 0 && avail - 1 - k < pages, "a column taken, and its page");
        }
        for (int r = 0; r < row.back(); ++r) {
            const int i = qlin::step_owner(row.data(), seqs, r), old = length[i] - (row[i + 1] - row[i]), pos = old + r - row[i];
            const int c = pos >> shift, fresh = c - qlin::step_columns(old, shift, shared);
            expect(pos >= 0 && pos < max_len && c < cols, "a row's place");
            expect(fresh < s[i].need && (fresh < 0 || avail - 1 - (need[i] + fresh) >= 0), "a row's page");
        }
    }
}

void refusals() {
    // rotary positions
    const qlin_rope_config good = {128, 64, 0, QLIN_ROPE_HALF, QLIN_ROPE_PLAIN, 0, 1e4, 0.0, 0.0, 0.0, 0.0, 0.0};
    qlin_rope* r = nullptr;
    const double nan = std::nan(""), inf = std::numeric_limits<double>::infinity();
    for (int i = 0; i < 30; ++i) {
        qlin_rope_config g = good;
        g.factor = 4.0;
        g.original_len = 8192;
        g.low = 1.0;
        g.high = 4.0;
        switch (i) {
            case 0: g.head_dim = 0; break;
            case 1: g.head_dim = -4; break;
            case 2: g.rotary_dim = 0; break;
            case 3: g.rotary_dim = 63; break;
            case 4: g.rotary_dim = 130; break;
            case 5: g.first = -2; break;
            case 6: g.first = 65; break;
            case 7: g.layout = 2; break;
            case 8: g.layout = -1; break;
            case 9: g.scaling = 5; break;
            case 10: g.scaling = -1; break;
            case 11: g.base = 1.0; break;
            case 12: g.base = nan; break;
            case 13: g.base = inf; break;
            case 14: g.amplitude = -1.0; break;
            case 15: g.amplitude = nan; break;
            case 16: g.scaling = QLIN_ROPE_LINEAR, g.factor = 0.5; break;
            case 17: g.scaling = QLIN_ROPE_BASE, g.factor = nan; break;
            case 18: g.scaling = QLIN_ROPE_BANDS, g.low = 0.0; break;
            case 19: g.scaling = QLIN_ROPE_BANDS, g.high = 1.0; break;
            case 20: g.scaling = QLIN_ROPE_RAMP, g.original_len = 0.0; break;
            case 21: g.scaling = QLIN_ROPE_RAMP, g.low = nan; break;
            case 22: g.scaling = QLIN_ROPE_RAMP, g.high = inf; break;
            case 23: g.scaling = QLIN_ROPE_BANDS, g.original_len = inf; break;
            case 24: g.first = kBig; break;
            case 25: g.rotary_dim = kLow; break;
            case 26: g.head_dim = 64, g.first = 2; break;
            case 27: g.scaling = QLIN_ROPE_LINEAR, g.factor = inf; break;
            case 28: g.amplitude = 1e39; break;
            case 29: g.amplitude = inf; break;
        }
        r = reinterpret_cast<qlin_rope*>(1);
        expect(qlin_rope_create(&g, &r) == QLIN_ERR_PARAM && !r, "a configuration that makes no sense");
    }
    qlin_rope_config wide = good;
    wide.head_dim = 257;
    expect(qlin_rope_create(&wide, &r) == QLIN_ERR_UNSUPPORTED && !r, "heads too wide");
    expect(qlin_rope_create(nullptr, &r) == QLIN_ERR_PARAM && qlin_rope_create(&good, nullptr) == QLIN_ERR_PARAM, "null");
    g_fail = 1;
    expect(qlin_rope_create(&good, &r) == QLIN_ERR_NOMEM && !r, "an allocation that fails");
    g_fail = 0;
    qlin_rope_free(nullptr);
    expect(qlin_rope_create(&good, &r) == QLIN_OK && r, "a rope");
    double w[32], a;
    expect(qlin_rope_query(r, w, &a) == QLIN_OK && w[0] == 1.0 && std::fabs(w[16] - 0.01) < 1e-15 && a == 1.0, "query");
    expect(qlin_rope_query(nullptr, w, &a) == QLIN_ERR_PARAM && qlin_rope_query(r, nullptr, &a) == QLIN_ERR_PARAM, "query of nothing");

    std::vector<float> x(4 * 6 * 128), y(x.size()), gamma(128, 1.0f);
    int32_t pos[4] = {0, 1, 2, 3};
    const int F = QLIN_F32;
    g_launches = 0;
    const auto turn = [&](int rows, int heads, int64_t ldx = 768, int64_t ldy = 768, int xt = QLIN_F32, int yt = QLIN_F32, uint32_t flags = 0) {
        return qlin_rope_run(r, rows, heads, x.data(), xt, ldx, pos, y.data(), yt, ldy, flags, nullptr);
    };
    expect(turn(-1, 6) == QLIN_ERR_PARAM && turn(4, 0) == QLIN_ERR_PARAM && turn(4, -1) == QLIN_ERR_PARAM, "sizes");
    expect(turn(4, 6, 767) == QLIN_ERR_PARAM && turn(4, 6, 768, 700) == QLIN_ERR_PARAM, "rows too narrow");
    expect(turn(4, 6, 768, 768, 2) == QLIN_ERR_PARAM && turn(4, 6, 768, 768, F, -1) == QLIN_ERR_PARAM, "unknown type");
    expect(turn(4, 6, 768, 768, F, F, QLIN_ROUND_HALF_EVEN) == QLIN_ERR_PARAM, "a flag of another call");
    expect(turn(4, 1025, 1 << 20, 1 << 20) == QLIN_ERR_UNSUPPORTED && turn(1 << 24, 6) == QLIN_ERR_UNSUPPORTED, "too much");
    expect(turn(4, kBig) == QLIN_ERR_PARAM, "heads of any number");
    expect(qlin_rope_run(nullptr, 4, 6, x.data(), F, 768, pos, y.data(), F, 768, 0, nullptr) == QLIN_ERR_PARAM, "no rope");
    expect(qlin_rope_run(r, 4, 6, nullptr, F, 768, pos, y.data(), F, 768, 0, nullptr) == QLIN_ERR_PARAM, "no rows");
    expect(qlin_rope_run(r, 4, 6, x.data(), F, 768, nullptr, y.data(), F, 768, 0, nullptr) == QLIN_ERR_PARAM, "no positions");
    expect(qlin_rope_run(r, 4, 6, x.data(), F, 768, pos, nullptr, F, 768, 0, nullptr) == QLIN_ERR_PARAM, "no output");
    const auto norm = [&](const qlin_rope* rope, int dim, int q, int k, float eps, const float* g, const int32_t* p) {
        return qlin_rope_run_norm(rope, 4, dim, q, k, g, g, eps, x.data(), F, 768, p, y.data(), F, 768, 0, nullptr);
    };
    expect(norm(r, 64, 4, 2, 1e-6f, gamma.data(), pos) == QLIN_ERR_PARAM, "heads of another width");
    expect(norm(r, 128, -1, 2, 1e-6f, gamma.data(), pos) == QLIN_ERR_PARAM && norm(r, 128, 0, 0, 1e-6f, gamma.data(), pos) == QLIN_ERR_PARAM &&
               norm(r, 128, kBig, kBig, 1e-6f, gamma.data(), pos) == QLIN_ERR_PARAM, "heads");
    for (float eps : {0.0f, -1.0f, (float)nan, (float)inf}) expect(norm(r, 128, 4, 2, eps, gamma.data(), pos) == QLIN_ERR_PARAM, "eps");
    expect(norm(nullptr, 257, 1, 1, 1e-6f, gamma.data(), nullptr) == QLIN_ERR_UNSUPPORTED, "heads too wide");
    expect(norm(r, 128, 4, 2, 1e-6f, gamma.data(), nullptr) == QLIN_ERR_PARAM, "no positions");
    g_device = 1;
    expect(turn(4, 6) == QLIN_ERR_PARAM, "another device");
    g_device = 0;
    expect(g_launches == 0, "nothing was launched");
    expect(turn(0, 6) == QLIN_OK && g_launches == 0, "no rows, nothing to do");
    expect(turn(4, 6) == QLIN_OK && turn(4, 6, 768, 768, F, F, QLIN_ROPE_INVERSE) == QLIN_OK && g_launches == 2, "turned");
    expect(norm(r, 128, 4, 2, 1e-6f, gamma.data(), pos) == QLIN_OK && norm(r, 128, 4, 2, 0.0f, nullptr, pos) == QLIN_OK &&
               norm(nullptr, 128, 4, 2, 1e-6f, gamma.data(), nullptr) == QLIN_OK && norm(r, 128, 0, 6, 1e-6f, gamma.data(), pos) == QLIN_OK, "normalized");
    for (int rows : {1, 100, 5000, (1 << 24) - 1}) {
        g_threads = 0;
        expect(qlin_rope_run(r, rows, 1024, x.data(), F, 1024 * 128, pos, y.data(), F, 1024 * 128, 0, nullptr) == QLIN_OK && g_threads < 1ull << 32, "what a launch covers");
    }

    // caches of 8 and 4 bits, the pass from the qkv projection
    qlin_kv_cache* c = nullptr;
    const qlin_kv_config cfg = {2, 128, 16, 8};
    for (int bits : {0, 2, 3, 5, 16, -4}) expect(qlin_kv_create_bits(&cfg, bits, &c) == QLIN_ERR_PARAM && !c, "bits");
    expect(qlin_kv_bits(nullptr) == QLIN_ERR_PARAM, "bits of nothing");
    qlin_workspace* ws = nullptr;
    expect(qlin_workspace_create(1, 8, 8, &ws) == QLIN_OK, "workspace");
    for (int bits : {8, 4}) {
        expect(qlin_kv_create_bits(&cfg, bits, &c) == QLIN_OK && qlin_kv_bits(c) == bits, "a cache");
        qlin_kv_info info;
        expect(qlin_kv_query(c, &info) == QLIN_OK && info.device_bytes == 8u * 2 * 16 * (bits == 8 ? 264 : 144), "bytes");
        const int32_t starts[2] = {0, 4}, length[1] = {20}, table[2] = {0, 1};
        const qlin_kv_batch b = {1, 4, 4, 32, starts, length, table, 2};
        std::vector<float> qkv(4 * 8 * 128), q(4 * 4 * 128);
        const auto pass = [&](const qlin_kv_batch& b, const qlin_rope* rope, int heads = 4, int64_t ld = 1024, int64_t ldq = 512, float eps = 1e-6f,
                              const float* g = nullptr, int t = QLIN_F32, uint32_t flags = 0) {
            return qlin_kv_append_qkv(ws, c, &b, rope, heads, g, g, eps, qkv.data(), t, ld, q.data(), F, ldq, flags, nullptr);
        };
        g_launches = 0;
        expect(pass(b, r, 0) == QLIN_ERR_PARAM && pass(b, r, -3) == QLIN_ERR_PARAM && pass(b, r, 1025, 1 << 20, 1 << 20) == QLIN_ERR_UNSUPPORTED, "heads");
        expect(pass(b, r, 4, 1023) == QLIN_ERR_PARAM && pass(b, r, 4, 1024, 511) == QLIN_ERR_PARAM, "rows too narrow");
        expect(pass(b, r, 4, 1024, 512, 0.0f, gamma.data()) == QLIN_ERR_PARAM, "eps");
        expect(pass(b, r, 4, 1024, 512, 1e-6f, nullptr, 7) == QLIN_ERR_PARAM && pass(b, r, 4, 1024, 512, 1e-6f, nullptr, F, QLIN_ROPE_INVERSE) == QLIN_ERR_PARAM, "type, flag");
        qlin_rope_config other = good;
        other.head_dim = 64;
        qlin_rope* r64 = nullptr;
        expect(qlin_rope_create(&other, &r64) == QLIN_OK && pass(b, r64) == QLIN_ERR_PARAM, "heads of another width");
        qlin_rope_free(r64);
        g_device = 1;
        qlin_rope* elsewhere = nullptr;
        expect(qlin_rope_create(&good, &elsewhere) == QLIN_OK, "a rope of another device");
        expect(pass(b, r) == QLIN_ERR_PARAM, "another device");
        g_device = 0;
        expect(pass(b, elsewhere) == QLIN_ERR_PARAM, "a rope of another device");
        qlin_rope_free(elsewhere);
        for (int i = 0; i < 4; ++i) {
            qlin_kv_batch z = b;
            if (i == 0) z.seqs = 0;
            if (i == 1) z.max_new = 5;
            if (i == 2) z.page_ld = 1;
            if (i == 3) z.row_start = nullptr;
            expect(pass(z, r) == QLIN_ERR_PARAM, "a batch that makes no sense");
        }
        qlin_kv_batch z = b;
        z.seqs = 1 << 12;
        z.rows = 1 << 24;
        z.max_new = 1 << 12;
        expect(pass(z, r) == QLIN_ERR_UNSUPPORTED, "more than a launch covers");
        expect(g_launches == 0, "nothing was launched");
        z.max_new = (1 << 12) - 1;
        g_threads = 0;
        expect(pass(z, r, 1024, 1 << 20, 1 << 20) == QLIN_OK && g_threads < 1ull << 32, "what a launch covers");
        expect(pass(b, r) == QLIN_OK && pass(b, nullptr) == QLIN_OK && pass(b, r, 4, 1024, 512, 1e-6f, gamma.data()) == QLIN_OK && g_launches == 4, "one launch each");
        const qlin_kv_batch idle = {1, 0, 0, 32, starts, length, table, 2};
        expect(qlin_kv_append_qkv(ws, c, &idle, r, 4, nullptr, nullptr, 0.0f, nullptr, F, 1024, nullptr, F, 512, 0, nullptr) == QLIN_OK && g_launches == 4, "idle");

        // tables
        int32_t change[2] = {1, 0}, len[2] = {0, 0}, tab[4] = {}, free_pages[8] = {}, free_count = 0, row_start[3];
        const qlin_kv_tables t = {2, 8, 4, 32, 16, 0, change, len, tab, 2, free_pages, &free_count, row_start, nullptr, nullptr, nullptr, nullptr};
        const int before = g_launches;
        for (int i = 0; i < 15; ++i) {
            qlin_kv_tables z = t;
            switch (i) {
                case 0: z.seqs = 0; break;
                case 1: z.rows = -1; break;
                case 2: z.max_new = -1; break;
                case 3: z.max_len = -1; break;
                case 4: z.prefix_tokens = 8; break;
                case 5: z.prefix_tokens = -16; break;
                case 6: z.prefix_tokens = 48; break;
                case 7: z.change = nullptr; break;
                case 8: z.length = nullptr; break;
                case 9: z.page_table = nullptr; break;
                case 10: z.page_ld = 1; break;
                case 11: z.free_pages = nullptr; break;
                case 12: z.free_count = nullptr; break;
                case 13: z.row_start = nullptr; break;
                case 14: z.page_ld = -1; break;
            }
            expect(qlin_kv_step(ws, c, &z, nullptr) == QLIN_ERR_PARAM, "tables that make no sense");
        }
        expect(qlin_kv_step(nullptr, c, &t, nullptr) == QLIN_ERR_PARAM && qlin_kv_step(ws, nullptr, &t, nullptr) == QLIN_ERR_PARAM &&
                   qlin_kv_step(ws, c, nullptr, nullptr) == QLIN_ERR_PARAM, "null");
        for (int i = 0; i < 4; ++i) {
            qlin_kv_tables z = t;
            if (i == 0) z.seqs = (1 << 20) + 1;
            if (i == 1) z.rows = (1 << 24) + 1;
            if (i == 2) z.max_len = (1 << 30) + 1, z.page_ld = 1 << 27;
            if (i == 3) z.seqs = 17, z.max_len = 1 << 30, z.page_ld = 1 << 26;
            expect(qlin_kv_step(ws, c, &z, nullptr) == QLIN_ERR_UNSUPPORTED, "too much");
        }
        g_device = 1;
        expect(qlin_kv_step(ws, c, &t, nullptr) == QLIN_ERR_PARAM, "another device");
        g_device = 0;
        expect(g_launches == before, "nothing was launched");
        expect(qlin_kv_step(ws, c, &t, nullptr) == QLIN_OK && g_launches == before + 1, "a small step is one launch");
        qlin_kv_free(c);
    }
    qlin_workspace_free(ws);
    qlin_rope_free(r);
}

}  // namespace

int main(int argc, char** argv) {
    const char* mode = argc > 1 ? argv[1] : "";
    if (!std::strcmp(mode, "rules")) rules();
    else if (!std::strcmp(mode, "tables")) tables();
    else if (!std::strcmp(mode, "refusals")) refusals();
    else return 2;
    if (!g_bad) std::printf("PASS %s\n", mode);
    return g_bad != 0;
}
