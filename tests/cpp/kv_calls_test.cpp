// Key/value cache without a GPU: the indexing that guards the kernels' reads, and what the entry
// points refuse.  The HIP calls of libqlinear.so bind to the definitions below (device memory is
// host memory, kernels do not run).
//
//   kv_calls_test index     row starts, lengths and page ids of any value stay inside the buffers
//   kv_calls_test refusals  arguments outside the documented limits are refused before any launch
//   kv_calls_test limits    the largest query heads and scales are taken, larger ones refused
//   kv_calls_test devices   each device that launches the kernel for many vectors has been asked for its LDS
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <limits>
#include <set>
#include <utility>
#include <vector>

#include <hip/hip_runtime_api.h>

#include "../../include/qlinear.h"
#include "../../open_rknpu2_lm_infer_amd/csrc/qlin_kv_index.hpp"

namespace {
int g_launches = 0, g_device = 0, g_fail = 0;
std::set<std::pair<const void*, int>> g_lds;  // functions whose dynamic LDS was raised, and on which device
hipError_t alloc(void** p, size_t n) {
    if (g_fail > 0 && --g_fail == 0) return hipErrorOutOfMemory;
    *p = std::calloc(1, n ? n : 1);
    return *p ? hipSuccess : hipErrorOutOfMemory;
}
}  // namespace

extern "C" {
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = g_device, hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) { return alloc(p, n); }
hipError_t hipFree(void* p) { return std::free(p), hipSuccess; }
hipError_t hipMemset(void* p, int v, size_t n) { return std::memset(p, v, n), hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) {
    void* p;
    const hipError_t e = alloc(&p, 1);
    *s = static_cast<hipStream_t>(p);
    return e;
}
hipError_t hipStreamDestroy(hipStream_t s) { return std::free(s), hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute a, int) {
    if (a == hipFuncAttributeMaxDynamicSharedMemorySize) g_lds.insert({f, g_device});
    return hipSuccess;
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode*) { return hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3, dim3, size_t, hipStream_t) { return hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* st) {
    *g = *b = dim3(1);
    *lds = 0;
    *st = nullptr;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3, dim3, void**, size_t, hipStream_t) { return ++g_launches, hipSuccess; }
}

namespace {

int g_bad = 0;
void expect(bool ok, const char* what) {
    if (!ok) {
        std::printf("FAILED: %s\n", what);
        ++g_bad;
    }
}

void index() {
    const int big = std::numeric_limits<int>::max(), low = std::numeric_limits<int>::min();
    const int vals[] = {low, low + 1, -4097, -1, 0, 1, 3, 7, 8, 9, 100, 4096, big - 1, big};
    for (int a : vals)
        for (int b : vals)
            for (int n : vals)
                for (int rows : {0, 1, 8, 100})
                    for (int max_new : {1, 8}) {
                        if (max_new > rows) continue;
                        const int starts[2] = {a, b};
                        const int max_len = 64;
                        const qlin::KvSeq s = qlin::kv_seq(starts, &n, 0, rows, max_new, max_len);
                        const bool good = a >= 0 && b >= a && b <= rows && b - a <= max_new && n >= 0 && n <= max_len;
                        expect(s.row0 >= 0 && s.rows >= 0 && s.rows <= max_new && s.row0 + s.rows <= rows, "rows in the tensor");
                        expect(s.len >= 0 && s.len <= max_len, "length in the table");
                        expect(s.bad == !good, "bad batches are flagged, good ones are not");
                        if (good) expect(s.row0 == a && s.rows == b - a && s.len == n, "good batches are taken as they are");
                        for (int t = 0; t < s.rows; ++t) {
                            const int seen = qlin::kv_visible(s, t);
                            expect(seen >= 0 && seen <= s.len, "visible tokens exist");
                            expect(seen == std::max(0, s.len - s.rows + t + 1), "causal");
                        }
                    }
    for (int id : vals) {
        bool bad = false;
        const int page = qlin::kv_page(id, 8, &bad);
        expect(page >= 0 && page < 8 && bad == (id < 0 || id >= 8), "pages in the cache");
    }
    for (int d : {1, 2, 3, 4, 5, 7, 8, 12, 31, 32, 33, 100, 127, 1000, 1 << 16, (1 << 16) + 1, (1 << 30) - 1, 1 << 30, big}) {
        const qlin::FastDiv f = qlin::fast_div(d);
        for (int64_t n : {0, 1, 2, 3, 30, 31, 32, 99, 100, 101, 4095, 4096, 1 << 20, (1 << 30) - 1, 1 << 30, big - 1, big})
            for (int64_t x : {n, n / d * d, n / d * d - 1, n / d * d + d - 1})
                if (x >= 0 && x <= big) expect(f.div((int)x) == x / d && f.mod((int)x) == x % d, "division by multiplication");
    }
    for (int tokens : {low, -5, 0, 1, 128, 129, 256, 1 << 30})
        expect(qlin::kv_parts(tokens, 128) == (tokens <= 128 ? 1 : (int)(((int64_t)tokens + 127) / 128)), "parts");
}

struct Made {
    qlin_kv_cache* c = nullptr;
    qlin_workspace* ws = nullptr;
    Made(int heads, int dim, int page, int pages) {
        const qlin_kv_config cfg = {heads, dim, page, pages};
        expect(qlin_kv_create(&cfg, &c) == QLIN_OK, "create");
        expect(qlin_workspace_create(1, 8, 8, &ws) == QLIN_OK, "workspace");
    }
    ~Made() {
        qlin_kv_free(c);
        qlin_workspace_free(ws);
    }
};

void refusals() {
    qlin_kv_cache* none = reinterpret_cast<qlin_kv_cache*>(1);
    const auto create = [&](int h, int d, int p, int n) {
        const qlin_kv_config cfg = {h, d, p, n};
        none = reinterpret_cast<qlin_kv_cache*>(1);
        return qlin_kv_create(&cfg, &none);
    };
    for (auto g : {std::vector<int>{0, 8, 16, 1}, {8, 0, 16, 1}, {8, 8, 0, 1}, {8, 8, 16, 0}, {-1, 8, 16, 1}, {8, 8, 24, 1}, {8, 8, -16, 1}})
        expect(create(g[0], g[1], g[2], g[3]) == QLIN_ERR_PARAM && !none, "geometry that makes no sense");
    for (auto g : {std::vector<int>{1025, 8, 16, 1}, {8, 257, 16, 1}, {8, 8, 8, 1}, {8, 8, 8192, 1}})
        expect(create(g[0], g[1], g[2], g[3]) == QLIN_ERR_UNSUPPORTED && !none, "geometry beyond the limits");
    expect(qlin_kv_create(nullptr, &none) == QLIN_ERR_PARAM && qlin_kv_create(nullptr, nullptr) == QLIN_ERR_PARAM, "null");
    g_fail = 1;
    expect(create(1, 64, 16, 1) == QLIN_ERR_NOMEM && !none, "an allocation that fails");
    g_fail = 0;
    expect(qlin_kv_query(nullptr, nullptr) == QLIN_ERR_PARAM, "query of nothing");
    qlin_kv_free(nullptr);

    Made m(2, 84, 16, 8);
    qlin_kv_info info;
    expect(qlin_kv_query(m.c, &info) == QLIN_OK && info.kv_heads == 2 && info.head_dim == 84 && info.head_dim_padded == 128 &&
               info.page_tokens == 16 && info.pages == 8 && info.device_bytes == 8 * 2 * 16 * (2 * 128 + 8), "query");
    const int32_t starts[3] = {0, 1, 4}, length[2] = {1, 30}, table[4] = {0, 1, 2, 3};
    const qlin_kv_batch good = {2, 4, 3, 32, starts, length, table, 2};
    std::vector<float> x(4 * 8 * 84), y(x.size());
    const int F = QLIN_F32;
    const auto append = [&](const qlin_kv_batch& b, int64_t ldk = 168, int64_t ldv = 168, int t = QLIN_F32, uint32_t flags = 0) {
        return qlin_kv_append(m.ws, m.c, &b, x.data(), ldk, x.data(), ldv, t, flags, nullptr);
    };
    const auto attend = [&](const qlin_kv_batch& b, int heads = 4, float scale = 1.0f, int64_t ldq = 336, int64_t ldo = 336) {
        return qlin_kv_attention(m.ws, m.c, &b, heads, x.data(), F, ldq, scale, y.data(), F, ldo, nullptr);
    };
    const auto prefix = [&](int tokens, const int32_t* pages) {
        return qlin_kv_attention_prefix(m.ws, m.c, &good, tokens, pages, 4, x.data(), F, 336, 1.0f, y.data(), F, 336, nullptr);
    };
    g_launches = 0;
    for (int i = 0; i < 12; ++i) {
        qlin_kv_batch b = good;
        switch (i) {
            case 0: b.seqs = 0; break;
            case 1: b.rows = -1; break;
            case 2: b.max_new = -1; break;
            case 3: b.max_new = 5; break;  // more than the rows
            case 4: b.max_len = -1; break;
            case 5: b.max_len = 33; break;  // two pages a sequence
            case 6: b.page_ld = 1; break;
            case 7: b.row_start = nullptr; break;
            case 8: b.length = nullptr; break;
            case 9: b.page_table = nullptr; break;
            case 10: b.seqs = -3; break;
            case 11: b.page_ld = -1; break;
        }
        expect(append(b) == QLIN_ERR_PARAM && attend(b) == QLIN_ERR_PARAM, "a batch that makes no sense");
    }
    qlin_kv_batch b = good;
    b.seqs = (1 << 20) + 1;
    expect(append(b) == QLIN_ERR_UNSUPPORTED && attend(b) == QLIN_ERR_UNSUPPORTED, "too many sequences");
    b = good;
    b.seqs = 1 << 20;
    b.rows = 1 << 24;
    b.max_new = 1 << 12;
    expect(append(b) == QLIN_ERR_UNSUPPORTED && attend(b) == QLIN_ERR_UNSUPPORTED, "more than a launch covers");
    b = good;
    b.rows = (1 << 24) + 1;
    expect(append(b) == QLIN_ERR_UNSUPPORTED && attend(b) == QLIN_ERR_UNSUPPORTED, "too many rows");
    b = good;
    b.max_len = (1 << 30) + 1;
    b.page_ld = 1 << 27;
    expect(append(b) == QLIN_ERR_UNSUPPORTED && attend(b) == QLIN_ERR_UNSUPPORTED, "too long");
    expect(append(good, 167) == QLIN_ERR_PARAM && append(good, 168, 100) == QLIN_ERR_PARAM, "rows too narrow");
    expect(append(good, 168, 168, 2) == QLIN_ERR_PARAM && append(good, 168, 168, -1) == QLIN_ERR_PARAM, "unknown type");
    expect(append(good, 168, 168, F, QLIN_SWIGLU) == QLIN_ERR_PARAM, "a flag of another call");
    expect(attend(good, 3) == QLIN_ERR_PARAM && attend(good, 0) == QLIN_ERR_PARAM && attend(good, -2) == QLIN_ERR_PARAM, "heads");
    expect(attend(good, 4, std::numeric_limits<float>::infinity()) == QLIN_ERR_PARAM, "scale");
    expect(attend(good, 4, std::numeric_limits<float>::quiet_NaN()) == QLIN_ERR_PARAM, "scale");
    expect(attend(good, 4, 1.0f, 335) == QLIN_ERR_PARAM && attend(good, 4, 1.0f, 336, 335) == QLIN_ERR_PARAM, "rows too narrow");
    expect(attend(good, 2048) == QLIN_ERR_PARAM || attend(good, 2048, 1.0f, 1 << 20, 1 << 20) == QLIN_ERR_UNSUPPORTED, "too many heads");
    expect(prefix(-16, table) == QLIN_ERR_PARAM && prefix(8, table) == QLIN_ERR_PARAM && prefix(16, nullptr) == QLIN_ERR_PARAM, "prefix");
    expect(qlin_kv_append(nullptr, m.c, &good, x.data(), 168, x.data(), 168, F, 0, nullptr) == QLIN_ERR_PARAM, "no workspace");
    expect(qlin_kv_append(m.ws, nullptr, &good, x.data(), 168, x.data(), 168, F, 0, nullptr) == QLIN_ERR_PARAM, "no cache");
    expect(qlin_kv_append(m.ws, m.c, nullptr, x.data(), 168, x.data(), 168, F, 0, nullptr) == QLIN_ERR_PARAM, "no batch");
    expect(qlin_kv_append(m.ws, m.c, &good, nullptr, 168, x.data(), 168, F, 0, nullptr) == QLIN_ERR_PARAM, "no rows");
    expect(qlin_kv_read(m.ws, m.c, &good, y.data(), 168, nullptr, 168, F, nullptr) == QLIN_ERR_PARAM, "no rows");
    expect(qlin_kv_attention(m.ws, m.c, &good, 4, nullptr, F, 336, 1.0f, y.data(), F, 336, nullptr) == QLIN_ERR_PARAM, "no rows");
    g_device = 1;  // another device is current
    expect(append(good) == QLIN_ERR_PARAM && attend(good) == QLIN_ERR_PARAM, "another device");
    g_device = 0;
    expect(g_launches == 0, "nothing was launched");
    // idle batches launch nothing; good ones run
    const qlin_kv_batch idle = {2, 0, 0, 32, starts, length, table, 2};
    expect(qlin_kv_append(m.ws, m.c, &idle, nullptr, 168, nullptr, 168, F, 0, nullptr) == QLIN_OK && attend(idle) == QLIN_OK, "idle");
    expect(g_launches == 0, "idle batches launch nothing");
    expect(append(good) == QLIN_OK && g_launches == 1, "append is one launch");
    expect(attend(good) == QLIN_OK && g_launches == 2, "short attention is one launch");
    expect(prefix(0, nullptr) == QLIN_OK && prefix(16, table) == QLIN_OK, "prefix");
}

void limits() {
    Made m(8, 16, 16, 8);
    const int32_t starts[2] = {0, 1}, length[1] = {1}, table[1] = {0};
    const qlin_kv_batch b = {1, 1, 1, 16, starts, length, table, 1};
    std::vector<float> x(2048 * 16), y(x.size());
    const auto attend = [&](int heads, float scale) {
        return qlin_kv_attention(m.ws, m.c, &b, heads, x.data(), QLIN_F32, heads * 16, scale, y.data(), QLIN_F32, heads * 16, nullptr);
    };
    g_launches = 0;
    expect(attend(1032, 1.0f) == QLIN_ERR_UNSUPPORTED && attend(2048, 1.0f) == QLIN_ERR_UNSUPPORTED, "too many query heads");
    expect(attend(8, std::ldexp(1.01f, 64)) == QLIN_ERR_UNSUPPORTED && attend(8, -std::numeric_limits<float>::max()) == QLIN_ERR_UNSUPPORTED, "too large a scale");
    expect(g_launches == 0, "nothing was launched");
    expect(attend(1024, 1.0f) == QLIN_OK && attend(8, std::ldexp(1.0f, 64)) == QLIN_OK && attend(8, -1.0f) == QLIN_OK && attend(8, 0.0f) == QLIN_OK, "the limits");
}

void devices() {
    const int32_t starts[2] = {0, 600}, length[1] = {600}, table[38] = {};
    const qlin_kv_batch b = {1, 600, 600, 600, starts, length, table, 38};
    for (int dim : {64, 84, 256}) {
        std::vector<float> q(600 * (size_t)dim), o(q.size());
        for (int dev : {0, 1, 2}) {
            g_device = dev;
            Made m(1, dim, 16, 38);
            const size_t before = g_lds.size();
            for (int i = 0; i < 2; ++i)
                expect(qlin_kv_attention(m.ws, m.c, &b, 1, q.data(), QLIN_F32, dim, 1.0f, o.data(), QLIN_F32, dim, nullptr) == QLIN_OK, "attention");
            expect(g_lds.size() == before + 1, "the kernel's LDS is asked for on this device");
        }
    }
    g_device = 0;
}

}  // namespace

int main(int argc, char** argv) {
    const char* mode = argc > 1 ? argv[1] : "";
    if (!std::strcmp(mode, "index")) index();
    else if (!std::strcmp(mode, "refusals")) refusals();
    else if (!std::strcmp(mode, "limits")) limits();
    else if (!std::strcmp(mode, "devices")) devices();
    else return 2;
    if (!g_bad) std::printf("PASS %s\n", mode);
    return g_bad != 0;
}
