// The tables of a serving step at their limits, without a GPU.
//
//   step_limits_test places   slots of rows: pages inside and outside the cache, a prefix's among them
//   step_limits_test room     the most slots find room in every workspace's scratch
#include <cstdio>
#include <cstring>
#include <initializer_list>
#include <limits>

#include "../../open_rknpu2_lm_infer_amd/csrc/qlin_kv_step.hpp"

namespace {

int g_bad = 0;
void expect(bool ok, const char* what) {
    if (!ok) {
        std::printf("FAILED: %s\n", what);
        ++g_bad;
    }
}

constexpr int kBig = std::numeric_limits<int>::max(), kLow = std::numeric_limits<int>::min();

void places() {
    for (int shift : {4, 6, 12})
        for (int shared : {0, 1, 3})
            for (int pages : {1, 40, 1 << 27})
                for (int id : {kLow, -1000000, -9, -1, 0, 39, 40, (1 << 27) - 1, 1 << 27, kBig})
                    for (int column : {0, 1, 2, 3, 7})
                        for (int off : {0, 5, (1 << shift) - 1})
                            for (bool before : {false, true}) {
                                const bool outside = id < 0 || id >= pages, own = column >= shared;
                                bool bad = before;
                                const int64_t at = qlin::step_place(id, column * (1 << shift) + off, shift, shared, pages, &bad);
                                expect(bad == (before || (outside && own)), "a page outside the cache is said, a prefix's is not looked at");
                                expect(at == (outside && own ? -1 : (int64_t)id * (1 << shift) + off), "the place of a row");
                            }
}

void room() {
    expect(qlin::kv_step_scratch(1 << 20) * (int64_t)sizeof(int32_t) <= (int64_t)64 << 20, "64 MiB of scratch");
    for (int seqs : {1, 2, 4096, 4097, 1 << 20})
        expect(qlin::kv_step_scratch(seqs) >= qlin::kStepTotals + 2 * ((int64_t)seqs + 1), "totals and two arrays of starts");
}

}  // namespace

int main(int argc, char** argv) {
    const char* mode = argc > 1 ? argv[1] : "";
    if (!std::strcmp(mode, "places")) places();
    else if (!std::strcmp(mode, "room")) room();
    else return 2;
    if (!g_bad) std::printf("PASS %s\n", mode);
    return g_bad != 0;
}
