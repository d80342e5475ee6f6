// Attention of few vectors over the 8-bit key/value cache, and which kernel a call takes.
#include "qlin_attend_kern.hpp"

namespace qlin {
namespace {

// Vectors of a workgroup, given how many share its tokens: one or two tiles here (two of 256 columns would
// not fit the registers), or the wide kernel's.  That one reads a token's bytes once for 128 vectors but
// waits at a barrier for every 32 tokens: with up to 256 vectors (512 where rows are f32 in or out) more workgroups of
// this one are faster.  One sequence, 4096 tokens, 8 KV heads, us here and there:
//   vectors           256          384          512          768         1024
//   fp16, 64       17.0 / 23.5  25.5 / 24.3  24.4 / 27.9  33.6 / 32.1  34.4 / 32.9
//   fp16, 128      21.6 / 32.3  34.1 / 34.7  30.9 / 37.8  45.7 / 46.9  48.4 / 46.5
//   fp16, 256      30.6 / 43.8  51.5 / 60.3  53.2 / 68.6  75.5 / 80.4  96.2 / 93.1
//   f32, 128       23.9 / 38.3  38.5 / 42.0  33.8 / 46.7  50.9 / 57.9  53.9 / 62.2
//   prefix, fp16   24.9 / 35.7  36.3 / 41.2  35.4 / 47.6  48.4 / 54.5  57.3 / 65.1   (128 columns)
//   prefix, f32    26.4 / 43.5  40.4 / 54.2  39.0 / 58.6  54.6 / 75.9  64.1 / 87.3
// What a batch holds beside that moves the crossing, and the limit on vectors alone is a middle: of 257 to 512 fp16 vectors
// in 36 random batches of 1 to 16 sequences this kernel takes 0.83 of the other's time on average, half of it for one
// sequence of a few hundred tokens, 1.35 of it for one of 15000 tokens and up to 1.85 for 16 sequences.
int tile_of(const AttendParams& p, int64_t vectors) {
    if (vectors > (p.q_f16 && p.o_f16 ? 256 : 512)) return kAttendWide;
    return vectors <= 16 || p.c.dim_padded > 128 ? 16 : 32;
}

}  // namespace

int attend_tile(const AttendParams& p) { return tile_of(p, (int64_t)p.b.max_new * p.group.d); }
int attend_tile_prefix(const AttendParams& p) { return tile_of(p, (int64_t)p.b.rows * p.group.d); }
int attend_classes_of(const AttendParams& p) {
    const int64_t vectors = (int64_t)p.b.max_new * p.group.d;
    if (p.c.bits != 4) return 1;
    return vectors <= 4 && p.c.shift >= 6 ? 4 : vectors <= 8 && p.c.shift >= 5 ? 2 : 1;
}

hipError_t launch_attend(const AttendParams& p, hipStream_t st) {
    return p.c.bits == 4 ? launch_attend_bits<4>(p, st) : launch_attend_bits<8>(p, st);
}

template hipError_t launch_attend_bits<8>(const AttendParams& p, hipStream_t st);

}  // namespace qlin
