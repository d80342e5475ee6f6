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
// In 4 bits the crossing lies where it does in 8, the same table of one sequence of 4096 tokens being
//   fp16, 64       17.1 / 23.5  26.4 / 24.5  25.1 / 27.9  36.4 / 33.8  37.2 / 33.7
//   fp16, 128      21.7 / 33.2  34.4 / 34.9  31.9 / 38.2  47.5 / 47.7  49.0 / 47.4
//   fp16, 256      32.3 / 42.6  49.0 / 62.9  50.1 / 71.2  72.6 / 83.5  92.5 / 96.3
//   f32, 128       23.9 / 38.8  39.1 / 43.5  34.4 / 47.7  52.6 / 58.3  54.6 / 63.8
// and 512 vectors of fp16 for each of 16 sequences of 1000 tokens, heads of 128, 88 / 48.
int tile_of(const AttendParams& p, int64_t vectors) {
    if (vectors > (p.q_f16 && p.o_f16 ? 256 : 512)) return kAttendWide;
    return vectors <= 16 || p.c.dim_padded > 128 ? 16 : 32;
}

}  // namespace

int attend_tile(const AttendParams& p) { return tile_of(p, (int64_t)p.b.max_new * p.group.d); }
int attend_tile_prefix(const AttendParams& p) { return tile_of(p, (int64_t)p.b.rows * p.group.d); }
// Two classes against none, fp16, us (one cache over and over), 4 KV heads with 8 query heads each, pages of 32 (of 150 batches of 4 to 8 vectors on pages of 32
// and 64, fp16 and f32, two take longer in none):
//                     64            128           256
//   1 x 300           4.9 / 6.0     6.0 / 7.6     8.3 / 10.8
//   1 x 32768         8.9 / 10.1   11.4 / 12.8   17.9 / 19.6
//   64, up to 4096   23.0 / 29.2   33.3 / 36.0   47.8 / 51.3
//   64 x 2048        16.4 / 19.8   24.8 / 25.2   33.5 / 37.4
// Four classes against two and none, 8 KV heads with 4 query heads each, pages of 64.  For one sequence of up to some thousand tokens two
// would be faster, and of 256 columns none as fast; batches and long sequences gain:
//   1 x 300           5.1 / 4.9 / 6.0      6.5 / 5.9 / 7.5      9.7 / 8.0 / 10.7
//   1 x 4096          7.6 / 7.1 / 7.7      8.4 / 7.6 / 8.4     11.5 / 9.9 / 11.0
//   1 x 32768        10.7 / 11.5 / 13.5   15.5 / 17.5 / 18.1   22.8 / 23.6 / 25.2
//   64, up to 4096   29.5 / 33.5 / 41.9   44.3 / 48.0 / 53.3   78 / 95 / 105
//   64 x 2048        18.5 / 20.4 / 27.0   28.4 / 30.6 / 33.8   52 / 55 / 56
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
