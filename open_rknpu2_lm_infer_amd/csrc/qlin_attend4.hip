// Attention of few vectors over the 4-bit key/value cache.
#include "qlin_attend_kern.hpp"

namespace qlin {
template hipError_t launch_attend_bits<4>(const AttendParams& p, hipStream_t st);
}  // namespace qlin
