// Attention of many rows over the 8-bit key/value cache.
#include "qlin_attend_wide_kern.hpp"

namespace qlin {
template hipError_t launch_attend_wide<8>(const AttendParams& p, bool prefix, hipStream_t st);
}  // namespace qlin
