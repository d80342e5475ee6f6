// Attention of many rows over the 4-bit key/value cache.
#include "qlin_attend_wide_kern.hpp"

namespace qlin {
template hipError_t launch_attend_wide<4>(const AttendParams& p, bool prefix, hipStream_t st);
}  // namespace qlin
