// Attention over a paged cache: rows and a cache of halves.
#include "attend_device.h"

namespace rpu_amd {
template void attend::launch<_Float16, _Float16>(const AttendArgs &a, hipStream_t s);
} // namespace rpu_amd
