// Attention over a paged cache: float rows beside a cache of halves.
#include "attend_device.h"

namespace rpu_amd {
template void attend::launch<float, _Float16>(const AttendArgs &a, hipStream_t s);
} // namespace rpu_amd
