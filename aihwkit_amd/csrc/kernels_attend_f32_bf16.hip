// Attention over a paged cache: float rows beside a bf16 cache.
#include "attend_device.h"

namespace rpu_amd {
template void attend::launch<float, __bf16>(const AttendArgs &a, hipStream_t s);
} // namespace rpu_amd
