// Attention over a paged cache: bf16 rows and a bf16 cache.
#include "attend_device.h"

namespace rpu_amd {
template void attend::launch<__bf16, __bf16>(const AttendArgs &a, hipStream_t s);
} // namespace rpu_amd
