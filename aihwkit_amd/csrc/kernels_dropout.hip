// Dropout whose mask is drawn again wherever it is needed and never stored: out = base + drop(x).  The backward pass is the
// same map of the gradient.
#include "digital.h"

#include <algorithm>

namespace rpu_amd {
namespace {

// A thread takes eight neighbouring elements, one Philox block, at a time.  Bound by memory: 16384 x 768 bf16 with a base in 12.6 us
// (75 MB, 6.0 TB/s); 64 x 256 floats in 5.2 us, a launch.
template <typename T, bool SHORT> __global__ __launch_bounds__(256) void k_dropout(DropoutArgs a) {
  const T *x = static_cast<const T *>(a.x.p), *base = static_cast<const T *>(a.base.p);
  T *out = static_cast<T *>(a.out.p);
  const uint32_t blocks = ((uint32_t)a.cols + 7u) / 8u, call = a.drop.on ? drop_call(a.drop) : 0;
  const uint64_t total = (uint64_t)a.rows * blocks;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
    const uint32_t row = (uint32_t)(i / blocks), block = (uint32_t)(i % blocks);
    const int left = a.cols - (int)(block * 8u);
    const long col = (long)block * 8;
    Packed8<T> x8 = ahead8<SHORT>(x + row * a.x.ld, col, a.cols), base8 = {};
    if (base) base8 = ahead8<SHORT>(base + row * a.base.ld, col, a.cols);
    const uint32_t kept = a.drop.on ? drop_kept(a.drop, call, row, block) : 0xffu;
    trim8(x8, col, a.cols);
    Values8 v = widen(x8);
    drop_apply(a.drop, kept, v);
    if (base) {
      trim8(base8, col, a.cols);
      const Values8 r = widen(base8);
#pragma unroll
      for (int h = 0; h < 8; ++h) v.v[h] += r.v[h];
    }
    write8(out + row * a.out.ld + col, v, left);
  }
}

} // namespace

void launch_dropout(const DropoutArgs &a, int dtype, int cus, hipStream_t s) {
  const uint64_t total = (uint64_t)a.rows * (((uint64_t)a.cols + 7) / 8);
  const dim3 grid((unsigned)std::min<uint64_t>((total + 255) / 256, (uint64_t)cus * 16));
  const auto launch = [&](auto x) {
    using T = decltype(x);
    if (a.cols < 8) hipLaunchKernelGGL((k_dropout<T, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_dropout<T, false>), grid, dim3(256), 0, s, a);
  };
  if (dtype == RPU_F32) launch(float{});
  else if (dtype == RPU_F16) launch(_Float16{});
  else launch(__bf16{});
}

} // namespace rpu_amd
