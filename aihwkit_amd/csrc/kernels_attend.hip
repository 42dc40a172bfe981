// Attention over a paged cache: the choice of the kernels (attend_device.h), and the join of what workgroups have of a line.
#include "cache.h"

namespace rpu_amd {
namespace {

constexpr float NONE = -__builtin_inff();

// out = sum over the parts 2^(m_p - m) sums_p / sum over the parts 2^(m_p - m) total_p.  A wave for a line; parts are shared by the lanes for
// their factors, columns for the sums.
__device__ __forceinline__ void join_line(const float *sums, const float2 *stats, long unit, long stride, int parts, int head, int lane, float (&v)[4], float &total) {
  const float2 mine = lane < parts ? stats[lane * stride + unit] : float2{NONE, 0.0f};
  float top = mine.x;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
  const float factor = mine.x == NONE ? 0.0f : __builtin_amdgcn_exp2f(mine.x - top);
  total = mine.x == NONE ? 0.0f : mine.y * factor;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) total += __shfl_xor(total, m);
  f32x4 r = {};
  const int d = lane * 4;
  for (int p = 0; p < parts; ++p) {
    const float f = __shfl(factor, p);
    if (f == 0.0f) continue; // nothing seen, or nothing left of it
    if (d < head) r += *reinterpret_cast<const f32x4 *>(sums + (p * stride + unit) * head + d) * f;
  }
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = total == 0.0f ? 0.0f : r[k] * inverse;
}

// Lines of sequences of few lines first, then those of rows.
template <typename T> __global__ __launch_bounds__(256) void k_attend_join(AttendArgs a, long few_units, long units) {
  const int lane = threadIdx.x & 63, q_heads = a.c.heads * a.group;
  long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  float v[4], total;
  int row, h;
  if (unit < few_units) {
    const int l = (int)(unit % a.few), head = (int)(unit / a.few % a.c.heads), which = (int)(unit / a.few / a.c.heads);
    const Sequence s = sequence_at(a.r, which);
    const int lines = (s.end - s.begin) * a.group;
    if (lines > a.few || l >= lines) return;
    row = s.begin + l / a.group;
    h = head * a.group + l % a.group;
    join_line(a.few_part, a.few_stats, unit, few_units, a.few_splits, a.c.head, lane, v, total);
  } else {
    unit -= few_units;
    if (unit >= units) return;
    row = (int)(unit / q_heads);
    h = (int)(unit % q_heads);
    const Sequence s = sequence_of(a.r, row);
    if (s.which < 0 || (long)(s.end - s.begin) * a.group <= a.few) return;
    join_line(a.part, a.stats, unit, units, a.splits, a.c.head, lane, v, total);
  }
  if (lane * 4 < a.c.head) store_first(static_cast<T *>(a.out.p) + row * a.out.ld + h * a.c.head + lane * 4, v, 4);
}

} // namespace

void launch_cache_attend(const AttendArgs &a, int dtype, int cache_dtype, hipStream_t s) {
  with_adapter_types(dtype, cache_dtype, [&](auto x, auto c) {
    using T = decltype(x);
    attend::launch<T, decltype(c)>(a, s);
    const long few = a.few_jobs && a.few_splits > 1 ? (long)a.r.n * a.c.heads * a.few : 0, rows = a.jobs && a.splits > 1 ? (long)a.r.rows * a.c.heads * a.group : 0;
    if (few + rows) hipLaunchKernelGGL(k_attend_join<T>, dim3((unsigned)((few + rows + 3) / 4)), dim3(256), 0, s, a, few, rows);
  });
}

} // namespace rpu_amd
