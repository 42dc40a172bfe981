// Attention of new rows over a paged cache: out = sum_j w_j v_j / sum_j w_j, w_j = exp(scale q k_j - max), over the positions that a row sees.
#include "cache.h"

#include <algorithm>

namespace rpu_amd {
namespace {

constexpr float NONE = -__builtin_inff();

// One wave for a head of a row: 64 positions at a time, a score to each lane, then the columns of the values to the lanes.
template <typename T, typename TC> __global__ __launch_bounds__(256) void k_attend_rows(AttendArgs a) {
  const int lane = threadIdx.x & 63, q_heads = a.c.heads * a.group, head = a.c.head;
  const long unit = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= (long)a.r.rows * q_heads) return;
  const int row = (int)(unit / q_heads), h = (int)(unit % q_heads), from = h / a.group;
  const Sequence s = sequence_of(a.r, row);
  if (s.which < 0) return;
  const long position = s.first + (row - s.begin);
  const long end = min(position + 1, (long)a.r.places), low = a.window ? max(position - a.window + 1, 0l) : 0;
  const int *table = a.r.tables + s.which * a.r.table_ld;
  const T *q = static_cast<const T *>(a.q.p) + row * a.q.ld + h * head;
  const TC *keys = static_cast<const TC *>(a.c.k), *values = static_cast<const TC *>(a.c.v);
  float most = NONE, total = 0.0f, mixed[4] = {};
  for (long tile = 0; tile < end; tile += 64) {
    if (tile >= a.sinks && tile + 64 <= low) {
      tile = low / 64 * 64;
      if (tile >= end) break;
    }
    const long j = tile + lane;
    const int page = j < end && (j >= low || j < a.sinks) ? page_of(a.c, a.r, table, j) : -1;
    const long place = page < 0 ? 0 : place_of(a.c, page, from, j);
    float score = 0.0f;
    if (page >= 0)
      for (int d = 0; d < head; d += 8) {
        const Values8 x = widen(load8(q + d)), y = widen(load8(keys + place + d));
#pragma unroll
        for (int k = 0; k < 8; ++k) score = fmaf(x.v[k], y.v[k], score);
      }
    score = page >= 0 ? score * a.scale : NONE;
    float now = score;
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) now = fmaxf(now, __shfl_xor(now, m));
    now = fmaxf(now, most);
    const float base = now == NONE ? 0.0f : now, shrink = expf(most - base);
    const float weight = page >= 0 ? expf(score - base) : 0.0f;
    float sum = weight;
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
    total = total * shrink + sum;
    most = now;
#pragma unroll
    for (int k = 0; k < 4; ++k) mixed[k] *= shrink;
    for (int i = 0; i < 64; ++i) {
      const int seen = __shfl(page, i);
      const long at = __shfl(place, i);
      const float w = __shfl(weight, i);
      if (seen < 0) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < head) mixed[k] = fmaf(w, to_float(values[at + lane + 64 * k]), mixed[k]);
    }
  }
  T *out = static_cast<T *>(a.out.p) + row * a.out.ld + h * head;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (lane + 64 * k < head) out[lane + 64 * k] = (T)(total == 0.0f ? 0.0f : mixed[k] / total);
}

} // namespace

void launch_cache_attend(const AttendArgs &a, int dtype, int cache_dtype, int cus, hipStream_t s) {
  (void)cus;
  const long units = (long)a.r.rows * a.c.heads * a.group;
  with_adapter_types(dtype, cache_dtype, [&](auto x, auto c) {
    using T = decltype(x);
    using TC = decltype(c);
    hipLaunchKernelGGL((k_attend_rows<T, TC>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, a);
  });
}

} // namespace rpu_amd
