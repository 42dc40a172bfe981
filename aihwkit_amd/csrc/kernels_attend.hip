// Attention over a paged cache: the choice of the kernels (attend_device.h), and the join of what workgroups have of a line.
#include "cache.h"

namespace rpu_amd {
namespace {

constexpr float NONE = -__builtin_inff();

// out = sum over the parts 2^(c m_p - c m) sums_p / sum over the parts 2^(c m_p - c m) total_p.  A workgroup for a line: the parts' factors to the lanes
// of every wave, their sums to the waves, four columns to a lane (and two parts to a wave, of heads of up to 128 columns).
constexpr int JOIN_WAVES = 4;
template <typename T> __device__ __forceinline__ bool join_line(const float *sums, const float2 *stats, long unit, long stride, int parts, int head, float c, f32x4 &v) {
  __shared__ f32x4 room[JOIN_WAVES][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float2 mine = lane < parts ? stats[lane * stride + unit] : float2{NONE, 0.0f};
  float top = mine.x;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
  const float factor = mine.x == NONE ? 0.0f : __builtin_amdgcn_exp2f(weight_between<References<T>>(mine.x, top, c));
  float total = mine.x == NONE ? 0.0f : mine.y * factor;
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) total += __shfl_xor(total, m);
  const int width = head <= 128 ? 32 : 64, d = lane % width * 4, columns = min(d, head - 4);
  const int first = wave * (64 / width) + lane / width, step = JOIN_WAVES * (64 / width);
  f32x4 r = {};
  for (int from = 0; from < parts; from += 4 * step) { // four loads under way together
    f32x4 part[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) part[u] = *reinterpret_cast<const f32x4 *>(sums + (min(from + first + u * step, parts - 1) * stride + unit) * head + columns);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int p = from + first + u * step;
      const float f = __shfl(factor, min(p, parts - 1));
      if (p < parts && f != 0.0f) r += part[u] * f; // 0: nothing seen, nothing left of it, or never written
    }
  }
  room[wave][lane] = r;
  __syncthreads();
  if ((int)threadIdx.x >= width || d >= head) return false;
  r = f32x4{};
  for (int w = 0; w < JOIN_WAVES; ++w)
    for (int k = lane; k < 64; k += width) r += room[w][k];
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = total == 0.0f ? 0.0f : r[k] * inverse;
  return true;
}

// Few parts: a wave for 64 times four columns of a row, whose parts' loads are all under way together.  (By a workgroup to a line, 29000 lines in four
// parts took 49 us, now 11.)
constexpr int JOIN_PARTS = 8;
template <typename T> __device__ __forceinline__ void join_row(const AttendArgs &a, int row, int i, bool with_few) {
  const Sequence s = sequence_of(a.r, row);
  const int q_heads = a.c.heads * a.group, head = a.c.head, pieces = head / 4, h = i / pieces, d = i % pieces * 4;
  const long lines = (long)(s.end - s.begin) * a.group;
  const bool few = lines <= a.few;
  const int parts = few ? with_few ? a.few_splits : 1 : a.splits;
  if (s.which < 0 || parts < 2 || h >= q_heads) return;
  const long stride = few ? (long)a.r.n * a.c.heads * a.few : (long)a.r.rows * q_heads;
  const long unit = few ? ((long)s.which * a.c.heads + h / a.group) * a.few + (row - s.begin) * a.group + h % a.group : (long)row * q_heads + h;
  const float *const sums = (few ? a.few_part : a.part) + unit * head + d;
  const float2 *const of = (few ? a.few_stats : a.stats) + unit;
  float2 stats[JOIN_PARTS];
  f32x4 part[JOIN_PARTS];
#pragma unroll
  for (int p = 0; p < JOIN_PARTS; ++p) stats[p] = of[min(p, parts - 1) * stride];
#pragma unroll
  for (int p = 0; p < JOIN_PARTS; ++p) part[p] = *reinterpret_cast<const f32x4 *>(sums + min(p, parts - 1) * stride * head);
  const float c = exponent_factor(a.scale);
  float top = NONE, total = 0.0f;
#pragma unroll
  for (int p = 0; p < JOIN_PARTS; ++p) top = fmaxf(top, stats[p].x);
  f32x4 v = {};
#pragma unroll
  for (int p = 0; p < JOIN_PARTS; ++p) {
    const bool seen = p < parts && stats[p].x != NONE;
    const float f = seen ? __builtin_amdgcn_exp2f(weight_between<References<T>>(stats[p].x, top, c)) : 0.0f;
    if (seen) total += stats[p].y * f;
    if (f != 0.0f) v += part[p] * f; // 0: nothing seen, nothing left of it, or never written
  }
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
  float r[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) r[k] = total == 0.0f ? 0.0f : v[k] * inverse;
  store_first(static_cast<T *>(a.out.p) + row * a.out.ld + h * head + d, r, 4);
}

// Lines of sequences of few lines first, then rows (`per_row` waves each) or, of many parts, their lines (0).
template <typename T> __global__ __launch_bounds__(64 * JOIN_WAVES) void k_attend_join(AttendArgs a, long few_units, int per_row) {
  const int q_heads = a.c.heads * a.group;
  long unit = blockIdx.x;
  const long units = gridDim.x - few_units;
  f32x4 v;
  int row, h;
  bool mine;
  if (unit < few_units) {
    const int l = (int)(unit % a.few), head = (int)(unit / a.few % a.c.heads), which = (int)(unit / a.few / a.c.heads);
    const Sequence s = sequence_at(a.r, which);
    const int lines = (s.end - s.begin) * a.group;
    if (lines > a.few || l >= lines) return;
    row = s.begin + l / a.group;
    h = head * a.group + l % a.group;
    mine = join_line<T>(a.few_part, a.few_stats, unit, few_units, a.few_splits, a.c.head, exponent_factor(a.scale), v);
  } else {
    unit -= few_units;
    if (per_row) {
      const long w = unit * JOIN_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
      row = (int)(w / per_row);
      if (row < a.r.rows) join_row<T>(a, row, (int)(w % per_row) * 64 + (threadIdx.x & 63), !few_units);
      return;
    }
    row = (int)(unit / q_heads);
    h = (int)(unit % q_heads);
    const Sequence s = sequence_of(a.r, row);
    if (s.which < 0 || (long)(s.end - s.begin) * a.group <= a.few) return;
    mine = join_line<T>(a.part, a.stats, unit, units, a.splits, a.c.head, exponent_factor(a.scale), v);
  }
  const float r[4] = {v[0], v[1], v[2], v[3]};
  if (mine) store_first(static_cast<T *>(a.out.p) + row * a.out.ld + h * a.c.head + threadIdx.x * 4, r, 4);
}

} // namespace

void launch_cache_attend(const AttendArgs &a, int dtype, int cache_dtype, hipStream_t s) {
  with_adapter_types(dtype, cache_dtype, [&](auto x, auto c) {
    using T = decltype(x);
    attend::launch<T, decltype(c)>(a, s);
    const int few = a.few_jobs ? a.few_splits : 1, many = a.jobs ? a.splits : 1;
    if (few < 2 && many < 2) return;
    const int q_heads = a.c.heads * a.group, per_row = many > JOIN_PARTS ? 0 : (q_heads * (a.c.head / 4) + 63) / 64;
    const long few_lines = (long)a.r.n * a.c.heads * a.few, units = per_row ? ((long)a.r.rows * per_row + JOIN_WAVES - 1) / JOIN_WAVES : (long)a.r.rows * q_heads;
    // (rows that have nothing to join cost their workgroups all the same)
    const bool by_line = few > JOIN_PARTS || !per_row || (many < 2 && few_lines < units);
    const long few_units = few > 1 && by_line ? few_lines : 0;
    hipLaunchKernelGGL(k_attend_join<T>, dim3((unsigned)(few_units + (many > 1 || !few_units ? units : 0))), dim3(64 * JOIN_WAVES), 0, s, a, few_units, per_row);
  });
}

} // namespace rpu_amd
