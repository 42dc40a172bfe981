// New keys and values into a paged cache; keys and queries are rotated by their positions on the way.
//   t = p f (turns; f: turns per position), (a, b) -> (a cos 2 pi t - b sin 2 pi t, a sin 2 pi t + b cos 2 pi t) of each pair
// t is taken in 64 bits and only what it has beyond whole turns goes on: far positions lose nothing.
#include "cache.h"

#include <algorithm>

namespace rpu_amd {
namespace {

// cosine and sine of a number of turns.  The fraction as a float and what that leaves, d: cos(x + d) = cos x - d sin x, d < 2^-24.
__device__ __forceinline__ float2 turned(double turns) {
  const double rest = turns - rint(turns);
  const float f = (float)rest;
  const float d = 6.2831853f * (float)(rest - (double)f);
  float sine, cosine;
  sincospif(2.0f * f, &sine, &cosine);
  return {cosine - d * sine, sine + d * cosine};
}

constexpr int THREADS = 256, MOST_ROWS_EACH = 2;

// A workgroup takes `each` rows: their places and angles go to LDS, once for all heads, then every thread moves groups of eight values (of
// both halves, where pairs lie apart).  A thread's first group is under way while places and angles, a chain of trips to memory (which sequence, its
// length, the page), are found.  SHORT: some part of a head is no row of eight columns and more.
// Bound by memory: 16384 rows of 32 query and 8 + 8 other heads of 128 bf16 in 80 us (403 MB, 5.0 TB/s; a copy of 2 GB takes 4.9), with 8 rows to a
// workgroup 89; few rows by the chain: 8 rows in 4.3 us, a launch, 3216 rows of 18 heads of 80 halves that are searched among 37 sequences in 9.1.
template <typename T, typename TC, bool SHORT> __global__ __launch_bounds__(THREADS) void k_cache_append(AppendArgs a, int each, int from) {
  __shared__ int page[MOST_ROWS_EACH];
  __shared__ long at[MOST_ROWS_EACH];
  __shared__ float2 angles[MOST_ROWS_EACH * (RPU_CACHE_MAX_HEAD / 2)];
  static_assert(MOST_ROWS_EACH <= THREADS / 64, "a wave has one row's entry");
  const int first = from + blockIdx.x * each, count = min(each, a.r.rows - first), tid = threadIdx.x;
  const int pairs = a.c.pairs, head = a.c.head, rest = head - 2 * pairs;
  // groups of a head: of its pairs, then of what is not rotated; values go over whole
  const int of_pairs = ((a.c.neighbours ? 2 * pairs : pairs) + 7) / 8, of_head = of_pairs + (rest + 7) / 8, of_value = head / 8;
  const int q_heads = a.q.p ? a.q_heads : 0, of_keys = (q_heads + a.c.heads) * of_head;
  const int of_row = of_keys + a.c.heads * of_value, groups = count * of_row;

  struct Group {
    int row, head, at; // of the workgroup's rows; of queries, then keys, then values (head < 0); number in the head
    Packed8<T> one, two;
  };
  const auto take = [&](int i) { // only loads
    Group p;
    p.row = i / of_row;
    int g = i - p.row * of_row;
    const long row = first + p.row;
    const T *in;
    int col, cols;
    bool both = false;
    if (g >= of_keys) {
      g -= of_keys;
      const int h = g / of_value;
      p.head = ~h;
      p.at = g - h * of_value;
      in = static_cast<const T *>(a.v.p) + row * a.v.ld + h * head;
      col = p.at * 8;
      cols = head;
    } else {
      const int h = p.head = g / of_head;
      p.at = g -= h * of_head;
      in = h < q_heads ? static_cast<const T *>(a.q.p) + row * a.q.ld + h * head : static_cast<const T *>(a.k.p) + row * a.k.ld + (h - q_heads) * head;
      both = g < of_pairs && !a.c.neighbours;
      if (g >= of_pairs) in += 2 * pairs;
      col = (g >= of_pairs ? g - of_pairs : g) * 8;
      cols = g >= of_pairs ? rest : both ? pairs : 2 * pairs;
    }
    p.one = ahead8<SHORT>(in, col, cols);
    if (both) p.two = ahead8<SHORT>(in + pairs, col, cols);
    return p;
  };
  const auto give = [&](Group &p) {
    const int r = p.row, g = p.at, h = p.head;
    if (page[r] == -2) return;
    const long row = first + r;
    if (h < 0) {
      if (page[r] >= 0) store8(static_cast<TC *>(a.c.v) + place_of(a.c, page[r], ~h, at[r]) + g * 8, widen(p.one));
      return;
    }
    const bool query = h < q_heads;
    if (!query && page[r] < 0) return;
    T *out = static_cast<T *>(a.out.p) + row * a.out.ld + h * head;
    TC *key = static_cast<TC *>(a.c.k) + (query ? 0 : place_of(a.c, page[r], h - q_heads, at[r]));
    const auto write = [&](int col, const Values8 &v, int n) {
      if (query) write8(out + col, v, n);
      else write8(key + col, v, n);
    };
    if (g >= of_pairs) {
      const int col = (g - of_pairs) * 8;
      trim8(p.one, col, rest);
      write(2 * pairs + col, widen(p.one), rest - col);
    } else if (a.c.neighbours) {
      const int col = g * 8;
      trim8(p.one, col, 2 * pairs);
      Values8 v = widen(p.one);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 t = angles[r * pairs + min(col / 2 + k, pairs - 1)];
        const float x = v.v[2 * k], y = v.v[2 * k + 1];
        v.v[2 * k] = fmaf(x, t.x, -(y * t.y));
        v.v[2 * k + 1] = fmaf(x, t.y, y * t.x);
      }
      write(col, v, 2 * pairs - col);
    } else {
      const int col = g * 8;
      trim8(p.one, col, pairs);
      trim8(p.two, col, pairs);
      Values8 x = widen(p.one), y = widen(p.two);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 t = angles[r * pairs + min(col + k, pairs - 1)];
        const float u = fmaf(x.v[k], t.x, -(y.v[k] * t.y));
        y.v[k] = fmaf(x.v[k], t.y, y.v[k] * t.x);
        x.v[k] = u;
      }
      write(col, x, pairs - col);
      write(pairs + col, y, pairs - col);
    }
  };

  Group now = take(min(tid, groups - 1));
  const double turn = pairs ? a.c.turns[tid % pairs] : 0.0;
  // (rows whose sequences are searched for by a wave each, others by a thread)
  const int by = a.r.starts ? 64 : 1;
  const int *entry = nullptr; // of the table
  for (int i = tid / by; i < count; i += THREADS / by) {
    const Sequence s = sequence_of(a.r, first + i);
    const long position = s.first + (first + i - s.begin);
    at[i] = position;
    page[i] = s.which < 0 ? -2 : -1; // no sequence, no page
    if (s.which >= 0 && position >= 0 && position < a.r.places) entry = a.r.tables + s.which * a.r.table_ld + (position >> a.c.page_shift);
  }
  const int number = entry ? *entry : -1;
  __syncthreads();
  for (int i = tid; i < count * pairs; i += THREADS) angles[i] = turned((double)at[i / pairs] * (i == tid ? turn : a.c.turns[i % pairs]));
  if (number >= 0 && number < a.c.pages && tid % by == 0) page[tid / by] = number;
  __syncthreads();
  for (int i = tid; i < groups; i += THREADS) {
    if (i != tid) now = take(i);
    give(now);
  }
}

} // namespace

void launch_cache_append(const AppendArgs &a, int dtype, int cache_dtype, int cus, hipStream_t s) {
  const int rotated = a.c.neighbours ? 2 * a.c.pairs : a.c.pairs, rest = a.c.head - 2 * a.c.pairs;
  const bool is_short = (rotated && rotated < 8) || (rest && rest < 8);
  const int each = (int)std::min<long>(MOST_ROWS_EACH, (a.r.rows + 8l * cus - 1) / (8l * cus));
  with_adapter_types(dtype, cache_dtype, [&](auto x, auto c) {
    using T = decltype(x);
    using TC = decltype(c);
    for (long from = 0; from < a.r.rows; from += MOST_GROUPS * each) {
      const dim3 grid((unsigned)std::min(MOST_GROUPS, (a.r.rows - from + each - 1) / each));
      if (is_short) hipLaunchKernelGGL((k_cache_append<T, TC, true>), grid, dim3(THREADS), 0, s, a, each, (int)from);
      else hipLaunchKernelGGL((k_cache_append<T, TC, false>), grid, dim3(THREADS), 0, s, a, each, (int)from);
    }
  });
}

} // namespace rpu_amd
