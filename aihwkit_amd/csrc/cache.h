// Attention over a paged cache: argument blocks, launches, and what the kernels share: where rows and positions lie.
#pragma once
#include "digital.h"

namespace rpu_amd {

struct CacheDev {
  void *k, *v;         // [pages][heads][page_size][head]
  const double *turns; // [pairs]
  int pages, page_shift, heads, head, pairs, neighbours;
};
struct CacheRowsDev {
  const int *tables, *lengths, *starts; // starts null: rows / n each
  long table_ld;
  int n, places, rows; // places: positions that a table holds
};

constexpr long MOST_GROUPS = 1 << 23; // workgroups of 256 threads in a launch: all threads are counted in 32 bits
struct AppendArgs {
  CacheDev c;
  CacheRowsDev r;
  MatrixDev k, v, q, out; // q.p null: none
  int q_heads;
};
void launch_cache_append(const AppendArgs &a, int dtype, int cache_dtype, int cus, hipStream_t s);

// How a call's work is shared among workgroups: sequences of few lines (a row's heads that share one of the cache count as lines of their own)
// have their positions shared by the waves of a workgroup, others have tiles of lines.  Of both, the positions may go in parts to several
// workgroups, whose sums are joined.
constexpr int ATTEND_FEW = 32, ATTEND_LINES = 128; // lines of a sequence that are few; of a tile
constexpr int ATTEND_FEW_HEAD = 128;               // of heads up to so many values; of longer ones of floats all go in tiles of lines
constexpr int ATTEND_FEW_LEAST = 4;                // tiles of 32 positions that a part has at least
struct AttendPlan {
  int few, few_splits, splits, tiles;              // few: the most lines of a sequence that goes that way, 0: none
  long few_jobs, jobs;                             // workgroups
  size_t few_part, few_stats, part, stats, bytes;  // offsets in the scratch memory, its size
};

struct AttendArgs {
  CacheDev c;
  CacheRowsDev r;
  MatrixDev q, out;
  int group;           // heads of a row that share one of the cache
  float scale;
  int window, sinks;   // window 0: none
  int few, few_splits, splits, tiles;
  long few_jobs, jobs;
  float *few_part, *part;      // sums of a part of the positions: [few_splits][n][heads][few][head], [splits][rows][q heads][head]
  float2 *few_stats, *stats;   // the score that weights are relative to (before the scale), and their sum
};
namespace attend {
template <typename T, typename TC> void launch(const AttendArgs &a, hipStream_t s);
}
void launch_cache_attend(const AttendArgs &a, int dtype, int cache_dtype, hipStream_t s);

#if defined(__HIPCC__)
// The rows of a sequence, and the position of the first.  Numbers on the GPU that are out of range leave it without rows or positions: nothing
// outside of the operands is touched.
struct Sequence {
  int which, begin, end;
  long first; // position of row `begin`
};
__device__ __forceinline__ Sequence sequence_at(const CacheRowsDev &r, int which) {
  Sequence s;
  s.which = which;
  if (r.starts) {
    s.begin = min(max(r.starts[which], 0), r.rows);
    s.end = min(max(r.starts[which + 1], s.begin), r.rows);
  } else {
    const int each = r.rows / r.n;
    s.begin = which * each;
    s.end = s.begin + each;
  }
  s.first = (long)r.lengths[which] - (s.end - s.begin);
  return s;
}
// The last of n numbers that `at_most` holds for, of numbers for which it holds up to some and then not; -1: none.  By a whole wave, 64 numbers at
// a time: two trips to memory for up to 4096 of them.
template <typename F> __device__ __forceinline__ int last_of(const int *numbers, int n, F &&at_most) {
  const int lane = threadIdx.x & 63;
  int low = -1, high = n; // holds for low, not for high
  while (high - low > 1) {
    const int step = max((high - low - 1 + 63) / 64, 1), i = low + 1 + lane * step;
    const int held = __popcll(__ballot(i < high && at_most(numbers[min(i, n - 1)], i)));
    const int from = low;
    if (held) low = from + 1 + (held - 1) * step;
    high = min(high, from + 1 + held * step);
  }
  return low;
}
// the sequence that a row belongs to (by a whole wave); which < 0: none
__device__ __forceinline__ Sequence sequence_of(const CacheRowsDev &r, int row) {
  if (!r.starts) return sequence_at(r, row / (r.rows / r.n));
  const int low = last_of(r.starts, r.n, [&](int start, int) { return start <= row; });
  if (low < 0) return {-1, 0, 0, 0};
  Sequence s = sequence_at(r, low);
  if (row < s.begin || row >= s.end) s.which = -1;
  return s;
}
// Weights are 2^(c score - c reference), c of the scale's magnitude.
constexpr float LOG2E = 1.44269504088896340736f;
__device__ __forceinline__ float exponent_factor(float scale) { return fabsf(scale * LOG2E); }
// Exponents have c reference + RAISED subtracted, rounded.  Scores may be up to SLACK powers of two above the reference: weights are at most 1 when they meet
// the values, so that the largest of these stay finite, of halves 2^15, so that small weights keep their bits.  (Floats are lifted afterwards.)
template <typename T> struct References { // of rows of T
  static constexpr float SLACK = 8.0f, RAISED = sizeof(T) == 4 ? 0.0f : __is_same(T, _Float16) ? SLACK - 15.0f : SLACK;
};
// The exponent of a weight relative to one score, relative to another.  Up to ATTEND_FAR, weights were made with the rounded reference (by up to 2^-8), so that
// this is the difference of those.  Beyond, where a float has c reference to 2^-7 at best (from 2^31 on to 128, and with scales up to 1e30 not at all),
// they were made of the difference of the scores.
constexpr float ATTEND_FAR = 0x1p16f;
template <typename R> __device__ __forceinline__ float weight_between(float of, float to, float c) {
  const float p = of * c, q = to * c;
  return fabsf(p) <= ATTEND_FAR && fabsf(q) <= ATTEND_FAR ? (p + R::RAISED) - (q + R::RAISED) : (of - to) * c;
}
// value 0 of a head at a position
__device__ __forceinline__ long place_of(const CacheDev &c, int page, int head, long position) {
  return ((((long)page * c.heads + head) << c.page_shift) + (position & ((1 << c.page_shift) - 1))) * c.head;
}
#endif

} // namespace rpu_amd
