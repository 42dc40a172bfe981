// Which tile of lines a workgroup has where sequences have unlike rows (`starts`), found on the GPU.  No HIP in here: the rule is checked on the CPU too.
#pragma once

#if defined(__HIPCC__)
#define RPU_TILES_FN __host__ __device__ inline __attribute__((always_inline))
#else
#define RPU_TILES_FN inline
#endif

namespace rpu_amd {
namespace attend {

// Sequence s has the numbers from (starts[s] * group) / lines + s on, up to those of the next: one more than it can need at most.  What lies before the
// first sequence's is nobody's: rows ahead of starts[0] belong to no sequence.
RPU_TILES_FN long first_number(int start, int which, int rows, int group, int lines) {
  const int row = start < 0 ? 0 : start > rows ? rows : start;
  return (long)row * group / lines + which;
}
RPU_TILES_FN long numbers_of(int rows, int group, int lines, int n) { return (long)rows * group / lines + n; }

// The sequence that has a number (-1: none) and which of its tiles that is.  last(f): the last s of n that f(starts[s], s) holds for, -1: none.
struct TileOf {
  int which;
  long tile;
};
template <typename Last> RPU_TILES_FN TileOf tile_of(long number, const int *starts, int rows, int group, int lines, Last &&last) {
  const int which = last([=](int start, int s) { return first_number(start, s, rows, group, lines) <= number; });
  if (which < 0) return {-1, 0};
  const long tile = number - first_number(starts[which], which, rows, group, lines);
  return {tile < 0 ? -1 : which, tile}; // (starts that decrease: a sequence that does not reach down to the number)
}

} // namespace attend
} // namespace rpu_amd
