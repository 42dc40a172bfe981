// The rule by which workgroups take tiles of lines, compiled for the CPU.
#include "../aihwkit_amd/csrc/attend_tiles.h"

using namespace rpu_amd::attend;

extern "C" long numbers(int rows, int group, int lines, int n) { return numbers_of(rows, group, lines, n); }

extern "C" void tiles(const int *starts, int n, int rows, int group, int lines, long count, int *which, long *tile) {
  for (long number = 0; number < count; ++number) {
    const TileOf t = tile_of(number, starts, rows, group, lines, [&](auto &&held) {
      int last = -1;
      while (last + 1 < n && held(starts[last + 1], last + 1)) ++last;
      return last;
    });
    which[number] = t.which;
    tile[number] = t.tile;
  }
}
