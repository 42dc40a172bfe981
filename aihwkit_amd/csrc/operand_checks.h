// What the C entry points of the digital operators check on the host before anything is launched: types, sizes, and that what is written
// lies apart from what is read.
#pragma once
#include "../../include/rpu_amd.h"
#include "entry.h"

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>

namespace rpu_amd {

// Grids, and indexes into rows, are 32-bit numbers: far more than a GPU's memory holds of one and the other together.
constexpr int MOST_ROWS = 1 << 28, MOST_COLS = 1 << 24, MOST_ADAPTER_COLS = 1 << 21;

inline size_t value_size(int dtype) { return dtype == RPU_F32 ? 4 : 2; }
inline void check_dtype(int dtype) {
  if (dtype != RPU_F32 && dtype != RPU_F16 && dtype != RPU_BF16) throw RpuError("Unknown data type.");
}
inline void check_rows(int rows) {
  if (rows < 0 || rows > MOST_ROWS) throw RpuError("The number of rows must be in 0 .. 2^28.");
}
inline void check_cols(int cols) {
  if (cols < 1 || cols > MOST_COLS) throw RpuError("The number of columns must be in 1 .. 2^24.");
}

// an operand's place in memory: rows of `width` bytes, `pitch` bytes apart
struct Span {
  const char *what;
  uintptr_t at;
  size_t rows, width, pitch;
  uintptr_t end() const { return at + (rows - 1) * pitch + width; }
};
inline Span matrix(const char *what, const void *p, long ld, int rows, int cols, size_t e) {
  if (!p && rows) throw RpuError(std::string(what) + " is null.");
  if (rows > 1 && ld < cols) throw RpuError(std::string("The rows of ") + what + " overlap.");
  if (ld > LONG_MAX / 8 / MOST_ROWS) throw RpuError(std::string("The rows of ") + what + " lie too far apart.");
  return {what, (uintptr_t)p, (size_t)rows, e * (size_t)cols, e * (size_t)(rows > 1 ? ld : cols)};
}
inline Span dense(const char *what, const void *p, size_t bytes) {
  if (!p && bytes) throw RpuError(std::string(what) + " is null.");
  return {what, (uintptr_t)p, bytes ? (size_t)1 : 0, bytes, bytes};
}
inline bool same_place(const Span &a, const Span &b) { return a.at == b.at && a.rows == b.rows && a.width == b.width && a.pitch == b.pitch; }
inline bool meet(const Span &a, const Span &b) {
  if (!a.rows || !b.rows || !a.width || !b.width) return false;
  if (a.end() <= b.at || b.end() <= a.at) return false;
  if (a.rows == 1 || b.rows == 1) { // one row against the rows of the other
    const Span &one = a.rows == 1 ? a : b, &many = a.rows == 1 ? b : a;
    if (many.rows == 1) return true;
    if (one.at < many.at) return true;
    const size_t from = (one.at - many.at) % many.pitch;
    return from < many.width || from + one.width > many.pitch;
  }
  if (a.pitch != b.pitch) return true;
  // column slices of one matrix lie apart if neither begins within the other's columns
  const size_t ahead = a.at >= b.at ? (a.at - b.at) % a.pitch : (a.pitch - (b.at - a.at) % a.pitch) % a.pitch;
  return ahead < b.width || ahead + a.width > a.pitch;
}
inline void apart(const Span &out, const Span &other, bool may_be_same = false) {
  if (meet(out, other) && !(may_be_same && same_place(out, other)))
    throw RpuError(std::string("The memory of ") + out.what + " overlaps that of " + other.what + ".");
}

struct Gpu { // the operands' GPU for the length of a call
  int device;
  DeviceGuard guard;
  explicit Gpu(int device_id) : device(pick(device_id)), guard(device) {}
  static int pick(int device_id) {
    int count = 0, current = 0;
    RPU_HIP_CHECK(hipGetDeviceCount(&count));
    if (device_id >= count) throw RpuError("There is no GPU of that number.");
    if (device_id < 0) RPU_HIP_CHECK(hipGetDevice(&current));
    return device_id < 0 ? current : device_id;
  }
  int cus() const {
    int n = 0;
    RPU_HIP_CHECK(hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device));
    return std::max(n, 1);
  }
};
inline void check_launch() { RPU_HIP_CHECK(hipGetLastError()); }

constexpr int MOST_CUS = 256; // that scratch sizes, which are asked for without a GPU, are for: an MI355X has so many

} // namespace rpu_amd
