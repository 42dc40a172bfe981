// The digital operators beside the tiles (dropout, layer norm, low-rank adapters): argument blocks, launches, and what their
// kernels share.  Tensors are rows of a unit column stride in one of three types; everything is computed in 32 bits.
#pragma once
#include "../../include/rpu_amd.h"
#include "bf16_parts.h"
#include "philox.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rpu_amd {

struct MatrixDev { // rows at p + row * ld; p null: not given
  void *p;
  long ld;
};

// Dropout of element (row, column): half column % 8 of the Philox block of counter (column / 8, row, call, RNG_DROPOUT), u,
// is dropped below the limit round(p 2^32): u < limit / 2^16, or u equal to it and the same half of the block of
// RNG_DROPOUT_LOW below limit % 2^16.  32 bits decide, at the price of 16: one element in 65536 needs the second block.
struct DropDev {
  uint32_t high, low; // the limit's halves (high = 65536: all)
  float scale;        // of what is kept, 1 / (1 - p)
  PhiloxKey key;
  uint32_t call;
  const int64_t *call_dev; // added to `call` when the kernel runs; null: nothing is
  int on;
};

struct DropoutArgs {
  MatrixDev x, base, out;
  int rows, cols;
  DropDev drop;
};
void launch_dropout(const DropoutArgs &a, int dtype, int cus, hipStream_t s);

struct NormArgs {
  MatrixDev x, out;
  const void *w, *b; // null: ones, zeros
  float *mean, *rstd;
  int rows, cols;
  float eps;
};
void launch_layer_norm(const NormArgs &a, int dtype, int w_dtype, int cus, hipStream_t s);

struct NormBackwardArgs {
  MatrixDev d, x, base, dx;
  const float *mean, *rstd;
  const void *w;       // null: ones
  void *dw, *db;       // null: not wanted (both)
  float *part;         // [parts][2][cols]
  int rows, cols, parts;
};
int layer_norm_parts(int rows, int cols, int cus); // workgroups of the backward pass, each of which leaves sums of its rows
void launch_layer_norm_backward(const NormBackwardArgs &a, int dtype, int w_dtype, hipStream_t s);

// Rows grouped by adapter: what launch_adapter_plan writes, one array of ints.
//   order [rows]       rows by adapter, in their order within each; those without one last
//   seg [n + 2]        seg[a]: where adapter a begins in `order`; seg[n]: the rows without one; seg[n + 1] = rows
//   tiles [4 * tiles]  {adapter or -1, first place in `order`, rows (0: none), 0}: at most ADAPTER_TILE_ROWS rows each
//   chunks [4 * chunks]  the same in longer pieces for the gradients, of adapters only; the last number is the slot for the
//                      chunk's sums, -1 if it holds all rows of its adapter
//   first [n + 1]      first[a]: the first chunk of adapter a
//   slot_first [n + 1]  the same of the slots
//   tile_first [n + 2], other [rows]  scratch of k_adapter_plan
constexpr int ADAPTER_TILE_ROWS = 64;
struct AdapterPlan {
  int rows, n;
  int chunk_rows;
  int max_tiles, max_chunks, max_slots;
  size_t order, seg, tiles, chunks, first, tile_first, slot_first, other, words; // offsets in ints, total
};
AdapterPlan adapter_plan(int rows, int n);
void launch_adapter_plan(const int *index, int *plan, const AdapterPlan &p, hipStream_t s);
// Turned matrices are made of adapters with rows.  Of fewer rows than adapters there are at most as many as rows: their matrices lie by the
// number of the adapter's first chunk, which is below `rows` then, the others' by the adapter.
inline bool adapter_listed(const AdapterPlan &p) { return p.n > p.rows; }
inline int adapter_turned(const AdapterPlan &p) { return p.n > p.rows ? p.rows : p.n; } // matrices that there is room for
constexpr int ADAPTER_FEW_ROWS = 64; // up to so many rows a forward call groups them by itself
constexpr int ADAPTER_MAX_RANK = 128;
constexpr int ADAPTER_MAX = 65535;

struct AdapterRowsArgs {
  MatrixDev in, base, out;     // forward: x, base, y; backward: d, base, dx
  const void *w_in, *w_out;    // [n][rank][in_size], [n][out_size][rank]: forward a, b; backward b, a with both exchanged
  const float *scale;
  float *hidden;               // [rows][rank]: a drop(x), or scale b^T d; without a plan it may be null
  const int *index;            // without a plan
  const int *plan;             // null: the rows are grouped from `index`
  AdapterPlan p;
  int rows, n, rank, in_size, out_size;
  int back;
  int listed;                  // the matrices lie by the adapters' first chunks (adapter_listed)
  int units_each;              // few rows: 32 columns of the output each, of a workgroup (set by the launch)
  DropDev drop;                // of the input (forward) or of the output (backward)
};
void launch_adapter_rows(const AdapterRowsArgs &a, int dtype, int w_dtype, int cus, hipStream_t s);

struct AdapterTurnArgs {
  const void *a, *b;
  void *a_turned, *b_turned;   // [in][rank], [rank][out] of adapters with rows
  const int *plan;
  AdapterPlan p;
  int n, rank, in_size, out_size;
  int listed;                  // as in AdapterRowsArgs
};
void launch_adapter_turn(const AdapterTurnArgs &a, int w_dtype, int cus, hipStream_t s);

struct AdapterGradArgs {
  MatrixDev x, d;
  const float *hidden, *up;    // [rows][rank]: a drop(x) and scale b^T d
  const float *scale;
  void *da, *db;               // [n][rank][in], [n][out][rank]
  float *part;                 // [max_slots][rank * (in + out)]
  const int *plan;
  AdapterPlan p;
  int rows, n, rank, in_size, out_size;
  DropDev drop;
};
void launch_adapter_grads(const AdapterGradArgs &a, int dtype, int w_dtype, int cus, hipStream_t s);

#if defined(__HIPCC__)
__device__ __forceinline__ int adapter_key(int index, int n) { return index >= 0 && index < n ? index : n; }

// ---- eight neighbouring values of a row -------------------------------------------------------------------------------
// Rows begin at any element: loads and stores of 16 bytes from any address that a value may have.
typedef uint32_t u32x4_from2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_from4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_from2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x2_from4 __attribute__((ext_vector_type(2), aligned(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
struct Values8 {
  float v[8];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__bf16 v) { return __uint_as_float((uint32_t)__builtin_bit_cast(uint16_t, v) << 16); }
__device__ __forceinline__ float to_float(_Float16 v) { return (float)v; }

template <typename T> struct Packed8; // the eight values as they are stored
template <> struct Packed8<float> {
  u32x4_from4 q[2];
};
template <> struct Packed8<__bf16> {
  u32x4_from2 q;
};
template <> struct Packed8<_Float16> {
  u32x4_from2 q;
};
__device__ __forceinline__ Packed8<float> load8(const float *p) {
  const u32x4_from4 *s = reinterpret_cast<const u32x4_from4 *>(p);
  return {{s[0], s[1]}};
}
__device__ __forceinline__ Packed8<__bf16> load8(const __bf16 *p) { return {*reinterpret_cast<const u32x4_from2 *>(p)}; }
__device__ __forceinline__ Packed8<_Float16> load8(const _Float16 *p) { return {*reinterpret_cast<const u32x4_from2 *>(p)}; }

__device__ __forceinline__ Values8 widen(const Packed8<float> &p) {
  Values8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = __uint_as_float(p.q[i >> 2][i & 3]);
  return r;
}
__device__ __forceinline__ Values8 widen(const Packed8<__bf16> &p) {
  Values8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.v[2 * i] = __uint_as_float(p.q[i] << 16);
    r.v[2 * i + 1] = __uint_as_float(p.q[i] & 0xffff0000u);
  }
  return r;
}
__device__ __forceinline__ Values8 widen(const Packed8<_Float16> &p) {
  Values8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 h = __builtin_bit_cast(f16x2, (uint32_t)p.q[i]);
    r.v[2 * i] = (float)h.x;
    r.v[2 * i + 1] = (float)h.y;
  }
  return r;
}
// a 16-bit value below seven others
__device__ __forceinline__ u32x4 shift_in(u32x4 q, uint16_t v) {
  return u32x4{q[0] << 16 | v, q[1] << 16 | q[0] >> 16, q[2] << 16 | q[1] >> 16, q[3] << 16 | q[2] >> 16};
}
// Eight values of a row from column `col` on, in two steps.  ahead8 only loads: where the row ends it begins earlier.  trim8, at the first
// use, moves the values down, with zeros behind the last column.  In one step, or with a branch around the load, every load would be
// waited for before the next begins: rows of fewer than eight columns, which cannot begin earlier, have kernels of their own (SHORT).
template <bool SHORT, typename T> __device__ __forceinline__ Packed8<T> ahead8(const T *row, long col, long cols) {
  if (!SHORT) return load8(row + min(col, cols - 8));
  if (cols >= 8) return load8(row + min(col, cols - 8)); // a matrix beside a short one
  Packed8<T> p = {};
#pragma unroll 1
  for (long i = cols - 1; i >= col; --i) {
    if constexpr (sizeof(T) == 4) {
      p.q[1] = u32x4{p.q[0][3], p.q[1][0], p.q[1][1], p.q[1][2]};
      p.q[0] = u32x4{__float_as_uint(row[i]), p.q[0][0], p.q[0][1], p.q[0][2]};
    } else {
      p.q = shift_in(p.q, __builtin_bit_cast(uint16_t, row[i]));
    }
  }
  return p;
}
template <typename T> __device__ __forceinline__ void trim8(Packed8<T> &p, long col, long cols) {
  if (cols < 8 || col + 8 <= cols) return;
  constexpr int WORDS = sizeof(T) == 4 ? 8 : 4;
  int by = (int)min(col + 8 - cols, 8l); // values
  uint32_t d[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    if constexpr (sizeof(T) == 4) d[i] = p.q[i >> 2][i & 3];
    else d[i] = p.q[i];
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) d[i] = by & 1 ? (d[i] >> 16 | (i + 1 < WORDS ? d[i + 1] << 16 : 0u)) : d[i];
    by >>= 1;
  }
#pragma unroll
  for (int step = 1; step <= WORDS; step *= 2)
#pragma unroll
    for (int i = 0; i < WORDS; ++i) d[i] = by & step ? (i + step < WORDS ? d[i + step] : 0u) : d[i];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    if constexpr (sizeof(T) == 4) p.q[i >> 2][i & 3] = d[i];
    else p.q[i] = d[i];
  }
}
template <bool SHORT, typename T> __device__ __forceinline__ Values8 read8(const T *row, long col, long cols) {
  Packed8<T> p = ahead8<SHORT>(row, col, cols);
  trim8(p, col, cols);
  return widen(p);
}

// ---- 16 bytes of neighbouring values of a row ---------------------------------------------------------------------------
template <typename T> constexpr int CHUNK = 16 / (int)sizeof(T); // values
template <typename T> struct Packed16 {
  u32x4 q;
};
template <typename T> __device__ __forceinline__ Packed16<T> load16(const T *p) {
  if constexpr (sizeof(T) == 4) return {*reinterpret_cast<const u32x4_from4 *>(p)};
  else return {*reinterpret_cast<const u32x4_from2 *>(p)};
}
// the same two steps as for eight values
template <bool SHORT, typename T> __device__ __forceinline__ Packed16<T> ahead16(const T *row, long col, long cols) {
  if (!SHORT) return load16(row + min(col, cols - CHUNK<T>));
  if (cols >= CHUNK<T>) return load16(row + min(col, cols - CHUNK<T>));
  Packed16<T> p = {};
#pragma unroll 1
  for (long i = cols - 1; i >= col; --i) {
    if constexpr (sizeof(T) == 4) p.q = u32x4{__float_as_uint(row[i]), p.q[0], p.q[1], p.q[2]};
    else p.q = shift_in(p.q, __builtin_bit_cast(uint16_t, row[i]));
  }
  return p;
}
template <typename T> __device__ __forceinline__ void trim16(Packed16<T> &p, long col, long cols) {
  if (cols < CHUNK<T> || col + CHUNK<T> <= cols) return;
  u32x4 q = p.q;
  int by = (int)min(col + CHUNK<T> - cols, (long)CHUNK<T>);
  if constexpr (sizeof(T) == 2) {
    if (by & 1) q = u32x4{q[0] >> 16 | q[1] << 16, q[1] >> 16 | q[2] << 16, q[2] >> 16 | q[3] << 16, q[3] >> 16};
    by >>= 1;
  }
  if (by & 1) q = u32x4{q[1], q[2], q[3], 0u};
  if (by & 2) q = u32x4{q[2], q[3], 0u, 0u};
  p.q = by & 4 ? u32x4{} : q;
}
template <typename T> __device__ __forceinline__ void widen16(float (&v)[CHUNK<T>], const Packed16<T> &p) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(p.q[i]);
  } else {
    const Values8 r = widen(Packed8<T>{p.q});
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r.v[i];
  }
}
template <typename T> __device__ __forceinline__ void add16(float (&v)[CHUNK<T>], const Packed16<T> &p) {
  float more[CHUNK<T>];
  widen16(more, p);
#pragma unroll
  for (int i = 0; i < CHUNK<T>; ++i) v[i] += more[i];
}

// what one wave wrote to LDS is there for its other lanes (whose instructions keep their order)
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// One rounding, to nearest even, from the 32 bits that everything was computed in.
__device__ __forceinline__ uint32_t pack2(float a, float b, __bf16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, _Float16) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
__device__ __forceinline__ void store8(float *p, const Values8 &r) {
  u32x4_from4 *d = reinterpret_cast<u32x4_from4 *>(p);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4_from4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(r.v[4 * h + i]);
    d[h] = q;
  }
}
template <typename T> __device__ __forceinline__ void store8(T *p, const Values8 &r) {
  u32x4_from2 q;
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = pack2(r.v[2 * i], r.v[2 * i + 1], T{});
  *reinterpret_cast<u32x4_from2 *>(p) = q;
}
// the first `count` of eight values
template <typename T> __device__ __forceinline__ void write8(T *p, const Values8 &r, int count) {
  if (count >= 8) {
    store8(p, r);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) p[i] = (T)r.v[i];
}

// types of rows and adapter weights, and a number, as arguments of a generic function
template <typename F> void with_adapter_types(int dtype, int w_dtype, F &&f) {
  if (dtype == RPU_BF16) f(__bf16{}, __bf16{});
  else if (dtype == RPU_F16) f(_Float16{}, _Float16{});
  else if (w_dtype == RPU_F32) f(float{}, float{});
  else if (w_dtype == RPU_F16) f(float{}, _Float16{});
  else f(float{}, __bf16{});
}
template <int V> struct Int {
  static constexpr int value = V;
};

// ---- products of 16-bit operands with floats ----------------------------------------------------------------------------
// 32 terms of 16 x 16 results
template <typename T> __device__ __forceinline__ f32x4 multiply32(u32x4 a, u32x4 b, f32x4 c) {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// what a part leaves of a value; nothing of an infinity
__device__ __forceinline__ float rest_of(float v, float part) { return __builtin_isfinite(v) ? v - part : 0.0f; }
// Two floats as three bf16 each, all of their 24 bits.  Cut off, not rounded: the largest float stays finite.
__device__ __forceinline__ void parts_of(float a, float b, uint32_t (&part)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    part[k] = (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u);
    a = rest_of(a, __uint_as_float(part[k] << 16));
    b = rest_of(b, __uint_as_float(part[k] & 0xffff0000u));
  }
}
// As three halves each, cut off too, the third 1 / HALF_THIRD times what it stands for: of floats that lift_of was found from all bits of those
// down to 2^-26 of the largest.  a and b become what is left of the others.  (An infinity leaves some finite number: where that is added, the
// infinity decides.)
constexpr float HALF_THIRD = 0x1p-11f;
__device__ __forceinline__ void halves_of(float &a, float &b, uint32_t (&part)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    part[k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    const f16x2 r = __builtin_bit_cast(f16x2, part[k]);
    a -= (float)r.x;
    b -= (float)r.y;
    if (k == 0) { // less than the 2^5 of the last bit, or a NaN
      a = fmaxf(a, -32.0f);
      b = fmaxf(b, -32.0f);
    }
    const float next = k == 1 ? 1.0f / HALF_THIRD : k == 2 ? HALF_THIRD : 1.0f;
    a *= next;
    b *= next;
  }
}
// Power of two that floats are multiplied by before halves_of, from their largest magnitude: they may leave the range of halves, the
// largest becomes 2^14 .. 2^15.  (Numbers of less than 2^-97 in steps of 2^-135.)
// What halves_of leaves is multiplied in another round, with a lift of its own, until nothing is left: a small value beside a large one that
// meets a zero keeps its 24 bits.  A round leaves less than 2^-48 of the largest value, so that there are at most six; of values of like
// size there is one.
constexpr int HALF_ROUNDS = 7;
__device__ __forceinline__ float lift_of(float most) {
  const int exponent = max((int)(__float_as_uint(most) >> 23), 30); // biased
  return __uint_as_float((uint32_t)(127 + 14 + 127 - exponent) << 23);
}
// the largest magnitude; of an infinity or a NaN, beside which nothing else counts, the largest number's
__device__ __forceinline__ float most_of(f32x4 v, float most = 0.0f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) most = fmaxf(most, fminf(fabsf(v[i]), 0x1.fffffep127f));
  return most;
}
// the largest of N = 4, 8, 16, 32 neighbouring lanes, in all of them; up to 16 without a trip through LDS
template <int N> __device__ __forceinline__ float most_of_lanes(float most) {
  static_assert(N == 4 || N == 8 || N == 16 || N == 32);
  const auto with = [&](auto ctrl) { // lanes of a row of 16 exchanged
    const int v = __float_as_int(most);
    most = fmaxf(most, __int_as_float(__builtin_amdgcn_update_dpp(v, v, decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  with(Int<0xb1>{});                   // 1 0 3 2 of every four
  with(Int<0x4e>{});                   // 2 3 0 1
  if (N > 4) with(Int<0x141>{});       // eight from behind
  if (N > 8) with(Int<0x140>{});       // sixteen from behind
  if (N > 16) most = fmaxf(most, __shfl_xor(most, 16));
  return most;
}
// something is left that a further round can take (less than 2^-120 is not)
__device__ __forceinline__ bool is_left(float most) { return most >= 0x1p-120f; }
// 1 over a power of two
__device__ __forceinline__ float inverse_of(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
// the first `count` of 4 or 8 values
template <typename T, int N> __device__ __forceinline__ void store_first(T *p, const float (&v)[N], int count) {
  static_assert(N == 4 || N == 8);
  if (count >= N) {
    if constexpr (N == 8) {
      store8(p, Values8{{v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]}});
    } else if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<f32x4_unaligned *>(p) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
      *reinterpret_cast<u32x2_from2 *>(p) = u32x2{pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{})};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < count) p[i] = (T)v[i];
}

// ---- dropout ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t drop_call(const DropDev &d) { return d.call + (d.call_dev ? (uint32_t)*d.call_dev : 0u); }

// bit h: element 8 * block + h of the row is kept
__device__ __forceinline__ uint32_t drop_kept(const DropDev &d, uint32_t call, uint32_t row, uint32_t block) {
  const Philox4 r = philox4x32_10(block, row, call, RNG_DROPOUT, d.key.k0, d.key.k1);
  uint32_t kept = 0, even = 0;
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    const uint32_t u = h & 1 ? r.v[h >> 1] >> 16 : r.v[h >> 1] & 0xffffu;
    kept |= u > d.high ? 1u << h : 0u;
    even |= u == d.high ? 1u << h : 0u;
  }
  if (even) {
    const Philox4 q = philox4x32_10(block, row, call, RNG_DROPOUT_LOW, d.key.k0, d.key.k1);
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      const uint32_t v = h & 1 ? q.v[h >> 1] >> 16 : q.v[h >> 1] & 0xffffu;
      kept |= v >= d.low ? even & (1u << h) : 0u;
    }
  }
  return kept;
}
// What is dropped is zero whatever it was (an infinity, a NaN), never zero times it.
__device__ __forceinline__ void drop_apply(const DropDev &d, uint32_t kept, Values8 &r) {
#pragma unroll
  for (int h = 0; h < 8; ++h) r.v[h] = kept & (1u << h) ? r.v[h] * d.scale : 0.0f;
}
#endif

} // namespace rpu_amd
