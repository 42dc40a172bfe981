// Low-rank adapters of many requests beside one projection: every row takes the adapter that its index names.
//   forward    hidden_t = A x_t,        y_t  = base_t + s B hidden_t
//   backward   up_t = s B^T d_t,        dx_t = base_t + A^T up_t,   dA = sum_t up_t x_t^T,   dB = s sum_t d_t hidden_t^T
// x goes through dropout first where that is on; its mask is drawn again in all three places.
//
//   k_adapter_plan   groups the rows by adapter (a stable counting sort) and cuts the groups into tiles and chunks
//   k_adapter_rows   a tile of rows through both thin products, hidden and up never leave the workgroup in between
//   k_adapter_turn   for the backward pass: the matrices with ranks and columns exchanged, so that it is the forward pass
//   k_adapter_grads  sums over the rows of a chunk, for 128 columns of dA or dB
//   k_adapter_join   adds the chunks of an adapter in their order, zeros for adapters without rows
#include "digital.h"

#include <algorithm>

namespace rpu_amd {
namespace {

template <int V> struct Int {
  static constexpr int value = V;
};

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;

__device__ __forceinline__ int adapter_key(int index, int n) { return index >= 0 && index < n ? index : n; }
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// lanes whose digit is this lane's (lanes with `valid` only)
__device__ __forceinline__ uint64_t same_digit(int digit, bool valid, int bits) {
  uint64_t mask = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool bit = (digit >> b) & 1;
    const uint64_t with = __ballot(valid && bit);
    mask &= bit ? with : ~with;
  }
  return mask;
}
// piece i of a list: key, first place, rows, slot
__device__ __forceinline__ int4 plan_piece(int i, const int *firsts, const int *seg, const int *slots, int keys, int n, int piece) {
  int lo = 0, hi = keys; // the last key that begins at or before piece i
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (firsts[mid + 1] <= i) lo = mid + 1;
    else hi = mid;
  }
  if (lo >= keys) return {-1, 0, 0, 0};
  const int at = seg[lo] + (i - firsts[lo]) * piece;
  return {lo < n ? lo : -1, at, min(piece, seg[lo + 1] - at), slots && slots[lo + 1] > slots[lo] ? slots[lo] + i - firsts[lo] : -1};
}

// Few adapters (a byte holds a key) and rows that LDS holds the keys of: one trip to memory for the index, everything else in
// LDS.
constexpr int PLAN_LDS_ROWS = 65536, PLAN_LDS_KEYS = 256;
__global__ __launch_bounds__(PLAN_THREADS) void k_adapter_plan_lds(const int *index, int *plan, AdapterPlan p) {
  __shared__ uint8_t key_of[PLAN_LDS_ROWS];
  __shared__ int hist[PLAN_WAVES][PLAN_LDS_KEYS], sums[4][4], firsts[4][PLAN_LDS_KEYS + 1]; // of rows, tiles, chunks, slots
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = p.n + 1, bits = 32 - __clz(p.n);
  const uint64_t below = (1ull << lane) - 1;
  const int share = (p.rows + PLAN_THREADS - 1) / PLAN_THREADS * 64, begin = min(wave * share, p.rows), end = min(begin + share, p.rows);
  for (int from = 0; from < p.rows; from += 8 * PLAN_THREADS) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = from + u * PLAN_THREADS + tid < p.rows ? index[from + u * PLAN_THREADS + tid] : 0;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (from + u * PLAN_THREADS + tid < p.rows) key_of[from + u * PLAN_THREADS + tid] = (uint8_t)adapter_key(v[u], p.n);
  }
  for (int i = tid; i < PLAN_WAVES * PLAN_LDS_KEYS; i += PLAN_THREADS) (&hist[0][0])[i] = 0;
  __syncthreads();
  for (int from = begin; from < end; from += 64) {
    const bool valid = from + lane < end;
    const int key = valid ? key_of[from + lane] : 0;
    const uint64_t same = same_digit(key, valid, bits);
    if (valid && !(same & below)) hist[wave][key] += __popcll(same);
    wave_sync();
  }
  __syncthreads();
  int count[4] = {};
  if (tid < PLAN_LDS_KEYS) { // a key's rows: those of wave 0 first
    for (int w = 0; w < PLAN_WAVES; ++w) {
      const int c = hist[w][tid];
      hist[w][tid] = count[0];
      count[0] += c;
    }
    count[1] = (count[0] + p.tile_rows - 1) / p.tile_rows;
    count[2] = tid < p.n ? (count[0] + p.chunk_rows - 1) / p.chunk_rows : 0;
    count[3] = count[2] > 1 ? count[2] : 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      int upto = count[c];
      for (int m = 1; m < 64; m <<= 1) {
        const int v = __shfl_up(upto, m);
        if (lane >= m) upto += v;
      }
      if (lane == 63) sums[wave][c] = upto;
      count[c] = upto - count[c];
    }
  }
  __syncthreads();
  if (tid < PLAN_LDS_KEYS) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      for (int w = 0; w < wave; ++w) count[c] += sums[w][c];
      firsts[c][tid] = count[c];
      if (tid == PLAN_LDS_KEYS - 1) firsts[c][PLAN_LDS_KEYS] = sums[0][c] + sums[1][c] + sums[2][c] + sums[3][c];
    }
  }
  __syncthreads();
  int *order = plan + p.order;
  for (int from = begin; from < end; from += 64) {
    const bool valid = from + lane < end;
    const int key = valid ? key_of[from + lane] : 0;
    const uint64_t same = same_digit(key, valid, bits);
    if (valid) order[firsts[0][key] + hist[wave][key] + __popcll(same & below)] = from + lane;
    wave_sync();
    if (valid && !(same & below)) hist[wave][key] += __popcll(same);
    wave_sync();
  }
  for (int i = tid; i < p.max_tiles; i += PLAN_THREADS)
    reinterpret_cast<int4 *>(plan + p.tiles)[i] = plan_piece(i, firsts[1], firsts[0], nullptr, keys, p.n, p.tile_rows);
  for (int i = tid; i < p.max_chunks; i += PLAN_THREADS)
    reinterpret_cast<int4 *>(plan + p.chunks)[i] = plan_piece(i, firsts[2], firsts[0], firsts[3], p.n, p.n, p.chunk_rows);
  for (int i = tid; i <= keys; i += PLAN_THREADS) plan[p.seg + i] = i < PLAN_LDS_KEYS + 1 ? firsts[0][i] : p.rows;
  for (int i = tid; i <= p.n; i += PLAN_THREADS) {
    plan[p.first + i] = firsts[2][i];
    plan[p.slot_first + i] = firsts[3][i];
  }
}

// Any number of rows and adapters: the lists go through memory, keys of more than a byte in two rounds of the sort.
__global__ __launch_bounds__(PLAN_THREADS) void k_adapter_plan(const int *index, int *plan, AdapterPlan p) {
  __shared__ int hist[PLAN_WAVES][256], start[256], sums[PLAN_WAVES][3];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, keys = p.n + 1;
  int *order = plan + p.order, *seg = plan + p.seg, *other = plan + p.other, *first = plan + p.first, *tile_first = plan + p.tile_first,
      *slot_first = plan + p.slot_first;
  const int share = (p.rows + PLAN_THREADS - 1) / PLAN_THREADS * 64; // rows of a wave
  const int begin = min(wave * (long)share, (long)p.rows), end = min(begin + (long)share, (long)p.rows);
  const uint64_t below = (1ull << lane) - 1;
  const int passes = keys <= 256 ? 1 : 2; // eight bits each
  for (int pass = 0; pass < passes; ++pass) {
    int *to = pass == passes - 1 ? order : other;
    const auto walk = [&](auto &&f) { // over the wave's rows, 64 at a time; the loads of eight times that are under way together
      for (int from = begin; from < end; from += 8 * 64) {
        int row[8], key[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) row[u] = pass && from + 64 * u + lane < end ? other[from + 64 * u + lane] : from + 64 * u + lane;
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = from + 64 * u + lane < end ? adapter_key(index[row[u]], p.n) : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const bool valid = from + 64 * u + lane < end;
          if (from + 64 * u >= end) break; // all lanes
          const int digit = (key[u] >> (8 * pass)) & 255;
          f(row[u], digit, same_digit(digit, valid, 8), valid);
        }
      }
    };
    for (int i = tid; i < PLAN_WAVES * 256; i += PLAN_THREADS) hist[i >> 8][i & 255] = 0;
    __syncthreads();
    walk([&](int, int digit, uint64_t same, bool valid) {
      if (valid && !(same & below)) hist[wave][digit] += __popcll(same);
      wave_sync();
    });
    __syncthreads();
    if (tid < 256) { // a digit's rows: those of wave 0 first
      int sum = 0;
      for (int w = 0; w < PLAN_WAVES; ++w) {
        const int c = hist[w][tid];
        hist[w][tid] = sum;
        sum += c;
      }
      start[tid] = sum;
    }
    __syncthreads();
    if (wave == 0) {
      int own[4], sum = 0;
      for (int i = 0; i < 4; ++i) {
        own[i] = sum;
        sum += start[4 * lane + i];
      }
      int upto = sum;
      for (int m = 1; m < 64; m <<= 1) {
        const int v = __shfl_up(upto, m);
        if (lane >= m) upto += v;
      }
      for (int i = 0; i < 4; ++i) start[4 * lane + i] = upto - sum + own[i];
    }
    __syncthreads();
    walk([&](int row, int digit, uint64_t same, bool valid) {
      if (valid) to[start[digit] + hist[wave][digit] + __popcll(same & below)] = row;
      wave_sync();
      if (valid && !(same & below)) hist[wave][digit] += __popcll(same);
      wave_sync();
    });
    __syncthreads();
  }
  // where every key begins: a key without rows where the next one does
  for (int i = tid; i <= p.rows; i += PLAN_THREADS) {
    const int before = i ? adapter_key(index[order[i - 1]], p.n) : -1, here = i < p.rows ? adapter_key(index[order[i]], p.n) : keys;
    for (int k = before + 1; k <= here; ++k) seg[k] = i;
  }
  __syncthreads();
  // tiles and chunks before every key
  const int keys_each = (keys + PLAN_THREADS - 1) / PLAN_THREADS;
  const int key0 = min(tid * keys_each, keys), key1 = min(key0 + keys_each, keys);
  const auto pieces = [&](int k, int piece) { return (seg[k + 1] - seg[k] + piece - 1) / piece; };
  int count[3] = {}; // tiles, chunks, and those chunks that are not all of their adapter
  const auto add = [&](int k) {
    count[0] += pieces(k, p.tile_rows);
    const int chunks = k < p.n ? pieces(k, p.chunk_rows) : 0;
    count[1] += chunks;
    count[2] += chunks > 1 ? chunks : 0;
  };
  for (int k = key0; k < key1; ++k) add(k);
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    int upto = count[c];
    for (int m = 1; m < 64; m <<= 1) {
      const int v = __shfl_up(upto, m);
      if (lane >= m) upto += v;
    }
    if (lane == 63) sums[wave][c] = upto;
    count[c] = upto - count[c];
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w)
    for (int c = 0; c < 3; ++c) count[c] += sums[w][c];
  for (int k = key0; k < key1; ++k) {
    tile_first[k] = count[0];
    if (k < p.n) {
      first[k] = count[1];
      slot_first[k] = count[2];
    }
    add(k);
  }
  if (tid == PLAN_THREADS - 1) { // the last thread's counts are those of all keys
    tile_first[keys] = count[0];
    first[p.n] = count[1];
    slot_first[p.n] = count[2];
  }
  __syncthreads();
  for (int i = tid; i < p.max_tiles; i += PLAN_THREADS)
    reinterpret_cast<int4 *>(plan + p.tiles)[i] = plan_piece(i, tile_first, seg, nullptr, keys, p.n, p.tile_rows);
  for (int i = tid; i < p.max_chunks; i += PLAN_THREADS)
    reinterpret_cast<int4 *>(plan + p.chunks)[i] = plan_piece(i, first, seg, slot_first, p.n, p.n, p.chunk_rows);
}

// ---- eight terms, or four ranks, of both operands of a product, as the matrix instructions take them ------------------
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// rows of float: products on the fp32 instructions, whatever the weights are stored as
template <typename T, typename TW, bool NARROW = __is_same(T, TW) && sizeof(T) == 2> struct Pipe {
  using X = Packed8<T>;
  using W = Packed8<TW>;
  using V = f32x4; // four ranks of hidden
  static __device__ __forceinline__ f32x4 multiply(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ f32x4 terms(const W &w, const X &x, f32x4 c) {
    const Values8 a = widen(w), b = widen(x);
    c = multiply(f32x4{a.v[0], a.v[1], a.v[2], a.v[3]}, f32x4{b.v[0], b.v[1], b.v[2], b.v[3]}, c);
    return multiply(f32x4{a.v[4], a.v[5], a.v[6], a.v[7]}, f32x4{b.v[4], b.v[5], b.v[6], b.v[7]}, c);
  }
  static __device__ __forceinline__ void keep(X &x, uint32_t kept) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x.q[i >> 2][i & 3] = kept & (1u << i) ? x.q[i >> 2][i & 3] : 0u;
  }
  template <int RT> static __device__ __forceinline__ float split(const f32x4 (&v)[RT], V (&to)[RT]) {
#pragma unroll
    for (int q = 0; q < RT; ++q) to[q] = v[q];
    return 1.0f;
  }
  using R = f32x4; // four ranks of a weight row
  static __device__ __forceinline__ R four(const float *p) { return *reinterpret_cast<const f32x4_unaligned *>(p); }
  template <typename H> static __device__ __forceinline__ R four(const H *p) {
    const u32x2_from2 w = *reinterpret_cast<const u32x2_from2 *>(p);
    const Values8 v = widen(Packed8<H>{u32x4_from2{w[0], w[1], 0u, 0u}});
    return R{v.v[0], v.v[1], v.v[2], v.v[3]};
  }
  static __device__ __forceinline__ void put(R &r, int i, TW w) { r[i] = to_float(w); }
  template <int RT> static __device__ __forceinline__ f32x4 ranks(const R (&w)[RT][2], int j, const V (&v)[RT], f32x4 c) {
#pragma unroll
    for (int q = 0; q < RT; ++q) c = multiply(w[q][j], v[q], c);
    return c;
  }
};

// 16-bit rows with weights of their type: exact products, sums in 32 bits.  hidden, which is not one of their numbers, goes into the
// second product as the sum of some that are, against the same weights again: three bf16 parts, which are all of its 24 bits; two
// halves, 22 bits (an error of 2^-23, twice that of a float, far below the 2^-11 of what is stored in the end).
template <typename T> struct Pipe<T, T, true> {
  using X = Packed8<T>;
  using W = Packed8<T>;
  struct V {
    u32x4 upper; // the first two parts
    u32x2 third;
  };
  static __device__ __forceinline__ f32x4 multiply(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (__is_same(T, __bf16)) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 terms(const W &w, const X &x, f32x4 c) { return multiply(w.q, x.q, c); }
  static __device__ __forceinline__ void keep(X &x, uint32_t kept) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.q[i] &= (kept & (1u << 2 * i) ? 0xffffu : 0u) | (kept & (2u << 2 * i) ? 0xffff0000u : 0u);
  }
  static __device__ __forceinline__ uint32_t cut(float a, float b) { return (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xffff0000u); }
  static __device__ __forceinline__ float rest(float v, float part) { return __builtin_isfinite(v) ? v - part : 0.0f; }
  // returns what the second product has to be multiplied by
  template <int RT> static __device__ __forceinline__ float split(const f32x4 (&v)[RT], V (&to)[RT]) {
    float lift = 1.0f, drop = 1.0f;
    if constexpr (__is_same(T, _Float16)) { // hidden may leave the range of halves: the largest of the row becomes 2^14 .. 2^15
      float most = 0.0f;
#pragma unroll
      for (int q = 0; q < RT; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = __builtin_isfinite(v[q][i]) ? fmaxf(most, fabsf(v[q][i])) : most;
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      const int exponent = max((int)(__float_as_uint(most) >> 23), 30); // biased; smaller rows than 2^-97 round to steps of 2^-135
      lift = __uint_as_float((uint32_t)(127 + 14 + 127 - exponent) << 23);
      drop = __uint_as_float((uint32_t)(exponent - 14) << 23);
    }
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float a = v[q][2 * h] * lift, b = v[q][2 * h + 1] * lift;
        if constexpr (__is_same(T, __bf16)) { // cut off, not rounded: the largest float stays finite
          const uint32_t high = cut(a, b);
          const float a1 = rest(a, __uint_as_float(high << 16)), b1 = rest(b, __uint_as_float(high & 0xffff0000u));
          const uint32_t mid = cut(a1, b1);
          to[q].upper[h] = high;
          to[q].upper[2 + h] = mid;
          to[q].third[h] = cut(a1 - __uint_as_float(mid << 16), b1 - __uint_as_float(mid & 0xffff0000u)); // eight bits are left
        } else {
          const uint32_t high = pack2(a, b, T{});
          const f16x2 r = __builtin_bit_cast(f16x2, high);
          to[q].upper[h] = high;
          to[q].upper[2 + h] = pack2(rest(a, (float)r.x), rest(b, (float)r.y), T{});
        }
      }
    return drop;
  }
  using R = u32x2;
  static __device__ __forceinline__ R four(const T *p) { return *reinterpret_cast<const u32x2_from2 *>(p); }
  static __device__ __forceinline__ void put(R &r, int i, T w) {
    const uint32_t bits = (uint32_t)__builtin_bit_cast(uint16_t, w);
    r[i >> 1] = i & 1 ? r[i >> 1] | bits << 16 : bits;
  }
  template <int RT> static __device__ __forceinline__ f32x4 ranks(const R (&w)[RT][2], int j, const V (&v)[RT], f32x4 c) {
#pragma unroll
    for (int q = 0; q < RT; ++q) c = multiply(u32x4{w[q][j][0], w[q][j][1], w[q][j][0], w[q][j][1]}, v[q].upper, c);
    if constexpr (__is_same(T, __bf16)) { // the third parts of two tiles of ranks at a time
#pragma unroll
      for (int q = 0; q < RT; q += 2) {
        const R next = q + 1 < RT ? w[q + 1 < RT ? q + 1 : q][j] : R{};
        const u32x2 more = q + 1 < RT ? v[q + 1 < RT ? q + 1 : q].third : u32x2{};
        c = multiply(u32x4{w[q][j][0], w[q][j][1], next[0], next[1]}, u32x4{v[q].third[0], v[q].third[1], more[0], more[1]}, c);
      }
    }
    return c;
  }
};

// the first `count` of eight stored values, zeros behind them
template <typename T> __device__ __forceinline__ Packed8<T> load8_first(const T *p, int count) {
  if (count >= 8) return load8(p);
  Packed8<T> r = {};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < count) {
      if constexpr (__is_same(T, float)) r.q[i >> 2][i & 3] = __float_as_uint(p[i]);
      else r.q[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << 16 * (i & 1);
    }
  return r;
}
template <typename T> __device__ __forceinline__ void clear_unless(Packed8<T> &r, bool kept) {
  if constexpr (__is_same(T, float)) {
    r.q[0] = kept ? r.q[0] : u32x4_from4{};
    r.q[1] = kept ? r.q[1] : u32x4_from4{};
  } else {
    r.q = kept ? r.q : u32x4_from2{};
  }
}

constexpr int WAVES = 8;

// A product of 16 x 16 results takes, per lane, row lane % 16 of one operand and column lane % 16 of the other, and of the terms
// those of lane / 16.  Terms may come in any order that both operands share: a lane reads eight neighbouring ones at once.  The
// result has, per lane, column lane % 16 and rows 4 (lane / 16) + 0 .. 3.  With the weights as rows that is: lane % 16 = the
// row of x, and four neighbouring ranks -- the very operand that the second product wants, and there four neighbouring columns
// of y, eight with the weights' rows dealt accordingly.
// The workgroup's waves share the terms of the first product, add their parts up in LDS, and share the columns of the second;
// nothing but x, base, y and the weights (which come from L2) is moved.  FULL: the rank fills its tiles of 16.
template <typename T, typename TW, int RT, int MT, bool FULL> __global__ __launch_bounds__(64 * WAVES) void k_adapter_rows(AdapterRowsArgs a) {
  using P = Pipe<T, TW>;
  constexpr int RP = 16 * RT, PITCH = RP + 4, TILES = MT * RT;
  constexpr int DEEP = RT <= 2 ? 4 / MT : RT == 4 ? 2 / MT : 1; // steps of 32 terms whose loads are under way together
  __shared__ float red[WAVES][16 * MT][PITCH];
  __shared__ int rows_of[64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, lm = lane & 15, kg = lane >> 4;
  int adapter, count;
  if (a.plan) {
    const int4 tile = reinterpret_cast<const int4 *>(a.plan + a.p.tiles)[blockIdx.x];
    adapter = tile.x;
    count = tile.z;
    if (!count) return;
    if ((int)threadIdx.x < count) rows_of[threadIdx.x] = a.plan[a.p.order + tile.y + threadIdx.x];
  } else { // the rows of the adapter of row blockIdx.x, unless an earlier row has it
    const int key = lane < a.rows ? adapter_key(a.index[lane], a.n) : -1;
    const int mine = __shfl(key, (int)blockIdx.x);
    const uint64_t same = __ballot(key == mine);
    if (same & ((1ull << blockIdx.x) - 1)) return;
    adapter = mine < a.n ? mine : -1;
    count = __popcll(same);
    if (wave == 0 && ((same >> lane) & 1)) rows_of[__popcll(same & ((1ull << lane) - 1))] = lane;
  }
  __syncthreads();
  const T *in = static_cast<const T *>(a.in.p), *base = static_cast<const T *>(a.base.p);
  T *out = static_cast<T *>(a.out.p);
  const int units = (a.out_size + 31) / 32; // of 32 columns, shared by the workgroups of the tile
  const int unit0 = (int)((long)units * blockIdx.y / gridDim.y), unit1 = (int)((long)units * (blockIdx.y + 1) / gridDim.y);
  if (adapter < 0) {
    if (base != out || !base)
      for (int m = wave; m < count; m += WAVES) {
        const long row = rows_of[m];
        for (int col = unit0 * 32 + lane * 8; col < min(unit1 * 32, a.out_size); col += 512) {
          Values8 v = {};
          if (base) v = read8(base + row * a.base.ld + col, a.out_size - col);
          write8(out + row * a.out.ld + col, v, a.out_size - col);
        }
      }
    if (a.hidden && !blockIdx.y)
      for (int i = (int)threadIdx.x; i < count * a.rank; i += 64 * WAVES) a.hidden[(long)rows_of[i / a.rank] * a.rank + i % a.rank] = 0.0f;
    return;
  }
  const TW *w_in = static_cast<const TW *>(a.w_in) + (long)adapter * a.rank * a.in_size;
  const TW *w_out = static_cast<const TW *>(a.w_out) + (long)adapter * a.rank * a.out_size;
  const float scale = a.scale[adapter];
  const bool drop_in = a.drop.on && !a.back, drop_out = a.drop.on && a.back;
  const uint32_t call = a.drop.on ? drop_call(a.drop) : 0;
  const int full_steps = a.in_size / 32;

  for (int m0 = 0; m0 < count; m0 += 16 * MT) {
    long row[MT];
    const T *x_at[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) { // rows beyond the last repeat it and are not stored
      row[mt] = rows_of[min(m0 + 16 * mt + lm, count - 1)];
      x_at[mt] = in + row[mt] * a.in.ld;
    }
    f32x4 sum[MT][RT] = {};
    // `n` steps, WAVES apart; not whole: the one that the terms end in; masked: of an input that goes through dropout
    const auto steps = [&](int step, auto n, auto whole, auto masked) {
      constexpr int N = decltype(n)::value;
      typename P::X x[N][MT];
      typename P::W w[N][RT];
#pragma unroll
      for (int s = 0; s < N; ++s) {
        const int col = (step + s * WAVES) * 32 + 8 * kg, left = decltype(whole)::value ? 8 : a.in_size - col;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) x[s][mt] = decltype(whole)::value ? load8(x_at[mt] + col) : load8_first(x_at[mt] + col, left);
#pragma unroll
        for (int q = 0; q < RT; ++q) {
          const int rank = 16 * q + lm;
          const TW *at = w_in + (long)(FULL ? rank : min(rank, a.rank - 1)) * a.in_size + col;
          w[s][q] = decltype(whole)::value ? load8(at) : load8_first(at, left);
          if (!FULL) clear_unless(w[s][q], rank < a.rank);
        }
      }
#pragma unroll
      for (int s = 0; s < N; ++s) {
        const uint32_t block = (uint32_t)(step + s * WAVES) * 4u + (uint32_t)kg;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          if (decltype(masked)::value) P::keep(x[s][mt], drop_kept(a.drop, call, (uint32_t)row[mt], block)); // scaled below
#pragma unroll
          for (int q = 0; q < RT; ++q) sum[mt][q] = P::terms(w[s][q], x[s][mt], sum[mt][q]);
        }
      }
    };
    int step = wave;
    if (drop_in) { // drawing the masks takes longer than the loads
      for (; step < full_steps; step += WAVES) steps(step, Int<1>{}, Int<1>{}, Int<1>{});
      if (step == full_steps && step * 32 < a.in_size) steps(step, Int<1>{}, Int<0>{}, Int<1>{});
    } else {
      for (; step + (DEEP - 1) * WAVES < full_steps; step += DEEP * WAVES) steps(step, Int<DEEP>{}, Int<1>{}, Int<0>{});
      if (DEEP > 1)
        for (; step < full_steps; step += WAVES) steps(step, Int<1>{}, Int<1>{}, Int<0>{});
      if (step == full_steps && step * 32 < a.in_size) steps(step, Int<1>{}, Int<0>{}, Int<0>{});
    }

    // the waves' parts, added in their order: tile t by wave t % WAVES
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int q = 0; q < RT; ++q) *reinterpret_cast<f32x4 *>(&red[wave][16 * mt + lm][16 * q + 4 * kg]) = sum[mt][q];
    __syncthreads();
    for (int t = wave; t < TILES; t += WAVES) {
      const int mt = t / RT, q = t % RT, m = m0 + 16 * mt + lm;
      float *at = &red[0][16 * mt + lm][16 * q + 4 * kg];
      f32x4 v = *reinterpret_cast<const f32x4 *>(at);
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v += *reinterpret_cast<const f32x4 *>(at + w * 16 * MT * PITCH);
      if (drop_in) v *= a.drop.scale;
      const f32x4 scaled = v * scale;
      if (a.hidden && !blockIdx.y && m < count) {
        float *to = a.hidden + (long)rows_of[m] * a.rank + 16 * q + 4 * kg;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (FULL || 16 * q + 4 * kg + i < a.rank) to[i] = a.back ? scaled[i] : v[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) // padding is zero also where a row holds an infinity, whose product with it is none
        at[i] = FULL || 16 * q + 4 * kg + i < a.rank ? scaled[i] : 0.0f;
    }
    __syncthreads();
    typename P::V hidden[MT][RT];
    float lift[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int q = 0; q < RT; ++q) sum[mt][q] = *reinterpret_cast<const f32x4 *>(&red[0][16 * mt + lm][16 * q + 4 * kg]);
      lift[mt] = P::split(sum[mt], hidden[mt]) * (drop_out ? a.drop.scale : 1.0f);
    }

    const auto columns = [&](int unit0, auto n, auto whole, auto masked) { // `n` units, WAVES apart
      constexpr int N = decltype(n)::value;
      Packed8<T> add[N][MT];
      typename P::R w[N][RT][2];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int unit = unit0 + u * WAVES, col = unit * 32 + 8 * kg;
        if (base) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            add[u][mt] = decltype(whole)::value ? load8(base + row[mt] * a.base.ld + col) : load8_first(base + row[mt] * a.base.ld + col, a.out_size - col);
        }
#pragma unroll
        for (int q = 0; q < RT; ++q)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            int c = unit * 32 + (lm >> 2) * 8 + j * 4 + (lm & 3); // the column whose result ends up beside its neighbours
            if (!decltype(whole)::value) c = min(c, a.out_size - 1);
            const int rank = 16 * q + 4 * kg;
            if (FULL) {
              w[u][q][j] = P::four(w_out + (long)c * a.rank + rank);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) P::put(w[u][q][j], i, rank + i < a.rank ? w_out[(long)c * a.rank + min(rank + i, a.rank - 1)] : (TW)0.0f);
            }
          }
      }
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int unit = unit0 + u * WAVES, col = unit * 32 + 8 * kg, left = decltype(whole)::value ? 8 : a.out_size - col;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          f32x4 acc[2] = {};
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[j] = P::ranks(w[u], j, hidden[mt], acc[j]);
          if (m0 + 16 * mt + lm >= count) continue;
          Values8 v;
#pragma unroll
          for (int h = 0; h < 8; ++h) v.v[h] = acc[h >> 2][h & 3] * lift[mt];
          if (decltype(masked)::value) {
            const uint32_t kept = drop_kept(a.drop, call, (uint32_t)row[mt], (uint32_t)unit * 4u + (uint32_t)kg);
#pragma unroll
            for (int h = 0; h < 8; ++h) v.v[h] = kept & (1u << h) ? v.v[h] : 0.0f;
          }
          if (base) {
            const Values8 b = widen(add[u][mt]);
#pragma unroll
            for (int h = 0; h < 8; ++h) v.v[h] += b.v[h];
          }
          if (decltype(whole)::value) store8(out + row[mt] * a.out.ld + col, v);
          else write8(out + row[mt] * a.out.ld + col, v, left);
        }
      }
    };
    constexpr int WIDE = RT * MT == 1 ? 4 : RT * MT == 2 ? 2 : 1; // units whose loads are under way together
    const int whole_units = min(unit1, a.out_size / 32);
    int unit = unit0 + wave;
    if (drop_out) {
      for (; unit < whole_units; unit += WAVES) columns(unit, Int<1>{}, Int<1>{}, Int<1>{});
      if (unit < unit1) columns(unit, Int<1>{}, Int<0>{}, Int<1>{});
    } else {
      for (; unit + (WIDE - 1) * WAVES < whole_units; unit += WIDE * WAVES) columns(unit, Int<WIDE>{}, Int<1>{}, Int<0>{});
      if (WIDE > 1)
        for (; unit < whole_units; unit += WAVES) columns(unit, Int<1>{}, Int<1>{}, Int<0>{});
      if (unit < unit1) columns(unit, Int<1>{}, Int<0>{}, Int<0>{});
    }
    __syncthreads();
  }
}

// The matrices of the adapters that have rows with ranks and columns exchanged: with them the backward pass of rows is the
// forward pass.
template <typename TW> __global__ __launch_bounds__(256) void k_adapter_turn(AdapterTurnArgs a) {
  __shared__ TW tile[64][65];
  const int *seg = a.plan + a.p.seg;
  const int t = (int)threadIdx.x, fast = t & 63, slow = t >> 6;
  const int a_tiles = (a.in_size + 63) / 64, b_tiles = (a.out_size + 63) / 64, rank_tiles = (a.rank + 63) / 64;
  for (int adapter = (int)blockIdx.y; adapter < a.n; adapter += (int)gridDim.y) {
    if (seg[adapter + 1] == seg[adapter]) continue;
    for (int k = (int)blockIdx.x; k < (a_tiles + b_tiles) * rank_tiles; k += (int)gridDim.x) {
      const int c = k / rank_tiles, r0 = k % rank_tiles * 64;
      const bool of_a = c < a_tiles;
      // a: [rank][in] -> [in][rank], b: [out][rank] -> [rank][out]
      const int rows = of_a ? a.rank : a.out_size, cols = of_a ? a.in_size : a.rank;
      const int row0 = of_a ? r0 : (c - a_tiles) * 64, col0 = of_a ? c * 64 : r0;
      const long at = (long)adapter * rows * cols;
      const TW *from = static_cast<const TW *>(of_a ? a.a : a.b) + at;
      TW *to = static_cast<TW *>(of_a ? a.a_turned : a.b_turned) + at;
      __syncthreads();
      TW v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = row0 + slow + 4 * i;
        v[i] = from[(long)min(r, rows - 1) * cols + min(col0 + fast, cols - 1)];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) tile[slow + 4 * i][fast] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = col0 + slow + 4 * i;
        if (c < cols && row0 + fast < rows) to[(long)c * rows + row0 + fast] = tile[fast][slow + 4 * i];
      }
    }
  }
}

constexpr int GRAD_WAVES = 4;

// 128 columns of dA (of x, against up) or of dB (of d, against scale hidden).  A wave takes 16 rows of its chunk at a time; lane
// % 16 reads eight neighbouring columns of four rows, and product j of a row takes column 8 (lane % 16) + j.
template <typename T, typename TW, int RT> __global__ __launch_bounds__(64 * GRAD_WAVES) void k_adapter_grads(AdapterGradArgs a) {
  __shared__ float sums[32 * RT][64];
  const int4 chunk = reinterpret_cast<const int4 *>(a.plan + a.p.chunks)[blockIdx.x];
  const int adapter = chunk.x, count = chunk.z;
  if (!count) return;
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, lm = lane & 15, kg = lane >> 4;
  const int *order = a.plan + a.p.order + chunk.y;
  const int x_slices = (a.in_size + 127) / 128;
  const bool of_a = (int)blockIdx.y < x_slices;
  const int c0 = ((int)blockIdx.y - (of_a ? 0 : x_slices)) * 128, width = of_a ? a.in_size : a.out_size;
  const MatrixDev m = of_a ? a.x : a.d;
  const float *factor = of_a ? a.up : a.hidden;
  const float scale = of_a ? 1.0f : a.scale[adapter];
  const bool drop = of_a && a.drop.on;
  const uint32_t call = drop ? drop_call(a.drop) : 0;
  const int col = c0 + 8 * lm, left = width - col, rank0 = 16 * RT * (int)blockIdx.z;
  f32x4 acc[8][RT] = {};
  for (int g = wave; g * 16 < count; g += GRAD_WAVES) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 16 * g + 4 * kg + i;
      const bool valid = at < count;
      const long row = order[min(at, count - 1)];
      Values8 x = read8(static_cast<const T *>(m.p) + row * m.ld + col, valid ? left : 0);
      if (drop) drop_apply(a.drop, drop_kept(a.drop, call, (uint32_t)row, (uint32_t)col / 8u), x);
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        const int rank = rank0 + 16 * q + lm;
        const float u = valid && rank < a.rank ? factor[row * a.rank + rank] * scale : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[j], u, acc[j][q], 0, 0, 0);
      }
    }
  }
  for (int from = 0; from < GRAD_WAVES; ++from) { // the waves' sums, added in their order
    if (wave == from) {
#pragma unroll
      for (int e = 0; e < 32 * RT; ++e) {
        const float v = acc[e & 7][e >> 5][(e >> 3) & 3] + (from ? sums[e][lane] : 0.0f);
        acc[e & 7][e >> 5][(e >> 3) & 3] = v;
        sums[e][lane] = v;
      }
    }
    __syncthreads();
  }
  if (wave != GRAD_WAVES - 1) return;
  const bool whole = chunk.w < 0; // nothing to join
  float *part = a.part + (long)chunk.w * a.rank * ((long)a.in_size + a.out_size) + (of_a ? 0 : (long)a.rank * a.in_size);
#pragma unroll
  for (int q = 0; q < RT; ++q) {
    const int rank = rank0 + 16 * q + lm;
    if (rank >= a.rank) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + 32 * kg + 8 * i;
      Values8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v.v[j] = acc[j][q][i];
      if (of_a) {
        const long at = (long)rank * a.in_size + c;
        if (whole) write8(static_cast<TW *>(a.da) + (long)adapter * a.rank * a.in_size + at, v, width - c);
        else write8(part + at, v, width - c);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (c + j >= width) continue;
          const long at = (long)(c + j) * a.rank + rank;
          if (whole) static_cast<TW *>(a.db)[(long)adapter * a.rank * a.out_size + at] = (TW)v.v[j];
          else part[at] = v.v[j];
        }
      }
    }
  }
}

template <typename TW> __global__ __launch_bounds__(256) void k_adapter_join(AdapterGradArgs a) {
  const long of_a = (long)a.rank * a.in_size, all = of_a + (long)a.rank * a.out_size;
  const int *first = a.plan + a.p.first, *slots = a.plan + a.p.slot_first;
  for (int adapter = (int)blockIdx.y; adapter < a.n; adapter += (int)gridDim.y) {
    if (first[adapter + 1] - first[adapter] == 1) continue;
    const int begin = slots[adapter], end = slots[adapter + 1];
    for (long e = (long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long)gridDim.x * 256) {
      float sum = 0.0f;
      int c = begin;
      for (; c + 8 <= end; c += 8) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = a.part[(c + u) * all + e];
#pragma unroll
        for (int u = 0; u < 8; ++u) sum += v[u];
      }
      for (; c < end; ++c) sum += a.part[c * all + e];
      if (e < of_a) static_cast<TW *>(a.da)[adapter * of_a + e] = (TW)sum;
      else static_cast<TW *>(a.db)[adapter * (all - of_a) + e - of_a] = (TW)sum;
    }
  }
}

template <typename F> void with_types(int dtype, int w_dtype, F &&f) {
  if (dtype == RPU_BF16) f(__bf16{}, __bf16{});
  else if (dtype == RPU_F16) f(_Float16{}, _Float16{});
  else if (w_dtype == RPU_F32) f(float{}, float{});
  else if (w_dtype == RPU_F16) f(float{}, _Float16{});
  else f(float{}, __bf16{});
}
template <typename F> void with_rank_tiles(int rank, F &&f) {
  if (rank <= 16) f(Int<1>{});
  else if (rank <= 32) f(Int<2>{});
  else if (rank <= 64) f(Int<4>{});
  else f(Int<8>{});
}

} // namespace

void launch_adapter_rows(const AdapterRowsArgs &a, int dtype, int w_dtype, int cus, hipStream_t s) {
  const int tile_rows = a.plan ? a.p.tile_rows : a.rows, tiles = a.plan ? a.p.max_tiles : a.rows;
  // tiles that leave CUs idle share their output columns among several workgroups, each of which makes hidden for itself
  const int units = (a.out_size + 31) / 32;
  const int slices = std::max(1, std::min(units / WAVES, cus / std::max(tiles, 1)));
  const dim3 grid((unsigned)tiles, (unsigned)slices);
  with_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    with_rank_tiles(a.rank, [&](auto rt) {
      constexpr int RT = decltype(rt)::value, MOST = RT <= 4 ? 2 : 1; // groups of 16 rows at a time: what registers and LDS hold
      const bool full = a.rank == 16 * RT;
      if (tile_rows <= 16 || MOST == 1) {
        if (full) hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, 1, true>), grid, dim3(64 * WAVES), 0, s, a);
        else hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, 1, false>), grid, dim3(64 * WAVES), 0, s, a);
      } else {
        if (full) hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, MOST, true>), grid, dim3(64 * WAVES), 0, s, a);
        else hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, MOST, false>), grid, dim3(64 * WAVES), 0, s, a);
      }
    });
  });
}

void launch_adapter_turn(const AdapterTurnArgs &a, int w_dtype, int cus, hipStream_t s) {
  const int tiles = ((a.in_size + 63) / 64 + (a.out_size + 63) / 64) * ((a.rank + 63) / 64);
  const dim3 grid((unsigned)std::min(tiles, std::max(1, cus * 8 / std::min(a.n, cus * 8))), (unsigned)std::min(a.n, cus * 8));
  if (w_dtype == RPU_F32) hipLaunchKernelGGL(k_adapter_turn<float>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_adapter_turn<uint16_t>, grid, dim3(256), 0, s, a);
}

AdapterPlan adapter_plan(int rows, int n) {
  AdapterPlan p{};
  p.rows = rows;
  p.n = n;
  p.tile_rows = rows <= 16384 ? 16 : 32;
  p.chunk_rows = 64;
  while (p.chunk_rows < 1024 && rows / p.chunk_rows > 32) p.chunk_rows *= 2;
  // every group of rows but for one may end with a piece that is not full
  p.max_tiles = (int)std::min<long>(rows, ((long)rows + p.tile_rows - 1) / p.tile_rows + std::min(n, rows));
  p.max_chunks = (int)std::min<long>(rows, ((long)rows + p.chunk_rows - 1) / p.chunk_rows + std::min(n, rows));
  p.max_slots = (int)std::min<long>(p.max_chunks, 2l * rows / p.chunk_rows); // of adapters with more rows than a chunk
  size_t at = 0;
  const auto take = [&](size_t words) {
    const size_t from = at;
    at += (words + 3) / 4 * 4;
    return from;
  };
  p.tiles = take(4 * (size_t)p.max_tiles);
  p.chunks = take(4 * (size_t)p.max_chunks);
  p.order = take((size_t)rows);
  p.seg = take((size_t)n + 2);
  p.first = take((size_t)n + 1);
  p.tile_first = take((size_t)n + 2);
  p.slot_first = take((size_t)n + 1);
  p.other = take(n + 1 > 256 ? (size_t)rows : 0);
  p.words = at;
  return p;
}

void launch_adapter_plan(const int *index, int *plan, const AdapterPlan &p, hipStream_t s) {
  if (p.rows <= PLAN_LDS_ROWS && p.n < PLAN_LDS_KEYS) hipLaunchKernelGGL(k_adapter_plan_lds, dim3(1), dim3(PLAN_THREADS), 0, s, index, plan, p);
  else hipLaunchKernelGGL(k_adapter_plan, dim3(1), dim3(PLAN_THREADS), 0, s, index, plan, p);
}

void launch_adapter_grads(const AdapterGradArgs &a, int dtype, int w_dtype, int cus, hipStream_t s) {
  const unsigned slices = (unsigned)(((long)a.in_size + 127) / 128 + ((long)a.out_size + 127) / 128);
  const long values = (long)a.rank * ((long)a.in_size + a.out_size);
  const dim3 join((unsigned)std::max<long>(1, std::min<long>((values + 255) / 256, std::max(1, cus * 8 / a.n))), (unsigned)std::min(a.n, 65535));
  with_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    if (a.rows)
      with_rank_tiles(a.rank, [&](auto rt) {
        constexpr int RT = decltype(rt)::value, AT_ONCE = RT < 4 ? RT : 4; // more sums than that of 64 ranks leave the registers
        hipLaunchKernelGGL((k_adapter_grads<T, TW, AT_ONCE>), dim3((unsigned)a.p.max_chunks, slices, RT / AT_ONCE), dim3(64 * GRAD_WAVES), 0, s, a);
      });
    hipLaunchKernelGGL(k_adapter_join<TW>, join, dim3(256), 0, s, a);
  });
}

} // namespace rpu_amd
