// The rows of low-rank adapters through their two thin products (kernels_adapter.hip says what is computed):
//   k_adapter_down  hidden = A x of 16 rows, the terms shared by the waves of a workgroup
//   k_adapter_up    y = base + s B hidden of 16 rows and 128 columns, every wave on columns of its own
//   k_adapter_few   both in one launch, for few rows
// The backward pass is the same with d for x, and the matrices turned (k_adapter_turn).
#include "digital.h"

#include <algorithm>

namespace rpu_amd {
namespace {

// ---- eight terms, or four ranks, of both operands of a product, as the matrix instructions take them ------------------

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
  static constexpr bool ROUNDS = false;
  static __device__ __forceinline__ float lift(float) { return 1.0f; }
  static __device__ __forceinline__ V split(const f32x4 &v, float) { return v; }
  using R = f32x4; // four ranks of a weight row
  static __device__ __forceinline__ R four(const float *p) { return *reinterpret_cast<const f32x4_unaligned *>(p); }
  template <typename H> static __device__ __forceinline__ R four(const H *p) {
    const u32x2_from2 w = *reinterpret_cast<const u32x2_from2 *>(p);
    const Values8 v = widen(Packed8<H>{u32x4_from2{w[0], w[1], 0u, 0u}});
    return R{v.v[0], v.v[1], v.v[2], v.v[3]};
  }
  template <typename H> static __device__ __forceinline__ R four_aligned(const H *p) { // in LDS
    if constexpr (sizeof(H) == 4) {
      return *reinterpret_cast<const f32x4 *>(p);
    } else {
      const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
      const Values8 v = widen(Packed8<H>{u32x4_from2{w[0], w[1], 0u, 0u}});
      return R{v.v[0], v.v[1], v.v[2], v.v[3]};
    }
  }
  static __device__ __forceinline__ void put(R &r, int i, TW w, uint32_t mask) { r[i] = __uint_as_float(__float_as_uint(to_float(w)) & mask); }
  template <int RT> static __device__ __forceinline__ f32x4 ranks(const R (&w)[RT], const V (&v)[RT], f32x4 c) {
#pragma unroll
    for (int q = 0; q < RT; ++q) c = multiply(w[q], v[q], c);
    return c;
  }
};

// 16-bit rows with weights of their type: exact products, sums in 32 bits.  hidden, which is not one of their numbers, goes into the
// second product as the sum of three that are, against the same weights again: all of its 24 bits.  Three bf16 always are; three halves,
// of which the third has a sum of its own, are of values down to 2^-26 of the largest, and what they leave of others takes another round.
template <typename T> struct Pipe<T, T, true> {
  using X = Packed8<T>;
  using W = Packed8<T>;
  struct V {
    u32x4 upper; // the first two parts
    u32x2 third;
  };
  static constexpr bool ROUNDS = __is_same(T, _Float16);
  static __device__ __forceinline__ f32x4 terms(const W &w, const X &x, f32x4 c) { return multiply32<T>(w.q, x.q, c); }
  static __device__ __forceinline__ void keep(X &x, uint32_t kept) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.q[i] &= (kept & (1u << 2 * i) ? 0xffffu : 0u) | (kept & (2u << 2 * i) ? 0xffff0000u : 0u);
  }
  static __device__ __forceinline__ float lift(float most) { return __is_same(T, __bf16) ? 1.0f : lift_of(most); }
  static __device__ __forceinline__ V split(f32x4 &v, float lift) { // v: what is left
    V to;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t part[3];
      if constexpr (ROUNDS) {
        const float back = inverse_of(lift);
        float a = v[2 * h] * lift, b = v[2 * h + 1] * lift;
        halves_of(a, b, part);
        v[2 * h] = a * back;
        v[2 * h + 1] = b * back;
      } else {
        parts_of(v[2 * h], v[2 * h + 1], part);
      }
      to.upper[h] = part[0];
      to.upper[2 + h] = part[1];
      to.third[h] = part[2];
    }
    return to;
  }
  // what an earlier round left of four ranks of a lane, those of lanes that are 16 apart together, against N tiles of weights
  template <int N> static __device__ __forceinline__ void add_left(const u32x2 (&w)[N], f32x4 left, f32x4 (&c)[N]) {
    for (int round = 1; round < HALF_ROUNDS; ++round) {
      float most = most_of(left);
      most = fmaxf(most, __shfl_xor(most, 16));
      most = fmaxf(most, __shfl_xor(most, 32));
      if (!__ballot(is_left(most))) break;
      const float lift = lift_of(most), back = inverse_of(lift);
      const V v[1] = {split(left, lift)};
#pragma unroll
      for (int t = 0; t < N; ++t) {
        const u32x2 w1[1] = {w[t]};
        c[t] += ranks(w1, v, f32x4{}) * back;
      }
    }
  }
  using R = u32x2;
  static __device__ __forceinline__ R four(const T *p) { return *reinterpret_cast<const u32x2_from2 *>(p); }
  static __device__ __forceinline__ R four_aligned(const T *p) { return *reinterpret_cast<const u32x2 *>(p); }
  static __device__ __forceinline__ void put(R &r, int i, T w, uint32_t mask) {
    const uint32_t bits = (uint32_t)__builtin_bit_cast(uint16_t, w) & mask;
    r[i >> 1] = i & 1 ? r[i >> 1] | bits << 16 : bits;
  }
  template <int RT> static __device__ __forceinline__ f32x4 ranks(const R (&w)[RT], const V (&v)[RT], f32x4 c) {
#pragma unroll
    for (int q = 0; q < RT; ++q) c = multiply32<T>(u32x4{w[q][0], w[q][1], w[q][0], w[q][1]}, v[q].upper, c);
    f32x4 third = ROUNDS ? f32x4{} : c;
#pragma unroll
    for (int q = 0; q < RT; q += 2) { // the third parts of two tiles of ranks at a time
      const R next = q + 1 < RT ? w[q + 1 < RT ? q + 1 : q] : R{};
      const u32x2 more = q + 1 < RT ? v[q + 1 < RT ? q + 1 : q].third : u32x2{};
      third = multiply32<T>(u32x4{w[q][0], w[q][1], next[0], next[1]}, u32x4{v[q].third[0], v[q].third[1], more[0], more[1]}, third);
    }
    return ROUNDS ? c + third * HALF_THIRD : third;
  }
};

// Ranks rank .. rank + 3 of a row of `ranks`, zeros behind the last.  Masked by bits: a choice between a load and zero becomes a branch
// around the load, and loads in branches wait for each other.
template <typename P, typename W> __device__ __forceinline__ typename P::R load_ranks(const W *row, int rank, int ranks) {
  W v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = row[min(rank + i, ranks - 1)];
  typename P::R r = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) P::put(r, i, v[i], (uint32_t)((rank + i - ranks) >> 31));
  return r;
}
template <typename T> __device__ __forceinline__ void clear_unless(Packed8<T> &r, bool kept) {
  const uint32_t mask = kept ? ~0u : 0u;
  if constexpr (sizeof(T) == 4) {
    r.q[0] &= mask;
    r.q[1] &= mask;
  } else {
    r.q &= mask;
  }
}

// A product of 16 x 16 results takes, per lane, row lane % 16 of one operand and column lane % 16 of the other, and of the terms
// those of lane / 16.  Terms may come in any order that both operands share: a lane reads eight neighbouring ones at once.  The
// result has, per lane, column lane % 16 and rows 4 (lane / 16) + 0 .. 3.  With the weights as rows that is: lane % 16 = the
// row of x, and four neighbouring ranks -- the very operand that the second product wants, and there four neighbouring columns
// of y, eight with the weights' rows dealt accordingly.
constexpr int WAVES = 8, UP_WAVES = 4; // of a workgroup: those that share the terms of the first product; those of the second alone

// Eight terms of a rank of A; trimmed: zeros behind the last term and the last rank.
template <bool SHORT, typename TW, bool FULL> __device__ __forceinline__ Packed8<TW> weight_terms(const TW *w, long in_size, int rank, int ranks, int col, bool whole) {
  const TW *row = w + (FULL ? rank : min(rank, ranks - 1)) * in_size;
  return whole ? load8(row + col) : ahead8<SHORT>(row, col, in_size);
}
template <typename TW, bool FULL> __device__ __forceinline__ void trim_terms(Packed8<TW> &w, long in_size, int rank, int ranks, int col) {
  trim8(w, col, in_size);
  if (!FULL) clear_unless(w, rank < ranks);
}

// Rank tile q of 16 rows: the waves' shares, added in their order.
template <int NW, int PITCH> __device__ __forceinline__ f32x4 add_shares(const float (*red)[16][PITCH], int q) {
  const int lane = (int)threadIdx.x & 63, lm = lane & 15, kg = lane >> 4;
  f32x4 v = *reinterpret_cast<const f32x4 *>(&red[0][lm][16 * q + 4 * kg]);
#pragma unroll
  for (int w = 1; w < NW; ++w) v += *reinterpret_cast<const f32x4 *>(&red[w][lm][16 * q + 4 * kg]);
  return v;
}

// What a workgroup makes: the columns `piece` of the rows `group` of a tile.  Workgroups b, b + 8, b + 16, .. meet the same XCD: they take the
// pieces of a group, one after another, then the groups of a tile.  (All rows of a piece first: 33.6 us instead of 32.4 for 8192 rows of
// 2304 floats, 26.5 instead of 25.0 for 4096 rows of 4096 bf16.)
struct Place {
  int4 tile;
  int group, piece;
};
__device__ __forceinline__ Place place_of(const AdapterRowsArgs &a, uint32_t groups, uint32_t pieces) {
  const uint32_t b = blockIdx.y * gridDim.x + blockIdx.x, j = b / 8, g = j / pieces, p = g / groups * 8 + b % 8;
  Place at = {{-1, 0, 0, 0}, (int)(g % groups), (int)(j % pieces)};
  if (p < (uint32_t)a.p.max_tiles) at.tile = reinterpret_cast<const int4 *>(a.plan + a.p.tiles)[p];
  return at;
}

__device__ __forceinline__ int matrix_of(const AdapterRowsArgs &a, int adapter) { return a.listed ? a.plan[a.p.first + adapter] : adapter; }

template <typename T> __device__ __forceinline__ void read8_lds(Packed8<T> &v, const uint32_t *at) {
  if constexpr (sizeof(T) == 4) {
    v.q[0] = *reinterpret_cast<const u32x4 *>(at);
    v.q[1] = *reinterpret_cast<const u32x4 *>(at + 4);
  } else {
    v.q = *reinterpret_cast<const u32x4 *>(at);
  }
}

// hidden of 16 rows.  The waves share the terms in segments of 256 bytes of x, each wave by itself up to the sum over all of them, so
// that they fall out of step and some always load.  x and A are read along their rows and turned into the operands' order in
// LDS of the wave's own: read in that order, 16 rows to every 16 lanes, they would take the address units four times as long.
// The workgroups begin at different segments: all those of an adapter read the same A.
// Bound by the reads of x, and the chain of loads before the first of them (tile, its rows, x).  8192 rows of 768 floats, rank 16: 11.2 us
// (28 MB); 8192 rows of 2304 floats: 21.0 us (75 MB, 3.6 TB/s); 4096 rows of 4096 bf16, rank 64: 14.9 us, where every 16 rows read all
// 0.5 MB of A from the L2, 134 MB.  With the stages of all waves in step (barriers around x in LDS) 15.5, 28 and 25 us; with 4 waves
// 13.6, 33 and 25 us, with 16 17.7, 30 and 16.4 us, both before loads went out together.  Registers: three or four waves of a SIMD without
// spills; six spill and take twice the time.
constexpr int DOWN_WAVES = 8;
template <typename T, typename TW, int RT, bool FULL, bool DROP, bool SHORT> __global__ __launch_bounds__(64 * DOWN_WAVES, RT == 8 ? 2 : DROP ? 3 : 4) void k_adapter_down(AdapterRowsArgs a) {
  using P = Pipe<T, TW>;
  constexpr int NW = DOWN_WAVES, SEG = 256 / (int)sizeof(T), STEPS = SEG / 32, X_LOADS = 4;
  constexpr int W_ROW = SEG * (int)sizeof(TW) / 16, W_LOADS = 16 * W_ROW / 64; // lanes of a rank; loads of a tile of 16 ranks
  constexpr int GROUP = RT < 4 ? RT : 4, PITCH = 16 * GROUP + 4;            // rank tiles that are added up at a time
  union Shared {
    uint32_t terms[NW][16][64 + 4];
    float red[NW][16][PITCH];
  };
  __shared__ Shared m;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, lm = lane & 15, kg = lane >> 4;
  const auto [tile, group, piece] = place_of(a, ADAPTER_TILE_ROWS / 16, 1);
  const int adapter = tile.x, count = min(tile.z - 16 * group, 16);
  if (count <= 0) return;
  const int *order = a.plan + a.p.order + tile.y + 16 * group;
  if (adapter < 0) {
    for (int i = tid; i < count * a.rank; i += 64 * NW) a.hidden[(long)order[i / a.rank] * a.rank + i % a.rank] = 0.0f;
    return;
  }
  const int row = order[min(lm, count - 1)]; // rows beyond the last repeat it and are not stored
  const T *x_at[X_LOADS];
#pragma unroll
  for (int j = 0; j < X_LOADS; ++j) x_at[j] = static_cast<const T *>(a.in.p) + (long)__shfl(row, 4 * j + kg) * a.in.ld;
  const TW *w_in = static_cast<const TW *>(a.w_in) + (long)matrix_of(a, adapter) * a.rank * a.in_size;
  const uint32_t call = DROP ? drop_call(a.drop) : 0;
  const int segments = (a.in_size + SEG - 1) / SEG, n = (segments - wave + NW - 1) / NW; // n of the wave
  const int first = n > 0 ? (int)(blockIdx.x / 8 % (unsigned)n) : 0;
  const auto segment = [&](int i) { return wave + NW * (first + i < n ? first + i : first + i - n); };
  const auto fetch_x = [&](Packed16<T> (&x)[X_LOADS], int seg) {
#pragma unroll
    for (int j = 0; j < X_LOADS; ++j) x[j] = ahead16<SHORT>(x_at[j], (long)seg * SEG + lm * CHUNK<T>, a.in_size);
  };
  const auto fetch_w = [&](Packed16<TW> (&w)[W_LOADS], int seg, int q) {
    int l = lane;
    asm volatile("" : "+v"(l)); // addresses made anew: kept for all tiles of ranks they spill
#pragma unroll
    for (int j = 0; j < W_LOADS; ++j) {
      const int rank = 16 * q + (l + 64 * j) / W_ROW;
      w[j] = ahead16<SHORT>(w_in + (uint32_t)(FULL ? rank : min(rank, a.rank - 1)) * (uint32_t)a.in_size, (long)seg * SEG + l % W_ROW * CHUNK<TW>, a.in_size);
    }
  };
  uint32_t(*const at)[64 + 4] = m.terms[wave];
  const auto turn_x = [&](Packed16<T> (&x)[X_LOADS], typename P::X (&v)[STEPS], int seg) {
    if (seg + 1 == segments) {
#pragma unroll
      for (int j = 0; j < X_LOADS; ++j) trim16(x[j], (long)seg * SEG + lm * CHUNK<T>, a.in_size);
    }
    wave_sync(); // the last weights have been read
#pragma unroll
    for (int j = 0; j < X_LOADS; ++j) *reinterpret_cast<u32x4 *>(&at[4 * j + kg][lm * 4]) = x[j].q;
    wave_sync();
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      read8_lds(v[u], &at[lm][(u * 32 + 8 * kg) * (int)sizeof(T) / 4]);
      if (DROP) P::keep(v[u], drop_kept(a.drop, call, (uint32_t)row, (uint32_t)((seg * STEPS + u) * 4 + kg))); // what is kept is scaled below
    }
  };
  const auto multiply = [&](Packed16<TW> (&w)[W_LOADS], const typename P::X (&v)[STEPS], int seg, int q, f32x4 sum) {
    int l = lane;
    asm volatile("" : "+v"(l));
    if (seg + 1 == segments) {
#pragma unroll
      for (int j = 0; j < W_LOADS; ++j) trim16(w[j], (long)seg * SEG + l % W_ROW * CHUNK<TW>, a.in_size);
    }
    if (!FULL) {
#pragma unroll
      for (int j = 0; j < W_LOADS; ++j) w[j].q &= (uint32_t)((16 * q + (l + 64 * j) / W_ROW - a.rank) >> 31);
    }
    wave_sync(); // what lay there has been read
#pragma unroll
    for (int j = 0; j < W_LOADS; ++j) *reinterpret_cast<u32x4 *>(&at[(lane + 64 * j) / W_ROW][lane % W_ROW * 4]) = w[j].q;
    wave_sync();
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      typename P::W t;
      read8_lds(t, &at[lm][(u * 32 + 8 * kg) * (int)sizeof(TW) / 4]);
      sum = P::terms(t, v[u], sum);
    }
    return sum;
  };
  f32x4 sum[RT] = {};
  Packed16<T> x[2][X_LOADS];
  Packed16<TW> w[2][W_LOADS];
  typename P::X v[STEPS];
  if constexpr (RT == 1) { // two segments under way
    if (n > 0) {
      fetch_x(x[0], segment(0));
      fetch_w(w[0], segment(0), 0);
    }
    if (n > 1) {
      fetch_x(x[1], segment(1));
      fetch_w(w[1], segment(1), 0);
    }
    const auto step = [&](Packed16<T> (&x)[X_LOADS], Packed16<TW> (&w)[W_LOADS], int i) {
      turn_x(x, v, segment(i));
      if (i + 2 < n) fetch_x(x, segment(i + 2));
      sum[0] = multiply(w, v, segment(i), 0, sum[0]);
      if (i + 2 < n) fetch_w(w, segment(i + 2), 0);
    };
    for (int i = 0; i < n; i += 2) {
      step(x[0], w[0], i);
      if (i + 1 < n) step(x[1], w[1], i + 1);
    }
  } else { // the next tile of ranks and the next segment
    if (n > 0) {
      fetch_x(x[0], segment(0));
      fetch_w(w[0], segment(0), 0);
    }
    for (int i = 0; i < n; ++i) {
      const int seg = segment(i);
      turn_x(x[0], v, seg);
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        if (q + 1 < RT) fetch_w(w[(q + 1) & 1], seg, q + 1);
        else if (i + 1 < n) fetch_w(w[0], segment(i + 1), 0);
        if (!q && i + 1 < n) fetch_x(x[0], segment(i + 1));
        sum[q] = multiply(w[q & 1], v, seg, q, sum[q]);
      }
    }
  }
  const float factor = a.back ? a.scale[adapter] : DROP ? a.drop.scale : 1.0f;
#pragma unroll
  for (int q0 = 0; q0 < RT; q0 += GROUP) {
    __syncthreads(); // the last terms or shares have been read
#pragma unroll
    for (int q = 0; q < GROUP; ++q) *reinterpret_cast<f32x4 *>(&m.red[wave][lm][16 * q + 4 * kg]) = sum[q0 + q];
    __syncthreads();
    if (wave >= GROUP || lm >= count) continue;
    const f32x4 v = add_shares<NW, PITCH>(m.red, wave) * factor;
    const int rank = 16 * (q0 + wave) + 4 * kg;
    float *to = a.hidden + (long)row * a.rank + rank;
    if (FULL) {
      *reinterpret_cast<f32x4_unaligned *>(to) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (rank + i < a.rank) to[i] = v[i];
    }
  }
}

// UP_ROWS rows x UP_COLS columns of y.  Everything comes and goes along the rows of its matrix and through LDS: hidden, in the form
// of the matrix instructions, for all waves; B, 16 columns of the wave at a time; the products, to which base is added as they are
// stored.  Loads in the lanes' order of the products, 16 rows to every 16 lanes, take the address units four times as long.
// Bound by base and y with small ranks: 8192 rows of 2304 floats, rank 16, in 30.5 us (151 MB, 4.9 TB/s; a copy of that size 5.4).  With larger
// ones by what comes from the L2: 4096 rows of 4096 bf16, rank 64, in 24.8 us, 67 MB of base and y (2.7 TB/s), and for every 8 KB of them 16
// of B and 4 of hidden.  16 x 256 took 32.0 and 25.0 us, 32 x 128 34.5 and 27.7 us where 16 x 128 took 32.4 and 25.0.
// Halves: registers for what is rare would leave a SIMD fewer waves, where no spill comes of it (rank 64 without a bound 41.0 us, with 39.0).
constexpr int up_waves_of_rounds(int rank_tiles, bool full) { return rank_tiles == 1 ? 8 : rank_tiles == 2 ? 7 : rank_tiles == 4 ? 5 + full : 1; }
constexpr int UP_ROWS = 16, UP_COLS = 128, UP_MT = UP_ROWS / 16, UP_PITCH = UP_COLS + 4, UP_T = UP_COLS / 16 / UP_WAVES;
template <typename T, typename TW, int RT, bool FULL, bool DROP, bool SHORT> __global__ __launch_bounds__(64 * UP_WAVES, (Pipe<T, TW>::ROUNDS ? up_waves_of_rounds(RT, FULL) : 1)) void k_adapter_up(AdapterRowsArgs a) {
  using P = Pipe<T, TW>;
  constexpr int EACH = CHUNK<T>, SHARE = UP_ROWS * UP_COLS / EACH / (64 * UP_WAVES); // values of a load; loads of a thread
  constexpr int QUADS = 4 * RT, H_SHARE = (UP_ROWS * QUADS + 64 * UP_WAVES - 1) / (64 * UP_WAVES);
  constexpr int W_PITCH = 16 * RT * (int)sizeof(TW), W_LOADS = (16 * W_PITCH / 16 + 63) / 64; // bytes of a full column of B; loads of a tile of 16
  __shared__ float products[UP_ROWS][UP_PITCH];
  __shared__ typename P::V hidden_of[UP_ROWS][QUADS + 1];
  __shared__ float back_of[UP_ROWS];
  __shared__ int left_of[UP_WAVES]; // whether the wave's values leave something for another round
  constexpr bool STAGED = RT > 1 || !FULL; // the 16 columns of one full tile of ranks lie side by side anyway
  __shared__ __align__(16) char weights[STAGED ? UP_WAVES : 1][STAGED ? 16 * (W_PITCH + 16) : 16];
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6, lm = lane & 15, kg = lane >> 4;
  const auto [tile, group, piece] = place_of(a, ADAPTER_TILE_ROWS / UP_ROWS, (a.out_size + UP_COLS - 1) / UP_COLS);
  const int adapter = tile.x, count = min(tile.z - UP_ROWS * group, UP_ROWS);
  if (count <= 0) return;
  const int *order = a.plan + a.p.order + tile.y + UP_ROWS * group;
  const int col0 = piece * UP_COLS, cols = min(a.out_size - col0, UP_COLS);
  const bool some = adapter >= 0;
  // B: 16 columns of ranks lie side by side
  const int mine = col0 + 16 * UP_T * wave; // the wave's first column
  const TW *w_out = static_cast<const TW *>(a.w_out) + (some ? (long)matrix_of(a, adapter) * a.rank * a.out_size : 0);
  const long w_all = (long)a.rank * a.out_size;
  Packed16<TW> w[UP_T][W_LOADS];
  typename P::R direct[UP_T];
  if (some) {
#pragma unroll
    for (int t = 0; t < UP_T; ++t) {
      if constexpr (STAGED) {
#pragma unroll
        for (int j = 0; j < W_LOADS; ++j) w[t][j] = ahead16<SHORT>(w_out, (long)(mine + 16 * t) * a.rank + (lane + 64 * j) * CHUNK<TW>, w_all);
      } else {
        const TW *at = w_out + (long)min(mine + 16 * t + lm, a.out_size - 1) * a.rank;
        direct[t] = FULL ? P::four(at + 4 * kg) : load_ranks<P>(at, 4 * kg, a.rank);
      }
    }
  }
  // base: threads of a row are a power of two that reaches its columns
  const int per_row = (cols + EACH - 1) / EACH, shift = per_row > 1 ? 32 - __clz(per_row - 1) : 0;
  const int rows_at_once = (64 * UP_WAVES) >> shift, my_row = tid >> shift, my_col = (tid & ((1 << shift) - 1)) * EACH;
  const bool in_row = my_col < cols;
  const T *base = static_cast<const T *>(a.base.p);
  int row[SHARE], h_row[H_SHARE];
#pragma unroll
  for (int k = 0; k < SHARE; ++k) row[k] = order[min(my_row + k * rows_at_once, count - 1)];
#pragma unroll
  for (int k = 0; k < H_SHARE; ++k) h_row[k] = order[min((tid + 64 * UP_WAVES * k) / QUADS, count - 1)];
  f32x4 h[H_SHARE];
  if (some) {
#pragma unroll
    for (int k = 0; k < H_SHARE; ++k) { // zeros behind the last rank, also where a row holds an infinity
      const float *from = a.hidden + (long)h_row[k] * a.rank;
      const int rank = tid % QUADS * 4;
      h[k] = FULL ? *reinterpret_cast<const f32x4_unaligned *>(from + rank) : load_ranks<Pipe<float, float>>(from, rank, a.rank);
    }
  }
  Packed16<T> add[SHARE];
  if (base && in_row) {
#pragma unroll
    for (int k = 0; k < SHARE; ++k) add[k] = ahead16<SHORT>(base + (long)row[k] * a.base.ld, col0 + my_col, a.out_size);
  }
  if (some) {
    const float scale = a.back ? 1.0f : a.scale[adapter];
    bool left = false;
#pragma unroll
    for (int k = 0; k < H_SHARE; ++k) {
      h[k] *= scale;
      const float lift = P::lift(most_of_lanes<QUADS>(most_of(h[k])));
      const int r = (tid + 64 * UP_WAVES * k) / QUADS;
      if (r < UP_ROWS) {
        hidden_of[r][tid % QUADS] = P::split(h[k], lift);
        if (tid % QUADS == 0) back_of[r] = inverse_of(lift);
        left |= P::ROUNDS && is_left(most_of(h[k]));
      }
    }
    if (P::ROUNDS) {
      const uint64_t of_wave = __ballot(left);
      if (lane == 0) left_of[wave] = of_wave != 0;
    }
    __syncthreads();
    typename P::V hidden[UP_MT][RT];
#pragma unroll
    for (int mt = 0; mt < UP_MT; ++mt)
#pragma unroll
      for (int q = 0; q < RT; ++q) hidden[mt][q] = hidden_of[16 * mt + lm][4 * q + kg];
#pragma unroll
    for (int t = 0; t < UP_T; ++t) {
      if (mine + 16 * t >= a.out_size) break;
      typename P::R r[RT];
      if constexpr (STAGED) {
        wave_sync(); // the last columns have been read
#pragma unroll
        for (int j = 0; j < W_LOADS; ++j) { // full ranks: columns apart by 16 bytes more, for the banks
          trim16(w[t][j], (long)(mine + 16 * t) * a.rank + (lane + 64 * j) * CHUNK<TW>, w_all);
          const int at = (lane + 64 * j) * 16;
          if (at < 16 * W_PITCH) *reinterpret_cast<u32x4 *>(&weights[wave][FULL ? at + at / W_PITCH * 16 : at]) = w[t][j].q;
        }
        wave_sync();
#pragma unroll
        for (int q = 0; q < RT; ++q) {
          const TW *from = reinterpret_cast<const TW *>(&weights[wave][lm * (FULL ? W_PITCH + 16 : a.rank * (int)sizeof(TW))]);
          r[q] = FULL ? P::four_aligned(from + 16 * q + 4 * kg) : load_ranks<P>(from, 16 * q + 4 * kg, a.rank);
        }
      } else {
        r[0] = direct[t];
      }
#pragma unroll
      for (int mt = 0; mt < UP_MT; ++mt) *reinterpret_cast<f32x4 *>(&products[16 * mt + lm][16 * (UP_T * wave + t) + 4 * kg]) = P::ranks(r, hidden[mt], f32x4{});
    }
    if constexpr (P::ROUNDS) { // rare: what the first round left, on operands that are read again rather than kept
      static_assert(UP_MT == 1);
      int more = 0;
#pragma unroll
      for (int w = 0; w < UP_WAVES; ++w) more |= left_of[w];
      if (more) {
        const float *from = a.hidden + (long)order[min(lm, count - 1)] * a.rank;
        const float lift = inverse_of(back_of[lm]);
        f32x4 c[UP_T] = {};
#pragma unroll 1
        for (int rank = 4 * kg; rank < 16 * RT; rank += 16) {
          typename P::R r[UP_T];
#pragma unroll
          for (int t = 0; t < UP_T; ++t) r[t] = load_ranks<P>(w_out + (long)min(mine + 16 * t + lm, a.out_size - 1) * a.rank, rank, a.rank);
          f32x4 v = load_ranks<Pipe<float, float>>(from, rank, a.rank) * scale;
          P::split(v, lift);
          P::add_left(r, v, c);
        }
#pragma unroll
        for (int t = 0; t < UP_T; ++t) *reinterpret_cast<f32x4 *>(&products[lm][16 * (UP_T * wave + t) + 4 * kg]) += c[t] * lift;
      }
    }
    __syncthreads();
  }
  const uint32_t call = DROP ? drop_call(a.drop) : 0;
#pragma unroll
  for (int k = 0; k < SHARE; ++k) {
    const int m = my_row + k * rows_at_once;
    if (m >= count || !in_row) continue;
    float v[EACH] = {};
    if (base) trim16(add[k], col0 + my_col, a.out_size);
    if (!some) { // rows without adapter: base goes through, zeros without it
      if (base) widen16(v, add[k]);
    } else {
      const float factor = back_of[m] * (DROP ? a.drop.scale : 1.0f);
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = products[m][my_col + i] * factor;
      if (DROP) {
        const uint32_t col = (uint32_t)(col0 + my_col), kept = drop_kept(a.drop, call, (uint32_t)row[k], col / 8u) >> (col & 7u);
#pragma unroll
        for (int i = 0; i < EACH; ++i) v[i] = kept & (1u << i) ? v[i] : 0.0f;
      }
      if (base) add16(v, add[k]);
    }
    store_first(static_cast<T *>(a.out.p) + (long)row[k] * a.out.ld + col0 + my_col, v, cols - my_col);
  }
}

// Up to ADAPTER_FEW_ROWS rows by their index alone.  4096 -> 4096 bf16, and a plan (6 us) with the two kernels above: 64 rows, rank 16, of 8
// adapters 12.1 and 17.4 us, of two 21.7 and 17.9, of one 47.7 and 18.5; rank 64 29.8 and 22.2, 56.7 and 22.6, 114.6 and 24.0; 16 rows of one
// adapter 11.3 and 17.5, rank 64 24.9 and 21.3.  (Rows of an adapter go through a workgroup 16 at a time, one group after another.)  Workgroup
// (i, s) makes the columns of slice s for all rows of the adapter of row
// i, unless an earlier row has it, and the hidden that it needs for them.
template <typename T, typename TW, int RT, bool FULL, bool SHORT> __global__ __launch_bounds__(64 * WAVES) void k_adapter_few(AdapterRowsArgs a) {
  using P = Pipe<T, TW>;
  constexpr int PITCH = 16 * RT + 4;
  __shared__ float red[WAVES][16][PITCH];
  __shared__ int rows_of[ADAPTER_FEW_ROWS];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, lm = lane & 15, kg = lane >> 4;
  const int key = lane < a.rows ? adapter_key(a.index[lane], a.n) : -1, adapter = __shfl(key, (int)blockIdx.x);
  const uint64_t same = __ballot(key == adapter);
  if (same & ((1ull << blockIdx.x) - 1)) return;
  const int count = __popcll(same);
  if (wave == 0 && ((same >> lane) & 1)) rows_of[__popcll(same & ((1ull << lane) - 1))] = lane;
  __syncthreads();
  const int units = (a.out_size + 31) / 32, unit0 = a.units_each * (int)blockIdx.y, unit1 = min(unit0 + a.units_each, units); // of 32 columns
  const bool some = adapter < a.n;
  const TW *w_in = static_cast<const TW *>(a.w_in) + (some ? (long)adapter * a.rank * a.in_size : 0);
  const TW *w_out = static_cast<const TW *>(a.w_out) + (some ? (long)adapter * a.rank * a.out_size : 0);
  const float scale = some ? a.scale[adapter] : 0.0f, kept_scale = a.drop.on ? a.drop.scale : 1.0f;
  const uint32_t call = a.drop.on ? drop_call(a.drop) : 0;
  const int steps = (a.in_size + 31) / 32, whole_steps = a.in_size / 32;
  const T *base = static_cast<const T *>(a.base.p);
  for (int m0 = 0; m0 < count; m0 += 16) {
    const long row = rows_of[min(m0 + lm, count - 1)]; // rows beyond the last repeat it and are not stored
    f32x4 sum[RT] = {};
    typename P::V hidden[RT] = {};
    if (some) {
      const T *x_at = static_cast<const T *>(a.in.p) + row * a.in.ld;
      constexpr int AT_ONCE = RT == 1 ? 4 : RT == 2 ? 2 : 1; // steps whose loads are under way together
      for (int first = wave; first < steps; first += AT_ONCE * WAVES) {
        typename P::X x[AT_ONCE];
        typename P::W w[AT_ONCE][RT];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) { // beyond the last step: that one again
          const int step = min(first + u * WAVES, steps - 1), col = step * 32 + 8 * kg;
          x[u] = step < whole_steps ? load8(x_at + col) : ahead8<SHORT>(x_at, col, a.in_size);
#pragma unroll
          for (int q = 0; q < RT; ++q) w[u][q] = weight_terms<SHORT, TW, FULL>(w_in, a.in_size, 16 * q + lm, a.rank, col, step < whole_steps);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u)
          if (first + u * WAVES < steps) {
            const int col = (first + u * WAVES) * 32 + 8 * kg;
            trim8(x[u], col, a.in_size);
#pragma unroll
            for (int q = 0; q < RT; ++q) trim_terms<TW, FULL>(w[u][q], a.in_size, 16 * q + lm, a.rank, col);
            if (a.drop.on) P::keep(x[u], drop_kept(a.drop, call, (uint32_t)row, (uint32_t)((first + u * WAVES) * 4 + kg)));
#pragma unroll
            for (int q = 0; q < RT; ++q) sum[q] = P::terms(w[u][q], x[u], sum[q]);
          }
      }
      __syncthreads(); // the last group's shares have been read
#pragma unroll
      for (int q = 0; q < RT; ++q) *reinterpret_cast<f32x4 *>(&red[wave][lm][16 * q + 4 * kg]) = sum[q];
      __syncthreads();
#pragma unroll
      for (int q = 0; q < RT; ++q) sum[q] = add_shares<WAVES, PITCH>(red, q) * kept_scale;
    }
#pragma unroll
    for (int q = 0; q < RT; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) { // padding is zero also where a row holds an infinity, whose product with it is none
        const int rank = 16 * q + 4 * kg + i;
        if (a.hidden && !blockIdx.y && !wave && m0 + lm < count && rank < a.rank) a.hidden[row * a.rank + rank] = sum[q][i];
        sum[q][i] = FULL || rank < a.rank ? sum[q][i] * scale : 0.0f;
      }
    float most = 0.0f;
#pragma unroll
    for (int q = 0; q < RT; ++q) most = most_of(sum[q], most);
    most = fmaxf(most, __shfl_xor(most, 16));
    most = fmaxf(most, __shfl_xor(most, 32));
    const float lift = P::lift(most), back = inverse_of(lift);
    bool left = false;
#pragma unroll
    for (int q = 0; q < RT; ++q) {
      hidden[q] = P::split(sum[q], lift);
      left |= P::ROUNDS && is_left(most_of(sum[q]));
    }
    const bool more = P::ROUNDS && __ballot(left) != 0;
    for (int unit = unit0 + wave; unit < unit1; unit += WAVES) {
      const int col = unit * 32 + 8 * kg; // the lane's results
      Packed8<T> add = {};
      if (base) add = ahead8<SHORT>(base + row * a.base.ld, col, a.out_size);
      f32x4 acc[2] = {};
      if (some) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          typename P::R w[RT];
          // row lm of the operand is the column whose result ends up beside its neighbours
          const TW *at = w_out + (long)min(unit * 32 + (lm >> 2) * 8 + j * 4 + (lm & 3), a.out_size - 1) * a.rank;
#pragma unroll
          for (int q = 0; q < RT; ++q) w[q] = FULL ? P::four(at + 16 * q + 4 * kg) : load_ranks<P>(at, 16 * q + 4 * kg, a.rank);
          acc[j] = P::ranks(w, hidden, acc[j]);
          if constexpr (P::ROUNDS) {
            if (__builtin_expect(more, 0)) { // what the first round left, found from the shares again, not kept
              f32x4 c[1] = {};
#pragma unroll 1
              for (int q = 0; q < RT; ++q) {
                f32x4 v = add_shares<WAVES, PITCH>(red, q) * kept_scale;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = FULL || 16 * q + 4 * kg + i < a.rank ? v[i] * scale : 0.0f;
                P::split(v, lift);
                const typename P::R of_tile[1] = {load_ranks<P>(at, 16 * q + 4 * kg, a.rank)};
                P::add_left(of_tile, v, c);
              }
              acc[j] += c[0] * lift;
            }
          }
        }
      }
      if (m0 + lm >= count) continue;
      if (base) trim8(add, col, a.out_size);
      const Values8 more = widen(add);
      Values8 v;
#pragma unroll
      for (int h = 0; h < 8; ++h) v.v[h] = some ? acc[h >> 2][h & 3] * back + more.v[h] : more.v[h];
      write8(static_cast<T *>(a.out.p) + row * a.out.ld + col, v, a.out_size - col);
    }
  }
}

// tiles of 16 ranks, whether the rank fills them, and whether a matrix has rows of fewer than eight columns.  Those are rare, and take the
// kernels of eight tiles whatever the rank, so that there is one more set of kernels and not four: 4096 rows, 4096 -> 7, rank 4, in 34 us
// (bf16) and 91 (floats), where 4096 -> 8 takes 14 and 20.
template <typename F> void with_sizes(int rank, int least, F &&f) {
  const auto full = [&](auto rt) { rank == 16 * decltype(rt)::value ? f(rt, Int<1>{}, Int<0>{}) : f(rt, Int<0>{}, Int<0>{}); };
  if (least < 8) f(Int<8>{}, Int<0>{}, Int<1>{});
  else if (rank <= 16) full(Int<1>{});
  else if (rank <= 32) full(Int<2>{});
  else if (rank <= 64) full(Int<4>{});
  else full(Int<8>{});
}

} // namespace

void launch_adapter_rows(const AdapterRowsArgs &args, int dtype, int w_dtype, int cus, hipStream_t s) {
  AdapterRowsArgs a = args;
  with_adapter_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    with_sizes(a.rank, std::min(a.in_size, a.out_size), [&](auto rt, auto full, auto small) {
      constexpr int RT = decltype(rt)::value, FULL = decltype(full)::value, SHORT = decltype(small)::value;
      if (!a.plan) {
        // rows that leave CUs idle share their columns among several workgroups, each of which makes hidden for itself: 8 rows of 768
        // and 2304 columns take 6.3 us, with a workgroup to an adapter 11.3; 64 rows 7.7 and 11.9
        const int units = (a.out_size + 31) / 32, pieces = std::max(1, cus / std::max(a.rows, 1));
        a.units_each = ((units + pieces - 1) / pieces + WAVES - 1) / WAVES * WAVES;
        const dim3 grid((unsigned)a.rows, (unsigned)((units + a.units_each - 1) / a.units_each));
        hipLaunchKernelGGL((k_adapter_few<T, TW, RT, FULL, SHORT>), grid, dim3(64 * WAVES), 0, s, a);
        return;
      }
      const auto grid = [&](int rows, int cols) { // the first dimension times the threads stays below 2^32
        const uint64_t all = (uint64_t)((a.p.max_tiles + 7) / 8 * 8) * (ADAPTER_TILE_ROWS / rows) * ((a.out_size + cols - 1) / cols), x = std::min<uint64_t>(all, 1u << 20);
        return dim3((unsigned)x, (unsigned)((all + x - 1) / x));
      };
      const dim3 down = grid(16, a.out_size), up = grid(UP_ROWS, UP_COLS);
      if (a.drop.on && !a.back) hipLaunchKernelGGL((k_adapter_down<T, TW, RT, FULL, true, SHORT>), down, dim3(64 * DOWN_WAVES), 0, s, a);
      else hipLaunchKernelGGL((k_adapter_down<T, TW, RT, FULL, false, SHORT>), down, dim3(64 * DOWN_WAVES), 0, s, a);
      if (a.drop.on && a.back) hipLaunchKernelGGL((k_adapter_up<T, TW, RT, FULL, true, SHORT>), up, dim3(64 * UP_WAVES), 0, s, a);
      else hipLaunchKernelGGL((k_adapter_up<T, TW, RT, FULL, false, SHORT>), up, dim3(64 * UP_WAVES), 0, s, a);
    });
  });
}

} // namespace rpu_amd
