// Attention of new rows over a paged cache: out = sum_j w_j v_j / sum_j w_j, w_j = exp(scale q k_j - max), over the positions that a row sees.
//
// The heads of a row that share one of the cache count as rows of their own beside each other ("lines": line = token * group + head of the group),
// so that keys and values are read once for all of them.  A wave has 32 lines, one to a lane and the lane 32 further on, and goes over tiles of
// positions with a running maximum and sum: scores S^T = K Q^T and sums O^T = V^T W^T in matrix instructions of 32 x 32 results, whose
// columns are the lines -- maximum, sum and rescaling stay in the lane, and the weights are the second product's operand as the first leaves
// them: its terms may come in any order, so that values are read (transposed, from LDS) in the order that the lanes have.
//
// Matrix operands are 16-bit.  Of 16-bit rows and caches they are the numbers themselves; weights of few lines, which memory bounds, are two of them (16 bits of
// bf16, 22 of halves: the result is as near as its own rounding lets it be), of tiles of lines they are rounded to that type: half a step of it, relative to each
// weight, in a mean of values, an error 1.27 times that of the result's rounding alone (8192 tokens, 32 heads of 128 bf16: 2.10e-3 for 1.65e-3 of the norm).
// In two parts there, products take half as many again: 810 us for 576, 16384 tokens under a window of 2048, 16 heads of 64 halves 266 for 212.
// Floats go in parts: beside bf16 and floats three bf16 each, beside halves two halves, lifted by a power of two; products of parts that add up to
// less than 2^-24 of the largest are left out (two halves have 22 to 23 bits).
//
// What bounds it, and what it reaches (us; MI355X):
//   one token a sequence   memory: keys and values are read once.  64 sequences of up to 8192 positions, 8 heads of 128 bf16 (1.3 GB): 240, 5.5 TB/s;
//                          one of 131072 positions (0.5 GB): 101; a window of 1024 (0.3 GB): 55; one of 1024 positions, 12 heads of 64: 9.2, two launches.
//                          (One wave for a line, without matrix instructions: 7551, 119976, 1026, 263.)  Heads of 256, 16 sequences of 4096, 8 heads bf16
//                          (0.3 GB): 79, in tiles of lines 113; one of 1024, 4 heads: 13, in tiles 35.
//   prompts                nothing alone: of the time of 8192 tokens, 32 heads of 128 bf16, 554 to 588 us (935 to 990 TFLOP/s; a large matrix product 1320), the matrix pipes are
//                          busy for 46 %, vector instructions take 50 %, LDS 45 %.  Of 565, without the loads of keys and values it takes 476,
//                          without exponentials 541, without barriers 551.  16384 tokens under a window of 2048, 16 heads of 64 halves: 205 to 215 (600 to 630 TFLOP/s).
//   float rows             the products of parts: 3 (bf16 cache), 2 (halves), 6 (floats).  8 x 1024 tokens, 12 heads of 64, bf16 cache: 54 (239 TFLOP/s, a matrix
//                          product of floats 152), halves 44 (293).  Floats throughout: 23 sequences, 15 heads of 80 under a window of 777: 107, of which few lines 14, the join 10.
// Not kept: 64 lines to a wave (half the reads of LDS; heads of 64 211 us for 203, heads of 128 spill), eight waves to a workgroup (618 for 563), the next
// tile's scores ahead for heads of 64 (a third wave to a SIMD is worth more: 254 for 219), waves' priorities and other orders of the instructions (1 %).
#pragma once
#include "attend_tiles.h"
#include "cache.h"

#include <algorithm>
#include <type_traits>

namespace rpu_amd {
namespace attend {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
constexpr float NONE = -__builtin_inff();

// How rows of T beside a cache of TC, heads of up to 32 D32 values, are worked on.
template <typename T, typename TC, int D32, bool FEW> struct Shape {
  static constexpr bool HALF = __is_same(TC, _Float16);
  using M = std::conditional_t<__is_same(TC, float), __bf16, TC>; // of matrix operands
  static constexpr int KP = sizeof(TC) == 4 ? 3 : 1;                         // parts of keys and values
  static constexpr int QP = sizeof(T) == 2 ? 1 : HALF ? 2 : 3;               // of queries
  static constexpr int WP = sizeof(T) == 2 && FEW ? 2 : QP;                  // of weights
  static constexpr int DP = D32 <= 2 ? 64 : D32 <= 4 ? 128 : 256, CHUNKS = DP / 8; // a head in LDS, and its pieces of 16 bytes
  static constexpr int TILE = FEW || KP == 3 || (DP == 256 && QP > 1) ? 32 : 64; // positions
  // Keys and values as they are go to LDS without a register in between (DIRECT), 1 KB to a wave's load: GROUP rows.
  static constexpr bool DIRECT = !FEW && KP == 1;
  // The scores of the next tile among the weights of this one, where a third wave to a SIMD has no registers anyway (of longer heads, 4 % in time, the
  // registers are all taken, and the compiler may spill).
  static constexpr bool AHEAD = DIRECT && DP == 128;
  static constexpr int GROUP = 64 / CHUNKS;
  static_assert(GROUP <= RPU_CACHE_MIN_PAGE, "a group of rows is of one page");
  static constexpr int BLOCKS = TILE / 32, STEPS = 2 * D32;
  // Registers are short: values are under way while the scores are multiplied, keys while the weights are (KEYS_LATE: while nothing is), not both;
  // queries are read and split again for every tile, or are in LDS, once for the waves of few lines.  (No kernel may spill: this compiler has stored
  // and reloaded three registers of a spilled four.)
  static constexpr bool LATE = FEW ? DP == 256 : KP == 3 && D32 > 2, KEYS_LATE = LATE && KP == 3 && D32 == 4;
  static constexpr bool QUERIES_AGAIN = QP == 3 && DP == 256, QUERIES_LDS = FEW && DP == 256;
  static_assert(!QUERIES_LDS || QP == 1, "queries as they are");
  // Where 16 bytes of a row lie in LDS: 16 rows that read the same chunk of keys, and four neighbouring rows that read four chunks of values,
  // touch every bank once, at distances that instructions mostly have as constants.  Through registers: rows 16 (keys) and 64 (values) bytes
  // more than their length apart.  DIRECT: chunk ^ turn of the row in its group, and groups at distances of more than 1 KB.
  static constexpr int K_ROW = DP + 8, V_ROW = DP + 32;
  static constexpr int K_GROUP = 512 + (DP == 256 ? 16 : 32), V_GROUP = 512 + (DP == 256 ? 64 : 0);
  static constexpr int K_PLANE = DIRECT ? TILE / GROUP * K_GROUP : TILE * K_ROW, V_PLANE = DIRECT ? TILE / GROUP * V_GROUP : TILE * V_ROW; // of one part
  static __device__ __forceinline__ int k_turn(int row) { return DP == 64 ? (row >> 1) & 3 : row & (GROUP - 1); }
  static __device__ __forceinline__ int v_turn(int row) { return (DP == 64 ? (row >> 1) & 1 : row & (GROUP - 1)) << 2; }
  static __device__ __forceinline__ int k_at(int row, int chunk) {
    return DIRECT ? row / GROUP * K_GROUP + row % GROUP * DP + (chunk ^ k_turn(row)) * 8 : row * K_ROW + chunk * 8;
  }
  static __device__ __forceinline__ int v_at(int row, int chunk) {
    return DIRECT ? row / GROUP * V_GROUP + row % GROUP * DP + (chunk ^ v_turn(row)) * 8 : row * V_ROW + chunk * 8;
  }
  // A wave that has its tile of float parts by itself puts the values where the keys were: four waves have room beside each other.
  static constexpr bool IN_TURN = FEW && KP == 3;
  static constexpr int TILE_VALUES = KP * (IN_TURN ? (K_PLANE > V_PLANE ? K_PLANE : V_PLANE) : K_PLANE + V_PLANE);
  static constexpr int KEY_WAVES = FEW ? 4 : 1; // that share a line's positions
  static constexpr int WAVES = FEW ? KEY_WAVES : 4, LINES = FEW ? 32 : 128, LOADERS = FEW ? 64 : 256;
  static constexpr int LOADS = TILE * CHUNKS / LOADERS;
  static constexpr int STAGES = FEW || KP == 3 ? 1 : 2; // tiles that there is room for
  static constexpr int PER_SIMD = D32 <= 4 && (KP == 1 ? QP == 1 || D32 <= 2 : !FEW) ? 2 : 1; // waves, as the registers allow
  static constexpr int TILES = FEW ? KEY_WAVES : STAGES, LDS = TILES * TILE_VALUES * 2 + (QUERIES_LDS ? STEPS * 1024 : 0);
  static_assert(!FEW || TILE_VALUES * 2 >= 32 * DP * 4, "the sums of a wave fit where its tile was");
};

template <typename M> __device__ __forceinline__ floatx16 multiply(u32x4 a, u32x4 b, floatx16 c) {
  if constexpr (__is_same(M, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// two floats as PARTS of type M each (rounded, what is left goes on); the largest floats stay finite, an infinity is in the second part (not SMALL: there are
// none)
template <typename M, bool SMALL = false, int PARTS> __device__ __forceinline__ void split2(float a, float b, uint32_t (&part)[PARTS]) {
#pragma unroll
  for (int k = 0; k < PARTS; ++k) {
    if constexpr (__is_same(M, __bf16)) {
      constexpr float MOST = 0x1.fep127f;
      part[k] = PARTS == 1 || k || SMALL ? pack2(a, b, __bf16{}) : pack2(__builtin_amdgcn_fmed3f(a, -MOST, MOST), __builtin_amdgcn_fmed3f(b, -MOST, MOST), __bf16{});
      if (k + 1 < PARTS) {
        a -= __uint_as_float(part[k] << 16);
        b -= __uint_as_float(part[k] & 0xffff0000u);
      }
    } else {
      part[k] = pack2(a, b, _Float16{});
      if (k + 1 < PARTS) {
        const f16x2 r = __builtin_bit_cast(f16x2, part[k]);
        a -= (float)r.x;
        b -= (float)r.y;
      }
    }
  }
}
template <typename M> __device__ __forceinline__ float value_of(uint16_t v) { return to_float(__builtin_bit_cast(M, v)); }
// a sum and two 16-bit values
template <typename M> __device__ __forceinline__ float add2(uint32_t two, float sum) {
  if constexpr (__is_same(M, __bf16)) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, two), __builtin_bit_cast(bf16x2, 0x3f803f80u), sum, false);
  else return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, two), __builtin_bit_cast(f16x2, 0x3c003c00u), sum, false);
}
// one of two 16-bit values is infinite or NaN
template <typename M> __device__ __forceinline__ bool not_finite2(uint32_t v) {
  constexpr uint32_t FIELD = __is_same(M, __bf16) ? 0x7f807f80u : 0x7c007c00u, STEP = __is_same(M, __bf16) ? 0x00800080u : 0x04000400u;
  return ((v & FIELD) + STEP) & 0x80008000u;
}
__device__ __forceinline__ float most(float a, float b) { return __builtin_elementwise_maximum(a, b); } // NaN if one is: no quieting before it
__device__ __forceinline__ float half_and_half(float v, float &other) { // of the lanes below 32, and of the others
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  other = __uint_as_float(r[1]);
  return __uint_as_float(r[0]);
}

// the next instructions that the compiler's scheduler puts: COUNT of a kind
enum { VECTOR = 0x2, PRODUCT = 0x8, READ = 0x100 };
template <int KIND, int COUNT> __device__ __forceinline__ void order(Int<COUNT>) { __builtin_amdgcn_sched_group_barrier(KIND, COUNT, 0); }

// Lines of a sequence, some of its heads and positions: what a workgroup does.
struct Job {
  Sequence s;
  int head, line, lines, split; // head of the cache; first line, lines of the sequence
};
__device__ __forceinline__ int lines_of(const Sequence &s, int group) { return (s.end - s.begin) * group; }

// The parts of one head of a sequence beside each other: of unlike sequences every L2 cache (neighbouring workgroups run on different ones) gets
// like shares.
__device__ __forceinline__ bool job_few(const AttendArgs &a, long at, Job &job) {
  if (at >= a.few_jobs) return false;
  job.split = (int)(at % a.few_splits);
  at /= a.few_splits;
  job.head = (int)(at % a.c.heads);
  job.s = sequence_at(a.r, (int)(at / a.c.heads));
  job.line = 0;
  job.lines = lines_of(job.s, a.group);
  return job.lines > 0 && job.lines <= a.few;
}
// Tiles of LINES lines, the last of the sequences first: they see most.  Where heads (of all sequences, if these have as many rows each) divide
// by the eight L2 caches, each cache has some of them; otherwise all go in turn.  Sequences of unlike rows: attend_tiles.h.
template <int LINES> __device__ __forceinline__ bool job_many(const AttendArgs &a, long at, Job &job) {
  if (at >= a.jobs) return false;
  const int each = a.r.starts ? a.tiles : a.tiles / a.r.n, sets = a.r.starts ? a.c.heads : a.c.heads * a.r.n; // tiles of a set
  int set, tile;
  if (sets % 8 == 0) {
    const int cache = (int)(at % 8), of_cache = sets / 8;
    at /= 8;
    job.split = (int)(at % a.splits);
    at /= a.splits;
    set = cache * of_cache + (int)(at % of_cache);
    tile = (int)(at / of_cache);
  } else {
    job.split = (int)(at % a.splits);
    at /= a.splits;
    set = (int)(at % sets);
    tile = (int)(at / sets);
  }
  tile = each - 1 - tile;
  job.head = set % a.c.heads;
  int which = set / a.c.heads;
  if (a.r.starts) {
    const TileOf t = tile_of(tile, a.r.starts, a.r.rows, a.group, LINES, [&](auto &&held) { return last_of(a.r.starts, a.r.n, held); });
    if (t.which < 0) return false;
    which = t.which;
    tile = (int)t.tile;
  }
  job.s = sequence_at(a.r, which);
  job.lines = lines_of(job.s, a.group);
  if ((long)tile * LINES >= job.lines || job.lines <= a.few) return false;
  job.line = tile * LINES;
  return true;
}

template <typename T, typename TC, int D32, bool FEW> __device__ __forceinline__ void attend_job(AttendArgs a, long from_job) {
  using S = Shape<T, TC, D32, FEW>;
  using M = typename S::M;
  constexpr int TILE = S::TILE, BLOCKS = S::BLOCKS, STEPS = S::STEPS, KP = S::KP, QP = S::QP, CHUNKS = S::CHUNKS, DP = S::DP, LOADS = S::LOADS;
  extern __shared__ __attribute__((aligned(16))) uint16_t attend_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  Job job;
  if (FEW ? !job_few(a, from_job + blockIdx.x, job) : !job_many<S::LINES>(a, from_job + blockIdx.x, job)) return;
  const int group = a.group, head = a.c.head;
  // (the same in all lanes, which the compiler does not see of what comes from memory)
  job.s.begin = __builtin_amdgcn_readfirstlane(job.s.begin);
  job.s.which = __builtin_amdgcn_readfirstlane(job.s.which);
  job.s.first = (long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(job.s.first >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)job.s.first));
  job.line = __builtin_amdgcn_readfirstlane(job.line);
  job.lines = __builtin_amdgcn_readfirstlane(job.lines);

  // the line of this lane
  const int line = job.line + (FEW ? 0 : 32 * wave) + (lane & 31);
  const bool live = line < job.lines;
  const int token = live ? line / group : 0, row = job.s.begin + token, q_head = job.head * group + (live ? line % group : 0);
  const auto place = [](long p) { return (int)min(max(p, -1l), 1l << 30); };
  const int last_seen = live ? place(job.s.first + token) : -1;                                     // positions <= last_seen
  const int before = a.window ? place(job.s.first + token - a.window) : -1;                         // and > before, or < sinks
  // positions that some line of the workgroup sees, and those that all of them do
  const int token0 = job.line / group, token1 = (min(job.line + S::LINES, job.lines) - 1) / group;
  const int end = min(place(job.s.first + token1) + 1, a.r.places), low = a.window ? min(place(job.s.first + token0 - a.window) + 1, end) : 0;
  const int all_last = place(job.s.first + token0), all_before = a.window ? place(job.s.first + token1 - a.window) : -1;
  // what the lines of this wave see at most
  const int wave_line = job.line + 32 * wave, wave_last = FEW || wave_line >= job.lines ? -1 : place(job.s.first + (min(wave_line + 32, job.lines) - 1) / group);
  const int sink_end = low > 0 ? min(a.sinks, end) : 0;
  const int sink_tiles = (sink_end + TILE - 1) / TILE, first_tile = max(low / TILE, sink_tiles), tiles = sink_tiles + max((end + TILE - 1) / TILE - first_tile, 0);
  const int splits = FEW ? a.few_splits : a.splits, each = max((tiles + splits - 1) / splits, FEW ? ATTEND_FEW_LEAST : 1);
  const int from = min(job.split * each, tiles), to = min(from + each, tiles), step = S::KEY_WAVES;
  const auto base_of = [&](int t) { return (t < sink_tiles ? t : first_tile + t - sink_tiles) * TILE; };

  // queries: 8 values of each 16 to a lane
  const T *const at_q = static_cast<const T *>(a.q.p) + (live ? row * a.q.ld + q_head * head : 0l);
  const auto query_at = [&](int i) { return load8(at_q + (16 * i + 8 * half < head ? 16 * i + 8 * half : 0)); };
  const bool none = a.scale == 0.0f;
  float lift = 1.0f;
  const auto parts_of_query = [&](const Packed8<T> &p, int i, auto &&put) { // (the scale's sign goes with them)
    const bool there = live && 16 * i + 8 * half < head && !none;
    if constexpr (QP == 1) {
      u32x4 v = p.q;
      if (a.scale < 0.0f) v ^= 0x80008000u;
      put(0, there ? v : u32x4{});
    } else {
      const Values8 v = widen(p);
      const float factor = a.scale < 0.0f ? -lift : lift;
      u32x4 out[QP];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t part[QP];
        split2<M>(there ? v.v[2 * k] * factor : 0.0f, there ? v.v[2 * k + 1] * factor : 0.0f, part);
#pragma unroll
        for (int j = 0; j < QP; ++j) out[j][k] = part[j];
      }
#pragma unroll
      for (int j = 0; j < QP; ++j) put(j, out[j]);
    }
  };
  u32x4 q[QP][S::QUERIES_AGAIN || S::QUERIES_LDS ? 1 : STEPS];
  uint16_t *const q_lds = attend_lds + S::TILES * S::TILE_VALUES + lane * 8;
  if constexpr (S::QUERIES_LDS) { // the waves' lines are the same
#pragma unroll
    for (int k = 0; k < STEPS / S::WAVES; ++k) {
      const int i = wave * (STEPS / S::WAVES) + k;
      parts_of_query(query_at(i), i, [&](int, u32x4 v) { *reinterpret_cast<u32x4 *>(q_lds + i * 512) = v; });
    }
    __syncthreads();
  } else if constexpr (!S::QUERIES_AGAIN) {
    Packed8<T> p[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) p[i] = query_at(i);
    if constexpr (QP == 2) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const Values8 v = widen(p[i]);
#pragma unroll
        for (int k = 0; k < 8; ++k) m = 16 * i + 8 * half < head ? fmaxf(m, fminf(fabsf(v.v[k]), 0x1.fffffep127f)) : m;
      }
      m = fmaxf(m, __shfl_xor(m, 32));
      lift = lift_of(m);
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) parts_of_query(p[i], i, [&](int j, u32x4 v) { q[j][i] = v; });
  }
  float c = none ? LOG2E : exponent_factor(a.scale) * inverse_of(lift); // of the exponents, in powers of two
  // A lift may take it out of the numbers that floats hold whole.  Lifted scores are less than 2^40 and multiples of 2^-48: with any factor below
  // 2^-126 all weights are 1, with any beyond floats only the largest score has one.
  if constexpr (QP == 2) c = __builtin_amdgcn_fmed3f(c, 0x1p-126f, 0x1.fffffep127f);

  // Tiles: page numbers are under way two tiles ahead, keys and values one.
  const int *table = a.r.tables + job.s.which * a.r.table_ld;
  const auto inside = [&](int t) { return t < to && lane < TILE && base_of(t) + lane < end; };
  const auto entry_at = [&](int t) { return table[inside(t) ? (base_of(t) + lane) >> a.c.page_shift : 0]; }; // (looked at later: not waited for)
  const auto page_at = [&](int t, int entry) { return inside(t) && entry >= 0 && entry < a.c.pages ? entry : -1; }; // of position `lane`; -1: not there
  const auto wanted = [&](int t, int page) { // positions of a tile that are there and that some line sees
    const int j = base_of(t) + lane;
    return __ballot(page >= 0 && (j >= low || j < sink_end));
  };
  // Row `lane` of a tile, in bytes from the first of the cache.  The rows of a group are of one page: their address is the wave's, read from the
  // lane of the first, and each lane has its place from there.
  const uint32_t row_bytes = head * (uint32_t)sizeof(TC), head_bytes = row_bytes << a.c.page_shift, page_bytes = head_bytes * a.c.heads, of_head = head_bytes * job.head;
  const auto rows_at = [&](int t, int page) {
    uint64_t at = (uint64_t)(uint32_t)max(page, 0) * page_bytes + of_head + ((base_of(t) + lane) & ((1 << a.c.page_shift) - 1)) * row_bytes;
    asm volatile("" : "+v"(at)); // made here, by all lanes: not in a branch that only some take, where others' are read from
    return at;
  };
  const auto address = [&](const void *from, uint64_t at, int r) {
    if (S::DIRECT && a.c.page_shift >= __builtin_ctz(TILE)) { // of one page
      from = static_cast<const char *>(from) + r * row_bytes;
      r = 0;
    }
    const uint32_t low = __builtin_amdgcn_readlane((int)(uint32_t)at, r), high = __builtin_amdgcn_readlane((int)(uint32_t)(at >> 32), r);
    const char *p = static_cast<const char *>(from) + ((uint64_t)high << 32 | low);
    asm volatile("" : "+s"(p)); // (in scalar registers)
    return p;
  };
  // DIRECT: from global memory to LDS, 16 bytes to a lane; columns beyond a head are zeros from the start.
  const int r_lane = lane / CHUNKS;
  const int k_lane = (lane % CHUNKS) ^ S::k_turn(r_lane), v_lane = (lane % CHUNKS) ^ S::v_turn(r_lane);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t *)attend_lds;
  const auto fetch = [&](const void *from, uint64_t at, int turned, int group_bytes, uint32_t to) {
    const uint32_t off = (r_lane * head + turned * 8) * 2;
    const char *p[TILE / S::GROUP / 4];
#pragma unroll
    for (int i = 0; i < TILE / S::GROUP / 4; ++i) p[i] = address(from, at, (4 * i + wave) * S::GROUP);
    if (turned * 8 < head)
#pragma unroll
      for (int i = 0; i < TILE / S::GROUP / 4; ++i) {
        const int to_group = __builtin_amdgcn_readfirstlane(to + (4 * i + wave) * group_bytes);
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(p[i]), "s"(to_group) : "memory", "m0");
      }
  };
  const auto fetch_keys = [&](uint64_t at, int stage) { fetch(a.c.k, at, k_lane, S::K_GROUP * 2, lds_at + stage * S::K_PLANE * 2); };
  const auto fetch_values = [&](uint64_t at, int stage) { fetch(a.c.v, at, v_lane, S::V_GROUP * 2, lds_at + (S::STAGES * S::K_PLANE + stage * S::V_PLANE) * 2); };
  // what this thread fetched: zeros where there is nothing; whether some value is not finite
  const auto clean = [&](uint16_t *values, uint64_t here) {
    bool bad = false;
    int column = lane * 8, r = r_lane;
    asm volatile("" : "+v"(column), "+v"(r)); // few tiles come here: no addresses and masks kept in registers for them
#pragma unroll
    for (int i = 0; i < TILE / S::GROUP / 4; ++i) {
      const int g = 4 * i + wave;
      u32x4 *const v = reinterpret_cast<u32x4 *>(values + g * S::V_GROUP + column);
      if (!((here >> (g * S::GROUP + r)) & 1)) *v = u32x4{};
      else {
        const u32x4 w = *v;
#pragma unroll
        for (int n = 0; n < 4; ++n) bad |= not_finite2<M>(w[n]);
      }
    }
    return bad;
  };
  // Through registers otherwise, by the same groups of rows.
  Packed8<TC> k_ahead[LOADS], v_ahead[LOADS];
  const int chunk = lane % CHUNKS, first_group = FEW ? 0 : wave;
  const uint32_t lane_at = (r_lane * head + (chunk * 8 < head ? chunk * 8 : 0)) * (uint32_t)sizeof(TC);
  const auto load = [&](Packed8<TC> (&ahead)[LOADS], const void *from, uint64_t at) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) ahead[i] = load8(reinterpret_cast<const TC *>(address(from, at, (S::LOADERS / 64 * i + first_group) * S::GROUP) + lane_at));
  };
  // into LDS, zeros where there is nothing
  const auto put = [&](Packed8<TC> (&ahead)[LOADS], auto at, int plane, uint16_t *tile, uint64_t here, bool whole) {
    if (!whole) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        if (!((here >> ((S::LOADERS / 64 * i + first_group) * S::GROUP + r_lane)) & 1) || chunk * 8 >= head) ahead[i] = {};
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      uint16_t *const to = tile + at((S::LOADERS / 64 * i + first_group) * S::GROUP + r_lane, chunk);
      if constexpr (KP == 1) {
        *reinterpret_cast<u32x4 *>(to) = ahead[i].q;
      } else {
        const Values8 v = widen(ahead[i]);
        u32x4 out[KP];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          uint32_t part[KP];
          split2<M>(v.v[2 * n], v.v[2 * n + 1], part);
#pragma unroll
          for (int j = 0; j < KP; ++j) out[j][n] = part[j];
        }
#pragma unroll
        for (int j = 0; j < KP; ++j) *reinterpret_cast<u32x4 *>(to + j * plane) = out[j];
      }
    }
  };
  const auto put_keys = [&](uint16_t *keys, uint64_t here, bool whole) {
    put(k_ahead, [](int r, int chunk) { return S::k_at(r, chunk); }, S::K_PLANE, keys, here, whole);
  };
  // whether some value is not finite, looked at where it matters
  const auto put_values = [&](uint16_t *values, uint64_t here, bool whole, bool look) {
    put(v_ahead, [](int r, int chunk) { return S::v_at(r, chunk); }, S::V_PLANE, values, here, whole);
    bool bad = false;
    if (look) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        if constexpr (KP == 1) {
#pragma unroll
          for (int n = 0; n < 4; ++n) bad |= not_finite2<M>(v_ahead[i].q[n]);
        } else {
          const Values8 v = widen(v_ahead[i]);
#pragma unroll
          for (int n = 0; n < 8; ++n) bad |= !__builtin_isfinite(v.v[n]);
        }
      }
    }
    return bad;
  };
  const auto all_there = [&] {
    if constexpr (FEW) wave_sync();
    else __syncthreads();
  };

  // scores of 32 positions each: 8 (i / 4) + 4 half + i % 4
  typedef floatx16 Scores[BLOCKS];
  constexpr int PRODUCTS = KP == 3 ? 6 : QP; // of a piece of keys or values, all parts
  const auto scores_of = [&](const uint16_t *tile, Scores &score) {
    const uint16_t *keys[2]; // of even and odd steps
#pragma unroll
    for (int i = 0; i < 2; ++i) keys[i] = tile + S::k_at(lane & 31, 2 * i + half) - (S::DIRECT ? 0 : 16 * i);
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) score[n] = floatx16{};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int slot = S::QUERIES_AGAIN || S::QUERIES_LDS ? 0 : i;
      if constexpr (S::QUERIES_LDS) q[0][0] = *reinterpret_cast<const u32x4 *>(q_lds + i * 512);
      if constexpr (S::QUERIES_AGAIN) parts_of_query(query_at(i), i, [&](int j, u32x4 v) { q[j][0] = v; });
#pragma unroll
      for (int n = 0; n < BLOCKS; ++n)
#pragma unroll
        for (int j = 0; j < KP; ++j) {
          const u32x4 k = *reinterpret_cast<const u32x4 *>(S::DIRECT ? keys[i & 1] + 32 / S::GROUP * n * S::K_GROUP + i / 2 * 32
                                                                     : keys[0] + j * S::K_PLANE + 32 * n * S::K_ROW + 16 * i);
#pragma unroll
          for (int l = 0; l < QP; ++l)
            if (j + l < 3) score[n] = multiply<M>(k, q[l][slot], score[n]);
        }
    }
  };
  // bit n: this lane's line sees position n of 32; the scores of the others leave
  typedef uint32_t Seen[BLOCKS];
  const auto mask = [&](int base, uint64_t here, Scores &score, Seen &seen) {
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n) {
      const int first = base + 32 * n;
      const auto below = [](int count) { return count >= 32 ? ~0u : (1u << max(count, 0)) - 1; };
      seen[n] = (uint32_t)(here >> (32 * n)) & below(last_seen - first + 1) & (~below(before - first + 1) | below(a.sinks - first));
      const uint32_t mine = seen[n] >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; ++i) score[n][i] = mine & (1u << (8 * (i / 4) + i % 4)) ? score[n][i] : NONE;
    }
  };
  // The score that weights are relative to, what their exponents have subtracted (it as a power of two, raised), and their sum (of this lane's positions).
  // It follows the maximum where that is more than 2^SLACK away: a maximum that grows by little with every tile, as of many like scores, rescales nothing.
  // Beyond ATTEND_FAR a power of two is too coarse to be subtracted from others; the reference is NaN then (and before anything is seen) and every tile's
  // scores have the score itself subtracted.
  using R = References<T>;
  float m = NONE, reference = __builtin_nanf(""), total = 0.0f;
  floatx16 sums[D32] = {};
  const auto raise = [&](Scores &score) {
    float now = score[0][0], other;
#pragma unroll
    for (int n = 0; n < BLOCKS; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) now = most(now, score[n][i]);
    now = half_and_half(now, other);
    now = most(now, other);
    const bool up = !(now * c <= (R::SLACK == R::RAISED ? reference : reference + (R::SLACK - R::RAISED)));
    if (__any(up)) {
      now = up ? most(now, m) : m;
      const float shrink = up ? __builtin_amdgcn_exp2f(m == NONE ? NONE : weight_between<R>(m, now, c)) : 1.0f;
      total *= shrink;
#pragma unroll
      for (int n = 0; n < D32; ++n) sums[n] *= shrink;
      m = now;
      const bool far = !(fabsf(m * c) <= ATTEND_FAR);
      reference = far ? __builtin_nanf("") : m * c + R::RAISED;
      if (__any(far)) {
        const float most_seen = far && m != NONE ? m : 0.0f;
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) score[n][i] -= most_seen;
      }
    }
    return reference != reference ? R::RAISED : reference;
  };
  // rare: what is not finite goes to the lines that see it by itself, and is zero for the product
  const auto repair = [&](uint16_t *values, const Seen &seen) {
#pragma unroll 1
    for (int r = 0; r < TILE; ++r) {
      const bool mine = (seen[BLOCKS - 1 ? r >> 5 : 0] >> (r & 31)) & 1;
#pragma unroll
      for (int n = 0; n < D32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float v = 0.0f;
#pragma unroll
          for (int j = 0; j < KP; ++j) v += value_of<M>(values[j * S::V_PLANE + S::v_at(r, 4 * n + i / 4) + 4 * half + i % 4]);
          if (mine && !__builtin_isfinite(v)) sums[n][i] += v;
        }
    }
    all_there();
    for (int i = FEW ? lane : tid; i < KP * S::V_PLANE / 2; i += S::LOADERS) { // (what lies between rows is never used)
      uint32_t *const two = reinterpret_cast<uint32_t *>(values) + i;
      const uint32_t v = *two;
      if (not_finite2<M>(v)) *two = (not_finite2<M>(v & 0xffffu) ? 0u : v & 0xffffu) | (not_finite2<M>(v & 0xffff0000u) ? 0u : v & 0xffff0000u);
    }
    all_there();
  };
  // Weights of 16 positions each (4 half + 8 (e / 4) + e % 4), and their products with four positions of 16 columns to 16 lanes.
  // Of floats they come from exponents near 0, which have more bits, and are lifted by a product; their `total` is of the weights before it.
  constexpr float LIFT = S::HALF ? 0x1p7f : 0x1p-8f;
  const auto add = [&](uint16_t *values, const Scores &score, float less) {
    constexpr int COLUMNS = S::DIRECT ? (DP == 64 ? 2 : 4) : 1;
    uint16_t *columns[COLUMNS];
#pragma unroll
    for (int n = 0; n < COLUMNS; ++n) columns[n] = values + S::v_at(4 * half + ((lane & 15) >> 2), 4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (lane & 1) * 4;
#pragma unroll
    for (int b = 0; b < 2 * BLOCKS; ++b) {
      u32x4 weights[S::WP];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const int at = 8 * (b & 1) + i;
        float w0 = __builtin_amdgcn_exp2f(fmaf(score[b / 2][at], c, -less)), w1 = __builtin_amdgcn_exp2f(fmaf(score[b / 2][at + 1], c, -less));
        if constexpr (S::WP > 1) total += w0 + w1;
        if constexpr (QP > 1) {
          w0 *= LIFT;
          w1 *= LIFT;
        }
        uint32_t part[S::WP];
        split2<M, true>(w0, w1, part);
        if constexpr (S::WP == 1) total = add2<M>(part[0], total); // of the rounded ones: those that the values are multiplied with
#pragma unroll
        for (int l = 0; l < S::WP; ++l) weights[l][i / 2] = part[l];
      }
#pragma unroll
      for (int n = 0; n < D32; ++n)
#pragma unroll
        for (int j = 0; j < KP; ++j) {
          s16x4 v[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint16_t *p = S::DIRECT ? columns[n % COLUMNS] + (16 * b + 8 * e) / S::GROUP * S::V_GROUP + n / 4 * 128
                                    : columns[0] + j * S::V_PLANE + (16 * b + 8 * e) * S::V_ROW + 32 * n;
            v[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p);
          }
          const u32x2 v0 = __builtin_bit_cast(u32x2, v[0]), v1 = __builtin_bit_cast(u32x2, v[1]);
          const u32x4 both = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
          for (int l = 0; l < S::WP; ++l)
            if (j + l < 3) sums[n] = multiply<M>(both, weights[l], sums[n]);
        }
    }
  };
  const auto zero_columns = [&] { // of DIRECT, beyond a head
    if (head == DP) return;
    for (int i = tid * 8; i < S::TILES * S::TILE_VALUES; i += S::WAVES * 64 * 8) *reinterpret_cast<u32x4 *>(attend_lds + i) = u32x4{};
    __syncthreads();
  };
  constexpr uint64_t ALL = TILE == 64 ? ~0ull : (1ull << TILE % 64) - 1;
  const auto is_masked = [&](int base, uint64_t here) { // some line does not see some position
    return here != ALL || base + TILE - 1 > all_last || (a.window && base <= all_before && base + TILE > a.sinks);
  };
  // what is not finite and not seen by all lines must not meet their weights of zero
  const auto everybody = [&](bool masked, bool bad) {
    if (!masked) {
      all_there();
      return false;
    }
    if constexpr (FEW) {
      bad = __any(bad);
      wave_sync();
      return bad;
    } else {
      return __syncthreads_or(bad) != 0;
    }
  };

  if constexpr (S::AHEAD) {
    // The scores of the next tile are multiplied among the weights of this one: keys are fetched two tiles ahead, values one.
    uint16_t *const all_keys = attend_lds, *const all_values = attend_lds + S::STAGES * S::K_PLANE;
    if (from < to) {
      zero_columns();
      const int entry0 = entry_at(from), entry1 = entry_at(from + 1);
      int entry = entry_at(from + 2), page = page_at(from, entry0);
      uint64_t here = wanted(from, page), at = rows_at(from, page);
      fetch_keys(at, 0);
      fetch_values(at, 0);
      page = page_at(from + 1, entry1);
      uint64_t next_here = wanted(from + 1, page);
      at = rows_at(from + 1, page);
      if (from + 1 < to) fetch_keys(at, 1);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      Scores even, odd;
      scores_of(all_keys, even);
      // one tile, whose scores are in `now`; those of the next come into `then` (of the last one there is nothing that needs them)
      const auto one = [&](int t, auto parity, Scores &now, Scores &then) {
        constexpr int turn = decltype(parity)::value;
        const int base = base_of(t);
        uint16_t *const values = all_values + turn * S::V_PLANE;
        const bool masked = is_masked(base, here);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const bool bad = everybody(masked, masked && clean(values, here));
        const uint64_t here_now = here;
        if (t + 1 < to) {
          fetch_values(at, turn ^ 1);
          here = next_here;
          const int page = page_at(t + 2, entry);
          next_here = wanted(t + 2, page);
          at = rows_at(t + 2, page);
          if (t + 2 < to) fetch_keys(at, turn);
          entry = entry_at(t + 3);
        }
        if (!bad && base > wave_last) return; // (the first lines of a workgroup do not see its last positions)
        Seen seen = {};
        if (masked) mask(base, here_now, now, seen);
        const float less = raise(now);
        if (bad) repair(values, seen);
        scores_of(all_keys + (turn ^ 1) * S::K_PLANE, then);
        add(values, now, less);
        order<READ>(Int<4>{});
#pragma unroll
        for (int i = 0; i < STEPS * BLOCKS; ++i) {
          order<PRODUCT>(Int<PRODUCTS>{});
          order<VECTOR>(Int<(112 * BLOCKS / 2) / (STEPS * BLOCKS)>{});
          order<READ>(Int<1>{});
        }
#pragma unroll
        for (int i = 0; i < 2 * BLOCKS * D32; ++i) {
          order<READ>(Int<2>{});
          order<PRODUCT>(Int<PRODUCTS>{});
        }
      };
      for (int t = from; t < to; t += 2) {
        one(t, Int<0>{}, even, odd);
        if (t + 1 < to) one(t + 1, Int<1>{}, odd, even);
      }
    }
  } else {
    int t = from + (FEW ? wave : 0), next_entry = 0;
    uint64_t there = 0, at_now = 0;
    if (t < to) {
      const int entry = entry_at(t);
      next_entry = entry_at(t + step);
      const int page = page_at(t, entry);
      there = wanted(t, page);
      at_now = rows_at(t, page);
      if constexpr (S::DIRECT) {
        zero_columns();
        fetch_keys(at_now, 0);
        fetch_values(at_now, 0);
      } else {
        if constexpr (!S::KEYS_LATE) load(k_ahead, a.c.k, at_now);
        if constexpr (!S::LATE) load(v_ahead, a.c.v, at_now);
      }
    }
    for (int turn = 0; t < to; t += step, turn ^= 1) {
      const int stage = FEW ? wave : S::STAGES == 2 ? turn : 0;
      uint16_t *const keys = attend_lds + stage * (S::IN_TURN ? S::TILE_VALUES : KP * S::K_PLANE);
      uint16_t *const values = S::IN_TURN ? keys : attend_lds + S::TILES * KP * S::K_PLANE + stage * KP * S::V_PLANE;
      const int base = base_of(t);
      const uint64_t here = there;
      const bool masked = is_masked(base, here), whole = here == ALL && head == DP, more = t + step < to;
      if (S::STAGES == 1 && !S::LATE) all_there(); // the tile before has been read (LATE: its keys before its values were put)
      uint64_t at = 0;
      if (more) {
        const int page = page_at(t + step, next_entry);
        there = wanted(t + step, page);
        at = rows_at(t + step, page);
        next_entry = entry_at(t + 2 * step);
      }
      bool bad = false;
      Scores score;
      if constexpr (S::IN_TURN) {
        put_keys(keys, here, whole);
        all_there();
        if (more) load(k_ahead, a.c.k, at);
        scores_of(keys, score);
        all_there();
        bad = everybody(masked, put_values(values, here, whole, masked));
        if (more) load(v_ahead, a.c.v, at);
      } else if constexpr (S::LATE) {
        if constexpr (S::KEYS_LATE) load(k_ahead, a.c.k, at_now);
        put_keys(keys, here, whole);
        all_there();
        load(v_ahead, a.c.v, at_now);
        if (FEW || base <= wave_last) scores_of(keys, score);
        bad = everybody(masked, put_values(values, here, whole, masked));
        if (!S::KEYS_LATE && more) load(k_ahead, a.c.k, at);
        at_now = at;
      } else {
        if constexpr (S::DIRECT) {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
          bad = masked && clean(values, here);
        } else {
          put_keys(keys, here, whole);
          bad = put_values(values, here, whole, masked);
        }
        bad = everybody(masked, bad);
        if (more) {
          at_now = at;
          if constexpr (S::DIRECT) {
            fetch_keys(at, turn ^ 1);
            fetch_values(at, turn ^ 1);
          } else {
            load(k_ahead, a.c.k, at);
            load(v_ahead, a.c.v, at);
          }
        }
      }
      if (!FEW && !bad && base > wave_last) continue; // (the first lines of a workgroup do not see its last positions)
      if constexpr (!S::IN_TURN && !S::LATE) scores_of(keys, score);
      // reads of LDS stay ahead of the products
      order<READ>(Int<4 * KP>{});
#pragma unroll
      for (int i = 0; i < STEPS * BLOCKS - 4; ++i) {
        order<PRODUCT>(Int<PRODUCTS>{});
        order<READ>(Int<KP>{});
      }
      order<PRODUCT>(Int<4 * PRODUCTS>{});
      Seen seen = {};
      if (masked) mask(base, here, score, seen);
      const float less = raise(score);
      if (bad) repair(values, seen);
      add(values, score, less);
    }
  }
  {
    float other;
    const float mine = half_and_half(total, other);
    total = mine + other;
  }
  if constexpr (QP > 1) total *= LIFT;
  if constexpr (!FEW) {
    if (!live) return;
    const long unit = (long)row * (a.c.heads * group) + q_head;
    if (a.splits > 1) {
      const long part = (long)job.split * a.r.rows * (a.c.heads * group) + unit;
      if (!half) a.stats[part] = float2{m * inverse_of(lift), total};
#pragma unroll
      for (int n = 0; n < D32; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 32 * n + 8 * i + 4 * half;
          if (d < head) *reinterpret_cast<f32x4 *>(a.part + part * head + d) = f32x4{sums[n][4 * i], sums[n][4 * i + 1], sums[n][4 * i + 2], sums[n][4 * i + 3]};
        }
      return;
    }
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    T *out = static_cast<T *>(a.out.p) + row * a.out.ld + q_head * head;
#pragma unroll
    for (int n = 0; n < D32; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * n + 8 * i + 4 * half;
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = total == 0.0f ? 0.0f : sums[n][4 * i + k] * inverse;
        if (d < head) store_first(out + d, v, 4);
      }
  } else {
    // the waves' parts meet in LDS, each where its tile was
    __shared__ float2 stats[S::KEY_WAVES][32];
    __shared__ float2 joined[32];
    if (!half) stats[wave][lane & 31] = float2{m, total};
    __syncthreads();
    float top = NONE, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < S::KEY_WAVES; ++w) top = most(top, stats[w][lane & 31].x);
    const auto shrink_of = [&](float of) { return of == NONE ? 0.0f : __builtin_amdgcn_exp2f(weight_between<R>(of, top, c)); };
#pragma unroll
    for (int w = 0; w < S::KEY_WAVES; ++w) sum = fmaf(stats[w][lane & 31].y, shrink_of(stats[w][lane & 31].x), sum);
    if (wave == 0 && !half) joined[lane & 31] = float2{top * inverse_of(lift), sum};
    const float shrink = shrink_of(m);
    float *const mine = reinterpret_cast<float *>(attend_lds + wave * S::TILE_VALUES) + (lane & 31) * DP;
    if (live)
#pragma unroll
      for (int n = 0; n < D32; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int piece = 8 * n + 2 * i + half; // of four values
          *reinterpret_cast<f32x4 *>(mine + (piece ^ (lane & (DP / 4 - 1) & 31)) * 4) =
              f32x4{sums[n][4 * i], sums[n][4 * i + 1], sums[n][4 * i + 2], sums[n][4 * i + 3]} * shrink;
        }
    __syncthreads();
    const int pieces = head / 4, count = job.lines * pieces;
    for (int i = tid; i < count; i += S::WAVES * 64) {
      const int l = i / pieces, piece = i % pieces;
      f32x4 v = {};
#pragma unroll
      for (int w = 0; w < S::KEY_WAVES; ++w)
        v += *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(attend_lds + w * S::TILE_VALUES) + l * DP + (piece ^ (l & (DP / 4 - 1) & 31)) * 4);
      const float2 both = joined[l];
      if (a.few_splits > 1) {
        const long part = (((long)job.split * a.r.n + job.s.which) * a.c.heads + job.head) * a.few + l;
        *reinterpret_cast<f32x4 *>(a.few_part + part * head + piece * 4) = v;
        if (piece == 0) a.few_stats[part] = both;
      } else {
        const float inverse = both.y == 0.0f ? 0.0f : 1.0f / both.y;
        float r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = both.y == 0.0f ? 0.0f : v[k] * inverse;
        store_first(static_cast<T *>(a.out.p) + (job.s.begin + l / group) * a.out.ld + (job.head * group + l % group) * head + piece * 4, r, 4);
      }
    }
  }
}

template <typename T, typename TC, int D32, bool FEW>
__global__ __launch_bounds__(256, (Shape<T, TC, D32, FEW>::PER_SIMD)) void k_attend(AttendArgs a, long from) {
  attend_job<T, TC, D32, FEW>(a, from);
}
// Sequences of many and of few lines in one launch, where both take as many waves to a SIMD: tiles, which take longest, first.  (bf16; 64 sequences of up
// to 40 and 16040 tokens, 8 heads of 128: 434 us, in two launches 546 (414 since); 16 of up to 100 and 600, 2 heads of 64: 17 and 23.)
template <typename T, typename TC, int D32>
__global__ __launch_bounds__(256, (Shape<T, TC, D32, false>::PER_SIMD)) void k_attend_mixed(AttendArgs a, long from) {
  if (from + blockIdx.x < a.jobs) attend_job<T, TC, D32, false>(a, from);
  else attend_job<T, TC, D32, true>(a, from - a.jobs);
}

template <typename T, typename TC> void launch(const AttendArgs &a, hipStream_t s) {
  const auto go = [&](auto kernel, long jobs, int lds) {
    for (long from = 0; from < jobs; from += MOST_GROUPS) hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(MOST_GROUPS, jobs - from)), dim3(256), lds, s, a, from);
  };
  const auto with = [&](auto d32) {
    constexpr int D32 = decltype(d32)::value;
    using Many = Shape<T, TC, D32, false>;
    static_assert(Many::WAVES == 4);
    if constexpr (D32 <= 4 || sizeof(T) == 2) { // (longer heads of floats have no few lines)
      using Few = Shape<T, TC, D32, true>;
      static_assert(Few::WAVES == 4);
      if constexpr (D32 <= 4 && Many::PER_SIMD == Few::PER_SIMD) { // (longer heads spill)
        if (a.jobs && a.few_jobs) return go(k_attend_mixed<T, TC, D32>, a.jobs + a.few_jobs, std::max(Many::LDS, Few::LDS));
      }
      go(k_attend<T, TC, D32, true>, a.few_jobs, Few::LDS);
    }
    go(k_attend<T, TC, D32, false>, a.jobs, Many::LDS);
  };
  if (a.c.head <= 64) with(Int<2>{});
  else if (a.c.head <= 96) with(Int<3>{});
  else if (a.c.head <= 128) with(Int<4>{});
  else with(Int<8>{});
}

} // namespace attend
} // namespace rpu_amd
