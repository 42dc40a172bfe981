// Low-rank adapters of many requests beside one projection: every row takes the adapter that its index names.
//   forward    hidden_t = A x_t,        y_t  = base_t + s B hidden_t
//   backward   up_t = s B^T d_t,        dx_t = base_t + A^T up_t,   dA = sum_t up_t x_t^T,   dB = s sum_t d_t hidden_t^T
// x goes through dropout first where that is on; its mask is drawn again in all three places.
//
//   k_adapter_plan   groups the rows by adapter (a stable counting sort) and cuts the groups into tiles and chunks
//   k_adapter_turn   for the backward pass: the matrices with ranks and columns exchanged, so that it is the forward pass
//   k_adapter_grads  sums over the rows of a chunk, for 128 columns of dA or dB
//   k_adapter_join   adds the chunks of an adapter in their order, zeros for adapters without rows
#include "digital.h"

#include <algorithm>

namespace rpu_amd {
namespace {

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;

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
// LDS.  A chain of latencies in one workgroup: 6 us for 256 rows, 9 for 8192, 75 for 100000, for which the other kernel takes 206.
constexpr int PLAN_LDS_ROWS = 131072, PLAN_LDS_KEYS = 256;
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
    count[1] = (count[0] + ADAPTER_TILE_ROWS - 1) / ADAPTER_TILE_ROWS;
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
    reinterpret_cast<int4 *>(plan + p.tiles)[i] = plan_piece(i, firsts[1], firsts[0], nullptr, keys, p.n, ADAPTER_TILE_ROWS);
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
    count[0] += pieces(k, ADAPTER_TILE_ROWS);
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
    reinterpret_cast<int4 *>(plan + p.tiles)[i] = plan_piece(i, tile_first, seg, nullptr, keys, p.n, ADAPTER_TILE_ROWS);
  for (int i = tid; i < p.max_chunks; i += PLAN_THREADS)
    reinterpret_cast<int4 *>(plan + p.chunks)[i] = plan_piece(i, first, seg, slot_first, p.n, p.n, p.chunk_rows);
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
    const int turned = a.listed ? a.plan[a.p.first + adapter] : adapter;
    for (int k = (int)blockIdx.x; k < (a_tiles + b_tiles) * rank_tiles; k += (int)gridDim.x) {
      const int c = k / rank_tiles, r0 = k % rank_tiles * 64;
      const bool of_a = c < a_tiles;
      // a: [rank][in] -> [in][rank], b: [out][rank] -> [rank][out]
      const int rows = of_a ? a.rank : a.out_size, cols = of_a ? a.in_size : a.rank;
      const int row0 = of_a ? r0 : (c - a_tiles) * 64, col0 = of_a ? c * 64 : r0;
      const long size = (long)rows * cols;
      const TW *from = static_cast<const TW *>(of_a ? a.a : a.b) + adapter * size;
      TW *to = static_cast<TW *>(of_a ? a.a_turned : a.b_turned) + turned * size;
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
// % 16 reads eight columns of four rows, 16 bytes beside those of its neighbours at a time, and product j of a row takes its column j.
// Rows of float: products on the fp32 instructions, bound by the reads of x and d up to rank 16 (8192 rows of 768 and 2304 columns in 25.1
// us, 101 MB, 4.0 TB/s; one group at a time, each waited for, 35 us).  Beyond, by too few waves: with rank 64 160 us, in which the matrix pipes
// are busy for 13 %; 256 registers leave less than one wave to a SIMD, and it waits for 45 % of its time, for loads and, at the end, for the
// waves before it to add 128 sums each in LDS.  A backward pass of those rows takes 79 us with rank 16, 256 with 64, 458 with 128.  16-bit
// rows: their numbers as they are on the 16-bit instructions, the factors in parts.  The same backward pass in bf16 takes 48 us with rank 16,
// 103 with 64, 188 with 128; on the fp32 instructions 53.8, 193 and 348; in f16 51, 114 and 205.
template <typename T, typename TW, int RT, bool SHORT> __global__ __launch_bounds__(64 * GRAD_WAVES, RT == 1 ? 3 : sizeof(T) == 2 ? 2 : 1) void k_adapter_grads(AdapterGradArgs a) {
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
  constexpr int EACH = CHUNK<T>, PIECES = 8 / EACH, STEP = 16 * EACH; // columns of a load, loads of a row, columns of a load of 16 lanes
  const int col = c0 + EACH * lm, rank0 = 16 * RT * (int)blockIdx.z;
  f32x4 acc[8][RT] = {};
  // the next group is under way, and the rows of the one after it
  constexpr bool NARROW = sizeof(T) == 2;
  constexpr int OWN = NARROW ? 8 : 4, GROUP = 4 * OWN; // rows of a lane, of a group
  struct Group {
    Packed16<T> x[OWN][PIECES];
    float u[OWN][RT];
  };
  const auto find = [&](int (&row)[OWN], int g) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) row[i] = order[min(GROUP * g + OWN * kg + i, count - 1)]; // rows beyond the last repeat it
  };
  const auto fetch = [&](Group &next, const int (&row)[OWN]) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
#pragma unroll
      for (int h = 0; h < PIECES; ++h) next.x[i][h] = ahead16<SHORT>(static_cast<const T *>(m.p) + (long)row[i] * m.ld, col + STEP * h, width);
#pragma unroll
      for (int q = 0; q < RT; ++q) next.u[i][q] = factor[(long)row[i] * a.rank + min(rank0 + 16 * q + lm, a.rank - 1)];
    }
  };
  // 16-bit rows: 32 terms to a product, the lane's 8 rows x 8 columns turned in its registers; the factors in three parts of the rows'
  // type, halves in as many rounds as they take
  const auto multiply_narrow = [&](Group &here, const int (&row)[OWN], int g) {
    u32x4 v[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
#pragma unroll
      for (int h = i; h < i + 2; ++h) {
        trim16(here.x[h][0], col, width);
        uint32_t kept = drop ? drop_kept(a.drop, call, (uint32_t)row[h], (uint32_t)col / 8u) : 0xffu;
        kept = GROUP * g + OWN * kg + h < count ? kept : 0u;
#pragma unroll
        for (int w = 0; w < 4; ++w) here.x[h][0].q[w] &= (kept & (1u << 2 * w) ? 0xffffu : 0u) | (kept & (2u << 2 * w) ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t x0 = here.x[i][0].q[j / 2], x1 = here.x[i + 1][0].q[j / 2];
        v[j][i / 2] = j & 1 ? x0 >> 16 | (x1 & 0xffff0000u) : (x0 & 0xffffu) | x1 << 16;
      }
    }
    const float factors = drop ? a.drop.scale : scale;
#pragma unroll
    for (int q = 0; q < RT; ++q) {
      float u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = GROUP * g + OWN * kg + i < count && rank0 + 16 * q + lm < a.rank ? here.u[i][q] * factors : 0.0f;
      u32x4 part[3];
      if constexpr (__is_same(T, __bf16)) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t p[3];
          parts_of(u[2 * w], u[2 * w + 1], p);
#pragma unroll
          for (int k = 0; k < 3; ++k) part[k][w] = p[k];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int k = 0; k < 3; ++k) acc[j][q] = multiply32<T>(v[j], part[k], acc[j][q]);
      } else {
        for (int round = 0; round < HALF_ROUNDS; ++round) {
          float most = 0.0f; // of the rank's factors in this group
#pragma unroll
          for (int i = 0; i < 8; i += 4) most = most_of(f32x4{u[i], u[i + 1], u[i + 2], u[i + 3]}, most);
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          if (round && !__ballot(is_left(most))) break;
          const float lift = lift_of(most), back = inverse_of(lift);
          bool left = false;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t p[3];
            float u0 = u[2 * w] * lift, u1 = u[2 * w + 1] * lift;
            halves_of(u0, u1, p);
            u[2 * w] = u0 * back;
            u[2 * w + 1] = u1 * back;
            left |= u0 != 0.0f || u1 != 0.0f;
#pragma unroll
            for (int k = 0; k < 3; ++k) part[k][w] = p[k];
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const f32x4 sum = multiply32<T>(v[j], part[1], multiply32<T>(v[j], part[0], f32x4{})), third = multiply32<T>(v[j], part[2], f32x4{});
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][q][i] = fmaf(fmaf(third[i], HALF_THIRD, sum[i]), back, acc[j][q][i]);
          }
          if (!__ballot(left)) break;
        }
      }
    }
  };
  const auto multiply = [&](Group &here, const int (&row)[OWN], int g) {
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const bool valid = GROUP * g + OWN * kg + i < count;
      Values8 x;
#pragma unroll
      for (int h = 0; h < PIECES; ++h) {
        trim16(here.x[i][h], col + STEP * h, width);
        float v[EACH];
        widen16(v, here.x[i][h]);
#pragma unroll
        for (int j = 0; j < EACH; ++j) x.v[EACH * h + j] = v[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x.v[j] = valid ? x.v[j] : 0.0f; // whatever the row that stands in for it holds
      if (drop) {
        uint32_t kept;
        if constexpr (PIECES == 1) {
          kept = drop_kept(a.drop, call, (uint32_t)row[i], (uint32_t)col / 8u);
        } else { // two neighbours hold half of two blocks each: each draws one
          const uint32_t mine = drop_kept(a.drop, call, (uint32_t)row[i], (uint32_t)(col + STEP * (lm & 1)) / 8u), other = (uint32_t)__shfl_xor((int)mine, 1);
          const uint32_t low = lm & 1 ? other : mine, high = lm & 1 ? mine : other, shift = col & 4;
          kept = (low >> shift & 15u) | (high >> shift & 15u) << 4;
        }
        drop_apply(a.drop, kept, x);
      }
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        const float u = valid && rank0 + 16 * q + lm < a.rank ? here.u[i][q] * scale : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[j], u, acc[j][q], 0, 0, 0);
      }
    }
  };
  const int groups = (count + GROUP - 1) / GROUP;
  if constexpr (NARROW) { // twice the rows to a group: the next one's would leave the registers
    int row[OWN];
    if (wave < groups) find(row, wave);
    for (int g = wave; g < groups; g += GRAD_WAVES) {
      Group here;
      fetch(here, row);
      int last[OWN];
#pragma unroll
      for (int i = 0; i < OWN; ++i) last[i] = row[i];
      if (g + GRAD_WAVES < groups) find(row, g + GRAD_WAVES);
      multiply_narrow(here, last, g);
    }
  } else {
    int rows[2][OWN], last[OWN];
    Group group[2];
    if (wave < groups) {
      find(rows[0], wave);
      fetch(group[0], rows[0]);
      find(rows[1], wave + GRAD_WAVES);
    }
    const auto step = [&](Group &here, Group &next, int (&row)[OWN], int (&ahead)[OWN], int g) {
      if (g + GRAD_WAVES < groups) fetch(next, ahead);
#pragma unroll
      for (int i = 0; i < OWN; ++i) last[i] = row[i];
      if (g + 2 * GRAD_WAVES < groups) find(row, g + 2 * GRAD_WAVES);
      multiply(here, last, g);
    };
    for (int g = wave; g < groups; g += 2 * GRAD_WAVES) {
      step(group[0], group[1], rows[0], rows[1], g);
      if (g + GRAD_WAVES < groups) step(group[1], group[0], rows[1], rows[0], g + GRAD_WAVES);
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
#pragma unroll
      for (int h = 0; h < PIECES; ++h) {
        const int c = c0 + STEP * h + EACH * (4 * kg + i);
        if (of_a) {
          const long at = (long)rank * a.in_size + c;
          float v[EACH];
#pragma unroll
          for (int j = 0; j < EACH; ++j) v[j] = acc[EACH * h + j][q][i];
          if (whole) store_first(static_cast<TW *>(a.da) + (long)adapter * a.rank * a.in_size + at, v, width - c);
          else store_first(part + at, v, width - c);
        } else {
#pragma unroll
          for (int j = 0; j < EACH; ++j) {
            if (c + j >= width) continue;
            const long at = (long)(c + j) * a.rank + rank;
            const float v = acc[EACH * h + j][q][i];
            if (whole) static_cast<TW *>(a.db)[(long)adapter * a.rank * a.out_size + at] = (TW)v;
            else part[at] = v;
          }
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

template <typename F> void with_rank_tiles(int rank, F &&f) {
  if (rank <= 16) f(Int<1>{});
  else if (rank <= 32) f(Int<2>{});
  else if (rank <= 64) f(Int<4>{});
  else f(Int<8>{});
}

} // namespace

void launch_adapter_turn(const AdapterTurnArgs &a, int w_dtype, int cus, hipStream_t s) {
  const int tiles = ((a.in_size + 63) / 64 + (a.out_size + 63) / 64) * ((a.rank + 63) / 64);
  // workgroups that wait for their loads, so many to a CU: 500 adapters of 4096 -> 4096, rank 16, 94 us; 8 workgroups to a CU 114
  const dim3 grid((unsigned)std::min(tiles, std::max(1, cus * 64 / std::min(a.n, cus * 8))), (unsigned)std::min(a.n, cus * 8));
  if (w_dtype == RPU_F32) hipLaunchKernelGGL(k_adapter_turn<float>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(k_adapter_turn<uint16_t>, grid, dim3(256), 0, s, a);
}

AdapterPlan adapter_plan(int rows, int n) {
  AdapterPlan p{};
  p.rows = rows;
  p.n = n;
  // A group of rows for every wave of the gradients' workgroups at least (128 rows; with 64 the backward pass of 1024 bf16 rows, rank 64, takes
  // 44.8 us instead of 38.0, of 512 rows of floats 29.7 and 27.8), and few enough chunks that their sums stay the lesser traffic.
  p.chunk_rows = 128;
  while (p.chunk_rows < 1024 && rows / p.chunk_rows > 32) p.chunk_rows *= 2;
  // every group of rows but for one may end with a piece that is not full
  p.max_tiles = (int)std::min<long>(rows, ((long)rows + ADAPTER_TILE_ROWS - 1) / ADAPTER_TILE_ROWS + std::min(n, rows));
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
  with_adapter_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    if (a.rows && std::min(a.in_size, a.out_size) < 8)
      hipLaunchKernelGGL((k_adapter_grads<T, TW, 1, true>), dim3((unsigned)a.p.max_chunks, slices, (unsigned)(a.rank + 15) / 16), dim3(64 * GRAD_WAVES), 0, s, a);
    else if (a.rows)
      with_rank_tiles(a.rank, [&](auto rt) {
        constexpr int RT = decltype(rt)::value, MOST = sizeof(T) == 2 ? 2 : 4, AT_ONCE = RT < MOST ? RT : MOST; // more sums, or rows under way, leave the registers
        hipLaunchKernelGGL((k_adapter_grads<T, TW, AT_ONCE, false>), dim3((unsigned)a.p.max_chunks, slices, RT / AT_ONCE), dim3(64 * GRAD_WAVES), 0, s, a);
      });
    hipLaunchKernelGGL(k_adapter_join<TW>, join, dim3(256), 0, s, a);
  });
}

} // namespace rpu_amd
