// Low-rank adapters of many requests beside one projection: every row takes the adapter that its index names.
//   forward    hidden_t = A x_t,        y_t  = base_t + s B hidden_t
//   backward   up_t = s B^T d_t,        dx_t = base_t + A^T up_t,   dA = sum_t up_t x_t^T,   dB = s sum_t d_t hidden_t^T
// x goes through dropout first where that is on; its mask is drawn again in all three places.
//
//   k_adapter_plan   groups the rows by adapter (a stable counting sort) and cuts the groups into tiles and chunks
//   k_adapter_rows   a tile of rows through both thin products, hidden and up never leave the workgroup in between
//   k_adapter_grads  sums over the rows of a chunk, for 128 columns of dA or dB
//   k_adapter_join   adds the chunks of an adapter in their order, zeros for adapters without rows
#include "digital.h"

#include <algorithm>

namespace rpu_amd {
namespace {

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;

__device__ __forceinline__ int adapter_key(int index, int n) { return index >= 0 && index < n ? index : n; }
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
// lanes whose digit is this lane's (lanes with `valid` only)
__device__ __forceinline__ uint64_t same_digit(int digit, bool valid) {
  uint64_t mask = __ballot(valid);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const bool bit = (digit >> b) & 1;
    const uint64_t with = __ballot(valid && bit);
    mask &= bit ? with : ~with;
  }
  return mask;
}

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
    for (int i = tid; i < PLAN_WAVES * 256; i += PLAN_THREADS) hist[i >> 8][i & 255] = 0;
    __syncthreads();
    for (int from = begin; from < end; from += 64) {
      const bool valid = from + lane < end;
      const int row = valid ? (pass ? other[from + lane] : from + lane) : 0;
      const int digit = (adapter_key(index[row], p.n) >> (8 * pass)) & 255;
      const uint64_t same = same_digit(digit, valid);
      if (valid && !(same & below)) hist[wave][digit] += __popcll(same);
      wave_sync();
    }
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
    for (int from = begin; from < end; from += 64) {
      const bool valid = from + lane < end;
      const int row = valid ? (pass ? other[from + lane] : from + lane) : 0;
      const int digit = (adapter_key(index[row], p.n) >> (8 * pass)) & 255;
      const uint64_t same = same_digit(digit, valid);
      if (valid) to[start[digit] + hist[wave][digit] + __popcll(same & below)] = row;
      wave_sync();
      if (valid && !(same & below)) hist[wave][digit] += __popcll(same);
      wave_sync();
    }
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
  const auto cut = [&](int *list, int most, const int *firsts, int n_keys, int piece, const int *slots) {
    for (int i = tid; i < most; i += PLAN_THREADS) {
      int lo = 0, hi = n_keys; // the last key that begins at or before piece i
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (firsts[mid + 1] <= i) lo = mid + 1;
        else hi = mid;
      }
      int4 entry = {-1, 0, 0, 0};
      if (lo < n_keys) {
        const int at = seg[lo] + (i - firsts[lo]) * piece;
        const int slot = slots && slots[lo + 1] > slots[lo] ? slots[lo] + i - firsts[lo] : -1;
        entry = {lo < p.n ? lo : -1, at, min(piece, seg[lo + 1] - at), slot};
      }
      reinterpret_cast<int4 *>(list)[i] = entry;
    }
  };
  cut(plan + p.tiles, p.max_tiles, tile_first, keys, p.tile_rows, nullptr);
  cut(plan + p.chunks, p.max_chunks, first, p.n, p.chunk_rows, slot_first);
}

constexpr int WAVES = 4;

__device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// A product of 16 x 16 results takes, per lane, column lane % 16 of one operand and row lane % 16 of the other, four terms at
// a time, of which the lane has term lane / 16.  Terms may come in any order that both operands share: a lane reads eight
// neighbouring terms at once and hands them out one by one.  The result has, per lane, column lane % 16 and rows
// 4 (lane / 16) + 0 .. 3.  With the weights as rows that is: lane % 16 = the row of x, and four neighbouring ranks -- the
// very operand that the second product wants, so hidden goes from one to the other through registers (and LDS where waves
// share the terms).
template <typename T, typename TW, int RT, int MT, bool BACK> __global__ __launch_bounds__(64 * WAVES) void k_adapter_rows(AdapterRowsArgs a) {
  constexpr int RP = 16 * RT, PITCH = RP + 4;
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
  const uint32_t call = a.drop.on ? drop_call(a.drop) : 0;

  for (int m0 = 0; m0 < count; m0 += 16 * MT) {
    long row[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) row[mt] = rows_of[min(m0 + 16 * mt + lm, count - 1)]; // rows beyond the last repeat it and are not stored
    f32x4 sum[MT][RT] = {};
    for (int k0 = 32 * wave; k0 < a.in_size; k0 += 32 * WAVES) {
      const int col = k0 + 8 * kg, left = a.in_size - col;
      Values8 w[RT];
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        const int rank = 16 * q + lm;
        if (BACK) {
#pragma unroll
          for (int j = 0; j < 8; ++j) w[q].v[j] = rank < a.rank && j < left ? to_float(w_in[(long)(col + j) * a.rank + rank]) : 0.0f;
        } else {
          w[q] = read8(w_in + (long)min(rank, a.rank - 1) * a.in_size + col, rank < a.rank ? left : 0);
        }
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        Values8 x = read8(in + row[mt] * a.in.ld + col, left);
        if (!BACK && a.drop.on) drop_apply(a.drop, drop_kept(a.drop, call, (uint32_t)row[mt], (uint32_t)col / 8u), x);
#pragma unroll
        for (int q = 0; q < RT; ++q)
#pragma unroll
          for (int j = 0; j < 8; ++j) sum[mt][q] = mfma(w[q].v[j], x.v[j], sum[mt][q]);
      }
    }
    // the waves' shares of the terms, added in their order by every wave
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int q = 0; q < RT; ++q) *reinterpret_cast<f32x4 *>(&red[wave][16 * mt + lm][16 * q + 4 * kg]) = sum[mt][q];
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = m0 + 16 * mt + lm;
#pragma unroll
      for (int q = 0; q < RT; ++q) {
        f32x4 v = *reinterpret_cast<const f32x4 *>(&red[0][16 * mt + lm][16 * q + 4 * kg]);
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += *reinterpret_cast<const f32x4 *>(&red[w][16 * mt + lm][16 * q + 4 * kg]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int rank = 16 * q + 4 * kg + i;
          const float scaled = v[i] * scale;
          if (a.hidden && !blockIdx.y && mt % WAVES == wave && m < count && rank < a.rank) a.hidden[row[mt] * a.rank + rank] = BACK ? scaled : v[i];
          sum[mt][q][i] = rank < a.rank ? scaled : 0.0f; // also where a row holds an infinity, whose product with the padding is none
        }
      }
    }
    for (int unit = unit0 + wave; unit < unit1; unit += WAVES) {
      f32x4 acc[MT][2] = {};
      const int col = unit * 32 + 8 * kg, left = a.out_size - col; // of the lane's results
#pragma unroll
      for (int q = 0; q < RT; ++q)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // row lm of the operand is the column whose result ends up beside its neighbours
          const int c = min(unit * 32 + (lm >> 2) * 8 + j * 4 + (lm & 3), a.out_size - 1);
          f32x4 w;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rank = 16 * q + 4 * kg + i;
            const long at = BACK ? (long)min(rank, a.rank - 1) * a.out_size + c : (long)c * a.rank + min(rank, a.rank - 1);
            w[i] = rank < a.rank ? to_float(w_out[at]) : 0.0f;
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[mt][j] = mfma(w[i], sum[mt][q][i], acc[mt][j]);
        }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        if (m0 + 16 * mt + lm >= count) continue;
        Values8 v;
#pragma unroll
        for (int h = 0; h < 8; ++h) v.v[h] = acc[mt][h >> 2][h & 3];
        if (BACK && a.drop.on) drop_apply(a.drop, drop_kept(a.drop, call, (uint32_t)row[mt], (uint32_t)col / 8u), v);
        if (base) {
          const Values8 add = read8(base + row[mt] * a.base.ld + col, left);
#pragma unroll
          for (int h = 0; h < 8; ++h) v.v[h] += add.v[h];
        }
        write8(out + row[mt] * a.out.ld + col, v, left);
      }
    }
    __syncthreads();
  }
}

// 128 columns of dA (of x, against up) or of dB (of d, against scale hidden).  A wave takes 16 rows of its chunk at a time; lane
// % 16 reads eight neighbouring columns of four rows, and product j of a row takes column 8 (lane % 16) + j.
template <typename T, typename TW, int RT> __global__ __launch_bounds__(64 * WAVES) void k_adapter_grads(AdapterGradArgs a) {
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
  for (int g = wave; g * 16 < count; g += WAVES) {
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
        for (int j = 0; j < 8; ++j) acc[j][q] = mfma(x.v[j], u, acc[j][q]);
      }
    }
  }
  for (int from = 0; from < WAVES; ++from) { // the waves' sums, added in their order
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
  if (wave != WAVES - 1) return;
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
      for (int c = begin; c < end; ++c) sum += a.part[c * all + e];
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
template <int V> struct Int {
  static constexpr int value = V;
};
template <typename F> void with_rank_tiles(int rank, F &&f) {
  if (rank <= 16) f(Int<1>{});
  else if (rank <= 32) f(Int<2>{});
  else if (rank <= 64) f(Int<4>{});
  else f(Int<8>{});
}

template <bool BACK> void launch_rows(const AdapterRowsArgs &a, int dtype, int w_dtype, int cus, hipStream_t s) {
  const int tile_rows = a.plan ? a.p.tile_rows : (a.rows + 15) / 16 * 16, tiles = a.plan ? a.p.max_tiles : a.rows;
  // tiles that leave CUs idle share their output columns among several workgroups, each of which makes hidden for itself
  const int units = (a.out_size + 31) / 32;
  const int slices = std::max(1, std::min(units / WAVES, cus / std::max(tiles, 1)));
  const dim3 grid((unsigned)tiles, (unsigned)slices);
  with_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    with_rank_tiles(a.rank, [&](auto rt) {
      constexpr int RT = decltype(rt)::value;
      constexpr int MOST = RT <= 2 ? 4 : 2; // groups of 16 rows at a time: what the registers and LDS hold
      if (tile_rows <= 16) hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, 1, BACK>), grid, dim3(64 * WAVES), 0, s, a);
      else if (tile_rows <= 32) hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, 2, BACK>), grid, dim3(64 * WAVES), 0, s, a);
      else hipLaunchKernelGGL((k_adapter_rows<T, TW, RT, MOST, BACK>), grid, dim3(64 * WAVES), 0, s, a);
    });
  });
}

} // namespace

AdapterPlan adapter_plan(int rows, int n) {
  AdapterPlan p{};
  p.rows = rows;
  p.n = n;
  p.tile_rows = rows <= 2048 ? 16 : rows <= 16384 ? 32 : 64;
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
  hipLaunchKernelGGL(k_adapter_plan, dim3(1), dim3(PLAN_THREADS), 0, s, index, plan, p);
}

void launch_adapter_forward(const AdapterRowsArgs &a, int dtype, int w_dtype, int cus, hipStream_t s) { launch_rows<false>(a, dtype, w_dtype, cus, s); }
void launch_adapter_backward_rows(const AdapterRowsArgs &a, int dtype, int w_dtype, int cus, hipStream_t s) { launch_rows<true>(a, dtype, w_dtype, cus, s); }

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
        hipLaunchKernelGGL((k_adapter_grads<T, TW, AT_ONCE>), dim3((unsigned)a.p.max_chunks, slices, RT / AT_ONCE), dim3(64 * WAVES), 0, s, a);
      });
    hipLaunchKernelGGL(k_adapter_join<TW>, join, dim3(256), 0, s, a);
  });
}

} // namespace rpu_amd
