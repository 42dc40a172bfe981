// Layer norm of rows, forward and backward.
//   forward   y = (x - mean) rstd w + b,  rstd = (mean((x - mean)^2) + eps)^-1/2
//   backward  h = (x - mean) rstd, g = d w:  dx = base + rstd (g - mean(g) - h mean(g h)),  dw = sum d h,  db = sum d
// A row stays in the registers of the threads that share it between its statistics and its use: one pass over the data.  The
// variance is that of the differences from the mean, never a difference of two sums.
#include "digital.h"

#include <algorithm>

namespace rpu_amd {
namespace {

// sum over the TPR threads of a row, the same value in all of them; `room`: a float per wave of the workgroup
template <int TPR> __device__ __forceinline__ float row_sum(float v, float *room) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  if (TPR > 64) {
    __syncthreads(); // the sums before this one have been read
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += room[w];
  }
  return v;
}

template <bool SHORT, typename T> __device__ __forceinline__ Values8 parameter8(const T *p, long col, long cols, float otherwise) {
  if (p) return read8<SHORT>(p, col, cols);
  Values8 r;
#pragma unroll
  for (int h = 0; h < 8; ++h) r.v[h] = otherwise;
  return r;
}

// Rows of up to 8 * TPR * V columns, TPR threads to a row; SHORT: of fewer than 8.  Bound by memory: 16384 x 1024 bf16 in 11.7 us (67 MB,
// 5.7 TB/s); one row of 768 floats in 6.7 us, a launch.
template <typename T, typename TW, int TPR, int V, bool SHORT = false> __global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_layer_norm(NormArgs a) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR;
  __shared__ float room[THREADS / 64];
  const int t = (int)threadIdx.x % TPR;
  const T *x = static_cast<const T *>(a.x.p);
  T *out = static_cast<T *>(a.out.p);
  Values8 w[V], b[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int col = (t + k * TPR) * 8;
    w[k] = parameter8<SHORT>(static_cast<const TW *>(a.w), col, a.cols, 1.0f);
    b[k] = parameter8<SHORT>(static_cast<const TW *>(a.b), col, a.cols, 0.0f);
  }
  const float n = (float)a.cols;
  for (long row = (long)blockIdx.x * ROWS + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * ROWS) {
    Packed8<T> p[V];
    Values8 v[V];
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) p[k] = ahead8<SHORT>(x + row * a.x.ld, (t + k * TPR) * 8, a.cols);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      trim8(p[k], (t + k * TPR) * 8, a.cols);
      v[k] = widen(p[k]);
#pragma unroll
      for (int h = 0; h < 8; ++h) sum += v[k].v[h];
    }
    const float mean = row_sum<TPR>(sum, room) / n;
    float squares = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int left = a.cols - (t + k * TPR) * 8;
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        v[k].v[h] = h < left ? v[k].v[h] - mean : 0.0f;
        squares = fmaf(v[k].v[h], v[k].v[h], squares);
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<TPR>(squares, room) / n + a.eps);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int col = (t + k * TPR) * 8;
#pragma unroll
      for (int h = 0; h < 8; ++h) v[k].v[h] = fmaf(v[k].v[h] * rstd, w[k].v[h], b[k].v[h]);
      write8(out + row * a.out.ld + col, v[k], a.cols - col);
    }
    if (t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Longer rows: a workgroup walks its row three times (the second and third time it comes from the caches).
constexpr int LONG = 1024;
template <typename T, typename TW> __global__ __launch_bounds__(LONG) void k_layer_norm_long(NormArgs a) {
  __shared__ float room[LONG / 64];
  const float n = (float)a.cols;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(a.x.p) + row * a.x.ld;
    T *out = static_cast<T *>(a.out.p) + row * a.out.ld;
    float sum = 0.0f;
    for (long col = (long)threadIdx.x * 8; col < a.cols; col += LONG * 8) {
      const Values8 v = read8<false>(x, col, a.cols);
#pragma unroll
      for (int h = 0; h < 8; ++h) sum += v.v[h];
    }
    const float mean = row_sum<LONG>(sum, room) / n;
    float squares = 0.0f;
    for (long col = (long)threadIdx.x * 8; col < a.cols; col += LONG * 8) {
      const int left = (int)(a.cols - col);
      const Values8 v = read8<false>(x, col, a.cols);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const float c = h < left ? v.v[h] - mean : 0.0f;
        squares = fmaf(c, c, squares);
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<LONG>(squares, room) / n + a.eps);
    for (long col = (long)threadIdx.x * 8; col < a.cols; col += LONG * 8) {
      const int left = (int)(a.cols - col);
      Values8 v = read8<false>(x, col, a.cols);
      const Values8 w = parameter8<false>(static_cast<const TW *>(a.w), col, a.cols, 1.0f), b = parameter8<false>(static_cast<const TW *>(a.b), col, a.cols, 0.0f);
#pragma unroll
      for (int h = 0; h < 8; ++h) v.v[h] = fmaf((v.v[h] - mean) * rstd, w.v[h], b.v[h]);
      write8(out + col, v, left);
    }
    if (threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

constexpr int backward_threads(int threads_of_a_row) { return threads_of_a_row == 64 ? 512 : threads_of_a_row; }
// Backward pass of rows of up to 8 * TPR * V columns.  A workgroup adds d and d h of its rows up in registers and leaves the
// sums in part[workgroup]; k_layer_norm_join adds those.  Bound by memory: 8192 x 768 floats with a base in 20.9 us (101 MB, 4.8 TB/s), and
// 3.9 for the join, 23.5 in a row.  The next row's loads under way while one is worked on took 21.4: the waves of a CU suffice.
template <typename T, typename TW, int TPR, int V, bool SHORT = false>
__global__ __launch_bounds__(backward_threads(TPR)) void k_layer_norm_backward(NormBackwardArgs a) {
  constexpr int THREADS = backward_threads(TPR), ROWS = THREADS / TPR;
  constexpr bool EARLY = TPR < 1024; // base under way with d and x, where the registers suffice
  __shared__ float room[THREADS / 64];
  __shared__ Values8 sums[ROWS > 1 ? 2 * TPR * V : 1];
  const int t = (int)threadIdx.x % TPR, group = (int)threadIdx.x / TPR;
  const T *d = static_cast<const T *>(a.d.p), *x = static_cast<const T *>(a.x.p), *base = static_cast<const T *>(a.base.p);
  T *dx = static_cast<T *>(a.dx.p);
  Values8 w[V], dw[V] = {}, db[V] = {};
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int col = (t + k * TPR) * 8;
    w[k] = parameter8<SHORT>(static_cast<const TW *>(a.w), col, a.cols, 1.0f);
  }
  const float n = (float)a.cols;
  for (long row = (long)blockIdx.x * ROWS + group; row < a.rows; row += (long)gridDim.x * ROWS) {
    Packed8<T> p[V], q[V], more[V];
    Values8 g[V], h[V];
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sum_g = 0.0f, sum_gh = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int col = (t + k * TPR) * 8;
      p[k] = ahead8<SHORT>(d + row * a.d.ld, col, a.cols);
      q[k] = ahead8<SHORT>(x + row * a.x.ld, col, a.cols);
      if (EARLY && base) more[k] = ahead8<SHORT>(base + row * a.base.ld, col, a.cols);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int col = (t + k * TPR) * 8, left = a.cols - col;
      trim8(p[k], col, a.cols);
      trim8(q[k], col, a.cols);
      g[k] = widen(p[k]);
      h[k] = widen(q[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hat = i < left ? (h[k].v[i] - mean) * rstd : 0.0f;
        h[k].v[i] = hat;
        dw[k].v[i] = fmaf(g[k].v[i], hat, dw[k].v[i]);
        db[k].v[i] += g[k].v[i];
        g[k].v[i] *= w[k].v[i];
        sum_g += g[k].v[i];
        sum_gh = fmaf(g[k].v[i], hat, sum_gh);
      }
    }
    const float mean_g = row_sum<TPR>(sum_g, room) / n, mean_gh = row_sum<TPR>(sum_gh, room) / n;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int col = (t + k * TPR) * 8, left = a.cols - col;
      Values8 r;
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = rstd * (g[k].v[i] - mean_g - h[k].v[i] * mean_gh);
      if (base) {
        if (!EARLY) more[k] = ahead8<SHORT>(base + row * a.base.ld, col, a.cols);
        trim8(more[k], col, a.cols);
        const Values8 add = widen(more[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] += add.v[i];
      }
      write8(dx + row * a.dx.ld + col, r, left);
    }
  }
  if (!a.dw) return;
  float *part = a.part + (long)blockIdx.x * 2 * a.cols;
  if (ROWS > 1) { // the groups of a workgroup one after the other
    for (int from = 0; from < ROWS; ++from) {
      if (group == from) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            dw[k].v[i] += from ? sums[t + k * TPR].v[i] : 0.0f;
            db[k].v[i] += from ? sums[(V + k) * TPR + t].v[i] : 0.0f;
          }
          sums[t + k * TPR] = dw[k];
          sums[(V + k) * TPR + t] = db[k];
        }
      }
      __syncthreads();
    }
    if (group != ROWS - 1) return;
  }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int col = (t + k * TPR) * 8, left = a.cols - col;
    write8(part + col, dw[k], left);
    write8(part + a.cols + col, db[k], left);
  }
}

// Longer rows: two walks over the row, the sums of the columns in `part` itself, each by the thread that has the column.
template <typename T, typename TW> __global__ __launch_bounds__(LONG) void k_layer_norm_backward_long(NormBackwardArgs a) {
  __shared__ float room[LONG / 64];
  const float n = (float)a.cols;
  float *part = a.part + (long)blockIdx.x * 2 * a.cols;
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T *d = static_cast<const T *>(a.d.p) + row * a.d.ld, *x = static_cast<const T *>(a.x.p) + row * a.x.ld;
    const T *base = a.base.p ? static_cast<const T *>(a.base.p) + row * a.base.ld : nullptr;
    T *dx = static_cast<T *>(a.dx.p) + row * a.dx.ld;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float sum_g = 0.0f, sum_gh = 0.0f;
    for (long col = (long)threadIdx.x * 8; col < a.cols; col += LONG * 8) {
      const int left = (int)(a.cols - col);
      const Values8 g = read8<false>(d, col, a.cols), v = read8<false>(x, col, a.cols), w = parameter8<false>(static_cast<const TW *>(a.w), col, a.cols, 1.0f);
      Values8 dw = {}, db = {};
      if (a.dw && row != (long)blockIdx.x) {
        dw = read8<false>(part, col, a.cols);
        db = read8<false>(part + a.cols, col, a.cols);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float hat = i < left ? (v.v[i] - mean) * rstd : 0.0f;
        dw.v[i] = fmaf(g.v[i], hat, dw.v[i]);
        db.v[i] += g.v[i];
        sum_g = fmaf(g.v[i], w.v[i], sum_g);
        sum_gh = fmaf(g.v[i] * w.v[i], hat, sum_gh);
      }
      if (a.dw) {
        write8(part + col, dw, left);
        write8(part + a.cols + col, db, left);
      }
    }
    const float mean_g = row_sum<LONG>(sum_g, room) / n, mean_gh = row_sum<LONG>(sum_gh, room) / n;
    for (long col = (long)threadIdx.x * 8; col < a.cols; col += LONG * 8) {
      const int left = (int)(a.cols - col);
      const Values8 g = read8<false>(d, col, a.cols), v = read8<false>(x, col, a.cols), w = parameter8<false>(static_cast<const TW *>(a.w), col, a.cols, 1.0f);
      Values8 r;
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = rstd * (g.v[i] * w.v[i] - mean_g - (v.v[i] - mean) * rstd * mean_gh);
      if (base) {
        const Values8 add = read8<false>(base, col, a.cols);
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] += add.v[i];
      }
      write8(dx + col, r, left);
    }
  }
}

// dw and db from the sums of the workgroups: 64 columns to a workgroup, its waves share the parts.
constexpr int JOIN_WAVES = 16;
template <typename TW> __global__ __launch_bounds__(64 * JOIN_WAVES) void k_layer_norm_join(NormBackwardArgs a) {
  __shared__ float sums[JOIN_WAVES][64];
  const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
  const long col = (long)blockIdx.x * 64 + lane, width = 2l * a.cols;
  float sum = 0.0f;
  if (col < width) {
    int p = wave;
    for (; p + 7 * JOIN_WAVES < a.parts; p += 8 * JOIN_WAVES) { // eight loads under way together
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = a.part[(p + u * JOIN_WAVES) * width + col];
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += v[u];
    }
    for (; p < a.parts; p += JOIN_WAVES) sum += a.part[p * width + col];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave || col >= width) return;
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < JOIN_WAVES; ++w) sum += sums[w][lane];
  if (col < a.cols) static_cast<TW *>(a.dw)[col] = (TW)sum;
  else static_cast<TW *>(a.db)[col - a.cols] = (TW)sum;
}

template <typename F> void with_types(int dtype, int w_dtype, F &&f) {
  if (dtype == RPU_F32) f(float{}, float{});
  else if (dtype == RPU_F16) w_dtype == RPU_F32 ? f(_Float16{}, float{}) : f(_Float16{}, _Float16{});
  else w_dtype == RPU_F32 ? f(__bf16{}, float{}) : f(__bf16{}, __bf16{});
}

// threads to a row of the backward pass, and their groups of eight columns each
constexpr int BACKWARD_LONGEST = 1024 * 16;
int backward_rows(int cols) { return cols <= 1024 ? 8 : 1; } // rows that a workgroup works on at a time

} // namespace

void launch_layer_norm(const NormArgs &a, int dtype, int w_dtype, int cus, hipStream_t s) {
  with_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    const auto grid = [&](int rows_each, int per_cu) { return dim3((unsigned)std::min(((long)a.rows + rows_each - 1) / rows_each, (long)cus * per_cu)); };
    if (a.cols < 8) hipLaunchKernelGGL((k_layer_norm<T, TW, 64, 1, true>), grid(4, 8), dim3(256), 0, s, a);
    else if (a.cols <= 512) hipLaunchKernelGGL((k_layer_norm<T, TW, 64, 1>), grid(4, 8), dim3(256), 0, s, a);
    else if (a.cols <= 1024) hipLaunchKernelGGL((k_layer_norm<T, TW, 64, 2>), grid(4, 6), dim3(256), 0, s, a);
    else if (a.cols <= 2048) hipLaunchKernelGGL((k_layer_norm<T, TW, 256, 1>), grid(1, 8), dim3(256), 0, s, a);
    else if (a.cols <= 4096) hipLaunchKernelGGL((k_layer_norm<T, TW, 256, 2>), grid(1, 6), dim3(256), 0, s, a);
    else if (a.cols <= 8192) hipLaunchKernelGGL((k_layer_norm<T, TW, 1024, 1>), grid(1, 2), dim3(1024), 0, s, a);
    else if (a.cols <= 16384) hipLaunchKernelGGL((k_layer_norm<T, TW, 1024, 2>), grid(1, 2), dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((k_layer_norm_long<T, TW>), grid(1, 2), dim3(LONG), 0, s, a);
  });
}

int layer_norm_parts(int rows, int cols, int cus) {
  // Workgroups of a CU.  Four waves each (1025 .. 4096 columns): 8192 rows of 1537 halves take 53 us with one, 33 with two, 28 with three,
  // 27 with four; of 4096 bf16 68, 46, 43 and 52.  Eight waves with rows of 513 .. 1024 columns in many registers: 16384 rows of 768
  // bf16 22.8 with one, 26.8 with two; shorter rows: 50000 of 64 floats 33.6 and 25.6, 16384 of 512 bf16 16.0 and 15.5.  Sixteen waves:
  // 4096 rows of 5000 halves 49.3 and 54.2.  Two rows each at least: of a column they read and write 12 bytes (16-bit rows without a base) to 32
  // (floats with one), their sums, written and read again, take 16.
  const int per_cu = cols <= 512 ? 2 : cols <= 1024 ? 1 : cols <= 4096 ? 3 : 1;
  const long groups = ((long)rows + backward_rows(cols) - 1) / backward_rows(cols);
  return (int)std::min((groups + 1) / 2, (long)cus * per_cu);
}

void launch_layer_norm_backward(const NormBackwardArgs &a, int dtype, int w_dtype, hipStream_t s) {
  with_types(dtype, w_dtype, [&](auto x, auto w) {
    using T = decltype(x);
    using TW = decltype(w);
    const dim3 grid((unsigned)a.parts);
    if (a.parts) {
      if (a.cols < 8) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 64, 1, true>), grid, dim3(512), 0, s, a);
      else if (a.cols <= 512) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 64, 1>), grid, dim3(512), 0, s, a);
      else if (a.cols <= 1024) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 64, 2>), grid, dim3(512), 0, s, a);
      else if (a.cols <= 2048) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 256, 1>), grid, dim3(256), 0, s, a);
      else if (a.cols <= 4096) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 256, 2>), grid, dim3(256), 0, s, a);
      else if (a.cols <= 8192) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 1024, 1>), grid, dim3(1024), 0, s, a);
      else if (a.cols <= BACKWARD_LONGEST) hipLaunchKernelGGL((k_layer_norm_backward<T, TW, 1024, 2>), grid, dim3(1024), 0, s, a);
      else hipLaunchKernelGGL((k_layer_norm_backward_long<T, TW>), grid, dim3(LONG), 0, s, a);
    }
    if (a.dw) hipLaunchKernelGGL(k_layer_norm_join<TW>, dim3((unsigned)((2l * a.cols + 63) / 64)), dim3(64 * JOIN_WAVES), 0, s, a);
  });
}

} // namespace rpu_amd
