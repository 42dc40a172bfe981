// C entry points of the digital operators beside the tiles: what they check on the host before anything is launched.
#include "digital.h"
#include "entry.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <vector>

namespace rpu_amd {
namespace {

// Grids, and indexes into rows, are 32-bit numbers: far more than a GPU's memory holds of one and the other together.
constexpr int MOST_ROWS = 1 << 28, MOST_COLS = 1 << 24, MOST_ADAPTER_COLS = 1 << 21;

size_t value_size(int dtype) { return dtype == RPU_F32 ? 4 : 2; }
void check_dtype(int dtype) {
  if (dtype != RPU_F32 && dtype != RPU_F16 && dtype != RPU_BF16) throw RpuError("Unknown data type.");
}
void check_rows(int rows) {
  if (rows < 0 || rows > MOST_ROWS) throw RpuError("The number of rows must be in 0 .. 2^28.");
}
void check_cols(int cols) {
  if (cols < 1 || cols > MOST_COLS) throw RpuError("The number of columns must be in 1 .. 2^24.");
}

// an operand's place in memory: rows of `width` bytes, `pitch` bytes apart
struct Span {
  const char *what;
  uintptr_t at;
  size_t rows, width, pitch;
  uintptr_t end() const { return at + (rows - 1) * pitch + width; }
};
Span matrix(const char *what, const void *p, long ld, int rows, int cols, size_t e) {
  if (!p && rows) throw RpuError(std::string(what) + " is null.");
  if (rows > 1 && ld < cols) throw RpuError(std::string("The rows of ") + what + " overlap.");
  if (ld > LONG_MAX / 8 / MOST_ROWS) throw RpuError(std::string("The rows of ") + what + " lie too far apart.");
  return {what, (uintptr_t)p, (size_t)rows, e * (size_t)cols, e * (size_t)(rows > 1 ? ld : cols)};
}
Span dense(const char *what, const void *p, size_t bytes) {
  if (!p && bytes) throw RpuError(std::string(what) + " is null.");
  return {what, (uintptr_t)p, bytes ? (size_t)1 : 0, bytes, bytes};
}
bool same_place(const Span &a, const Span &b) { return a.at == b.at && a.rows == b.rows && a.width == b.width && a.pitch == b.pitch; }
bool meet(const Span &a, const Span &b) {
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
void apart(const Span &out, const Span &other, bool may_be_same = false) {
  if (meet(out, other) && !(may_be_same && same_place(out, other)))
    throw RpuError(std::string("The memory of ") + out.what + " overlaps that of " + other.what + ".");
}

DropDev drop_dev(const rpu_dropout_params *d) {
  DropDev r{};
  if (!d) return r;
  if (!(d->p >= 0.0 && d->p <= 1.0)) throw RpuError("The dropout probability must be in [0, 1].");
  if (d->reserved) throw RpuError("A reserved field of the dropout parameters is not 0.");
  const uint64_t limit = (uint64_t)std::floor(d->p * 4294967296.0 + 0.5);
  r.high = (uint32_t)(limit >> 16);
  r.low = (uint32_t)(limit & 0xffffu);
  r.scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.0f;
  r.key = {(uint32_t)d->seed, (uint32_t)(d->seed >> 32)};
  r.call = d->call;
  r.call_dev = d->call_dev;
  r.on = d->p > 0.0;
  return r;
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
void check_launch() { RPU_HIP_CHECK(hipGetLastError()); }

constexpr int MOST_CUS = 256; // that scratch sizes, which are asked for without a GPU, are for: an MI355X has so many

void check_adapters(const rpu_adapters *a, int dtype) {
  check_dtype(dtype);
  if (!a) throw RpuError("The adapters are null.");
  if (a->reserved) throw RpuError("A reserved field of the adapters is not 0.");
  if (a->n < 1 || a->n > RPU_ADAPTER_MAX) throw RpuError("The number of adapters must be in 1 .. 65535.");
  if (a->in_size < 1 || a->out_size < 1 || a->in_size > MOST_ADAPTER_COLS || a->out_size > MOST_ADAPTER_COLS)
    throw RpuError("The sizes of the adapters must be in 1 .. 2^21.");
  if (a->rank < 1 || a->rank > RPU_ADAPTER_MAX_RANK) throw RpuError("The rank of the adapters must be in 1 .. 128.");
  check_dtype(a->w_dtype);
  if (dtype != RPU_F32 && a->w_dtype != dtype) throw RpuError("Adapters beside 16-bit rows must be of the rows' type.");
  if (!a->a_dev || !a->b_dev || !a->scale_dev) throw RpuError("The adapters' matrices or scales are null.");
}
void check_plan(const void *plan, size_t bytes, const AdapterPlan &p) {
  if (!plan) throw RpuError("The row plan is null.");
  if (bytes < p.words * sizeof(int)) throw RpuError("The row plan is too small for this many rows and adapters.");
  if ((uintptr_t)plan % 16) throw RpuError("The row plan is not aligned to 16 bytes.");
}
struct BackwardScratch { // offsets in bytes
  size_t up, part, a_turned, b_turned, bytes;
  BackwardScratch(const rpu_adapters *a, int rows) {
    const AdapterPlan p = adapter_plan(rows, a->n);
    const size_t e = value_size(a->w_dtype);
    bytes = 0;
    up = take(4 * (size_t)rows * a->rank);
    part = take(4 * (size_t)p.max_slots * a->rank * ((size_t)a->in_size + a->out_size));
    a_turned = take(e * adapter_turned(p) * a->rank * a->in_size);
    b_turned = take(e * adapter_turned(p) * a->rank * a->out_size);
  }
  size_t take(size_t n) {
    const size_t from = bytes;
    bytes += (n + 15) / 16 * 16;
    return from;
  }
};

} // namespace
} // namespace rpu_amd

using namespace rpu_amd;

extern "C" {

int rpu_dropout(const void *x_dev, long x_ld, const void *base_dev, long base_ld, void *out_dev, long out_ld, int dtype,
                int rows, int cols, const rpu_dropout_params *params, int device_id, void *stream) {
  return guarded([&] {
    check_dtype(dtype);
    check_rows(rows);
    check_cols(cols);
    if (!params) throw RpuError("The dropout parameters are null.");
    const size_t e = value_size(dtype);
    const Span out = matrix("the output", out_dev, out_ld, rows, cols, e);
    apart(out, matrix("x", x_dev, x_ld, rows, cols, e), true);
    if (base_dev) apart(out, matrix("the base", base_dev, base_ld, rows, cols, e), true);
    DropoutArgs a{{const_cast<void *>(x_dev), x_ld}, {const_cast<void *>(base_dev), base_ld}, {out_dev, out_ld}, rows, cols, drop_dev(params)};
    if (!rows) return;
    const Gpu gpu(device_id);
    launch_dropout(a, dtype, gpu.cus(), (hipStream_t)stream);
    check_launch();
  });
}

int rpu_layer_norm(const void *x_dev, long x_ld, const void *w_dev, const void *b_dev, int w_dtype, void *out_dev, long out_ld,
                   float *mean_dev, float *rstd_dev, int dtype, int rows, int cols, float eps, int device_id, void *stream) {
  return guarded([&] {
    check_dtype(dtype);
    check_rows(rows);
    check_cols(cols);
    if (w_dtype != RPU_F32 && w_dtype != dtype) throw RpuError("Weight and bias must be float or of the rows' type.");
    if (!(eps >= 0.0f) || std::isinf(eps)) throw RpuError("eps must be finite and not negative.");
    const size_t e = value_size(dtype), we = value_size(w_dtype);
    const Span out = matrix("the output", out_dev, out_ld, rows, cols, e), mean = dense("mean", mean_dev, 4 * (size_t)rows),
               rstd = dense("rstd", rstd_dev, 4 * (size_t)rows), x = matrix("x", x_dev, x_ld, rows, cols, e);
    apart(out, x, true);
    apart(out, mean);
    apart(out, rstd);
    apart(mean, rstd);
    apart(mean, x);
    apart(rstd, x);
    for (const void *p : {w_dev, b_dev})
      if (p)
        for (const Span &s : {out, mean, rstd}) apart(s, dense("weight or bias", p, we * (size_t)cols));
    if (!rows) return;
    const Gpu gpu(device_id);
    launch_layer_norm({{const_cast<void *>(x_dev), x_ld}, {out_dev, out_ld}, w_dev, b_dev, mean_dev, rstd_dev, rows, cols, eps}, dtype, w_dtype,
                      gpu.cus(), (hipStream_t)stream);
    check_launch();
  });
}

size_t rpu_layer_norm_backward_scratch(int rows, int cols) {
  if (rows < 0 || rows > MOST_ROWS || cols < 1 || cols > MOST_COLS) return 0;
  return (size_t)layer_norm_parts(rows, cols, MOST_CUS) * 2 * (size_t)cols * sizeof(float);
}

int rpu_layer_norm_backward(const void *d_dev, long d_ld, const void *x_dev, long x_ld, const float *mean_dev,
                            const float *rstd_dev, const void *w_dev, int w_dtype, const void *base_dev, long base_ld,
                            void *dx_dev, long dx_ld, void *dw_dev, void *db_dev, int dtype, int rows, int cols,
                            void *scratch_dev, size_t scratch_bytes, int device_id, void *stream) {
  return guarded([&] {
    check_dtype(dtype);
    check_rows(rows);
    check_cols(cols);
    if (w_dtype != RPU_F32 && w_dtype != dtype) throw RpuError("Weight and bias must be float or of the rows' type.");
    if (!dw_dev != !db_dev) throw RpuError("The gradients of weight and bias come together.");
    const size_t e = value_size(dtype), we = value_size(w_dtype), stats = 4 * (size_t)rows;
    const Span dx = matrix("dx", dx_dev, dx_ld, rows, cols, e), d = matrix("d", d_dev, d_ld, rows, cols, e), x = matrix("x", x_dev, x_ld, rows, cols, e),
               mean = dense("mean", mean_dev, stats), rstd = dense("rstd", rstd_dev, stats);
    std::vector<Span> read{d, x};
    if (base_dev) read.push_back(matrix("the base", base_dev, base_ld, rows, cols, e));
    for (const Span &s : read) apart(dx, s, true); // a row is read before it is written
    read.push_back(mean);
    read.push_back(rstd);
    if (w_dev) read.push_back(dense("the weight", w_dev, we * (size_t)cols));
    std::vector<Span> written;
    if (dw_dev) {
      if (scratch_bytes < rpu_layer_norm_backward_scratch(rows, cols)) throw RpuError("The scratch memory is too small.");
      written = {dense("dw", dw_dev, we * (size_t)cols), dense("db", db_dev, we * (size_t)cols),
                 dense("the scratch memory", scratch_dev, rpu_layer_norm_backward_scratch(rows, cols))};
      if ((uintptr_t)scratch_dev % 4) throw RpuError("The scratch memory is not aligned to 4 bytes.");
    }
    for (size_t k = 0; k < written.size(); ++k) {
      for (const Span &s : read) apart(written[k], s);
      for (size_t i = 0; i < k; ++i) apart(written[k], written[i]);
      apart(written[k], dx);
    }
    for (size_t k = base_dev ? 3 : 2; k < read.size(); ++k) apart(dx, read[k]);
    if (!rows && !dw_dev) return;
    const Gpu gpu(device_id);
    const int parts = layer_norm_parts(rows, cols, std::min(gpu.cus(), MOST_CUS));
    launch_layer_norm_backward({{const_cast<void *>(d_dev), d_ld}, {const_cast<void *>(x_dev), x_ld}, {const_cast<void *>(base_dev), base_ld},
                                {dx_dev, dx_ld}, mean_dev, rstd_dev, w_dev, dw_dev, db_dev, (float *)scratch_dev, rows, cols, parts},
                               dtype, w_dtype, (hipStream_t)stream);
    check_launch();
  });
}

size_t rpu_adapter_plan_bytes(int rows, int n) {
  if (rows < 0 || rows > MOST_ROWS || n < 1 || n > RPU_ADAPTER_MAX) return 0;
  return adapter_plan(rows, n).words * sizeof(int);
}

int rpu_adapter_plan(const int32_t *index_dev, int rows, int n, void *plan_dev, size_t plan_bytes, int device_id, void *stream) {
  return guarded([&] {
    check_rows(rows);
    if (n < 1 || n > RPU_ADAPTER_MAX) throw RpuError("The number of adapters must be in 1 .. 65535.");
    const AdapterPlan p = adapter_plan(rows, n);
    check_plan(plan_dev, plan_bytes, p);
    apart(dense("the row plan", plan_dev, p.words * sizeof(int)), dense("the index", index_dev, sizeof(int32_t) * (size_t)rows));
    const Gpu gpu(device_id);
    launch_adapter_plan(index_dev, (int *)plan_dev, p, (hipStream_t)stream);
    check_launch();
  });
}

int rpu_adapter_forward(const rpu_adapters *adapters, const void *x_dev, long x_ld, const int32_t *index_dev,
                        const void *plan_dev, size_t plan_bytes, const rpu_dropout_params *drop, const void *base_dev,
                        long base_ld, void *y_dev, long y_ld, float *hidden_dev, int dtype, int rows, int device_id,
                        void *stream) {
  return guarded([&] {
    check_adapters(adapters, dtype);
    check_rows(rows);
    const rpu_adapters &w = *adapters;
    const AdapterPlan p = adapter_plan(rows, w.n);
    const size_t e = value_size(dtype), we = value_size(w.w_dtype);
    const Span y = matrix("y", y_dev, y_ld, rows, w.out_size, e);
    std::vector<Span> written{y}, read{matrix("x", x_dev, x_ld, rows, w.in_size, e),
                                       dense("a", w.a_dev, we * w.n * w.rank * (size_t)w.in_size),
                                       dense("b", w.b_dev, we * w.n * w.rank * (size_t)w.out_size), dense("the scales", w.scale_dev, 4 * (size_t)w.n)};
    if (plan_dev) {
      check_plan(plan_dev, plan_bytes, p);
      read.push_back(dense("the row plan", plan_dev, p.words * sizeof(int)));
    } else {
      if (rows > RPU_ADAPTER_FEW_ROWS) throw RpuError("So many rows need a row plan.");
      read.push_back(dense("the index", index_dev, sizeof(int32_t) * (size_t)rows));
    }
    if (hidden_dev) written.push_back(dense("hidden", hidden_dev, 4 * (size_t)rows * w.rank));
    if (base_dev) {
      const Span base = matrix("the base", base_dev, base_ld, rows, w.out_size, e);
      apart(y, base, true);
      if (hidden_dev) apart(written[1], base);
    }
    for (const Span &o : written)
      for (const Span &s : read) apart(o, s);
    if (hidden_dev) apart(y, written[1]);
    const DropDev d = drop_dev(drop);
    if (!rows) return;
    if (plan_dev && !hidden_dev) throw RpuError("hidden is null.");
    const Gpu gpu(device_id);
    AdapterRowsArgs a{};
    a.in = {const_cast<void *>(x_dev), x_ld};
    a.base = {const_cast<void *>(base_dev), base_ld};
    a.out = {y_dev, y_ld};
    a.w_in = w.a_dev;
    a.w_out = w.b_dev;
    a.scale = w.scale_dev;
    a.hidden = hidden_dev;
    a.index = index_dev;
    a.plan = (const int *)plan_dev;
    a.p = p;
    a.rows = rows;
    a.n = w.n;
    a.rank = w.rank;
    a.in_size = w.in_size;
    a.out_size = w.out_size;
    a.drop = d;
    launch_adapter_rows(a, dtype, w.w_dtype, gpu.cus(), (hipStream_t)stream);
    check_launch();
  });
}

size_t rpu_adapter_backward_scratch(const rpu_adapters *adapters, int rows) {
  if (!adapters || rows < 0 || rows > MOST_ROWS || adapters->n < 1 || adapters->n > RPU_ADAPTER_MAX || adapters->rank < 1 ||
      adapters->rank > RPU_ADAPTER_MAX_RANK || adapters->in_size < 1 || adapters->out_size < 1 || adapters->in_size > MOST_ADAPTER_COLS ||
      adapters->out_size > MOST_ADAPTER_COLS || (adapters->w_dtype != RPU_F32 && adapters->w_dtype != RPU_F16 && adapters->w_dtype != RPU_BF16))
    return 0;
  return BackwardScratch(adapters, rows).bytes;
}

int rpu_adapter_backward(const rpu_adapters *adapters, const void *d_dev, long d_ld, const void *x_dev, long x_ld,
                         const float *hidden_dev, const void *plan_dev, size_t plan_bytes, const rpu_dropout_params *drop,
                         const void *base_dev, long base_ld, void *dx_dev, long dx_ld, void *da_dev, void *db_dev, int dtype,
                         int rows, void *scratch_dev, size_t scratch_bytes, int device_id, void *stream) {
  return guarded([&] {
    check_adapters(adapters, dtype);
    check_rows(rows);
    const rpu_adapters &w = *adapters;
    const AdapterPlan p = adapter_plan(rows, w.n);
    check_plan(plan_dev, plan_bytes, p);
    const BackwardScratch s(adapters, rows);
    const size_t e = value_size(dtype), we = value_size(w.w_dtype), need = s.bytes;
    if (scratch_bytes < need) throw RpuError("The scratch memory is too small.");
    if ((uintptr_t)scratch_dev % 4) throw RpuError("The scratch memory is not aligned to 4 bytes.");
    const size_t of_a = we * w.n * w.rank * (size_t)w.in_size, of_b = we * w.n * w.rank * (size_t)w.out_size;
    const std::vector<Span> read{matrix("d", d_dev, d_ld, rows, w.out_size, e), matrix("x", x_dev, x_ld, rows, w.in_size, e),
                                 dense("a", w.a_dev, of_a), dense("b", w.b_dev, of_b), dense("the scales", w.scale_dev, 4 * (size_t)w.n),
                                 dense("hidden", hidden_dev, 4 * (size_t)rows * w.rank), dense("the row plan", plan_dev, p.words * sizeof(int))};
    const std::vector<Span> written{matrix("dx", dx_dev, dx_ld, rows, w.in_size, e), dense("da", da_dev, of_a), dense("db", db_dev, of_b),
                                    dense("the scratch memory", scratch_dev, need)};
    for (size_t k = 0; k < written.size(); ++k) {
      for (const Span &r : read) apart(written[k], r);
      for (size_t i = 0; i < k; ++i) apart(written[k], written[i]);
      if (base_dev) apart(written[k], matrix("the base", base_dev, base_ld, rows, w.in_size, e), k == 0);
    }
    const DropDev drop_of_x = drop_dev(drop);
    const Gpu gpu(device_id);
    float *up = (float *)((char *)scratch_dev + s.up), *part = (float *)((char *)scratch_dev + s.part);
    AdapterGradArgs g{};
    g.x = {const_cast<void *>(x_dev), x_ld};
    g.d = {const_cast<void *>(d_dev), d_ld};
    g.hidden = hidden_dev;
    g.up = up;
    g.scale = w.scale_dev;
    g.da = da_dev;
    g.db = db_dev;
    g.part = part;
    g.plan = (const int *)plan_dev;
    g.p = p;
    g.rows = rows;
    g.n = w.n;
    g.rank = w.rank;
    g.in_size = w.in_size;
    g.out_size = w.out_size;
    g.drop = drop_of_x;
    if (rows) {
      AdapterTurnArgs turn{w.a_dev, w.b_dev, (char *)scratch_dev + s.a_turned, (char *)scratch_dev + s.b_turned, g.plan, p, w.n, w.rank, w.in_size, w.out_size, adapter_listed(p)};
      launch_adapter_turn(turn, w.w_dtype, gpu.cus(), (hipStream_t)stream);
      AdapterRowsArgs a{};
      a.in = g.d;
      a.base = {const_cast<void *>(base_dev), base_ld};
      a.out = {dx_dev, dx_ld};
      a.w_in = turn.b_turned;
      a.w_out = turn.a_turned;
      a.scale = w.scale_dev;
      a.hidden = up;
      a.plan = g.plan;
      a.p = p;
      a.rows = rows;
      a.n = w.n;
      a.rank = w.rank;
      a.in_size = w.out_size;
      a.out_size = w.in_size;
      a.drop = drop_of_x;
      a.back = 1;
      a.listed = adapter_listed(p);
      launch_adapter_rows(a, dtype, w.w_dtype, gpu.cus(), (hipStream_t)stream);
    }
    launch_adapter_grads(g, dtype, w.w_dtype, gpu.cus(), (hipStream_t)stream);
    check_launch();
  });
}

} // extern "C"
