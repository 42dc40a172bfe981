// C entry points of attention over a paged cache: what they check on the host before anything is launched.
#include "attend_tiles.h"
#include "cache.h"
#include "operand_checks.h"

#include <cmath>
#include <vector>

namespace rpu_amd {
namespace {

constexpr int MOST_PLACES = 1 << 30, MOST_HEADS = 1 << 16;

CacheDev cache_dev(const rpu_cache *cache, int dtype) {
  if (!cache) throw RpuError("The cache is null.");
  const rpu_cache &c = *cache;
  check_dtype(dtype);
  check_dtype(c.dtype);
  if (c.reserved) throw RpuError("A reserved field of the cache is not 0.");
  if (dtype != RPU_F32 && c.dtype != dtype) throw RpuError("A cache beside 16-bit rows must be of the rows' type.");
  if (c.pages < 1 || c.heads < 1 || c.heads > MOST_HEADS) throw RpuError("A cache has pages, and 1 .. 65536 heads.");
  if (c.page_size < RPU_CACHE_MIN_PAGE || c.page_size > RPU_CACHE_MAX_PAGE || (c.page_size & (c.page_size - 1)))
    throw RpuError("The size of a page must be a power of two, 8 to 65536.");
  if (c.head_size < 8 || c.head_size > RPU_CACHE_MAX_HEAD || c.head_size % 8) throw RpuError("The size of a head must be a multiple of 8 up to 256.");
  if (value_size(c.dtype) * c.head_size * c.page_size * (size_t)c.heads > INT_MAX) throw RpuError("The keys of a page must take less than 2 GB.");
  if (c.pairs < 0 || 2 * (long)c.pairs > c.head_size) throw RpuError("A head cannot have so many pairs.");
  if (c.pairs && !c.turns_dev) throw RpuError("The rotation's turns are null.");
  if (!c.k_dev || !c.v_dev) throw RpuError("The cache's keys or values are null.");
  if ((uintptr_t)c.k_dev % 16 || (uintptr_t)c.v_dev % 16) throw RpuError("The cache's keys and values must be aligned to 16 bytes.");
  return {c.k_dev, c.v_dev, c.turns_dev, c.pages, __builtin_ctz((unsigned)c.page_size), c.heads, c.head_size, c.pairs, c.neighbours != 0};
}
CacheRowsDev rows_dev(const rpu_cache &c, const rpu_cache_rows *rows) {
  if (!rows) throw RpuError("The rows' sequences are null.");
  const rpu_cache_rows &r = *rows;
  if (r.reserved) throw RpuError("A reserved field of the rows' sequences is not 0.");
  check_rows(r.rows);
  if (r.n < 1 || r.n > MOST_ROWS) throw RpuError("The number of sequences must be in 1 .. 2^28.");
  if (!r.starts_dev && r.rows % r.n) throw RpuError("Without starts, the sequences have as many rows each.");
  if (r.table_width < 1 || (long)r.table_width * c.page_size > MOST_PLACES) throw RpuError("A table must hold 1 .. 2^30 positions.");
  if (!r.tables_dev || !r.lengths_dev) throw RpuError("The tables or lengths are null.");
  if (r.n > 1 && (r.table_ld < r.table_width || r.table_ld > LONG_MAX / 8 / MOST_ROWS)) throw RpuError("The tables overlap or lie too far apart.");
  return {r.tables_dev, r.lengths_dev, r.starts_dev, r.n > 1 ? r.table_ld : r.table_width, r.n, r.table_width * c.page_size, r.rows};
}
std::vector<Span> numbers(const rpu_cache &c, const rpu_cache_rows &r) { // what the kernels are steered by
  std::vector<Span> all{matrix("the tables", r.tables_dev, r.table_ld, r.n, r.table_width, 4), dense("the lengths", r.lengths_dev, 4 * (size_t)r.n)};
  if (r.starts_dev) all.push_back(dense("the starts", r.starts_dev, 4 * ((size_t)r.n + 1)));
  if (c.pairs) all.push_back(dense("the turns", c.turns_dev, 8 * (size_t)c.pairs));
  return all;
}
size_t cache_bytes(const rpu_cache &c) { return value_size(c.dtype) * (size_t)c.pages * c.heads * c.page_size * c.head_size; }
int width_of(int heads, const rpu_cache &c) {
  const long width = (long)heads * c.head_size;
  if (heads < 1 || width > MOST_COLS) throw RpuError("A row must have at least one head, and at most 2^24 values.");
  return (int)width;
}

// Parts that `units` of work are split into, over up to `longest` positions: as long as there are fewer workgroups than the GPU runs together, of
// at least `least` positions; beyond that, so that units of unlike length do not wait for the longest, of at least 1024.  (64 sequences, 8 heads of 128
// bf16: lengths up to 8192, in 512, 2048 and 4096 workgroups 251, 248 and 244 us; a window of 1024 in 512, 1024 and 2048 57, 67 and 71 us.)
int splits_for(long units, long longest, long least, long together, long many) {
  const long fill = std::min(together / units, (longest + least - 1) / least), more = std::min(many / units, longest / 1024);
  return (int)std::max(1l, std::min(64l, std::max(fill, more)));
}
AttendPlan attend_plan(const rpu_cache &c, const rpu_cache_rows &r, int q_heads, int dtype, int window, int sinks, int longest) {
  AttendPlan p{};
  if ((long)r.rows * (q_heads / c.heads) > (1 << 30)) throw RpuError("So many rows and heads are too many for a call.");
  const long group = q_heads / c.heads, places = (long)r.table_width * c.page_size;
  const long lines = r.starts_dev ? 0 : r.rows / r.n * group; // of every sequence
  // positions that a workgroup goes over, whose lines are of up to so many neighbouring tokens
  const auto seen = [&](long tokens) {
    const long all = longest && longest < places ? longest : places;
    return window ? std::min(all, (long)window + sinks + tokens + 64) : all;
  };
  const bool all_tiles = c.head_size > ATTEND_FEW_HEAD && dtype == RPU_F32;
  if (!all_tiles && (r.starts_dev || lines <= ATTEND_FEW)) {
    p.few = r.starts_dev ? ATTEND_FEW : (int)lines;
    // Parts cost a join, 3 us, which so few positions do not take.  (us without and with parts.  36 units, heads of 64 bf16: 384 positions 7.7 and 8.8,
    // 768 10.9 and 8.9; float rows: 256 7.2 and 9.0, 512 9.8 and 9.1; floats: 256 10.3 and 10.7, 512 16 and 11.  144 units: bf16 768 11.8 and 12.5, 1024 14.8
    // and 13.7; floats 768 23 and 26, 1024 29 and 29.)
    const long units = (long)r.n * c.heads, most = seen(ATTEND_FEW / group + 1);
    const long alone = units >= 128 ? 768 : c.dtype == RPU_F32 ? 128 : dtype == RPU_F32 ? 256 : 384;
    p.few_splits = most <= alone ? 1 : splits_for(units, most, 32 * ATTEND_FEW_LEAST, 512, 4096);
    p.few_jobs = (long)r.n * c.heads * p.few_splits;
  }
  if (all_tiles || r.starts_dev || lines > ATTEND_FEW) {
    const long tiles = r.starts_dev ? attend::numbers_of(r.rows, (int)group, ATTEND_LINES, r.n) : (lines + ATTEND_LINES - 1) / ATTEND_LINES * r.n;
    if (tiles > INT_MAX) throw RpuError("So many rows and heads are too many for a call.");
    p.tiles = (int)tiles;
    // (tiles that there are if the rows are of one sequence, at most about as many workgroups without work as with it)
    const long least = r.starts_dev ? r.rows * group / ATTEND_LINES + 1 : tiles;
    // (Positions of floats cost most, so shorter parts pay: of at least 256 in 768 workgroups 109 and 36 us, of 512 in 256 137 and 49, for 23 sequences
    // of up to 275 tokens, 15 heads of 80 under a window of 777, and for 760 tokens of one, 14 heads of 72.  Of 16 bits the same parts lose: 84 to 108
    // and 13.6 to 16.6 us for 2865 tokens of 18 heads of 232 and 2 sequences of 261, 10 heads of 104.)
    const bool costly = c.dtype == RPU_F32 && !all_tiles;
    p.splits = splits_for(least * c.heads, seen(ATTEND_LINES / group + 1), costly ? 256 : 512, costly ? 768 : c.dtype == RPU_F32 ? 256 : 512, all_tiles ? 2048 : 0);
    p.splits = (int)std::max(1l, std::min<long>(p.splits, 2048 / (tiles * c.heads)));
    p.jobs = tiles * c.heads * p.splits;
  }
  // (sequences, tiles and parts are counted in 32 bits)
  if (std::max(p.few_jobs, p.jobs) > (1l << 30)) throw RpuError("So many sequences, rows and heads are too many for a call.");
  const auto take = [&](size_t n) {
    const size_t at = p.bytes;
    p.bytes += (n + 15) / 16 * 16;
    return at;
  };
  const size_t few = p.few_splits > 1 ? (size_t)p.few_jobs * p.few : 0, many = p.splits > 1 ? (size_t)p.splits * r.rows * q_heads : 0;
  p.few_part = take(few * 4 * c.head_size);
  p.few_stats = take(few * 8);
  p.part = take(many * 4 * c.head_size);
  p.stats = take(many * 8);
  return p;
}

} // namespace
} // namespace rpu_amd

using namespace rpu_amd;

extern "C" {

int rpu_cache_append(const rpu_cache *cache, const rpu_cache_rows *rows, const void *k_dev, long k_ld, const void *v_dev, long v_ld,
                     const void *q_dev, long q_ld, void *out_dev, long out_ld, int q_heads, int dtype, int device_id, void *stream) {
  return guarded([&] {
    AppendArgs a{};
    a.c = cache_dev(cache, dtype);
    a.r = rows_dev(*cache, rows);
    const size_t e = value_size(dtype), bytes = cache_bytes(*cache);
    const int width = width_of(cache->heads, *cache);
    std::vector<Span> read = numbers(*cache, *rows), written{dense("the cache's keys", cache->k_dev, bytes), dense("the cache's values", cache->v_dev, bytes)};
    read.push_back(matrix("k", k_dev, k_ld, a.r.rows, width, e));
    read.push_back(matrix("v", v_dev, v_ld, a.r.rows, width, e));
    apart(written[0], written[1]);
    if (q_dev) {
      const int q_width = width_of(q_heads, *cache);
      const Span q = matrix("q", q_dev, q_ld, a.r.rows, q_width, e), out = matrix("the output", out_dev, out_ld, a.r.rows, q_width, e);
      apart(out, q, true);
      for (const Span &w : written) {
        apart(w, q);
        apart(out, w);
      }
      for (const Span &r : read) apart(out, r);
    }
    for (const Span &w : written)
      for (const Span &r : read) apart(w, r);
    if (!a.r.rows) return;
    a.k = {const_cast<void *>(k_dev), k_ld};
    a.v = {const_cast<void *>(v_dev), v_ld};
    a.q = {const_cast<void *>(q_dev), q_ld};
    a.out = {out_dev, out_ld};
    a.q_heads = q_heads;
    const Gpu gpu(device_id);
    launch_cache_append(a, dtype, cache->dtype, gpu.cus(), (hipStream_t)stream);
    check_launch();
  });
}

size_t rpu_cache_attend_scratch(const rpu_cache *cache, const rpu_cache_rows *rows, int q_heads, int dtype, int window, int sinks, int longest) {
  size_t bytes = 0; // of operands that the call refuses: none
  (void)guarded([&] {
    (void)cache_dev(cache, dtype);
    if (rows_dev(*cache, rows).rows && width_of(q_heads, *cache) && q_heads % cache->heads == 0 && window >= 0 && sinks >= 0 && longest >= 0)
      bytes = attend_plan(*cache, *rows, q_heads, dtype, window, sinks, longest).bytes;
  });
  return bytes;
}

int rpu_cache_attend(const rpu_cache *cache, const rpu_cache_rows *rows, const void *q_dev, long q_ld, void *out_dev, long out_ld, int q_heads,
                     int dtype, float scale, int window, int sinks, int longest, void *scratch_dev, size_t scratch_bytes, int device_id,
                     void *stream) {
  return guarded([&] {
    AttendArgs a{};
    a.c = cache_dev(cache, dtype);
    a.r = rows_dev(*cache, rows);
    const size_t e = value_size(dtype), bytes = cache_bytes(*cache);
    const int width = width_of(q_heads, *cache);
    if (q_heads % cache->heads) throw RpuError("The heads of a row must be a multiple of the cache's.");
    if (!(std::fabs(scale) <= 1e30f)) throw RpuError("The scale must be finite, and at most 1e30.");
    if (window < 0 || sinks < 0) throw RpuError("window and sinks must not be negative.");
    if (sinks && !window) throw RpuError("Only a window has first tokens that stay visible.");
    if (longest < 0) throw RpuError("longest must not be negative.");
    const AttendPlan p = a.r.rows ? attend_plan(*cache, *rows, q_heads, dtype, window, sinks, longest) : AttendPlan{};
    const size_t need = p.bytes;
    if (scratch_bytes < need) throw RpuError("The scratch memory is too small.");
    const Span q = matrix("q", q_dev, q_ld, a.r.rows, width, e), out = matrix("the output", out_dev, out_ld, a.r.rows, width, e),
               scratch = dense("the scratch memory", scratch_dev, need);
    if (need && (uintptr_t)scratch_dev % 16) throw RpuError("The scratch memory is not aligned to 16 bytes.");
    std::vector<Span> read = numbers(*cache, *rows);
    read.push_back(dense("the cache's keys", cache->k_dev, bytes));
    read.push_back(dense("the cache's values", cache->v_dev, bytes));
    for (const Span &r : read) {
      apart(out, r);
      apart(scratch, r);
    }
    apart(out, q, true);
    apart(scratch, q);
    apart(scratch, out);
    if (!a.r.rows) return;
    a.q = {const_cast<void *>(q_dev), q_ld};
    a.out = {out_dev, out_ld};
    a.group = q_heads / cache->heads;
    a.scale = scale;
    a.window = window;
    a.sinks = sinks;
    a.few = p.few;
    a.few_splits = p.few_splits;
    a.splits = p.splits;
    a.tiles = p.tiles;
    a.few_jobs = p.few_jobs;
    a.jobs = p.jobs;
    char *const at = (char *)scratch_dev;
    a.few_part = (float *)(at + p.few_part);
    a.few_stats = (float2 *)(at + p.few_stats);
    a.part = (float *)(at + p.part);
    a.stats = (float2 *)(at + p.stats);
    const Gpu gpu(device_id);
    launch_cache_attend(a, dtype, cache->dtype, (hipStream_t)stream);
    check_launch();
  });
}

} // extern "C"
