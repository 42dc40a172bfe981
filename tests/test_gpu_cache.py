"""Attention over a paged cache and what fills the cache, against their formulas in 64 bits (cache_oracle has the bounds)."""
import random

import pytest
import torch

from aihwkit_amd import _cabi, digital
from cache_oracle import U, attended, bound_of, rotated
from test_gpu_digital import BF16, F16, F32, NAMES, close, half_step, rand

pytestmark = pytest.mark.gpu

PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]      # rows, cache
PAIR_IDS = [f"{NAMES[a]}-{NAMES[b]}" for a, b in PAIRS]
NAN, INF = float("nan"), float("inf")


def numbers(values, **kw):
    return torch.tensor(values, dtype=torch.int32, device="cuda", **kw)


class Batch:
    """Sequences of (new, earlier) tokens on pages in any order; places that no sequence has are NaN."""

    def __init__(self, layout, heads, kv, head, page, dtype, cache_dtype, seed=0, before=0, behind=0, spread=2.0):
        rng = random.Random(seed)
        self.new, self.lengths = [m for m, _ in layout], [m + c for m, c in layout]
        self.head, self.kv, self.heads, self.dtype = head, kv, heads, dtype
        counts = [-(-length // page) for length in self.lengths]
        pages = sum(counts) + 2
        order = list(range(pages))
        rng.shuffle(order)
        width = max(counts) + 1
        self.tables_host = torch.full((len(layout), width), -1, dtype=torch.int32)
        self.keys = torch.full((pages, kv, page, head), NAN, dtype=cache_dtype)
        self.values = torch.full((pages, kv, page, head), NAN, dtype=cache_dtype)
        for s, count in enumerate(counts):
            mine, order = order[:count], order[count:]
            for k, at in enumerate(mine):
                self.tables_host[s, k] = at
                filled = min(page, self.lengths[s] - k * page)
                self.keys[at, :, :filled] = rand(seed * 1000 + 31 * s + k, kv, filled, head, dtype=cache_dtype).cpu()
                self.values[at, :, :filled] = rand(seed * 1000 + 31 * s + k + 500, kv, filled, head, dtype=cache_dtype).cpu()
        self.starts_host = [before + sum(self.new[:s]) for s in range(len(layout) + 1)]
        self.rows = self.starts_host[-1] + behind
        self.q = rand(seed + 7, self.rows, heads, head, dtype=dtype, std=spread)

    def gpu(self):
        self.cache = digital.PagedCache(self.keys.cuda(), self.values.cuda())
        self.tables, self.lengths_gpu, self.starts = self.tables_host.cuda(), numbers(self.lengths), numbers(self.starts_host)
        return self

    def attend(self, starts=True, **kw):
        return self.cache.attend(self.q, self.tables, self.lengths_gpu, starts=self.starts if starts else None, **kw)

    def expected(self, **kw):
        kw.setdefault("scale", self.head ** -0.5)
        return attended(self.q.double().cpu(), self.keys.double(), self.values.double(), self.tables_host, self.lengths, self.starts_host, **kw)

    def check(self, out, rows=None, **kw):
        expected, parts = self.expected(**kw)
        limit = bound_of(parts, self.head, self.dtype)
        within = slice(self.starts_host[0], self.starts_host[-1]) if rows is None else rows
        close(out[within], expected[within], limit[within])


# -- attend --------------------------------------------------------------------------------------------------------------

LAYOUTS = {
    "token": [(1, 0)], "tokens": [(1, 30), (1, 0), (1, 64), (1, 129), (1, 500)], "few": [(3, 61), (3, 0), (3, 200)], "prompt": [(97, 0)],
    "prompts": [(65, 0), (65, 0)], "chunks": [(40, 300), (40, 24), (40, 88)], "mixed": [(1, 700), (0, 40), (130, 70), (1, 0), (0, 0), (33, 31), (2, 126)],
}
HEADS = [(1, 1, 8), (12, 12, 64), (8, 2, 128), (14, 2, 80), (3, 1, 256), (5, 5, 24), (9, 3, 136), (40, 1, 64)]      # heads of rows and cache, size


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("heads, kv, head", HEADS)
def test_attend(layout, heads, kv, head, dtype, cache_dtype):
    batch = Batch(LAYOUTS[layout], heads, kv, head, 16, dtype, cache_dtype, seed=3).gpu()
    batch.check(batch.attend())
    if layout not in ("mixed",):
        batch.check(batch.attend(starts=False, longest=max(batch.lengths)))


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (64, 4), (100, 64), (130, 70), (5000, 3), (200, 4000), (3, 130)])
@pytest.mark.parametrize("heads, kv, head", [(4, 2, 64), (6, 1, 128)])
def test_windows_and_first_tokens(window, sinks, heads, kv, head, dtype, cache_dtype):
    for layout in ("tokens", "mixed", "prompt"):
        batch = Batch(LAYOUTS[layout], heads, kv, head, 32, dtype, cache_dtype, seed=5).gpu()
        batch.check(batch.attend(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("page", [8, 16, 64, 128, 1024])
@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_sizes_of_pages(page, dtype, cache_dtype):
    batch = Batch(LAYOUTS["mixed"], 4, 2, 64, page, dtype, cache_dtype, seed=6, before=3, behind=5).gpu()
    batch.check(batch.attend())
    batch.check(batch.attend(window=50, sinks=2), window=50, sinks=2)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_long_caches(dtype, cache_dtype):
    """Work that is split over the positions: one token and few rows over thousands of them, and beside short sequences."""
    for layout, heads, kv, head in (([(1, 9999)], 8, 2, 128), ([(5, 7001)], 3, 3, 64), ([(1, 6000), (1, 3), (1, 4095), (1, 64)], 4, 1, 72),
                                    ([(70, 5000)], 2, 1, 128), ([(1, 5555), (60, 2000), (0, 10), (9, 0)], 4, 2, 64)):
        batch = Batch(layout, heads, kv, head, 64, dtype, cache_dtype, seed=8).gpu()
        batch.check(batch.attend())
        if len(set(batch.new)) == 1:
            batch.check(batch.attend(starts=False))
        batch.check(batch.attend(window=1500, sinks=5), window=1500, sinks=5)
        batch.check(batch.attend(longest=100))      # too small a number costs time only


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("kv, group, head", [(48, 1, 64), (16, 3, 40), (7, 7, 8)])
def test_batches_of_many_rows(kv, group, head, dtype):
    """Thousands of rows of unlike sequences: the same bits as sequence by sequence, and (some rows) the formula."""
    layout = [(400, 90), (331, 0), (0, 17), (1, 499), (500, 12), (450, 3), (470, 1), (2, 300), (390, 100), (420, 20)]
    batch = Batch(layout, kv * group, kv, head, 16, dtype, dtype, seed=18, before=1, behind=3)
    batch.tables_host = batch.tables_host[:, :32].contiguous()      # 512 positions: no parts
    at = int(batch.tables_host[0, 3])
    batch.values[at, 0, 5, 2:5] = INF
    batch.gpu()
    for kw in (dict(), dict(window=70, sinks=5)):
        whole = batch.attend(**kw)
        assert (whole[:1] == 0).all() and (whole[-3:] == 0).all()
        for s in range(len(layout)):
            rows = slice(batch.starts_host[s], batch.starts_host[s + 1])
            if batch.new[s] > 2:       # (few rows go another way)
                alone = batch.cache.attend(batch.q[rows], batch.tables[s:s + 1], batch.lengths_gpu[s:s + 1], **kw)
                assert torch.equal(torch.nan_to_num(alone), torch.nan_to_num(whole[rows]))
        short = Batch.__new__(Batch)
        short.__dict__.update(batch.__dict__)
        for s, i in ((1, 0), (1, 330), (4, 255), (4, 256), (5, 100), (8, 389)):     # one row: of as many positions as there are up to it
            row = batch.starts_host[s] + i
            short.q, short.rows = batch.q[row:row + 1], 1
            short.tables_host, short.lengths, short.starts_host = batch.tables_host[s:s + 1], [batch.lengths[s] - batch.new[s] + i + 1], [0, 1]
            short.check(whole[row:row + 1], **kw)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("heads, kv, head", [(6, 2, 72), (5, 5, 8), (2, 1, 128), (2, 1, 200)])
@pytest.mark.parametrize("context", [700, 1300, 5000])
def test_joins_of_few_and_of_many_parts(context, heads, kv, head, dtype, cache_dtype):
    """Parts of rows beside parts of few tokens, empty sequences and rows of none; a window leaves most parts nothing."""
    batch = Batch([(70, context), (1, context - 90), (0, 5), (33, 0), (2, 600), (40, 129)], heads, kv, head, 16, dtype, cache_dtype, seed=21, before=2, behind=3).gpu()
    for kw in (dict(), dict(window=90, sinks=1)):
        out = batch.attend(**kw)
        batch.check(out, **kw)
        assert (out[:2] == 0).all() and (out[-3:] == 0).all()
    batch.tables[0, :40] = -1       # the first 640 positions of all of the rows: nothing for the first parts
    batch.tables_host[0, :40] = -1
    batch.check(batch.attend())
    alike = Batch([(70, context), (70, 0)], heads, kv, head, 16, dtype, cache_dtype, seed=22).gpu()
    alike.check(alike.attend(starts=False))


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 30.0])
def test_scales(scale, dtype, cache_dtype):
    batch = Batch(LAYOUTS["mixed"], 4, 2, 64, 16, dtype, cache_dtype, seed=9, spread=1.0).gpu()
    batch.check(batch.attend(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_scores_of_any_order_of_size(dtype, cache_dtype):
    """The largest score comes first, last, or grows from place to place; some differ by hundreds."""
    for order in (1, -1):
        batch = Batch([(3, 400), (200, 0)], 2, 1, 64, 16, dtype, cache_dtype, seed=10, spread=1.0)
        for s in range(2):
            for j in range(batch.lengths[s]):
                at = int(batch.tables_host[s, j // 16])
                batch.keys[at, :, j % 16, 0] = order * (j - 200) * 0.25
        batch.q[:, :, 0] = 8.0
        batch.gpu()
        batch.check(batch.attend())


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_rows_that_see_nothing_are_zeros(dtype, cache_dtype):
    batch = Batch([(6, 0), (70, 10), (1, 40)], 4, 2, 64, 16, dtype, cache_dtype, seed=11).gpu()
    # fewer positions than rows, none at all, fewer than none
    for lengths in ([2, 30, 0], [0, 0, 0], [-5, -(2 ** 31), -1]):
        batch.lengths, batch.lengths_gpu = lengths, numbers(lengths)
        out = batch.attend()
        batch.check(out)
        for s in range(3):
            none = max(0, min(batch.new[s], batch.new[s] - lengths[s]))
            assert (out[batch.starts_host[s]:batch.starts_host[s] + none] == 0).all()


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_pages_that_are_not_there(dtype, cache_dtype):
    """Holes in tables, and lengths beyond them: positions without a page are not seen."""
    batch = Batch([(1, 200), (80, 150), (4, 60)], 4, 2, 64, 16, dtype, cache_dtype, seed=12)
    batch.tables_host[0, 3], batch.tables_host[0, 0], batch.tables_host[1, 5] = -1, 2 ** 31 - 1, batch.keys.size(0)
    batch.tables_host[1, 8:] = -7
    batch.tables_host[2, :] = -(2 ** 31)
    batch.gpu()
    out = batch.attend()
    batch.check(out)
    assert (out[batch.starts_host[2]:] == 0).all()
    batch.check(batch.attend(window=40, sinks=20), window=40, sinks=20)
    batch.tables_host, batch.tables = batch.tables_host[:, :6].contiguous(), batch.tables[:, :6]
    batch.check(batch.attend())
    batch.lengths = [2 ** 31 - 1, 150, 64]
    batch.lengths_gpu = numbers(batch.lengths)
    batch.check(batch.attend())


def test_starts_and_lengths_out_of_range_touch_nothing_else():
    batch = Batch([(4, 30), (4, 0), (40, 9)], 4, 2, 64, 16, BF16, BF16, seed=13).gpu()
    whole = torch.full((batch.rows + 20, 4, 64), 7.0, dtype=BF16, device="cuda")
    out = whole[10:10 + batch.rows]
    keys = torch.nan_to_num(batch.cache.keys, nan=3.0)
    for starts in ([-5, 4, 8, 1000], [40, 30, 20, 10], [2 ** 31 - 1, -(2 ** 31), 0, 5], [48, 48, 48, 48]):
        for lengths in ([2 ** 31 - 1] * 3, [-(2 ** 31)] * 3, [34, 4, 49]):
            batch.cache.attend(batch.q, batch.tables, numbers(lengths), starts=numbers(starts), out=out)
            batch.cache.append(torch.zeros(batch.rows, 2, 64, dtype=BF16, device="cuda"), torch.zeros(batch.rows, 2, 64, dtype=BF16, device="cuda"),
                               batch.tables, numbers(lengths), starts=numbers(starts), queries=batch.q, out=out)
            assert (whole[:10] == 7).all() and (whole[10 + batch.rows:] == 7).all()
    assert keys.shape == batch.cache.keys.shape


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_what_is_not_seen_does_not_reach_a_row(bad, dtype, cache_dtype):
    """Values and keys of later positions, of positions behind the window, of another head and of unused places."""
    check_poisoned(bad, 64, dtype, cache_dtype)


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("head", [40, 80, 128, 176, 256])
@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_what_is_not_seen_does_not_reach_rows_of_other_heads(head, bad, dtype, cache_dtype):
    check_poisoned(bad, head, dtype, cache_dtype)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("window, sinks", [(1, 1), (64, 4), (100, 64), (3, 130)])
@pytest.mark.parametrize("heads, kv, head", [(5, 5, 80), (2, 1, 200), (3, 1, 256)])
def test_windows_of_other_heads(heads, kv, head, window, sinks, dtype, cache_dtype):
    for layout in ("tokens", "mixed"):
        batch = Batch(LAYOUTS[layout], heads, kv, head, 32, dtype, cache_dtype, seed=23).gpu()
        batch.check(batch.attend(window=window, sinks=sinks), window=window, sinks=sinks)


def check_poisoned(bad, head, dtype, cache_dtype):
    batch = Batch([(140, 60), (3, 130), (1, 300)], 4, 2, head, 16, dtype, cache_dtype, seed=14)
    poisoned = {0: [100, 127, 150, 199], 1: [132, 5], 2: [7, 100]}
    for s, places in poisoned.items():
        for j in places:
            at = int(batch.tables_host[s, j // 16])
            batch.values[at, :, j % 16, 3:30] = bad
            batch.keys[at, 1, j % 16, 5] = bad
    batch.gpu()
    for kw in (dict(), dict(window=33, sinks=4), dict(window=70, sinks=0)):
        out = batch.attend(**kw).double().cpu()
        expected, parts = batch.expected(**kw)
        limit = bound_of(parts, head, dtype)
        fine = torch.ones(batch.rows, dtype=torch.bool)
        for s, places in poisoned.items():
            for i in range(batch.new[s]):
                p = batch.lengths[s] - batch.new[s] + i
                for j in places:
                    if j <= p and ("window" not in kw or j > p - kw["window"] or j < kw["sinks"]):
                        fine[batch.starts_host[s] + i] = False
        assert int(fine.sum()) > 20
        close(out[fine].to(dtype), expected[fine], limit[fine])
        # where such values are seen the columns beside them are what they are, and the columns themselves not numbers
        seen = ~fine
        close(out[seen][:, :2, 30:].to(dtype), expected[seen][:, :2, 30:], limit[seen][:, :2, 30:])
        assert not torch.isfinite(out[seen][:, :2, 3:30]).any()


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_infinite_and_undefined_queries_stay_with_their_row(dtype, cache_dtype):
    batch = Batch([(40, 100), (1, 70)], 4, 2, 64, 16, dtype, cache_dtype, seed=15).gpu()
    clean = batch.attend()
    batch.q[7, 1, 5], batch.q[30, 2, 0] = NAN, INF
    out = batch.attend()
    assert torch.isnan(out[7, 1]).all()
    same = torch.ones(41, 4, dtype=torch.bool)
    same[7, 1] = same[30, 2] = False
    assert torch.equal(out[same], clean[same])


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_layouts_of_operands(dtype, cache_dtype):
    """Queries as a column slice of a joint projection that begins at any value, outputs in a slice whose other columns stay, wide tables, and
    in place."""
    batch = Batch(LAYOUTS["mixed"], 4, 2, 64, 16, dtype, cache_dtype, seed=16, before=2, behind=3).gpu()
    plain = batch.attend()
    assert (plain[:2] == 0).all() and (plain[-3:] == 0).all()
    wide = torch.full((batch.rows, 3 + 256 + 9), NAN, dtype=dtype, device="cuda")
    wide[:, 3:259] = batch.q.view(batch.rows, 256)
    sliced = wide[:, 3:259].unflatten(1, (4, 64))
    space = torch.full((batch.rows, 5 + 256 + 2), 9.0, dtype=dtype, device="cuda")
    out = space[:, 5:261].unflatten(1, (4, 64))
    tables = torch.full((len(batch.lengths), batch.tables.size(1) + 7), 10 ** 6, dtype=torch.int32, device="cuda")
    tables[:, 4:-3] = batch.tables
    given = batch.cache.attend(sliced, tables[:, 4:-3], batch.lengths_gpu, starts=batch.starts, out=out)
    assert given is out and torch.equal(out[2:-3], plain[2:-3])
    assert (space[:, :5] == 9).all() and (space[:, 261:] == 9).all() and (space[:2] == 9).all() and (space[-3:] == 9).all()
    turned = batch.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(batch.cache.attend(turned, batch.tables, batch.lengths_gpu, starts=batch.starts), plain)
    mine = batch.q.clone()
    batch.cache.attend(mine, batch.tables, batch.lengths_gpu, starts=batch.starts, out=mine)
    assert torch.equal(mine[2:-3], plain[2:-3]) and torch.equal(mine[:2], batch.q[:2]) and torch.equal(mine[-3:], batch.q[-3:])
    assert torch.equal(batch.attend(), plain)      # the same bits at every run


def test_offsets_beyond_32_bits():
    """A cache of 4.4 GB of keys and as many of values whose last pages are used."""
    pages = (1 << 31) // (8 * 64 * 128) + 300
    keys, values = torch.empty(2, pages, 8, 64, 128, dtype=BF16, device="cuda")
    small = Batch([(1, 700), (50, 100)], 16, 8, 128, 64, BF16, BF16, seed=17).gpu()
    n = small.keys.size(0)
    keys[pages - n:], values[pages - n:] = small.cache.keys, small.cache.values
    tables = torch.where(small.tables >= 0, small.tables + (pages - n), small.tables)
    cache = digital.PagedCache(keys, values)
    assert torch.equal(cache.attend(small.q, tables, small.lengths_gpu, starts=small.starts), small.attend())
    k, v = rand(1, small.rows, 8, 128, dtype=BF16), rand(2, small.rows, 8, 128, dtype=BF16)
    cache.append(k, v, tables, small.lengths_gpu, starts=small.starts)
    small.cache.append(k, v, small.tables, small.lengths_gpu, starts=small.starts)
    assert torch.equal(torch.nan_to_num(keys[pages - n:]), torch.nan_to_num(small.cache.keys))
    assert torch.equal(torch.nan_to_num(values[pages - n:]), torch.nan_to_num(small.cache.values))


# -- append --------------------------------------------------------------------------------------------------------------

def test_more_workgroups_than_a_launch_has():
    """Of 256 threads each, 2^24 workgroups: what they do is the same as in a small call, all the way to the last."""
    n, period = (1 << 24) + 37, 512
    keys, values = (rand(seed, 3, 1, 8, 8, dtype=F16).cuda() for seed in (51, 52))
    cache = digital.PagedCache(keys, values)
    tables = numbers([[k % 4 - 1] for k in range(period)])
    lengths, q = numbers([k % 9 for k in range(period)]), rand(53, period, 1, 8, dtype=F16).cuda()
    times = -(-n // period)
    few = cache.attend(q, tables, lengths)
    many = cache.attend(q.repeat(times, 1, 1)[:n], tables.repeat(times, 1)[:n], lengths.repeat(times)[:n])
    assert torch.equal(many, few.repeat(times, 1, 1)[:n])
    # rows of a key and a value each: two to a workgroup
    rows = (1 << 25) + 37
    pages = -(-rows // 65536)
    k = torch.arange(8 * rows, dtype=torch.int32, device="cuda").remainder_(2039).to(F16).view(rows, 1, 8)
    cache = digital.PagedCache(torch.full((pages, 1, 65536, 8), -1.0, dtype=F16, device="cuda"), torch.full((pages, 1, 65536, 8), -1.0, dtype=F16, device="cuda"))
    cache.append(k, k, numbers([list(range(pages))]), numbers([rows]))
    for held in (cache.keys, cache.values):
        assert torch.equal(held.view(-1, 1, 8)[:rows], k) and (held.view(-1, 8)[rows:] == -1).all()


def check_append(batch, frequencies, neighbours, starts=True, layout=lambda t: t):
    """Against the formula; what is not a new row's place keeps its bits."""
    cache = digital.PagedCache(batch.keys.cuda(), batch.values.cuda(), frequencies, neighbours)
    total, dtype, cache_dtype = batch.rows, batch.dtype, batch.keys.dtype
    k, v = rand(21, total, batch.kv, batch.head, dtype=dtype), rand(22, total, batch.kv, batch.head, dtype=dtype)
    out = cache.append(layout(k), layout(v), batch.tables_host.cuda(), numbers(batch.lengths), starts=numbers(batch.starts_host) if starts else None,
                       queries=layout(batch.q))
    f = torch.zeros(0, dtype=torch.float64) if frequencies is None else frequencies
    page_size = batch.keys.size(2)
    untouched = torch.ones(batch.keys.shape[0], page_size, dtype=torch.bool)
    for s, m in enumerate(batch.new):
        if not m:
            continue
        rows = slice(batch.starts_host[s], batch.starts_host[s + 1])
        positions = torch.arange(batch.lengths[s] - m, batch.lengths[s])
        # cosine and sine are off by 4 U each, the products and their sum by a rounding each
        for source, got in ((batch.q, out[rows].cpu()), (k, None)):
            x = source[rows].double().cpu()
            expected = rotated(x, positions, f, neighbours)
            size = rotated(x.abs(), torch.zeros(m), f, neighbours)
            partner = size.clone()
            pairs = f.numel()
            a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
            partner[..., a], partner[..., b] = size[..., b], size[..., a]
            limit = 8 * U * (size + partner)
            limit[..., 2 * pairs:] = 0.0
            if got is not None:
                close(got, expected, limit)
                continue
            for i, p in enumerate(positions.tolist()):
                page = int(batch.tables_host[s, p // page_size]) if 0 <= p < batch.tables_host.size(1) * page_size else -1
                if 0 <= page < batch.keys.size(0):
                    untouched[page, p % page_size] = False
                    close(cache.keys[page, :, p % page_size], expected[i], limit[i])
                    assert torch.equal(cache.values[page, :, p % page_size].cpu(), v[rows][i].cpu().to(cache_dtype))
    for now, then in ((cache.keys, batch.keys), (cache.values, batch.values)):
        now, then = now.cpu().permute(0, 2, 1, 3)[untouched], then.permute(0, 2, 1, 3)[untouched]
        assert torch.equal(now.view(torch.int16 if cache_dtype != F32 else torch.int32), then.view(torch.int16 if cache_dtype != F32 else torch.int32))
    return cache, out


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("heads, kv, head", HEADS)
@pytest.mark.parametrize("pairs", ["none", "one", "some", "all"])
@pytest.mark.parametrize("neighbours", [False, True], ids=["halves", "neighbours"])
def test_append(heads, kv, head, pairs, neighbours, dtype, cache_dtype):
    count = {"none": 0, "one": 1, "some": head // 4 + 1, "all": head // 2}[pairs]
    f = digital.rotation_frequencies(head)[:count] if count else None
    batch = Batch(LAYOUTS["mixed"], heads, kv, head, 16, dtype, cache_dtype, seed=20, before=1, behind=4)
    _, out = check_append(batch, f, neighbours)
    assert (out[:1] == 0).all() and (out[-4:] == 0).all()


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_append_of_equal_shares_far_positions_and_bad_places(dtype, cache_dtype):
    f = digital.rotation_frequencies(64)
    check_append(Batch([(3, 5), (3, 0), (3, 77)], 4, 2, 64, 8, dtype, cache_dtype, seed=23), f, False, starts=False)
    # on a table of pages that are not there but for the last: positions around 2^29
    page = 65536
    batch = Batch([(2, 0)], 4, 2, 64, page, dtype, cache_dtype, seed=24)
    batch.tables_host = torch.full((1, 8192), -1, dtype=torch.int32)
    batch.tables_host[0, 8191] = 1
    for length in (2 ** 29 + 5, 2 ** 29, 2 ** 29 + 1, 2 ** 31 - 1, 1, 0, -(2 ** 31)):
        batch.lengths = [length]
        check_append(batch, f, True)
    batch = Batch([(40, 60), (1, 5)], 4, 2, 64, 16, dtype, cache_dtype, seed=25)
    batch.tables_host[0, 4], batch.tables_host[0, 5], batch.tables_host[1, 0] = -2, 2 ** 31 - 1, batch.keys.size(0)
    check_append(batch, f, False)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_append_of_slices_and_in_place(dtype, cache_dtype):
    f = digital.rotation_frequencies(80)[:19]

    def slice_of(t):
        wide = torch.full((t.size(0), 5 + t[0].numel() + 2), NAN, dtype=t.dtype, device="cuda")
        wide[:, 5:-2] = t.flatten(1)
        return wide[:, 5:-2].unflatten(1, t.shape[1:])

    batch = Batch(LAYOUTS["mixed"], 4, 2, 80, 16, dtype, cache_dtype, seed=26)
    for neighbours in (False, True):
        _, out = check_append(batch, f, neighbours, layout=slice_of)
        cache = digital.PagedCache(batch.keys.cuda(), batch.values.cuda(), f, neighbours)
        k, mine = rand(21, batch.rows, 2, 80, dtype=dtype), batch.q.clone()
        args = (k, k, batch.tables_host.cuda(), numbers(batch.lengths))
        assert cache.append(*args, starts=numbers(batch.starts_host), queries=mine, out=mine) is mine and torch.equal(mine, out)
        assert cache.append(*args, starts=numbers(batch.starts_host)) is None


def test_values_beyond_a_half_become_infinite_and_nan_stays():
    cache = digital.PagedCache(*torch.zeros(2, 2, 1, 8, 8, dtype=F16, device="cuda"))
    k = torch.tensor([[1e6, -1e6, NAN, 65519.0, 65520.0, 1e-9, -0.0, INF]], device="cuda").view(1, 1, 8)
    cache.append(k, k, numbers([[1]]), numbers([2]))
    for t in (cache.keys, cache.values):
        assert torch.equal(torch.nan_to_num(t[1, 0, 1]), torch.nan_to_num(k[0, 0].half()))


# -- calls ---------------------------------------------------------------------------------------------------------------

def steps(batch, k, v, f):
    """One append and attend on a fresh cache: everything that they give."""
    cache = digital.PagedCache(torch.nan_to_num(batch.keys).cuda(), torch.nan_to_num(batch.values).cuda(), f)
    rotated_q = cache.append(k, v, batch.tables, batch.lengths_gpu, starts=batch.starts, queries=batch.q)
    same = cache.append(k[:4], v[:4], batch.tables[:2], batch.lengths_gpu[:2], queries=batch.q[:4])
    out = cache.attend(rotated_q, batch.tables, batch.lengths_gpu, starts=batch.starts, window=90, sinks=3, longest=800)
    few = cache.attend(rotated_q[:4], batch.tables[:2], batch.lengths_gpu[:2], scale=0.2)
    return cache.keys, cache.values, rotated_q, same, out, few


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
def test_the_general_path_gives_the_same_results(dtype, cache_dtype, monkeypatch):
    batch = Batch(LAYOUTS["mixed"], 4, 2, 64, 16, dtype, cache_dtype, seed=30, behind=2).gpu()
    k, v, f = rand(1, batch.rows, 2, 64, dtype=dtype), rand(2, batch.rows, 2, 64, dtype=dtype), digital.rotation_frequencies(64)
    native = steps(batch, k, v, f)
    with monkeypatch.context() as patch:
        patch.setattr(_cabi, "_torch_calls", _cabi._GeneralPath())
        general = steps(batch, k, v, f)
    for a, b in zip(native, general):
        assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)


def test_what_the_native_calls_take_and_what_is_refused(monkeypatch):
    m, batch = _cabi.torch_calls(), Batch([(1, 40), (1, 9)], 4, 2, 64, 16, BF16, BF16, seed=31).gpu()
    c, k = batch.cache, rand(1, 2, 2, 64, dtype=BF16)
    t, lengths = batch.tables, batch.lengths_gpu
    assert m.cache_attend(c.keys, c.values, c._shape, batch.q, t, lengths, None, None, 0, 0, None, None, True) is not None
    assert m.cache_attend(c.keys, c.values, c._shape, batch.q.float(), t, lengths, batch.starts, 0.5, 9, 2, 50, None, True) is not None
    assert m.cache_append(c.keys, c.values, c._shape, None, False, k, k, t, lengths, None, batch.q, None, True) is not None
    assert m.cache_append(c.keys, c.values, c._shape, None, False, k, k, t, lengths, batch.starts, None, None, True) == (None,)
    for path in ("native", "general"):
        with monkeypatch.context() as patch:
            if path == "general":
                patch.setattr(_cabi, "_torch_calls", _cabi._GeneralPath())
            for error, text, call in (
                    (RuntimeError, "multiple of the cache", lambda: c.attend(batch.q[:, :3], t, lengths)),
                    (RuntimeError, "rows' type", lambda: c.attend(batch.q.half(), t, lengths)),
                    (RuntimeError, "expected", lambda: c.attend(batch.q[..., :56], t, lengths)),
                    (RuntimeError, "expected", lambda: c.attend(batch.q.flatten(1), t, lengths)),
                    (RuntimeError, "int32", lambda: c.attend(batch.q, t.long(), lengths)),
                    (RuntimeError, "int32", lambda: c.attend(batch.q, t, lengths.cpu())),
                    (TypeError, "starts", lambda: c.attend(batch.q, t, lengths, starts=[0, 1, 2])),
                    (RuntimeError, "starts", lambda: c.attend(batch.q, t, lengths, starts=batch.starts[:2])),
                    (RuntimeError, "as many rows each", lambda: c.attend(batch.q[:1], t, lengths)),
                    (RuntimeError, "as many sequences", lambda: c.attend(batch.q, t, lengths[:1])),
                    (RuntimeError, "dimension", lambda: c.attend(batch.q, t[0], lengths)),
                    (RuntimeError, "0 .. 2", lambda: c.attend(batch.q, t, lengths, window=-1)),
                    (RuntimeError, "0 .. 2", lambda: c.attend(batch.q, t, lengths, longest=1 << 40)),
                    (RuntimeError, "Only a window", lambda: c.attend(batch.q, t, lengths, sinks=2)),
                    (RuntimeError, "scale", lambda: c.attend(batch.q, t, lengths, scale=NAN)),
                    (RuntimeError, "out", lambda: c.attend(batch.q, t, lengths, out=batch.q[:1].clone())),
                    (RuntimeError, "out", lambda: c.attend(batch.q, t, lengths, out=batch.q.float())),
                    (RuntimeError, "lie in a row", lambda: c.attend(batch.q, t, lengths, out=torch.empty(4, 2, 64, dtype=BF16, device="cuda").transpose(0, 1))),
                    (RuntimeError, "overlaps", lambda: c.attend(batch.q, t, lengths, out=c.keys.view(-1)[:512].view(2, 4, 64))),
                    (RuntimeError, "cache's 2 heads", lambda: c.append(k[:, :1], k[:, :1], t, lengths)),
                    (RuntimeError, "cache's 2 heads", lambda: c.append(k, k[:1], t, lengths)),
                    (RuntimeError, "type", lambda: c.append(k, k.float(), t, lengths)),
                    (RuntimeError, "no queries", lambda: c.append(k, k, t, lengths, out=batch.q)),
                    (RuntimeError, "queries", lambda: c.append(k, k, t, lengths, queries=batch.q[:1])),
                    (RuntimeError, "overlaps", lambda: c.append(k, c.values.view(-1)[:256].view(2, 2, 64), t, lengths))):
                with pytest.raises(error, match=text):
                    call()
    for error, text, make in (
            (RuntimeError, "power of two", lambda: digital.PagedCache(c.keys[:, :, :12].contiguous(), c.values[:, :, :12].contiguous())),
            (RuntimeError, "multiple of 8", lambda: digital.PagedCache(c.keys[..., :12].contiguous(), c.values[..., :12].contiguous())),
            (RuntimeError, "dense", lambda: digital.PagedCache(c.keys[:, :1], c.values[:, :1])),
            (RuntimeError, "dense", lambda: digital.PagedCache(c.keys, c.values[:1])),
            (RuntimeError, "one type", lambda: digital.PagedCache(c.keys, c.values.half())),
            (RuntimeError, "CUDA", lambda: digital.PagedCache(c.keys, c.values.cpu())),
            (RuntimeError, "half a head", lambda: digital.PagedCache(c.keys, c.values, digital.rotation_frequencies(80))),
            (TypeError, "frequencies", lambda: digital.PagedCache(c.keys, c.values, [1.0]))):
        with pytest.raises((error, RuntimeError), match=text):
            make()
    other = digital.PagedCache(c.keys, c.values)
    other.keys = c.keys[:1].contiguous()
    with pytest.raises(RuntimeError, match="dense"):
        other.attend(batch.q, t, lengths)


def test_no_rows():
    batch = Batch([(1, 40)], 4, 2, 64, 16, F32, BF16, seed=32).gpu()
    none = batch.q[:0]
    assert batch.cache.attend(none, batch.tables, batch.lengths_gpu).shape == (0, 4, 64)
    assert batch.cache.append(none[:, :2], none[:, :2], batch.tables, batch.lengths_gpu, queries=none).shape == (0, 4, 64)


def test_streams():
    """Calls on streams of their own at the same time, each with scratch of its own."""
    batches = [Batch([(1, 5000 + 700 * i), (30, 1000)], 4, 2, 64, 16, BF16, BF16, seed=33 + i).gpu() for i in range(3)]
    expected = [b.attend() for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for b, s in zip(batches, streams):
            with torch.cuda.stream(s):
                got.append(b.attend(non_blocking=True))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


def test_captured_steps_follow_their_numbers():
    """Two captured steps with tables, lengths and rows of their own, replayed in turn with eager calls between them."""
    f = digital.rotation_frequencies(64)
    graphs = []
    for seed, dtype, cache_dtype in ((40, BF16, BF16), (41, F32, BF16)):
        batch = Batch([(1, 3000), (1, 17)], 4, 2, 64, 16, dtype, cache_dtype, seed=seed).gpu()
        cache = digital.PagedCache(torch.nan_to_num(batch.cache.keys), torch.nan_to_num(batch.cache.values), f)
        k, v, lengths = rand(seed, 2, 2, 64, dtype=dtype), rand(seed + 1, 2, 2, 64, dtype=dtype), batch.lengths_gpu.clone()

        def step(cache=cache, batch=batch, k=k, v=v, lengths=lengths):
            q = cache.append(k, v, batch.tables, lengths, queries=batch.q, non_blocking=True)
            return cache.attend(q, batch.tables, lengths, longest=3100, non_blocking=True)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, step, k, lengths))
    for turn in range(4):
        for graph, out, step, k, lengths in graphs:
            k.copy_(rand(100 + turn, *k.shape, dtype=k.dtype))
            lengths.copy_(numbers([3001 - 40 * turn, 18 - turn]))
            graph.replay()
            torch.cuda.synchronize()
            replayed = out.clone()
            assert torch.equal(replayed, step()) and torch.isfinite(replayed).all()


def test_captured_mixed_batches():
    """The padded batch of a serving step: starts, lengths and tables change from replay to replay."""
    batch = Batch(LAYOUTS["mixed"], 4, 2, 64, 16, BF16, BF16, seed=44, behind=40).gpu()
    out = torch.full_like(batch.q, 5.0)
    batch.attend(out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.attend(out=out, non_blocking=True)
    for new in (LAYOUTS["mixed"], [(0, 1), (0, 0), (1, 5), (1, 30), (20, 0), (3, 60), (1, 0)], [(0, 0)] * 7):
        batch.new = [min(m, length) for (m, _), length in zip(new, batch.lengths)]
        batch.starts_host = [sum(batch.new[:s]) for s in range(8)]
        batch.starts.copy_(numbers(batch.starts_host))
        for _ in range(2):
            out.fill_(5.0)
            graph.replay()
            torch.cuda.synchronize()
            if batch.starts_host[-1]:
                batch.check(out)
            assert (out[batch.starts_host[-1]:] == 5).all()


def test_a_run_beside_tiles():
    """A transformer block's attention as it is served: projections as inference tiles, layer norm, append and attend between them.  Prompts in
    one call, then token by token, against the whole prompts at once."""
    from aihwkit_amd.inference import InferenceTile
    from aihwkit_amd.rpu_base import devices as dv
    io = dv.AnalogTileInputOutputParameter()
    io.is_perfect = True
    heads, head, width = 4, 16, 64

    def tile(out_size, in_size, seed):
        t = InferenceTile(out_size, in_size, forward_io=io)
        t.set_weights(rand(seed, out_size, in_size, std=0.1).cpu())
        t.cuda()
        return t

    project, merge = tile(3 * width, width, 1), tile(width, width, 2)
    w, b = 1 + rand(3, width, std=0.1), rand(4, width, std=0.1)
    cache = digital.PagedCache(*torch.full((2, 12, heads, 8, head), NAN, dtype=F32, device="cuda"), digital.rotation_frequencies(head))
    tables = numbers([[7, 2, 9, -1], [0, 11, 5, -1]])
    x = rand(5, 2, 20, width)      # two sequences of 20 tokens

    def block(rows, lengths, starts=None):
        z, _, _ = digital.layer_norm(rows, w, b, 1e-5)
        joint = project.forward(z, is_test=True).view(-1, 3, heads, head)
        q = cache.append(joint[:, 1], joint[:, 2], tables, lengths, starts=starts, queries=joint[:, 0])
        mixed = cache.attend(q, tables, lengths, starts=starts)
        return digital.dropout(merge.forward(mixed.view(-1, width), is_test=True), 0.0, 0, base=rows)

    whole = block(x.reshape(40, width), numbers([20, 20])).view(2, 20, width)
    cache.keys.fill_(NAN)
    cache.values.fill_(NAN)
    first = block(torch.cat((x[0, :13], x[1, :7])), numbers([13, 7]), numbers([0, 13, 20]))
    got = [[first[:13]], [first[13:]]]
    for t in range(7):
        one = block(torch.stack((x[0, 13 + t], x[1, 7 + t])), numbers([14 + t, 8 + t]))
        got[0].append(one[:1])
        got[1].append(one[1:])
    # against the definition in 64 bits; values of order one through sums of 64 terms in four stages
    f, wq, wm = x.double().cpu(), project.get_weights().double(), merge.get_weights().double()
    c = f - f.mean(-1, keepdim=True)
    z = c * (c.square().mean(-1, keepdim=True) + 1e-5) ** -0.5 * w.double().cpu() + b.double().cpu()
    q, k, v = (z @ wq.T).view(2, 20, 3, heads, head).unbind(2)
    position, freq = torch.arange(20), digital.rotation_frequencies(head)
    for s in range(2):
        qs, ks = rotated(q[s], position, freq, False), rotated(k[s], position, freq, False)
        scores = torch.einsum("ihd,jhd->hij", qs, ks) * head ** -0.5
        scores = scores.masked_fill(torch.triu(torch.ones(20, 20, dtype=torch.bool), 1), -INF)
        mixed = torch.einsum("hij,jhd->ihd", torch.softmax(scores, -1), v[s]).reshape(20, width)
        expected = f[s] + mixed @ wm.T
        limit = 1000 * U * max(1.0, float(expected.abs().max()))
        assert float((whole[s].double().cpu() - expected).abs().max()) <= limit
        mine = torch.cat(got[s])
        assert float((mine.double().cpu() - expected[:mine.size(0)]).abs().max()) <= limit
    assert half_step(F32) == U
