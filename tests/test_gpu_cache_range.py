"""Calls of the paged cache that its documentation allows at the ends of their range, against the formula in 64 bits."""
import pytest
import torch

from aihwkit_amd import digital
from cache_oracle import U, bound_of
from test_gpu_cache import BF16, F16, F32, LAYOUTS, PAIR_IDS, PAIRS, Batch, numbers
from test_gpu_digital import close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("heads, kv, head", [(64, 16, 64), (24, 12, 128), (16, 16, 200)])
def test_many_rows_of_no_sequence_before_the_first(heads, kv, head, dtype, cache_dtype):
    """Tables of 256 positions, so that nothing goes in parts; in place, where a tile that two workgroups took would read its own output."""
    batch = Batch([(150, 60), (0, 9), (2, 30), (70, 5)], heads, kv, head, 16, dtype, cache_dtype, seed=61, before=900, behind=300).gpu()
    given = batch.q.clone()
    out = batch.attend()
    batch.check(out)
    assert (out[:900] == 0).all() and (out[-300:] == 0).all()
    mine = batch.q.clone()
    assert batch.attend(out=mine) is mine
    assert torch.equal(mine[900:-300], out[900:-300]) and torch.equal(mine[:900], given[:900]) and torch.equal(mine[-300:], given[-300:])


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("heads, kv, head", [(4, 2, 64), (2, 1, 128), (2, 1, 200)])
def test_scales_near_zero(heads, kv, head, dtype, cache_dtype):
    """The mean of what a row sees, of rows of zeros too (whose lift beside halves is the largest that there is)."""
    for layout in ("tokens", "mixed", "prompt"):
        batch = Batch(LAYOUTS[layout], heads, kv, head, 16, dtype, cache_dtype, seed=62).gpu()
        batch.q[::2] = 0.0
        batch.q[1::3, 1] = 1e-30
        for scale in (1e-12, -1e-20, 1e-37, 1e-42, 2.0 ** -149):
            batch.check(batch.attend(scale=scale), scale=scale)
        batch.check(batch.attend(scale=scale, window=50, sinks=3), scale=scale, window=50, sinks=3)


LONG = {"parts": ([(1, 5555), (60, 2000), (0, 10), (9, 0)], 4, 2, 64), "token": ([(1, 3000)], 4, 4, 64), "rows": ([(70, 5000)], 2, 1, 128), "long heads": ([(1, 2500), (30, 900)], 2, 2, 200),
        "mixed": (LAYOUTS["mixed"], 6, 2, 80)}


def whole_scores(name, dtype, cache_dtype, offset=lambda j: 0.0):
    """Queries and keys of whole numbers, so that scores are exact in any order of their terms, and an offset to the scores of position j."""
    layout, heads, kv, head = LONG[name]
    batch = Batch(layout, heads, kv, head, 16, dtype, cache_dtype, seed=63)
    gen = torch.Generator().manual_seed(64)
    keys = torch.randint(-2, 3, batch.keys.shape, generator=gen).to(cache_dtype)
    batch.keys = torch.where(batch.keys.isnan(), batch.keys, keys)
    batch.q = torch.randint(-2, 3, batch.q.shape, generator=gen).to(dtype).cuda()
    batch.q[..., 0] = 256.0
    for s, length in enumerate(batch.lengths):
        for j in range(length):
            batch.keys[int(batch.tables_host[s, j // 16]), :, j % 16, 0] = offset(j)
    return batch.gpu()


def check_exact(batch, difference, **kw):
    """As ``Batch.check``, of scores without an error: exponents are off by four roundings (the scale, log2 e, the score's distance to another and the product) of
    what counts of their difference."""
    expected, parts = batch.expected(**kw)
    parts["magnitude"].fill_(4 * difference / (batch.head + 6))
    within = slice(batch.starts_host[0], batch.starts_host[-1])
    close(batch.attend(**kw)[within], expected[within], bound_of(parts, batch.head, batch.dtype)[within])


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("name", LONG)
def test_large_scales(name, dtype, cache_dtype):
    """Only the largest scores count, all of them alike: they are whole numbers."""
    batch = whole_scores(name, dtype, cache_dtype)
    for scale in (300.0, 1e5, -1e9, 1e10, 3e17, -1e30):
        check_exact(batch, 0.0, scale=scale)
    check_exact(batch, 0.0, scale=scale, window=90, sinks=2)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("name", LONG)
def test_scores_far_from_zero(name, dtype, cache_dtype):
    """2^18 and more beside differences of a few: 2^-64 and less of a weight does not count."""
    for offset in (lambda j: 1024.0, lambda j: -1024.0, lambda j: -1024.0 if j < 700 else 1024.0, lambda j: 1024.0 if j % 64 == 7 else -8.0):
        batch = whole_scores(name, dtype, cache_dtype, offset)
        for scale in (0.05, 0.25, 1.0):
            check_exact(batch, 64.0, scale=scale)


@pytest.mark.parametrize("dtype, cache_dtype", [(F32, F32), (F32, BF16), (BF16, BF16)], ids=["f32-f32", "f32-bf16", "bf16-bf16"])
@pytest.mark.parametrize("heads, kv, head", [(4, 2, 64), (2, 1, 128), (2, 1, 200)])
@pytest.mark.parametrize("rise", [0.5, 1.375, 5.375])
def test_largest_values_under_rising_scores(rise, heads, kv, head, dtype, cache_dtype):
    """Two values of 1.5e38 in a head's column, whose scores are above the first that a row meets."""
    batch = Batch([(70, 200), (1, 300), (2, 5000), (40, 2000)], heads, kv, head, 16, dtype, cache_dtype, seed=65)
    batch.keys = torch.where(batch.keys.isnan(), batch.keys, torch.zeros((), dtype=cache_dtype))
    batch.q.zero_()
    batch.q[..., 0] = 1.0
    for s, length in enumerate(batch.lengths):
        for j in (100, batch.lengths[s] - batch.new[s] - 20):
            at = int(batch.tables_host[s, j // 16])
            batch.keys[at, :, j % 16, 0] = rise
            batch.values[at, :, j % 16, 5] = 1.5e38
    batch.gpu()
    assert torch.isfinite(batch.attend(scale=1.0)[batch.starts_host[0]:batch.starts_host[-1]]).all()
    check_exact(batch, 64.0, scale=1.0)


def named_places(batch, starts, lengths):
    """What rows of those starts and lengths, clamped to the rows and tables that there are, may be written to."""
    named = torch.zeros(batch.keys.shape[0], batch.keys.shape[2], dtype=torch.bool)
    page_size = batch.keys.size(2)
    for s in range(len(lengths)):
        begin = min(max(starts[s], 0), batch.rows)
        m = min(max(starts[s + 1], begin), batch.rows) - begin
        for p in range(max(lengths[s] - m, 0), min(lengths[s], batch.tables_host.size(1) * page_size)):
            page = int(batch.tables_host[s, p // page_size])
            if 0 <= page < batch.keys.size(0):
                named[page, p % page_size] = True
    return named


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("neighbours", [False, True], ids=["halves", "neighbours"])
def test_starts_lengths_and_tables_out_of_range_write_nowhere_else(neighbours, dtype, cache_dtype):
    """Cache, queries and output lie in larger memory: what is beside them, and every place of the cache that no row's sequence names, keeps its bits."""
    batch = Batch([(4, 30), (4, 0), (40, 9)], 4, 2, 64, 16, dtype, cache_dtype, seed=66)
    batch.tables_host[0, 1], batch.tables_host[2, 2] = 2 ** 31 - 1, batch.keys.size(0)
    count, bits = batch.keys.numel(), torch.int32 if cache_dtype == F32 else torch.int16
    room = torch.randint(-2 ** 15, 2 ** 15, (3 * 4096 + 2 * count,), generator=torch.Generator().manual_seed(67)).to(bits).cuda()
    keys, values = (room[4096 + k * (4096 + count):][:count].view(cache_dtype).view(batch.keys.shape) for k in range(2))
    cache = digital.PagedCache(keys, values, digital.rotation_frequencies(64)[:19], neighbours)
    whole = torch.full((batch.rows + 20, 4, 64), 7.0, dtype=dtype, device="cuda")
    out = whole[10:10 + batch.rows]
    rows = torch.ones(batch.rows, 2, 64, dtype=dtype, device="cuda")
    tables = batch.tables_host.cuda()
    for starts in ([-5, 4, 8, 1000], [40, 30, 20, 10], [2 ** 31 - 1, -(2 ** 31), 0, 5], [48, 48, 48, 48], [0, 4, 8, 48]):
        for lengths in ([2 ** 31 - 1] * 3, [-(2 ** 31)] * 3, [34, 4, 49]):
            given = dict(starts=numbers(starts), out=out)
            before = room.clone()
            cache.attend(batch.q, tables, numbers(lengths), **given)
            assert torch.equal(room, before)
            cache.append(rows, rows, tables, numbers(lengths), queries=batch.q, **given)
            named = named_places(batch, starts, lengths)
            if starts == [0, 4, 8, 48] and lengths == [34, 4, 49]:
                assert int(named.sum()) > 20 and (values.cpu().permute(0, 2, 1, 3)[named] == 1).all()
            for k, now in enumerate((keys, values)):
                then = before[4096 + k * (4096 + count):][:count].view(batch.keys.shape)
                now = now.view(bits)
                assert torch.equal(now.cpu().permute(0, 2, 1, 3)[~named], then.cpu().permute(0, 2, 1, 3)[~named])
                now.copy_(then)
            assert torch.equal(room, before)          # beside the cache
            assert (whole[:10] == 7).all() and (whole[10 + batch.rows:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("heads, kv, head", [(12, 12, 64), (14, 2, 80), (8, 2, 128), (3, 1, 256)])
def test_few_rows_of_16_bits_have_what_their_rounding_leaves(heads, kv, head, dtype):
    """Weights in two parts: each is off by half a step of what its rounding leaves, a quarter of eps squared, of halves at least 2^-25 / 2^7 of the largest
    (which is 2^7 and more when it is rounded).  What is stored is the number nearest to some value that near."""
    step = torch.finfo(dtype).eps ** 2 / 4
    for layout in ([(1, 0), (1, 30), (1, 129), (1, 500), (1, 1000)], [(3, 61), (2, 0), (2, 200)], [(1, 2500), (4, 40)]):
        batch = Batch(layout, heads, kv, head, 16, dtype, dtype, seed=68).gpu()
        for kw in (dict(), dict(window=70, sinks=3)):
            expected, parts = batch.expected(**kw)
            each = (head + 6) * U * parts["magnitude"] + 12 * U + parts["count"] * U
            limit = (2 * each + step) * parts["plain"] * (1 + 2 * each + step) + (2.0 ** -32 * parts["flat"] if dtype == F16 else 0.0) + 2 * U * expected.abs()
            got = batch.attend(**kw).cpu()
            assert (got >= (expected - limit).to(dtype)).all() and (got <= (expected + limit).to(dtype)).all()
