"""Calls of the paged cache that its documentation allows at the ends of their range, against the formula in 64 bits."""
import pytest
import torch

from cache_oracle import bound_of
from test_gpu_cache import BF16, F32, LAYOUTS, PAIR_IDS, PAIRS, Batch
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
@pytest.mark.parametrize("scale", [1e-12, -1e-20, 1e-37, 1e-42, 2.0 ** -149])
def test_scales_near_zero(scale, heads, kv, head, dtype, cache_dtype):
    """The mean of what a row sees, of rows of zeros too (whose lift beside halves is the largest that there is)."""
    for layout in ("tokens", "mixed", "prompt"):
        batch = Batch(LAYOUTS[layout], heads, kv, head, 16, dtype, cache_dtype, seed=62).gpu()
        batch.q[::2] = 0.0
        batch.q[1::3, 1] = 1e-30
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
@pytest.mark.parametrize("scale", [300.0, 1e5, -1e9, 1e10, 3e17, -1e30])
def test_large_scales(scale, name, dtype, cache_dtype):
    """Only the largest scores count, all of them alike: they are whole numbers."""
    batch = whole_scores(name, dtype, cache_dtype)
    check_exact(batch, 0.0, scale=scale)
    check_exact(batch, 0.0, scale=scale, window=90, sinks=2)


@pytest.mark.parametrize("dtype, cache_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("name", LONG)
@pytest.mark.parametrize("offset", [lambda j: 1024.0, lambda j: -1024.0, lambda j: -1024.0 if j < 700 else 1024.0, lambda j: 1024.0 if j % 64 == 7 else -8.0],
                         ids=["high", "low", "rising", "few"])
@pytest.mark.parametrize("scale", [0.05, 0.25, 1.0])
def test_scores_far_from_zero(scale, offset, name, dtype, cache_dtype):
    """2^18 and more beside differences of a few: 2^-64 and less of a weight does not count."""
    check_exact(whole_scores(name, dtype, cache_dtype, offset), 64.0, scale=scale)


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
