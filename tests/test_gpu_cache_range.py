"""Calls of the paged cache that its documentation allows at the ends of their range, against the formula in 64 bits."""
import pytest
import torch

from test_gpu_cache import LAYOUTS, PAIR_IDS, PAIRS, Batch

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
