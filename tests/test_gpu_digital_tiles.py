"""Inference tiles with low-rank adapters: a call that is refused leaves the tile as it was."""
import pytest
import torch

from aihwkit_amd import digital
from aihwkit_amd.inference import InferenceTile
from test_gpu_digital import rand

pytestmark = pytest.mark.gpu


def noisy_tile():
    tile = InferenceTile(40, 33)                                 # the default periphery draws output noise in every call
    tile.set_weights(rand(70, 40, 33, std=0.1).cpu())
    tile.cuda().tile.set_seed(11)
    return tile


def test_refused_adapters_draw_nothing_from_the_tile():
    x, index = rand(71, 30, 32), (torch.arange(30, device="cuda") % 3).to(torch.int32)
    adapters = digital.LowRankAdapters(rand(72, 3, 4, 32), rand(73, 3, 40, 4))
    replaced = digital.LowRankAdapters(rand(72, 3, 4, 32), rand(73, 3, 40, 4))
    replaced.a = replaced.a[:, :3]
    mixed = digital.LowRankAdapters(rand(72, 3, 4, 32), rand(73, 3, 40, 4))
    mixed.b = mixed.b.half()
    scaled = digital.LowRankAdapters(rand(72, 3, 4, 32), rand(73, 3, 40, 4))
    scaled.scale = scaled.scale.double()
    tile, fresh = noisy_tile(), noisy_tile()
    for wrong, rows, error in (
            (digital.LowRankAdapters(rand(72, 3, 4, 32), rand(73, 3, 41, 4)), index, RuntimeError),       # another number of outputs
            (digital.LowRankAdapters(rand(72, 3, 4, 31), rand(73, 3, 40, 4)), index, RuntimeError),       # of inputs
            (adapters, index[:29], RuntimeError), (adapters, index.long(), RuntimeError), (adapters, index.cpu(), RuntimeError),
            (adapters, list(range(30)), TypeError),
            (adapters, digital.AdapterRows(index, 4), RuntimeError), (adapters, digital.AdapterRows(index[:29], 3), RuntimeError),
            (replaced, index, RuntimeError), (mixed, index, RuntimeError), (scaled, index, RuntimeError)):
        with pytest.raises(error):
            tile.forward(x, bias=True, adapters=wrong, rows=rows)
    for given in (x.half(), x.cpu(), x[:, :31], x.double(), None):
        with pytest.raises((RuntimeError, TypeError)):
            tile.forward(given, bias=True, adapters=adapters, rows=index)
    y = tile.forward(x, bias=True, adapters=adapters, rows=index)
    base = fresh.forward(x, bias=True)
    assert torch.equal(y, adapters.forward(x, index, base=base))
    assert not torch.equal(fresh.forward(x, bias=True), base)    # it does draw


def test_adapters_on_a_tile_take_rows_of_other_layouts():
    x, index = rand(74, 32, 90).t(), (torch.arange(90, device="cuda") % 4 - 1).to(torch.int32)
    adapters = digital.LowRankAdapters(rand(72, 3, 4, 32), rand(73, 3, 40, 4))
    base = noisy_tile().forward(x.contiguous(), bias=True)
    expected = adapters.forward(x.contiguous(), index, base=base)
    for rows in (index, digital.AdapterRows(index, 3)):
        assert torch.equal(noisy_tile().forward(x, bias=True, adapters=adapters, rows=rows), expected)
    one = noisy_tile().forward(x[4].contiguous(), bias=True)
    assert torch.equal(noisy_tile().forward(x[4], bias=True, adapters=adapters, rows=index[4:5]),
                       adapters.forward(x[4], index[4:5], base=one))
