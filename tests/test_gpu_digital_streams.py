"""Rows grouped on one stream and used on others, and in captures."""
import pytest
import torch

from aihwkit_amd import _cabi, digital
from test_gpu_digital import Set

pytestmark = pytest.mark.gpu


def step(s, rows):
    y, hidden = s.adapters.forward(s.x, rows, base=s.base, return_hidden=True, non_blocking=True, **s.drop)
    return (y, hidden, *s.adapters.backward(s.d, s.x, rows, hidden, base=s.dx_base, non_blocking=True, **s.drop))


@pytest.mark.parametrize("general", [False, True], ids=["native", "general"])
def test_rows_grouped_on_another_stream_are_waited_for(general, monkeypatch):
    """The grouping is queued behind other work on its stream; calls on a second stream come after it all the same, and its memory is not
    given away while they are under way."""
    s = Set(3000, 64, 80, 8, 4, p=0.1)
    expected = s.step()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    if general:
        monkeypatch.setattr(_cabi, "_torch_calls", _cabi._GeneralPath())
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(first):
            torch.cuda._sleep(4000000)
            rows = digital.AdapterRows(s.index, s.n)
        with torch.cuda.stream(second):
            got = step(s, rows)
            again = step(s, rows)
            torch.cuda._sleep(4000000)
            late = step(s, rows)
        size = rows._bytes
        del rows
        with torch.cuda.stream(first):                        # what is free of the first stream's memory is written
            spoilt = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(20)]
        torch.cuda.synchronize()
        for results in (got, again, late):
            assert all(torch.equal(p, q) for p, q in zip(results, expected))
        del spoilt


def test_rows_grouped_before_a_capture():
    s = Set(300, 64, 80, 8, 4, p=0.1)
    expected = s.step()
    rows = digital.AdapterRows(s.index, s.n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(s, rows)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(s, rows)
    for _ in range(4):
        for t in results:
            t.zero_()
        graph.replay()
        eager = step(s, rows)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) and torch.equal(r, q) for p, q, r in zip(results, expected, eager))
