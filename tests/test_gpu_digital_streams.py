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


def test_rows_grouped_within_a_capture_and_used_on_a_stream_of_it():
    """Two streams of one capture: the second, which joined before the rows were grouped, comes after that all the same."""
    s = Set(300, 64, 80, 8, 4, p=0.1)
    index = s.index.clone()
    second = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = torch.cuda.current_stream()
        second.wait_stream(first)
        rows = digital.AdapterRows(index, s.n)
        with torch.cuda.stream(second):
            results = step(s, rows)
        first.wait_stream(second)
    for k in range(4):
        s.index.copy_((s.index + 1) % 4)
        index.copy_(s.index)
        for t in results:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(results, s.step())), k


def test_rows_whose_stream_is_being_captured_are_refused_elsewhere():
    s = Set(300, 64, 80, 8, 4)
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(first):
        rows = digital.AdapterRows(s.index, s.n)
    torch.cuda.synchronize()
    x = torch.ones(64, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=first):
        y = digital.dropout(x, 0.5, 1, non_blocking=True)
        with torch.cuda.stream(second), pytest.raises(RuntimeError, match="captured"):
            s.adapters.forward(s.x, rows, non_blocking=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, digital.dropout(x, 0.5, 1))
