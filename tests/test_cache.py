"""Attention over a paged cache without a GPU: every refusal of the C entry points and of the Python calls comes before anything is
launched; and the oracle that the GPU tests hold the kernels against, against its definition."""
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from aihwkit_amd import _cabi, digital
from cache_oracle import attended, bound_of, rotated

F32, F16, BF16 = 0, 1, 2
AT = 1 << 40          # an address that nothing reads: all of these calls are refused
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def place(k):
    return AT + (k << 32)


def refused(code, text):
    message = _cabi.lib().rpu_last_error().decode()
    assert code != 0 and text in message, (code, message)


def cache(**kw):
    given = dict(k_dev=place(0), v_dev=place(1), turns_dev=place(2), pages=4, page_size=16, heads=2, head_size=64, dtype=F32, pairs=32, neighbours=0,
                 reserved=0)
    return _cabi.Cache(**dict(given, **kw))


def rows(**kw):
    given = dict(tables_dev=place(3), lengths_dev=place(4), starts_dev=None, table_ld=2, n=2, table_width=2, rows=8, reserved=0)
    return _cabi.CacheRows(**dict(given, **kw))


def append(c=None, r=None, k=place(5), k_ld=128, v=place(6), v_ld=128, q=place(7), q_ld=256, out=place(8), out_ld=256, heads=4, dtype=F32):
    c, r = cache() if c is None else c, rows() if r is None else r
    return _cabi.lib().rpu_cache_append(C.byref(c), C.byref(r), k, k_ld, v, v_ld, q, q_ld, out, out_ld, heads, dtype, -1, None)


def attend(c=None, r=None, q=place(7), q_ld=256, out=place(8), out_ld=256, heads=4, dtype=F32, scale=0.125, window=0, sinks=0, longest=0,
           scratch=place(9), scratch_bytes=1 << 31):
    c, r = cache() if c is None else c, rows() if r is None else r
    return _cabi.lib().rpu_cache_attend(C.byref(c), C.byref(r), q, q_ld, out, out_ld, heads, dtype, scale, window, sinks, longest, scratch,
                                        scratch_bytes, -1, None)


@pytest.mark.parametrize("kw, text", [
    (dict(pages=0), "has pages"), (dict(heads=0), "has pages"), (dict(heads=65537), "has pages"), (dict(pages=-1), "has pages"),
    (dict(page_size=0), "power of two"), (dict(page_size=4), "power of two"), (dict(page_size=24), "power of two"), (dict(page_size=131072), "power of two"),
    (dict(page_size=-16), "power of two"),
    (dict(head_size=0), "multiple of 8"), (dict(head_size=60), "multiple of 8"), (dict(head_size=264), "multiple of 8"),
    (dict(pairs=-1), "pairs"), (dict(pairs=33), "pairs"), (dict(turns_dev=None), "turns"), (dict(k_dev=None), "null"), (dict(v_dev=None), "null"),
    (dict(k_dev=place(0) + 8), "aligned"), (dict(v_dev=place(1) + 2), "aligned"), (dict(dtype=3), "Unknown data type"), (dict(reserved=1), "reserved"),
    (dict(heads=1024, page_size=65536), "2 GB"),
])
def test_caches_that_are_refused(kw, text):
    refused(append(c=cache(**kw)), text)
    refused(attend(c=cache(**kw)), text)


@pytest.mark.parametrize("kw, text", [
    (dict(n=0), "number of sequences"), (dict(n=-1), "number of sequences"), (dict(rows=-1), "number of rows"), (dict(rows=(1 << 28) + 2), "number of rows"),
    (dict(rows=7), "as many rows each"), (dict(table_width=0), "2^30"), (dict(table_width=1 << 27, table_ld=1 << 27), "2^30"),
    (dict(tables_dev=None), "null"), (dict(lengths_dev=None), "null"), (dict(table_ld=1), "tables overlap"), (dict(table_ld=1 << 60), "too far apart"),
    (dict(reserved=5), "reserved"),
])
def test_rows_that_are_refused(kw, text):
    refused(append(r=rows(**kw)), text)
    refused(attend(r=rows(**kw)), text)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=4), "Unknown data type"), (dict(dtype=BF16), "16-bit rows"), (dict(dtype=F16, c=cache(dtype=BF16)), "16-bit rows"),
    (dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(out=None), "output is null"), (dict(k_ld=127), "overlap"), (dict(v_ld=0), "overlap"),
    (dict(q_ld=255), "overlap"), (dict(out_ld=255), "overlap"), (dict(heads=0), "at least one head"), (dict(heads=1 << 19), "at most 2^24"),
    (dict(out=place(7) + 8), "overlaps"), (dict(out=place(0)), "overlaps"), (dict(out=place(1) + 64), "overlaps"), (dict(out=place(5) + 64), "overlaps"),
    (dict(out=place(3)), "overlaps"), (dict(out=place(4) + 4), "overlaps"), (dict(out=place(2)), "overlaps"), (dict(k=place(0)), "overlaps"),
    (dict(v=place(1) + 4 * 2 * 16 * 64 * 4 - 4), "overlaps"), (dict(q=place(0) + 32), "overlaps"), (dict(c=cache(v_dev=place(0) + 1024)), "overlaps"),
    (dict(c=cache(turns_dev=place(0))), "overlaps"), (dict(r=rows(tables_dev=place(1))), "overlaps"), (dict(r=rows(starts_dev=place(1))), "overlaps"),
])
def test_append_refusals(kw, text):
    refused(append(**kw), text)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=4), "Unknown data type"), (dict(dtype=BF16), "16-bit rows"), (dict(q=None), "q is null"), (dict(out=None), "output is null"),
    (dict(heads=3), "multiple of the cache's"), (dict(heads=0), "at least one head"), (dict(q_ld=255), "overlap"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=-2e30), "scale"), (dict(r=rows(rows=1 << 28), c=cache(head_size=8, pairs=0, heads=1), heads=16), "too many"), (dict(window=-1), "negative"), (dict(sinks=-1, window=4), "negative"), (dict(sinks=4), "Only a window"),
    (dict(longest=-1), "longest"), (dict(out=place(7) + 8), "overlaps"), (dict(out=place(0)), "overlaps"), (dict(out=place(1)), "overlaps"),
    (dict(out=place(3)), "overlaps"), (dict(out=place(4)), "overlaps"), (dict(r=rows(starts_dev=place(8))), "overlaps"),
])
def test_attend_refusals(kw, text):
    refused(attend(**kw), text)


def test_null_structures_are_refused():
    lib, c, r = _cabi.lib(), cache(), rows()
    refused(lib.rpu_cache_append(None, C.byref(r), AT, 128, AT, 128, None, 0, None, 0, 0, F32, -1, None), "cache is null")
    refused(lib.rpu_cache_append(C.byref(c), None, AT, 128, AT, 128, None, 0, None, 0, 0, F32, -1, None), "sequences are null")
    refused(lib.rpu_cache_attend(None, C.byref(r), AT, 128, AT, 128, 2, F32, 1.0, 0, 0, 0, None, 0, -1, None), "cache is null")
    assert lib.rpu_cache_attend_scratch(None, C.byref(r), 4, F32, 0, 0, 0) == 0
    assert lib.rpu_cache_attend_scratch(C.byref(c), None, 4, F32, 0, 0, 0) == 0


def test_calls_without_rows_need_no_gpu():
    assert append(r=rows(rows=0)) == 0 and attend(r=rows(rows=0)) == 0


def test_python_refusals():
    host = torch.zeros(4, 2, 16, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        digital.PagedCache(host, host)
    with pytest.raises(TypeError, match="keys"):
        digital.PagedCache(None, host)
    f = digital.rotation_frequencies(64, 100.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and float(f[0]) == 1.0 and abs(float(f[16]) - 0.1) < 1e-15


SCRIPT = """
import sys
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from aihwkit_amd._cabi import torch_calls

transform, m = sys.argv[1], torch_calls()

def f(x):
    k = torch.empty(4, 2, 16, 8, device="cuda")
    i = torch.empty(3, dtype=torch.int32, device="cuda")
    t = torch.empty(3, 2, dtype=torch.int32, device="cuda")
    assert m.cache_append(k, k, (4, 2, 16, 8), None, False, x, x, t, i, None, None, None, True) is None
    assert m.cache_attend(k, k, (4, 2, 16, 8), x, t, i, None, None, 0, 0, None, None, True) is None
    return x + 1

with FakeTensorMode():
    x = torch.empty(2, 3, 2, 8, device="cuda")
    if transform == "vmap":
        torch.vmap(f)(x)
    else:
        f(x[0])
print("done")
"""


@pytest.mark.parametrize("transform", ["vmap", "none"])
def test_tensors_without_storage_are_left_to_the_general_path(transform):
    run = subprocess.run([sys.executable, "-c", SCRIPT, transform], env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=240)
    assert run.returncode == 0 and run.stdout.strip().endswith("done"), run.stdout + run.stderr[-1500:]


def test_native_calls_refuse_host_tensors_by_doing_nothing():
    m, k, x, i, t = _cabi.torch_calls(), torch.zeros(4, 2, 16, 8), torch.zeros(3, 2, 8), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    assert m.cache_append(k, k, k.shape, None, False, x, x, t, i, None, None, None, True) is None
    assert m.cache_attend(k, k, k.shape, x, t, i, None, None, 0, 0, None, None, True) is None
    for call in (m.cache_append, m.cache_attend):
        with pytest.raises(TypeError, match="13"):
            call()


# -- the oracle ----------------------------------------------------------------------------------------------------------

def test_oracle_against_its_definition():
    """Position by position: two sequences on pages in any order, a page that is not there, a window with first tokens."""
    gen = torch.Generator().manual_seed(1)
    keys, values = torch.randn(5, 1, 4, 8, generator=gen).double(), torch.randn(5, 1, 4, 8, generator=gen).double()
    tables = [[3, 0, 9], [1, -1, 4]]
    lengths, starts = [10, 9], [1, 3, 6]
    q = torch.randn(7, 2, 8, generator=gen).double()
    out, _ = attended(q, keys, values, torch.tensor(tables), lengths, starts, scale=0.3, window=4, sinks=2)
    for s in range(2):
        m = starts[s + 1] - starts[s]
        for i in range(m):
            p = lengths[s] - m + i
            for h in range(2):
                weights, mixed = 0.0, torch.zeros(8).double()
                for j in range(p + 1):
                    page = tables[s][j // 4]
                    if 0 <= page < 5 and (j > p - 4 or j < 2):
                        w = float(torch.exp(0.3 * (q[starts[s] + i, h] * keys[page, 0, j % 4]).sum()))
                        weights += w
                        mixed += w * values[page, 0, j % 4]
                assert torch.allclose(out[starts[s] + i, h], mixed / weights, rtol=1e-12, atol=1e-12)
    assert torch.isnan(out[0]).all() and torch.isnan(out[6]).all()      # of no sequence


def test_oracle_of_rotations():
    f = torch.tensor([0.5, 0.25], dtype=torch.float64)
    x = torch.arange(1.0, 9.0).double().view(1, 1, 8)
    for neighbours, (a, b) in ((False, (0, 2)), (True, (0, 1))):
        y = rotated(x, torch.tensor([7]), f, neighbours)[0, 0]
        angle = torch.tensor(3.5).double()
        assert torch.allclose(y[a], x[0, 0, a] * angle.cos() - x[0, 0, b] * angle.sin())
        assert torch.allclose(y[b], x[0, 0, a] * angle.sin() + x[0, 0, b] * angle.cos())
        assert torch.equal(y[4:], x[0, 0, 4:])


def test_bounds_grow_with_what_they_are_bounds_of():
    """A weight that is rounded moves the result by no more than the bound."""
    gen = torch.Generator().manual_seed(2)
    keys, values, q = (torch.randn(*s, generator=gen).double() for s in ((3, 1, 16, 8), (3, 1, 16, 8), (4, 1, 8)))
    args = (torch.tensor([[0, 1, 2]]), [48], [0, 4])
    out, parts = attended(q, keys, values, *args, scale=1.0)
    limit = bound_of(parts, 8, torch.bfloat16)
    for k in range(20):
        noise = 1 + (torch.rand(3, 1, 16, 1, generator=gen).double() - 0.5) * 2 ** -8
        moved, _ = attended(q, keys, values, *args, scale=1.0, weigh=noise)
        assert ((moved - out).abs() <= limit).all()
