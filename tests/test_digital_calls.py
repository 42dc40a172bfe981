"""The native calls of the digital operators and the general path in Python give the same results, the same errors, and leave
the same tensors to each other."""
import os
import subprocess
import sys

import pytest
import torch

from aihwkit_amd import _cabi, digital

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = """
import sys
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from aihwkit_amd._cabi import torch_calls

transform, m = sys.argv[1], torch_calls()

CALLS = {
    "dropout": lambda x, a, b, s, i: m.dropout(x, 0.5, 1, 0, None, None, True),
    "layer_norm": lambda x, a, b, s, i: m.layer_norm(x, None, None, 1e-5, None, True),
    "layer_norm_backward": lambda x, a, b, s, i: m.layer_norm_backward(x, x, s, s, None, None, None, True),
    "adapter_plan": lambda x, a, b, s, i: m.adapter_plan(i, 3),
    "adapter_forward": lambda x, a, b, s, i: m.adapter_forward(a, b, s, x, i, None, None, None, True, 0.0, 0, 0, True),
    "adapter_backward": lambda x, a, b, s, i: m.adapter_backward(a, b, s, x, x, i, None, s, None, None, 0.0, 0, 0, True),
}

def f(x):
    a, b, s = torch.empty(3, 4, 8, device="cuda"), torch.empty(3, 8, 4, device="cuda"), torch.empty(3, device="cuda")
    i = torch.empty(3, dtype=torch.int32, device="cuda")
    for name, call in CALLS.items():
        print(name, flush=True)
        assert call(x, a, b, s, i) is None
    return x + 1

with FakeTensorMode():
    x = torch.empty(2, 3, 8, device="cuda")
    if transform == "vmap":
        torch.vmap(f)(x)
    elif transform == "jvp":
        torch.func.jvp(f, (x[0],), (x[1],))
    else:
        f(x[0])
print("done")
"""


@pytest.mark.parametrize("transform", ["vmap", "jvp", "none"])
def test_tensors_without_storage_are_left_to_the_general_path(transform):
    run = subprocess.run([sys.executable, "-c", SCRIPT, transform], env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True,
                         text=True, timeout=240)
    assert run.returncode == 0 and run.stdout.strip().endswith("done"), run.stdout + run.stderr[-1500:]


def test_native_calls_refuse_host_tensors_by_doing_nothing():
    m, x, v = _cabi.torch_calls(), torch.zeros(3, 8), torch.zeros(3)
    assert m.dropout(x, 0.5, 1, 0, None, None, True) is None
    assert m.layer_norm(x, None, None, 1e-5, None, True) is None
    assert m.layer_norm_backward(x, x, v, v, None, None, None, True) is None
    assert m.adapter_plan(torch.zeros(3, dtype=torch.int32), 2) is None
    for call, n in ((m.dropout, 7), (m.layer_norm, 6), (m.layer_norm_backward, 8), (m.adapter_plan, 2), (m.adapter_forward, 13),
                    (m.adapter_backward, 14)):
        with pytest.raises(TypeError, match=str(n)):
            call()


class Calls:
    """Every digital operator once, on tensors of the GPU."""

    def __init__(self, dtype):
        gen = torch.Generator("cuda").manual_seed(3)

        def rand(*shape):
            return torch.randn(shape, generator=gen, device="cuda").to(dtype)

        self.x, self.d, self.w, self.b = rand(80, 40), rand(80, 40), rand(40), rand(40)
        self.adapters = digital.LowRankAdapters(rand(3, 6, 40), rand(3, 24, 6), torch.rand(3, generator=gen, device="cuda"))
        self.y = rand(80, 24)
        self.index = (torch.arange(80, device="cuda") % 4).to(torch.int32)

    def run(self, p=0.25, seed=5, call=2, base=True):
        x, d, y, add = self.x, self.d, self.y, self.d if base else None
        drop = dict(p=p, seed=seed, call=call)
        results = [digital.dropout(x, base=add, **drop)]
        norm = digital.layer_norm(x, self.w, self.b, 1e-3)
        results += [*norm, *digital.layer_norm_backward(d, x, norm[1], norm[2], self.w, base=add)]
        rows = digital.AdapterRows(self.index, 3)
        out, hidden = self.adapters.forward(x, rows, base=y if base else None, return_hidden=True, **drop)
        results += [out, hidden, *self.adapters.backward(y, x, rows, hidden, base=add, **drop)]
        results += [self.adapters.forward(x, self.index, **drop), self.adapters.forward(x[:9], self.index[:9], **drop)]
        results += self.adapters.backward(y, x, self.index, hidden, **drop)
        return results


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_the_general_path_gives_the_same_results(dtype, monkeypatch):
    calls = Calls(dtype)
    for kw in (dict(), dict(base=False), dict(seed=2 ** 64 - 1, call=2 ** 32 - 1), dict(p=0.0)):
        native = calls.run(**kw)
        with monkeypatch.context() as patch:
            patch.setattr(_cabi, "_torch_calls", _cabi._GeneralPath())
            general = calls.run(**kw)
        assert len(native) == len(general)
        for a, b in zip(native, general):
            assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a, b)


@pytest.mark.gpu
def test_what_the_native_calls_take():
    """The plain cases do not reach the general path: it is slower by several times."""
    m, c = _cabi.torch_calls(), Calls(torch.bfloat16)
    wide = torch.empty(80, 100, dtype=torch.bfloat16, device="cuda")
    assert m.dropout(wide[:, 8:48], 0.1, 1, 0, c.x, wide[:, 50:90], True) is not None
    assert m.layer_norm(c.x, c.w, None, 1e-5, None, True) is not None
    assert m.layer_norm(c.x, c.w.float(), c.b.float(), 1e-5, None, True) is not None
    assert m.adapter_plan(c.index, 3) is not None
    a = c.adapters
    assert m.adapter_forward(a.a, a.b, a.scale, c.x, c.index, None, c.y, None, True, 0.0, 0, 0, True) is not None
    # these are for the general path to convert or to word the errors of
    assert m.dropout(c.x.t(), 0.1, 1, 0, None, None, True) is None
    assert m.dropout(c.x, 0.1, 1 << 64, 0, None, None, True) is None and m.dropout(c.x, 0.1, 1, -1, None, None, True) is None
    assert m.dropout(c.x, 2.0, 1, 0, None, None, True) is None
    assert m.dropout(c.x, 0.1, 1, torch.zeros(1, dtype=torch.int64, device="cuda"), None, None, True) is None
    assert m.dropout(c.x, 0.1, 1, 0, c.x.float(), None, True) is None
    assert m.layer_norm(c.x, c.w.half(), None, 1e-5, None, True) is None
    assert m.adapter_forward(a.a.float(), a.b, a.scale, c.x, c.index, None, None, None, True, 0.0, 0, 0, True) is None
    assert m.adapter_forward(a.a, a.b, a.scale, c.x, c.index[:79], None, None, None, True, 0.0, 0, 0, True) is None
    assert m.adapter_forward(a.a, a.b, a.scale, c.x, c.index.long(), None, None, None, True, 0.0, 0, 0, True) is None
    with pytest.raises(RuntimeError, match="overlaps"):
        m.dropout(wide[:, 8:48], 0.1, 1, 0, None, wide[:, 20:60], True)
