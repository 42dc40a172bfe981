"""Scratch memory of the digital operators: calls with exactly as much as is asked for, between guards that stay as they are."""
import ctypes as C

import pytest
import torch

from aihwkit_amd import _cabi, digital
from test_gpu_digital import BF16, F16, F32, PAIR_IDS, PAIRS, Set, close, norm_backward_reference, rand

pytestmark = pytest.mark.gpu

TYPE = {F32: 0, F16: 1, BF16: 2}
GUARD = 4096


class Scratch:
    def __init__(self, size):
        self.size, self.memory = size, torch.full((size + 2 * GUARD,), 90, dtype=torch.uint8, device="cuda")

    @property
    def at(self):
        return self.memory.data_ptr() + GUARD

    def check(self):
        assert (self.memory[:GUARD] == 90).all() and (self.memory[GUARD + self.size:] == 90).all()


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows, n, used, rank", [
    (500, 700, (3, 690, 0, -1), 16), (60, 61, (60,), 5), (1, 65535, (65534,), 3), (300, 300, (0, 299, 7), 40), (700, 3, (2, 0), 8), (300, 301, (-1,), 4),
])
def test_adapters_backward(rows, n, used, rank, dtype, w_dtype):
    """More adapters than rows and fewer, one of them with several chunks of rows."""
    choice = torch.tensor(used, dtype=torch.int32, device="cuda")
    index = choice[(torch.arange(rows, device="cuda") * torch.arange(rows, device="cuda") // 3) % (2 * len(used)) % len(used)]
    s = Set(rows, 40, 24, rank, n, dtype, w_dtype, p=0.2, index=index, seed=940)
    rows_of = digital.AdapterRows(index, n)
    y, hidden = s.adapters.forward(s.x, rows_of, base=s.base, return_hidden=True, **s.drop)
    w = s.adapters._operand(s.x)
    drop = _cabi.DropoutParams(p=s.p, seed=s.drop["seed"], call=s.drop["call"])
    scratch = Scratch(_cabi.lib().rpu_adapter_backward_scratch(C.byref(w), rows))
    dx, da, db = torch.empty_like(s.x), torch.empty_like(s.a), torch.empty_like(s.b)
    _cabi.check(_cabi.lib().rpu_adapter_backward(
        C.byref(w), s.d.data_ptr(), 24, s.x.data_ptr(), 40, hidden.data_ptr(), rows_of._plan.data_ptr(), rows_of._bytes, C.byref(drop),
        s.dx_base.data_ptr(), 40, dx.data_ptr(), 40, da.data_ptr(), db.data_ptr(), TYPE[dtype], rows, scratch.at, scratch.size, 0, stream()))
    torch.cuda.synchronize()
    scratch.check()
    s.check((y, hidden, dx, da, db))


@pytest.mark.parametrize("rows, cols", [(1, 8), (3000, 70), (9000, 512), (5000, 700), (2500, 1537), (1700, 4096), (700, 5000), (600, 16400)])
def test_layer_norm_backward(rows, cols):
    x, d, w = rand(24, rows, cols), rand(25, rows, cols), rand(26, cols)
    _, mean, rstd = digital.layer_norm(x)
    scratch = Scratch(_cabi.lib().rpu_layer_norm_backward_scratch(rows, cols))
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    _cabi.check(_cabi.lib().rpu_layer_norm_backward(
        d.data_ptr(), cols, x.data_ptr(), cols, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), 0, None, 0, dx.data_ptr(), cols,
        dw.data_ptr(), db.data_ptr(), 0, rows, cols, scratch.at, scratch.size, 0, stream()))
    torch.cuda.synchronize()
    scratch.check()
    ref = norm_backward_reference(d, x, mean, rstd, w, None)
    for got, expected, bound in zip((dx, dw, db), ref[:3], ref[3:]):
        close(got, expected, bound)
