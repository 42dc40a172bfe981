"""Digital operators beside the tiles, without a GPU: every refusal of the C entry points and of the Python calls comes before
anything is launched, and the sizes of what a caller provides."""
import ctypes as C

import pytest
import torch

from aihwkit_amd import _cabi, digital

F32, F16, BF16 = 0, 1, 2
AT = 1 << 40          # an address that nothing reads: all of these calls are refused


def refused(code, text):
    message = _cabi.lib().rpu_last_error().decode()
    assert code != 0 and text in message, (code, message)


def drop(p=0.5, **kw):
    return _cabi.DropoutParams(p=p, seed=1, **kw)


def dropout(x=AT, x_ld=64, base=None, base_ld=0, out=AT + (1 << 30), out_ld=64, dtype=F32, rows=8, cols=64, params=None):
    params = drop() if params is None else params
    return _cabi.lib().rpu_dropout(x, x_ld, base, base_ld, out, out_ld, dtype, rows, cols, C.byref(params), -1, None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=3), "Unknown data type"), (dict(dtype=-1), "Unknown data type"),
    (dict(rows=-1), "number of rows"), (dict(rows=(1 << 28) + 1), "number of rows"),
    (dict(cols=0), "number of columns"), (dict(cols=(1 << 24) + 1), "number of columns"),
    (dict(x=None), "x is null"), (dict(out=None), "output is null"),
    (dict(x_ld=63), "rows of x overlap"), (dict(out_ld=0), "rows of the output overlap"), (dict(x_ld=-64), "rows of x overlap"),
    (dict(x_ld=1 << 60), "too far apart"),
    (dict(params=drop(-0.1)), "probability"), (dict(params=drop(1.5)), "probability"), (dict(params=drop(float("nan"))), "probability"),
    (dict(params=drop(0.5, reserved=1)), "reserved"),
    (dict(out=AT + 4), "overlaps"), (dict(out=AT, out_ld=65), "overlaps"), (dict(out=AT + 64 * 4), "overlaps"),
    (dict(base=AT + (1 << 30) + 4, base_ld=64), "overlaps"),
    # column slices of one matrix: the second begins inside the first
    (dict(x_ld=128, out_ld=128, out=AT + 63 * 4), "overlaps"), (dict(x_ld=100, out_ld=100, out=AT + 64 * 4), "overlaps"),
    # one row against the rows of another matrix
    (dict(rows=8, out=AT + 7 * 64 * 4), "overlaps"),
])
def test_dropout_refusals(kw, text):
    refused(dropout(**kw), text)


def test_null_parameters_are_refused():
    lib = _cabi.lib()
    refused(lib.rpu_dropout(AT, 64, None, 0, AT + (1 << 30), 64, F32, 8, 64, None, -1, None), "null")
    refused(lib.rpu_adapter_forward(None, AT, 64, AT, None, 0, None, None, 0, AT + 1, 64, None, F32, 8, -1, None), "null")
    assert lib.rpu_adapter_backward_scratch(None, 8) == 0


def test_calls_without_rows_need_no_gpu():
    assert dropout(rows=0) == 0 and dropout(rows=0, x=None, out=None) == 0
    assert _cabi.lib().rpu_layer_norm(None, 8, None, None, F32, None, 8, None, None, F32, 0, 8, 1e-5, -1, None) == 0


def norm(x=AT, out=AT + (1 << 30), w=None, b=None, w_dtype=F32, mean=AT + (2 << 30), rstd=AT + (3 << 30), dtype=F32, rows=8, cols=64,
         eps=1e-5):
    return _cabi.lib().rpu_layer_norm(x, cols, w, b, w_dtype, out, cols, mean, rstd, dtype, rows, cols, eps, -1, None)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=7), "Unknown data type"), (dict(w_dtype=BF16), "Weight and bias"), (dict(dtype=F16, w_dtype=BF16), "Weight and bias"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(mean=None), "mean is null"), (dict(rstd=None), "rstd is null"), (dict(rstd=AT + (2 << 30)), "overlaps"),
    (dict(mean=AT), "overlaps"), (dict(rstd=AT + (1 << 30) + 8), "overlaps"), (dict(w=AT + (1 << 30)), "overlaps"),
    (dict(b=AT + (2 << 30) - 8), "overlaps"), (dict(out=AT + 8), "overlaps"), (dict(cols=0), "number of columns"),
])
def test_layer_norm_refusals(kw, text):
    refused(norm(**kw), text)


def norm_backward(d=AT, x=AT + (1 << 30), mean=AT + (2 << 30), rstd=AT + (3 << 30), w=AT + (4 << 30), base=None, dx=AT + (5 << 30),
                  dw=AT + (6 << 30), db=AT + (7 << 30), dtype=F32, w_dtype=F32, rows=8, cols=64, scratch=AT + (8 << 30), scratch_bytes=1 << 20):
    return _cabi.lib().rpu_layer_norm_backward(d, cols, x, cols, mean, rstd, w, w_dtype, base, cols, dx, cols, dw, db, dtype, rows,
                                               cols, scratch, scratch_bytes, -1, None)


@pytest.mark.parametrize("kw, text", [
    (dict(db=None), "come together"), (dict(dw=None), "come together"), (dict(scratch_bytes=3), "too small"),
    (dict(scratch=None), "null"), (dict(scratch=AT + (8 << 30) + 2), "aligned"), (dict(scratch=AT), "overlaps"),
    (dict(scratch=AT + (5 << 30)), "overlaps"), (dict(db=AT + (6 << 30) + 4), "overlaps"), (dict(dx=AT + 4), "overlaps"),
    (dict(dx=AT + (3 << 30)), "overlaps"), (dict(dw=AT + (4 << 30)), "overlaps"), (dict(d=None), "d is null"), (dict(x=None), "x is null"),
    (dict(base=AT + (5 << 30) + 4), "overlaps"), (dict(w_dtype=F16), "Weight and bias"),
])
def test_layer_norm_backward_refusals(kw, text):
    refused(norm_backward(**kw), text)


def adapters(**kw):
    given = dict(a_dev=AT, b_dev=AT + (1 << 30), scale_dev=AT + (2 << 30), n=4, in_size=64, out_size=48, rank=8, w_dtype=F32, reserved=0)
    return _cabi.Adapters(**dict(given, **kw))


def forward(w=None, x=AT + (3 << 30), x_ld=64, index=AT + (4 << 30), plan=None, plan_bytes=0, params=None, base=None, y=AT + (5 << 30),
            y_ld=48, hidden=None, dtype=F32, rows=8):
    w = adapters() if w is None else w
    return _cabi.lib().rpu_adapter_forward(C.byref(w), x, x_ld, index, plan, plan_bytes, None if params is None else C.byref(params),
                                           base, 48, y, y_ld, hidden, dtype, rows, -1, None)


BAD_ADAPTERS = [
    (dict(n=0), "number of adapters"), (dict(n=65536), "number of adapters"), (dict(rank=0), "rank"), (dict(rank=129), "rank"),
    (dict(in_size=0), "sizes"), (dict(out_size=(1 << 21) + 1), "sizes"), (dict(w_dtype=9), "Unknown data type"),
    (dict(a_dev=None), "null"), (dict(b_dev=None), "null"), (dict(scale_dev=None), "null"), (dict(reserved=1), "reserved"),
]


@pytest.mark.parametrize("kw, text", BAD_ADAPTERS)
def test_adapter_refusals(kw, text):
    refused(forward(w=adapters(**kw)), text)
    refused(backward(w=adapters(**kw)), text)


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=5), "Unknown data type"), (dict(dtype=BF16), "16-bit rows"), (dict(dtype=F16, w=adapters(w_dtype=BF16)), "16-bit rows"),
    (dict(rows=65), "need a row plan"), (dict(index=None), "index is null"), (dict(x=None), "x is null"), (dict(y=None), "y is null"),
    (dict(x_ld=63), "rows of x overlap"), (dict(y_ld=47), "rows of y overlap"), (dict(params=drop(2.0)), "probability"),
    (dict(plan=AT + (6 << 30), plan_bytes=8), "too small"), (dict(plan=AT + (6 << 30) + 4, plan_bytes=1 << 20), "aligned"),
    (dict(y=AT + (3 << 30)), "overlaps"), (dict(y=AT), "overlaps"), (dict(y=AT + (1 << 30)), "overlaps"), (dict(y=AT + (4 << 30)), "overlaps"),
    (dict(base=AT + (5 << 30) + 4), "overlaps"), (dict(hidden=AT + (5 << 30)), "overlaps"), (dict(hidden=AT + (3 << 30)), "overlaps"),
    (dict(hidden=AT + (7 << 30), base=AT + (7 << 30)), "overlaps"), (dict(rows=-1), "number of rows"),
    (dict(rows=100, plan=AT + (5 << 30), plan_bytes=1 << 20), "overlaps"),
])
def test_adapter_forward_refusals(kw, text):
    refused(forward(**kw), text)


def backward(w=None, d=AT + (3 << 30), x=AT + (4 << 30), hidden=AT + (5 << 30), plan=AT + (6 << 30), plan_bytes=1 << 20, base=None,
             dx=AT + (7 << 30), da=AT + (8 << 30), db=AT + (9 << 30), dtype=F32, rows=8, scratch=AT + (10 << 30), scratch_bytes=1 << 24):
    w = adapters() if w is None else w
    return _cabi.lib().rpu_adapter_backward(C.byref(w), d, 48, x, 64, hidden, plan, plan_bytes, None, base, 64, dx, 64, da, db, dtype,
                                            rows, scratch, scratch_bytes, -1, None)


@pytest.mark.parametrize("kw, text", [
    (dict(plan=None), "plan is null"), (dict(plan_bytes=16), "too small"), (dict(hidden=None), "hidden is null"), (dict(da=None), "da is null"),
    (dict(db=None), "db is null"), (dict(scratch_bytes=16), "too small"), (dict(scratch=None), "null"), (dict(scratch=AT + (10 << 30) + 1), "aligned"),
    (dict(dx=AT + (3 << 30)), "overlaps"), (dict(dx=AT + (4 << 30)), "overlaps"), (dict(da=AT), "overlaps"), (dict(db=AT + (1 << 30)), "overlaps"),
    (dict(db=AT + (8 << 30)), "overlaps"), (dict(scratch=AT + (7 << 30)), "overlaps"), (dict(base=AT + (8 << 30)), "overlaps"),
    (dict(base=AT + (7 << 30) + 4), "overlaps"), (dict(dtype=F16), "16-bit rows"), (dict(da=AT + (6 << 30)), "overlaps"),
])
def test_adapter_backward_refusals(kw, text):
    refused(backward(**kw), text)


def test_plan_refusals_and_sizes():
    lib = _cabi.lib()
    assert lib.rpu_adapter_plan_bytes(-1, 4) == lib.rpu_adapter_plan_bytes(8, 0) == lib.rpu_adapter_plan_bytes(8, 65536) == 0
    for rows, n in ((0, 1), (1, 1), (64, 65535), (1000, 7), (100000, 300)):
        size = lib.rpu_adapter_plan_bytes(rows, n)
        assert size >= 4 * (rows + 4 * n) and size % 16 == 0
        refused(lib.rpu_adapter_plan(AT + (1 << 36), rows, n, AT, size - 1, -1, None), "too small")
    refused(lib.rpu_adapter_plan(AT + (1 << 36), 8, 4, AT + 8, 1 << 20, -1, None), "aligned")
    refused(lib.rpu_adapter_plan(AT + 64, 8, 4, AT, 1 << 20, -1, None), "overlaps")
    refused(lib.rpu_adapter_plan(None, 8, 4, AT, 1 << 20, -1, None), "null")
    refused(lib.rpu_adapter_plan(AT, 8, 4, None, 0, -1, None), "null")


def test_scratch_sizes_do_not_grow_with_rows_without_end():
    lib = _cabi.lib()
    assert lib.rpu_layer_norm_backward_scratch(0, 768) == 0
    assert lib.rpu_layer_norm_backward_scratch(1, 768) == 2 * 768 * 4
    assert lib.rpu_layer_norm_backward_scratch(1 << 24, 768) == lib.rpu_layer_norm_backward_scratch(1 << 20, 768) <= 16 << 20
    # as many adapters as rows: nothing has to be joined; up [8][8] and the matrices turned, [8][8][64 + 48] floats
    assert lib.rpu_adapter_backward_scratch(C.byref(adapters(n=8)), 8) == 4 * 8 * 8 * (1 + 64 + 48)


def test_python_calls_refuse_host_tensors_and_wrong_types():
    x = torch.zeros(4, 8)
    for call in (lambda: digital.dropout(x, 0.5, 1), lambda: digital.layer_norm(x), lambda: digital.layer_norm_backward(x, x, x, x),
                 lambda: digital.AdapterRows(torch.zeros(4, dtype=torch.int32), 2), lambda: digital.AdapterRows(torch.zeros(4), 2),
                 lambda: digital.LowRankAdapters(torch.zeros(1, 2, 8), torch.zeros(1, 8, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        digital.dropout([1.0], 0.5, 1)
    with pytest.raises(RuntimeError, match="float32"):
        digital.dropout(torch.zeros(4, 8, dtype=torch.int32), 0.5, 1)
