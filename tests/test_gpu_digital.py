"""Digital operators beside the tiles (dropout, layer norm, low-rank adapters) against their formulas in 64 bits.

Tolerances are worst cases of 32-bit arithmetic in any order: a sum of n terms is off by at most n U times the sum of their
magnitudes (U = 2^-24, half a step of float32), and a stored result by half a step of its type on top."""
import numpy as np
import pytest
import torch

from aihwkit_amd import digital
from aihwkit_amd.inference import InferenceTile
from aihwkit_amd.rpu_base import devices as dv

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
IDS = [NAMES[t] for t in TYPES]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(seed, *shape, dtype=F32, std=1.0):
    gen = torch.Generator("cpu").manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std).to(dtype).cuda()


def sliced(tensor, left=3, right=5):
    """The same matrix as a column slice of a wider one, whose other columns are NaN."""
    rows, cols = tensor.shape
    whole = torch.full((rows, left + cols + right), float("nan"), dtype=tensor.dtype, device=tensor.device)
    whole[:, left:left + cols] = tensor
    return whole[:, left:left + cols]


def close(got, expected, bound):
    """Every value within ``bound`` (64 bits), stored in the type of ``got``: half a step, or half the smallest number.  What is
    rounded lies beyond the largest number of the type (by half a step of it) where ``expected`` less ``bound`` does: then, and
    only then, an infinity of its sign is the nearest number; nearer to it than ``bound`` both may be."""
    dtype, got, expected, bound = got.dtype, got.double().cpu(), expected.cpu(), bound.cpu()
    info = torch.finfo(dtype)
    limit = bound + half_step(dtype) * (expected.abs() + bound) + info.smallest_normal * info.eps / 2
    most = info.max * (1 + info.eps / 4)     # half a step beyond the largest number
    outside = torch.isinf(got) & (expected.sign() == got.sign()) & (expected.abs() + bound >= most)
    assert (torch.isinf(got) | (expected.abs() - bound < most)).all()
    over = torch.where(outside, torch.zeros(()).double(), (got - expected).abs() - limit)
    assert not torch.isnan(over).any()
    assert (over <= 0).all(), (float(over.max()), int((over > 0).sum()), over.numel())


# -- dropout -----------------------------------------------------------------------------------------------------------

def half_words(rows, cols, seed, call, purpose):
    """Half-words of the Philox4x32-10 blocks of counters (column / 8, row, call, purpose), as numpy integers."""
    row, block = np.meshgrid(np.arange(rows, dtype=np.uint64), np.arange(-(-cols // 8), dtype=np.uint64), indexing="ij")
    c = [block, row, np.full_like(row, call % (1 << 32)), np.full_like(row, purpose)]
    k0, k1, low = seed % (1 << 32), seed >> 32, np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) % (1 << 32), (k1 + 0xBB67AE85) % (1 << 32)
    halves = np.stack([w for v in c for w in (v & np.uint64(0xFFFF), v >> np.uint64(16))], -1)
    return halves.reshape(rows, -1)[:, :cols].astype(np.int64)


def kept(rows, cols, p, seed, call):
    limit = int(np.floor(p * 2.0 ** 32 + 0.5))
    both = half_words(rows, cols, seed, call, 18) * 65536 + half_words(rows, cols, seed, call, 19)
    return torch.from_numpy(both >= limit)


def dropped(x, p, seed, call, base=None):
    """Bit for bit: one product, one sum, one rounding to the stored type."""
    x = x.cpu()
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1 else 0.0, dtype=F32)
    y = torch.where(kept(*x.shape, p, seed, call), x.float() * scale, torch.zeros(()))
    if base is not None:
        y = y + base.cpu().float()
    return y.to(x.dtype)


def test_half_words_are_the_librarys_generator():
    import ctypes as C

    from aihwkit_amd import _cabi
    out = (C.c_uint32 * 4)()
    _cabi.check(_cabi.lib().rpu_philox4x32_10((C.c_uint32 * 4)(2, 5, 77, 18), (C.c_uint32 * 2)(9, 3), out))
    words = half_words(6, 24, 9 + (3 << 32), 77, 18)[5, 16:24]
    assert [int(words[2 * k] + 65536 * words[2 * k + 1]) for k in range(4)] == list(out)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 8), (3, 7), (5, 9), (64, 256), (129, 785), (1000, 24), (2, 40000)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_is_bit_equal_to_its_definition(dtype, rows, cols, p):
    x, base = rand(1, rows, cols, dtype=dtype), rand(2, rows, cols, dtype=dtype)
    seed, call = 0xFEDCBA9876543210, 0xFFFFFFFF
    assert torch.equal(digital.dropout(x, p, seed, call).cpu(), dropped(x, p, seed, call))
    assert torch.equal(digital.dropout(x, p, seed, call, base=base).cpu(), dropped(x, p, seed, call, base))


def test_dropout_limits_of_32_bits():
    """A probability between two neighbouring 16-bit limits: elements that the first half-word leaves undecided go by the
    second, to the last bit of the limit."""
    rows, cols, seed, call = 64, 512, 5, 9
    high, low = half_words(rows, cols, seed, call, 18), half_words(rows, cols, seed, call, 19)
    x = torch.ones(rows, cols, device="cuda")
    for row, col in ((0, 0), (3, 13), (17, 255), (63, 511)):
        limit = int(high[row, col] * 65536 + low[row, col])
        for step, stays in ((0, True), (1, False)):
            y = digital.dropout(x, (limit + step) / 2.0 ** 32, seed, call).cpu()
            assert bool(y[row, col] != 0) is stays
            assert torch.equal(y != 0, torch.from_numpy(high * 65536 + low >= limit + step))


def test_dropout_of_infinities_and_nan():
    x = torch.full((40, 64), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep = kept(40, 64, 0.5, 3, 0)
    y = digital.dropout(x, 0.5, 3).cpu()
    assert (y[~keep] == 0).all() and torch.isinf(y[::2][keep[::2]]).all() and torch.isnan(y[1::2][keep[1::2]]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_dropout_in_place_slices_and_dimensions(dtype):
    x, base = rand(3, 33, 45, dtype=dtype), rand(4, 33, 45, dtype=dtype)
    expected = dropped(x, 0.3, 8, 2, base)
    out = sliced(torch.zeros_like(x))
    assert digital.dropout(sliced(x), 0.3, 8, 2, base=sliced(base, 1, 2), out=out) is out
    assert torch.equal(out.cpu(), expected)
    assert torch.isnan(out._base[:, :3]).all() and torch.isnan(out._base[:, 48:]).all()
    for where in (x.clone(), base.clone()):
        given = where.clone()
        same = digital.dropout(where if torch.equal(given, x) else x, 0.3, 8, 2, base=where if torch.equal(given, base) else base, out=where)
        assert torch.equal(same.cpu(), expected)
    assert torch.equal(digital.dropout(x.view(3, 11, 45), 0.3, 8, 2).cpu(), dropped(x, 0.3, 8, 2).view(3, 11, 45))
    assert torch.equal(digital.dropout(x.t(), 0.3, 8, 2).cpu(), dropped(x.t(), 0.3, 8, 2))   # copied first
    assert torch.equal(digital.dropout(x[7], 0.3, 8, 2).cpu(), dropped(x[7:8], 0.3, 8, 2)[0])
    assert digital.dropout(x[:0], 0.3, 8).shape == (0, 45)


def test_dropout_call_on_the_gpu_and_mask_statistics():
    x = torch.ones(512, 1000, device="cuda")
    count = torch.tensor([41], device="cuda")
    a = digital.dropout(x, 0.25, 7, count)
    assert torch.equal(a, digital.dropout(x, 0.25, 7, 41))
    count += 1
    b = digital.dropout(x, 0.25, 7, count)
    assert torch.equal(b, digital.dropout(x, 0.25, 7, 42)) and not torch.equal(a, b)
    n = x.numel()
    for y in (a, b):       # five standard deviations of a binomial count
        assert abs(int((y == 0).sum()) - 0.25 * n) < 5 * (n * 0.25 * 0.75) ** 0.5
    both = int(((a == 0) & (b == 0)).sum())
    assert abs(both - n / 16) < 5 * (n * (1 / 16) * (15 / 16)) ** 0.5


def test_rows_beyond_32_bit_offsets():
    """Rows that lie 2^20 values apart: the last ones begin beyond 2^32 values."""
    whole = torch.empty((4100, 1 << 20), dtype=F16, device="cuda")
    x = whole[:, 5:45]
    x.copy_(rand(5, 4100, 40, dtype=F16))
    assert torch.equal(digital.dropout(x, 0.2, 4).cpu(), dropped(x, 0.2, 4, 0))
    y, mean, rstd = digital.layer_norm(x)
    assert torch.equal(y, digital.layer_norm(x.contiguous())[0])
    a, b = rand(6, 2, 4, 40, dtype=F16), rand(7, 2, 24, 4, dtype=F16)
    index = (torch.arange(4100, device="cuda") % 2).to(torch.int32)
    out = whole[:, 64:88]
    digital.LowRankAdapters(a, b).forward(x, index, out=out)
    assert torch.equal(out, digital.LowRankAdapters(a, b).forward(x.contiguous(), index))


# -- layer norm --------------------------------------------------------------------------------------------------------

COLS = [1, 2, 7, 8, 63, 511, 512, 513, 768, 1000, 1024, 1025, 1537, 2048, 2049, 4096, 4097, 8192, 8200, 16384, 16385, 40007]


def norm_reference(x, w, b, eps):
    """y, mean, rstd in 64 bits, and how far 32-bit sums may be off.  Here the order is part of the bound, so that it says
    something about rows with a large offset: a thread adds up to 40 values of a row (40007 columns over 1024 threads, eight at
    a time), the lanes of a wave come together in 6 steps and up to 16 waves one after the other, so that no value goes through
    more than 62 roundings on its way, and a sum of n values is off by at most min(n, 62) U times their magnitudes."""
    n = min(x.size(1), 62)
    x, w, b = x.double().cpu(), w.double().cpu(), b.double().cpu()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = c.square().mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    d_mean = (n + 2) * U * x.abs().mean(1, keepdim=True)
    d_c = d_mean + U * c.abs()                                              # of x - mean
    d_var = (n + 3) * U * var + 2 * (c.abs() * d_c).mean(1, keepdim=True) + (d_c ** 2).mean(1, keepdim=True)
    d_rstd = rstd * (0.5 * d_var / (var + eps) + 4 * U) * 1.01              # first order; second order is covered by 1 %
    ok = d_var < 0.01 * (var + eps)
    y = c * rstd * w + b
    d_y = (c.abs() * d_rstd + d_c * (rstd + d_rstd)) * w.abs() + 4 * U * (y.abs() + b.abs())
    return y, mean[:, 0], rstd[:, 0], d_y, d_mean[:, 0], d_rstd[:, 0], ok[:, 0]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype, w_dtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)],
                         ids=["f32", "f16", "f16_f32", "bf16", "bf16_f32"])
def test_layer_norm(cols, dtype, w_dtype):
    rows = 1 if cols > 8192 else 37
    x = rand(10, rows, cols, dtype=dtype) + 0.25
    w, b = 1 + rand(11, cols, dtype=w_dtype, std=0.2), rand(12, cols, dtype=w_dtype)
    y, mean, rstd = digital.layer_norm(x, w, b, 1e-3)
    ref, mean64, rstd64, d_y, d_mean, d_rstd, ok = norm_reference(x, w, b, 1e-3)
    assert ok.all()
    close(y, ref, d_y)
    close(mean, mean64, d_mean)
    close(rstd, rstd64, d_rstd)
    assert y.dtype == dtype and mean.shape == rstd.shape == (rows,)


@pytest.mark.parametrize("rows", [1, 2, 5, 63, 1030, 5000])
def test_layer_norm_rows_slices_and_missing_parameters(rows):
    x = rand(13, rows, 130, dtype=BF16)
    w, b = rand(14, 130), rand(15, 130)
    ones, zeros = torch.ones(130), torch.zeros(130)
    for ww, bb in ((None, None), (w, None), (None, b), (w, b)):
        y = digital.layer_norm(sliced(x), ww, bb)[0]
        ref, _, _, d_y, _, _, ok = norm_reference(x, ones if ww is None else ww, zeros if bb is None else bb, 1e-5)
        assert ok.all()
        close(y, ref, d_y)
    out = sliced(x)
    same, mean, rstd = digital.layer_norm(out, w, b, out=out)                 # in place, inside a larger matrix
    assert same is out and torch.equal(out, y) and torch.isnan(out._base[:, :3]).all()
    y3, mean3, _ = digital.layer_norm(x.view(rows, 1, 130), w, b)
    assert torch.equal(y3.view(rows, 130), y) and mean3.shape == (rows, 1) and torch.equal(mean3[:, 0], mean)
    assert digital.layer_norm(x[:0])[1].shape == (0,)


def test_layer_norm_keeps_small_differences_of_large_values():
    """An offset of 1000 and differences of one: the variance is that of the differences, not a difference of squares."""
    x = rand(16, 16, 768) + 1000.0
    y, mean, rstd = digital.layer_norm(x, eps=0.0)
    ref, _, _, d_y, _, _, ok = norm_reference(x, torch.ones(768), torch.zeros(768), 0.0)
    assert ok.all()
    close(y, ref, d_y)
    # the squares of 1000 in 32 bits alone would move y by a hundredth and more
    assert (y.double().cpu() - ref).abs().max() < 1e-3


def test_layer_norm_of_constant_rows_infinities_and_nan():
    x = torch.ones(8, 300, device="cuda")
    x[3] = float("nan")
    x[4, 7] = float("inf")
    w, b = rand(17, 300), rand(18, 300)
    y, mean, rstd = digital.layer_norm(x, w, b)
    for row in (0, 1, 2, 5, 6, 7):      # no spread: bias alone
        assert torch.equal(y[row], b)
    assert torch.isnan(y[3]).all() and torch.isnan(y[4]).all()
    dx, dw, db = digital.layer_norm_backward(torch.ones_like(x), x, mean, rstd, w)
    assert torch.isfinite(dx[[0, 1, 2, 5, 6, 7]]).all() and torch.isfinite(db).all()


def norm_backward_reference(d, x, mean, rstd, w, base):
    n, rows = x.size(1), x.size(0)
    d, x, mean, rstd, w = (t.double().cpu() for t in (d, x, mean[:, None], rstd[:, None], w))
    h = (x - mean) * rstd
    d_h = 2.01 * U * h.abs()
    g = d * w
    s1, s2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    d_s1 = (n + 2) * U * g.abs().mean(1, keepdim=True)
    d_s2 = (n + 6) * U * (g * h).abs().mean(1, keepdim=True)
    dx = rstd * (g - s1 - h * s2)
    size = rstd * (g.abs() + s1.abs() + (h * s2).abs())
    d_dx = rstd * (d_s1 + h.abs() * d_s2 + d_h * s2.abs()) + 6 * U * size
    if base is not None:
        dx = dx + base.double().cpu()
        d_dx = d_dx + U * (dx.abs() + d_dx)
    dw, db = (d * h).sum(0), d.sum(0)
    return dx, dw, db, d_dx, (rows + 4) * U * (d * h).abs().sum(0), (rows + 1) * U * d.abs().sum(0)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype, w_dtype", [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)],
                         ids=["f32", "f16", "f16_f32", "bf16", "bf16_f32"])
def test_layer_norm_backward(cols, dtype, w_dtype):
    rows = 3 if cols > 8192 else 41
    x, d, base = rand(20, rows, cols, dtype=dtype), rand(21, rows, cols, dtype=dtype), rand(22, rows, cols, dtype=dtype)
    w = 1 + rand(23, cols, dtype=w_dtype, std=0.2)
    _, mean, rstd = digital.layer_norm(x, w, w)
    for add in (None, base):
        dx, dw, db = digital.layer_norm_backward(d, x, mean, rstd, w, base=add)
        ref = norm_backward_reference(d, x, mean, rstd, w, add)
        for got, expected, bound in zip((dx, dw, db), ref[:3], ref[3:]):
            close(got, expected, bound)
        assert dx.dtype == dtype and dw.dtype == db.dtype == w_dtype


@pytest.mark.parametrize("rows, cols", [(0, 70), (1, 70), (2, 1030), (9, 768), (700, 768), (3000, 70), (20000, 40), (2500, 1537), (1100, 5000),
                                        (1500, 16600)])
def test_layer_norm_backward_rows(rows, cols):
    x, d, w = rand(24, rows, cols), rand(25, rows, cols), rand(26, cols)
    _, mean, rstd = digital.layer_norm(x)
    dx, dw, db = digital.layer_norm_backward(d, x, mean, rstd, w)
    if not rows:
        assert dx.shape == (0, cols) and (dw == 0).all() and (db == 0).all()
        return
    ref = norm_backward_reference(d, x, mean, rstd, w, None)
    for got, expected, bound in zip((dx, dw, db), ref[:3], ref[3:]):
        close(got, expected, bound)
    again = digital.layer_norm_backward(d, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))        # sums in a fixed order
    plain, none, none2 = digital.layer_norm_backward(d, x, mean, rstd)
    assert none is None and none2 is None
    close(plain, *(norm_backward_reference(d, x, mean, rstd, torch.ones(cols), None)[k] for k in (0, 3)))


@pytest.mark.parametrize("cols", [130, 1300, 16400])
def test_layer_norm_backward_in_place_and_slices(cols):
    x, d, base, w = rand(27, 9, cols), rand(28, 9, cols), rand(29, 9, cols), rand(30, cols)
    _, mean, rstd = digital.layer_norm(x)
    dx, dw, db = digital.layer_norm_backward(d, x, mean, rstd, w, base=base)
    for k in range(3):
        given = [x.clone(), d.clone(), base.clone()]
        got = digital.layer_norm_backward(given[1], given[0], mean, rstd, w, base=given[2], out=given[k])
        assert got[0] is given[k] and all(torch.equal(p, q) for p, q in zip(got, (dx, dw, db)))
    out = sliced(torch.zeros_like(x))
    got = digital.layer_norm_backward(sliced(d), sliced(x, 2, 2), mean, rstd, w, base=sliced(base, 1, 8), out=out)
    assert all(torch.equal(p, q) for p, q in zip(got, (dx, dw, db))) and torch.isnan(out._base[:, :3]).all()


def test_layer_norm_gradients_against_differences():
    """Difference quotients of the forward pass: what the formula's own quotient is off by, and 32-bit outputs over the step."""
    rows, cols, step = 6, 96, 2.0 ** -6
    x, w, b, d = rand(31, rows, cols), 1 + rand(32, cols, std=0.1), rand(33, cols), rand(34, rows, cols)
    _, mean, rstd = digital.layer_norm(x, w, b)
    dx, dw, db = digital.layer_norm_backward(d, x, mean, rstd, w)
    for k, gradient in enumerate((dx, dw, db)):
        given = [x, w, b]
        way = rand(35 + k, *given[k].shape)
        losses, exact, allowed = [], [], 0.0
        for sign in (1.0, -1.0):
            moved = list(given)
            moved[k] = given[k] + sign * step * way
            losses.append((digital.layer_norm(*moved)[0].double() * d.double()).sum().item())
            ref = norm_reference(*moved, 1e-5)
            exact.append((ref[0] * d.double().cpu()).sum().item())
            allowed += ((ref[3] + U * ref[0].abs()) * d.double().cpu().abs()).sum().item() / (2 * step)
        along = (gradient.double() * way.double()).sum().item()
        ref = norm_backward_reference(d, x, mean, rstd, w, None)
        bound = ((ref[3 + k] + U * ref[k].abs()) * way.double().cpu().abs()).sum().item()
        truncated = abs((exact[0] - exact[1]) / (2 * step) - (ref[k] * way.double().cpu()).sum().item())
        assert abs((losses[0] - losses[1]) / (2 * step) - along) <= allowed + bound + truncated
        assert abs(along) > 10 * (allowed + bound + truncated)


# -- low-rank adapters -------------------------------------------------------------------------------------------------

PAIRS = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]
PAIR_IDS = ["f32", "f32_bf16", "f32_f16", "bf16", "f16"]


class Set:
    """Adapters, operands, and the results in 64 bits with the worst cases of 32-bit sums beside them."""

    def __init__(self, rows, x, d, rank, n, dtype=F32, w_dtype=F32, p=0.0, index=None, seed=100):
        self.p, self.n, self.rank = p, n, rank
        self.a, self.b = rand(seed, n, rank, x, dtype=w_dtype, std=x ** -0.5), rand(seed + 1, n, d, rank, dtype=w_dtype)
        self.scale = rand(seed + 2, n)
        self.x, self.base = rand(seed + 3, rows, x, dtype=dtype), rand(seed + 4, rows, d, dtype=dtype)
        self.d, self.dx_base = rand(seed + 5, rows, d, dtype=dtype), rand(seed + 6, rows, x, dtype=dtype)
        if index is None:
            gen = torch.Generator("cpu").manual_seed(seed + 7)
            index = torch.randint(-1, n, (rows,), generator=gen, dtype=torch.int32).cuda()
        self.index = index
        self.adapters = digital.LowRankAdapters(self.a, self.b, self.scale)
        self.drop = dict(p=p, seed=12345678901234, call=6)

    def forward(self, rows=None, **kw):
        return self.adapters.forward(self.x, self.index if rows is None else rows, base=self.base, **dict(self.drop, **kw))

    def step(self, rows=None):
        rows = digital.AdapterRows(self.index, self.n) if rows is None else rows
        y, hidden = self.adapters.forward(self.x, rows, base=self.base, return_hidden=True, **self.drop)
        return (y, hidden, *self.adapters.backward(self.d, self.x, rows, hidden, base=self.dx_base, **self.drop))

    def reference(self):
        """y, hidden, dx, da, db and their bounds.  Every sum: its terms' magnitudes, with the errors of the factors."""
        x, d = self.x.double().cpu(), self.d.double().cpu()
        keep = torch.ones_like(x)
        if self.p:
            keep = kept(*x.shape, self.p, self.drop["seed"], self.drop["call"]).double() / (1 - self.p)
            x = torch.where(keep > 0, x * keep, torch.zeros(()).double())
        rows, k, n_out, r = x.size(0), x.size(1), d.size(1), self.rank
        y, dx = self.base.double().cpu().clone(), self.dx_base.double().cpu().clone()
        d_y, d_dx = torch.zeros_like(y), torch.zeros_like(dx)
        hidden, d_hidden = torch.zeros(rows, r).double(), torch.zeros(rows, r).double()
        da, db = torch.zeros(self.a.shape).double(), torch.zeros(self.b.shape).double()
        d_da, d_db = torch.zeros_like(da), torch.zeros_like(db)
        index = self.index.cpu()
        for i in sorted(set(index.tolist())):
            if not 0 <= i < self.n:
                continue
            at = torch.nonzero(index == i)[:, 0]
            a, b, s = self.a[i].double().cpu(), self.b[i].double().cpu(), self.scale[i].double().cpu()
            xi, di, m = x[at], d[at], at.numel()
            v = xi @ a.T
            d_v = (k + 2) * U * (xi.abs() @ a.abs().T)
            hidden[at], d_hidden[at] = v, d_v
            term = s.abs() * ((v.abs() + d_v) @ b.abs().T)
            y[at] += s * (v @ b.T)
            d_y[at] = s.abs() * (d_v @ b.abs().T) + (r + 3) * U * term + U * (y[at].abs() + term)
            u = s * (di @ b)
            d_u = (n_out + 2) * U * s.abs() * (di.abs() @ b.abs())
            term = (u.abs() + d_u) @ a.abs()
            dx[at] += (u @ a) * keep[at]
            d_dx[at] = (d_u @ a.abs() + (r + 3) * U * term) * keep[at] + U * (dx[at].abs() + term * keep[at])
            da[i], d_da[i] = u.T @ xi, d_u.T @ xi.abs() + (m + 3) * U * ((u.abs() + d_u).T @ xi.abs())
            db[i] = s * (di.T @ v)
            d_db[i] = s.abs() * (di.abs().T @ d_v + (m + 3) * U * (di.abs().T @ (v.abs() + d_v)))
        return (y, hidden, dx, da, db), (d_y, d_hidden, d_dx, d_da, d_db)

    def check(self, results):
        for got, expected, bound in zip(results, *self.reference()):
            assert got.shape == expected.shape
            close(got, expected, bound)


SHAPES = [  # rows, x, d, rank, adapters
    (1, 1, 1, 1, 1), (1, 768, 2304, 16, 3), (2, 7, 9, 3, 2), (8, 64, 33, 16, 32), (16, 100, 31, 5, 1), (17, 31, 100, 17, 2),
    (33, 129, 257, 33, 4), (64, 40, 24, 8, 64), (65, 785, 300, 5, 7), (200, 96, 64, 64, 3), (300, 70, 50, 65, 2), (129, 33, 130, 128, 2),
    (2100, 64, 48, 16, 1), (2500, 40, 72, 24, 300), (5000, 24, 16, 2, 1000), (17000, 16, 24, 4, 3),
]


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows, x, d, rank, n", SHAPES)
def test_adapters_forward_and_backward(rows, x, d, rank, n, dtype, w_dtype):
    s = Set(rows, x, d, rank, n, dtype, w_dtype, p=0.25 if (rows + rank) % 2 else 0.0)
    s.check(s.step())
    close(s.forward(), *(t[0] for t in s.reference()))                        # the index alone, few rows without a plan
    again = s.step()
    assert all(torch.equal(p, q) for p, q in zip(s.step(), again))            # sums in a fixed order


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows, x, d, rank, n", [
    (70, 7, 300, 128, 2), (70, 300, 5, 64, 3), (90, 3, 2, 20, 2), (66, 1, 8, 16, 1), (80, 8, 1, 33, 2), (64, 6, 700, 16, 2),  # fewer than 8 columns
    (40, 5003, 4100, 16, 2), (20, 4099, 2050, 128, 1), (65, 2050, 1111, 40, 2),                                            # many segments
    (70000, 9, 10, 3, 3), (140000, 4, 3, 2, 2), (66000, 12, 5, 17, 400),                                                   # long lists of rows
])
def test_adapters_of_extreme_sizes(rows, x, d, rank, n, dtype, w_dtype):
    s = Set(rows, x, d, rank, n, dtype, w_dtype, p=0.0 if x % 2 else 0.3)
    results = s.step()
    s.check(results)
    if rows <= 64:
        close(s.forward(), *(t[0] for t in s.reference()))
    assert all(torch.equal(p, q) for p, q in zip(s.step(), results))


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rows", [9, 200])
@pytest.mark.parametrize("d", [5, 200])
def test_base_goes_through_rows_without_adapter_bit_by_bit(dtype, rows, d):
    s = Set(rows, 24, d, 4, 2, dtype, dtype, index=(torch.arange(rows, device="cuda") % 3).to(torch.int32))
    none = s.index == 2
    s.base[none] = torch.tensor([-0.0, 0.0, float("inf"), -1.5], dtype=dtype, device="cuda").repeat(d)[:d]
    bits = {2: torch.int16, 4: torch.int32}[dtype.itemsize]
    for rows_of in (s.index, digital.AdapterRows(s.index, 2)):
        y = s.forward(rows_of)
        assert torch.equal(y[none].view(bits), s.base[none].view(bits))


@pytest.mark.parametrize("rows", [1, 15, 64, 65, 500])
def test_rows_without_adapter(rows):
    """Numbers outside of 0 .. n - 1 mean none: base goes through, and nothing of such a row reaches a gradient."""
    for numbers in ([-1], [4], [2 ** 31 - 1], [-2 ** 31], [-1, 0, 4, 3]):
        index = torch.tensor([numbers[k % len(numbers)] for k in range(rows)], dtype=torch.int32, device="cuda")
        s = Set(rows, 40, 56, 6, 4, index=index)
        none = (index < 0) | (index >= 4)
        y, hidden, dx, da, db = s.step()
        assert torch.equal(y[none], s.base[none]) and torch.equal(dx[none], s.dx_base[none]) and (hidden[none] == 0).all()
        s.check((y, hidden, dx, da, db))
        assert (s.adapters.forward(s.x, index)[none] == 0).all()              # without a base
        out = s.base.clone()
        assert s.adapters.forward(s.x, index, base=out, out=out, **s.drop) is out and torch.equal(out, y if rows > 64 else s.forward())
        s.x[none] = float("nan")
        s.d[none] = float("inf")
        after = s.step()
        assert torch.equal(after[0], y) and all(torch.equal(p, q) for p, q in zip(after[2:], (dx, da, db)))


@pytest.mark.parametrize("rows", [40, 300])
def test_nan_and_infinities_stay_with_their_row_and_adapter(rows):
    s = Set(rows, 50, 45, 7, 3, index=(torch.arange(rows, device="cuda") % 3).to(torch.int32))
    clean = s.step()
    s.x[4, 3], s.d[7, 9] = float("nan"), float("-inf")                        # both of adapter 1
    y, hidden, dx, da, db = s.step()
    other = torch.arange(rows, device="cuda") != 4
    assert torch.equal(y[other], clean[0][other]) and torch.isnan(y[4]).all()
    other = torch.arange(rows, device="cuda") != 7
    assert torch.equal(dx[other], clean[2][other]) and not torch.isfinite(dx[7]).any()
    for k in (0, 2):
        assert torch.equal(da[k], clean[3][k]) and torch.equal(db[k], clean[4][k])
    assert torch.isnan(da[1, :, 3]).all() and not torch.isfinite(db[1, 9]).any()
    few = s.forward()
    assert torch.isnan(few[4]).all() and torch.isfinite(few[torch.arange(rows, device="cuda") != 4]).all()


def test_infinite_inputs_meet_no_padding():
    """A rank that fills no matrix tile: an infinity times the padding would be NaN."""
    s = Set(20, 16, 12, 3, 1, index=torch.zeros(20, dtype=torch.int32, device="cuda"))
    s.a.fill_(1.0)
    s.b.fill_(1.0)
    s.scale.fill_(1.0)
    s.x.fill_(1.0)
    s.x[5, 2] = float("inf")
    y, hidden = s.adapters.forward(s.x, digital.AdapterRows(s.index, 1), return_hidden=True)
    assert torch.isinf(y[5]).all() and torch.isinf(hidden[5]).all() and (y[6] == 48).all()
    assert torch.isinf(s.adapters.forward(s.x, s.index)[5]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
def test_large_hidden_values_keep_their_range(dtype):
    """hidden far outside of half precision: it never leaves 32 bits (as two 16-bit numbers it would be infinite)."""
    s = Set(70, 64, 40, 8, 2, dtype, dtype)
    s.a.mul_(4000.0)
    s.b.mul_(2.0 ** -10)
    s.x.mul_(64.0)
    s.check(s.step())
    assert s.step()[1].abs().max() > 65504


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
def test_adapters_on_slices_and_more_dimensions(dtype, w_dtype):
    s = Set(90, 77, 58, 9, 3, dtype, w_dtype, p=0.1)
    y, hidden, dx, da, db = s.step()
    rows = digital.AdapterRows(s.index, 3)
    out, dx_out = sliced(torch.zeros_like(s.base)), sliced(torch.zeros_like(s.x))
    got, hidden2 = s.adapters.forward(sliced(s.x), rows, base=sliced(s.base, 1, 1), out=out, return_hidden=True, **s.drop)
    back = s.adapters.backward(sliced(s.d, 2, 9), sliced(s.x, 1, 7), rows, hidden2, base=sliced(s.dx_base), out=dx_out, **s.drop)
    assert got is out and torch.equal(out, y) and torch.equal(hidden2, hidden) and back[0] is dx_out
    assert all(torch.equal(p, q) for p, q in zip(back, (dx, da, db)))
    assert torch.isnan(out._base[:, :3]).all() and torch.isnan(dx_out._base[:, -5:]).all()
    many = s.adapters.forward(s.x.view(9, 10, 77), s.index.view(9, 10), base=s.base.view(9, 10, 58), **s.drop)
    assert torch.equal(many.view(90, 58), y)
    one = s.adapters.forward(s.x[4], s.index[4:5], base=s.base[4])
    assert one.shape == (58,)
    assert s.adapters.forward(s.x[:0], s.index[:0]).shape == (0, 58)
    none = digital.AdapterRows(s.index[:0], 3)
    y0, h0 = s.adapters.forward(s.x[:0], none, return_hidden=True)
    dx0, da0, db0 = s.adapters.backward(s.d[:0], s.x[:0], none, h0)
    assert dx0.shape == (0, 77) and (da0 == 0).all() and (db0 == 0).all()


def test_most_adapters():
    index = torch.tensor([65534, 3, 65534, 70000, 256, 255, 3, -5] * 20, dtype=torch.int32, device="cuda")
    s = Set(160, 8, 8, 2, 65535, index=index)
    s.check(s.step())


def test_plan_is_shared_and_checked():
    s = Set(100, 32, 40, 4, 5)
    rows = digital.AdapterRows(s.index, 5)
    wide = Set(100, 48, 24, 20, 5, F32, BF16, index=s.index, seed=300)
    s.check(s.step(rows))
    wide.check(wide.step(rows))
    s.index.fill_(-1)                                                         # the plan is of what the index held
    assert not torch.equal(s.step(rows)[0], s.base)
    with pytest.raises(RuntimeError, match="grouped for 5"):
        Set(100, 8, 8, 2, 4).adapters.forward(torch.zeros(100, 8, device="cuda"), rows)
    with pytest.raises(RuntimeError, match="expected 99 rows"):
        s.adapters.forward(s.x[:99], rows)
    with pytest.raises(RuntimeError, match="int32"):
        s.adapters.forward(s.x, s.index.long())
    with pytest.raises(RuntimeError, match="columns"):
        s.adapters.forward(s.x[:, :31], rows)
    with pytest.raises(RuntimeError, match="base"):
        s.adapters.forward(s.x, rows, base=s.base[:, :39])
    with pytest.raises(RuntimeError, match="type"):
        s.adapters.forward(s.x, rows, base=s.base.half())
    with pytest.raises(RuntimeError, match="16-bit rows"):
        s.adapters.forward(s.x.half(), rows)
    with pytest.raises(RuntimeError, match="hidden"):
        s.adapters.backward(s.d, s.x, rows, torch.zeros(100, 5, device="cuda"))
    with pytest.raises(RuntimeError, match="overlaps"):
        s.adapters.backward(s.d, s.x, rows, torch.zeros(100, 4, device="cuda"), out=s.x)
    with pytest.raises(RuntimeError, match="call"):
        s.adapters.forward(s.x, rows, p=0.1, call=torch.zeros(1, device="cuda"))
    with pytest.raises(RuntimeError, match="Invalid a"):
        s.adapters.a = s.a[:, :3]
        s.adapters.forward(s.x, rows)


def test_adapter_matrices_are_used_as_they_are_at_the_call():
    s = Set(20, 32, 40, 4, 2)
    before = s.forward()
    s.a.mul_(2.0)
    assert not torch.equal(s.forward(), before)
    s.adapters.a = s.a / 2.0
    assert torch.equal(s.forward(), before)


def test_adapter_gradients_against_differences():
    """y is linear in x, a and b each: a difference quotient of any step is exact but for the rounding of y."""
    s = Set(70, 48, 36, 6, 3)
    y, hidden, dx, da, db = s.step()
    dx = dx - s.dx_base
    d = s.d.double()
    for given, gradient in ((s.x, dx), (s.a, da), (s.b, db)):
        way, start = rand(400, *given.shape, std=0.5), given.clone()
        losses, allowed = [], 0.0
        for sign in (1.0, -1.0):
            given.copy_(start + sign * way)
            moved = (given.double() - start.double()) * sign                  # as the sum was rounded
            losses.append((s.adapters.forward(s.x, s.index, base=s.base).double() * d).sum().item())
            ref, bound = s.reference()
            allowed += ((bound[0] + U * (ref[0].abs() + bound[0])) * d.cpu().abs()).sum().item() / 2
            allowed += ((moved - way.double()).abs() * gradient.double().abs()).sum().item()
        given.copy_(start)
        ref, bound = s.reference()
        k = {id(s.x): 2, id(s.a): 3, id(s.b): 4}[id(given)]
        slack = bound[k] + 2 * U * ref[k].abs() + (U * s.dx_base.double().cpu().abs() if k == 2 else 0)
        allowed += (slack * way.double().cpu().abs()).sum().item()
        along = (gradient.double() * way.double()).sum().item()
        assert abs((losses[0] - losses[1]) / 2 - along) <= allowed
        assert abs(along) > 3 * allowed


# -- streams, graphs, together -----------------------------------------------------------------------------------------

def test_other_streams():
    s = Set(300, 64, 80, 8, 4, p=0.1)
    expected = s.step()
    x = rand(50, 500, 300)
    plain = digital.dropout(x, 0.4, 1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for stream in streams:                                                    # both at once, each with scratch of its own
        with torch.cuda.stream(stream):
            rows = digital.AdapterRows(s.index, s.n)
            y, hidden = s.adapters.forward(s.x, rows, base=s.base, return_hidden=True, non_blocking=True, **s.drop)
            back = s.adapters.backward(s.d, s.x, rows, hidden, base=s.dx_base, non_blocking=True, **s.drop)
            results.append((y, hidden, *back, digital.dropout(x, 0.4, 1, non_blocking=True)))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(p, q) for p, q in zip(got, (*expected, plain)))


class Block:
    """Norm, a tile with adapters, dropout and the residual sum: forward and the digital part of the backward pass."""

    def __init__(self, rows=130, size=64, dropout=0.2):
        io = dv.AnalogTileInputOutputParameter()
        io.is_perfect = True
        self.tile = InferenceTile(size, size, forward_io=io)
        self.tile.set_weights(rand(60, size, size, std=0.1).cpu())
        self.tile.cuda()
        self.adapters = digital.LowRankAdapters(rand(61, 3, 8, size, std=0.1), rand(62, 3, size, 8, std=0.1), rand(63, 3))
        self.x, self.d = rand(64, rows, size), rand(65, rows, size, std=0.1)
        self.w, self.b = 1 + rand(66, size, std=0.1), rand(67, size)
        self.index = (torch.arange(rows, device="cuda") % 4 - 1).to(torch.int32)
        self.call = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.p = dropout

    def step(self):
        drop = dict(p=self.p, seed=9, call=self.call, non_blocking=True)
        rows = digital.AdapterRows(self.index, 3)
        n, mean, rstd = digital.layer_norm(self.x, self.w, self.b, non_blocking=True)
        y = self.tile.tile.forward(n, False, False, False, True, True)
        y, hidden = self.adapters.forward(n, rows, base=y, out=y, return_hidden=True, **drop)
        out = digital.dropout(y, base=self.x, **drop)
        d_y = digital.dropout(self.d, **drop)
        d_n = self.tile.tile.backward(d_y, False, False, False, True)
        d_n, da, db = self.adapters.backward(d_y, n, rows, hidden, base=d_n, out=d_n, **drop)
        dx, dw, dbias = digital.layer_norm_backward(d_n, self.x, mean, rstd, self.w, base=self.d, non_blocking=True)
        return out, dx, da, db, dw, dbias


def test_a_block_against_its_formulas():
    """Forward and backward of the whole block in 64 bits by torch's autograd on the same masks.  The results are sums over
    up to 64 terms in each of five stages and 130 rows in the gradients; 400 U of the largest value covers any order of them
    (values are of order one, the weights' rows of order 0.8, so that no stage makes an error of another grow)."""
    block = Block()
    got = block.step()
    torch.cuda.synchronize()
    f = [t.detach().double().cpu().requires_grad_() for t in (block.x, block.adapters.a, block.adapters.b, block.w, block.b)]
    x, a, b, w, bias = f
    tile = block.tile.get_weights().double()
    keep = kept(130, 64, block.p, 9, 0).double() / (1 - block.p)
    mean = x.mean(1, keepdim=True)
    n = (x - mean) * ((x - mean).square().mean(1, keepdim=True) + 1e-5) ** -0.5 * w + bias
    y = n @ tile.T
    parts = []
    for k in range(130):
        i = k % 4 - 1
        parts.append(y[k] if i < 0 else y[k] + block.scale64(i) * (b[i] @ (a[i] @ (n[k] * keep[k]))))
    out = x + torch.stack(parts) * keep
    (out * block.d.double().cpu()).sum().backward()
    for result, expected in zip(got, [out.detach()] + [t.grad for t in f]):
        limit = 400 * U * max(1.0, float(expected.abs().max()))
        assert float((result.double().cpu() - expected).abs().max()) <= limit


Block.scale64 = lambda self, i: self.adapters.scale[i].double().cpu()


def test_captured_steps_draw_new_masks_and_keep_apart():
    """Two captured steps, replayed in turn with eager work in between: each replay is bit-equal to the eager step at its count."""
    blocks = [Block(), Block(rows=40, size=48, dropout=0.5)]
    side = torch.cuda.Stream()
    captured = []
    for block in blocks:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                block.step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results = block.step()
        captured.append((graph, results))
    seen = []
    for count in range(5):
        for block, (graph, results) in zip(blocks, captured):
            block.call.fill_(count)
            graph.replay()
            replayed = [r.clone() for r in results]
            eager = block.step()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(replayed, eager)), count
            seen.append(replayed[0])
    assert not torch.equal(seen[0], seen[2])


def test_inference_tile_with_adapters():
    io = dv.AnalogTileInputOutputParameter()
    io.is_perfect = True
    tile = InferenceTile(40, 33, forward_io=io)
    tile.set_weights(rand(70, 40, 33, std=0.1).cpu())
    tile.cuda()
    s = Set(30, 32, 40, 4, 3, seed=500)
    base = tile.forward(s.x, is_test=True, bias=True)
    y = tile.forward(s.x, is_test=True, bias=True, adapters=s.adapters, rows=s.index)
    assert torch.equal(y, s.adapters.forward(s.x, s.index, base=base))
    rows = digital.AdapterRows(s.index, 3)
    assert torch.equal(tile.forward(s.x, True, True, adapters=s.adapters, rows=rows), s.adapters.forward(s.x, rows, base=base))
    tile.alpha = 1.5       # drift compensation is of the tile alone
    assert torch.equal(tile.forward(s.x, True, True, adapters=s.adapters, rows=rows), s.adapters.forward(s.x, rows, base=base * 1.5))
    with pytest.raises(RuntimeError, match="rows"):
        tile.forward(s.x, True, True, adapters=s.adapters)
