"""Low-rank adapters whose factors differ by many powers of two, and infinities and NaN beside 16-bit rows.

What the second products take (hidden, up, and the factors of the gradients) is computed in 32 bits: a large value that meets a zero
leaves what a small one beside it gives with 24 bits.  The bounds are those of ``Set``: worst cases of 32-bit sums."""
import pytest
import torch

from aihwkit_amd import digital
from test_gpu_digital import BF16, F16, F32, IDS, PAIR_IDS, PAIRS, TYPES, Set, close, rand

pytestmark = pytest.mark.gpu

HIGH, LOW = 2.0 ** 8, 2.0 ** -8


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rows", [40, 70])
@pytest.mark.parametrize("rank", [2, 16, 40])
def test_a_large_hidden_value_beside_small_ones(rows, rank, dtype, w_dtype):
    """Rank 0 is 2^32 times the others and meets zeros in b."""
    s = Set(rows, 48, 40, rank, 2, dtype, w_dtype, seed=900)
    s.x[:, :8], s.x[:, 8:] = rand(901, rows, 8, dtype=dtype, std=HIGH), rand(902, rows, 40, dtype=dtype, std=LOW)
    s.a.zero_()
    s.a[:, 0, :8], s.a[:, 1:, 8:] = rand(903, 2, 8, dtype=w_dtype, std=HIGH), rand(904, 2, rank - 1, 40, dtype=w_dtype, std=LOW)
    s.b.copy_(rand(905, 2, 40, rank, dtype=w_dtype, std=2.0 ** 12))
    s.b[:, :, 0] = 0
    s.base.zero_()
    y, hidden, *_ = results = s.step()
    known = (s.index >= 0)
    assert (hidden[known, 0].abs().median() > 2.0 ** 28 * hidden[known, 1:].abs().median())
    s.check(results)
    s.check((s.forward(),))


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rank", [2, 16, 40])
def test_a_large_gradient_of_hidden_beside_small_ones(rank, dtype, w_dtype):
    """b^T d of rank 0 is 2^36 times the others' and meets zeros in a."""
    rows = 70
    s = Set(rows, 48, 40, rank, 2, dtype, w_dtype, seed=910)
    s.d[:, :8], s.d[:, 8:] = rand(911, rows, 8, dtype=dtype, std=2.0 ** 10), rand(912, rows, 32, dtype=dtype, std=2.0 ** -10)
    s.b.zero_()
    s.b[:, :8, 0], s.b[:, 8:, 1:] = rand(913, 2, 8, dtype=w_dtype, std=HIGH), rand(914, 2, 32, rank - 1, dtype=w_dtype, std=LOW)
    s.a.zero_()
    s.a[:, 0, :8], s.a[:, 1:, 8:] = rand(915, 2, 8, dtype=w_dtype, std=2.0 ** -10), rand(916, 2, rank - 1, 40, dtype=w_dtype, std=2.0 ** 11)
    s.dx_base.zero_()
    s.x.mul_(2.0 ** -8)
    s.check(s.step())


@pytest.mark.parametrize("dtype, w_dtype", PAIRS, ids=PAIR_IDS)
@pytest.mark.parametrize("rank", [1, 16, 40])
@pytest.mark.parametrize("rows", [70, 700])
@pytest.mark.parametrize("of", ["a", "b"])
def test_rows_with_large_factors_beside_rows_with_small_ones(of, rows, rank, dtype, w_dtype):
    """Gradients add up rows of one adapter.  Every other row has a factor (b^T d for a's gradient, hidden for b's) 2^36 times its
    neighbours', and zeros in the columns where those have their values."""
    s = Set(rows, 48, 40, rank, 2, dtype, w_dtype, seed=920)
    large, small, half = slice(0, None, 2), slice(1, None, 2), (rows + 1) // 2
    s.index.copy_((torch.arange(rows, device="cuda") // 4 % 2).to(torch.int32))
    factor_of, other, matrix = (s.d, s.x, s.b) if of == "a" else (s.x, s.d, s.a.transpose(1, 2))
    width = factor_of.size(1)
    matrix[:, :20] = rand(921, 2, 20, rank, dtype=w_dtype, std=HIGH)
    matrix[:, 20:] = rand(922, 2, width - 20, rank, dtype=w_dtype, std=LOW)
    for t, of_large, of_small in ((factor_of, 2.0 ** 10, 2.0 ** -10), (other, 1.0, 2.0 ** 12)):
        t.zero_()
        t[large, :20] = rand(923 + t.size(1), half, 20, dtype=dtype, std=of_large)
        t[small, 20:] = rand(924 + t.size(1), rows - half, t.size(1) - 20, dtype=dtype, std=of_small)
    results, (values, bounds) = s.step(), s.reference()
    if of == "b":
        assert results[1][large].abs().median() > 2.0 ** 28 * results[1][small].abs().median()
    k, part = (3, (slice(None), slice(None), slice(20, None))) if of == "a" else (4, (slice(None), slice(20, None)))
    assert values[k][part].abs().median() > 2.0 ** -8          # well within half precision
    close(results[k][part], values[k][part], bounds[k][part])


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows", [40, 300])
def test_nan_and_infinities_of_16_bit_rows_stay_with_their_row_and_adapter(rows, dtype):
    s = Set(rows, 50, 45, 7, 3, dtype, dtype, index=(torch.arange(rows, device="cuda") % 3).to(torch.int32))
    clean, few = s.step(), s.forward()
    s.x[4, 3], s.x[10, 5], s.d[7, 9], s.d[13, 2] = float("nan"), float("inf"), float("-inf"), float("nan")      # all of adapter 1
    y, hidden, dx, da, db = s.step()
    sound = torch.ones(rows, dtype=torch.bool, device="cuda")
    sound[[4, 10]] = False
    assert torch.equal(y[sound], clean[0][sound]) and torch.isnan(y[4]).all() and not torch.isfinite(y[10]).any()
    assert torch.equal(s.forward()[sound], few[sound]) and torch.isnan(s.forward()[4]).all()
    sound[:] = True
    sound[[7, 13]] = False
    assert torch.equal(dx[sound], clean[2][sound]) and not torch.isfinite(dx[7]).any() and torch.isnan(dx[13]).all()
    for k in (0, 2):
        assert torch.equal(da[k], clean[3][k]) and torch.equal(db[k], clean[4][k])
    assert not torch.isfinite(da[1, :, 3]).any() and not torch.isfinite(db[1, 9]).any()


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("rank", [3, 16, 40])
@pytest.mark.parametrize("rows", [20, 90])
def test_infinite_rows_give_infinities_beside_ones(rows, rank, dtype):
    """Weights of one, whose product with an infinity is the infinity: neither padding nor the parts that numbers are taken apart into
    make it a NaN."""
    s = Set(rows, 16, 24, rank, 1, dtype, dtype, index=torch.zeros(rows, dtype=torch.int32, device="cuda"))
    for t in (s.a, s.b, s.scale, s.x, s.d):
        t.fill_(1.0)
    s.x[5, 2], s.d[6, 4] = float("inf"), float("-inf")
    s.base.zero_()
    s.dx_base.zero_()
    y, hidden, dx, da, db = s.step()
    assert (y[5] == float("inf")).all() and (hidden[5] == float("inf")).all() and (y[6] == 16 * rank).all()
    assert (s.forward()[5] == float("inf")).all()
    assert (dx[6] == float("-inf")).all() and (dx[5] == 24 * rank).all()
    sound = torch.arange(16, device="cuda") != 2
    assert (da[0][:, sound] == float("-inf")).all()            # of row 6; column 2 adds an infinity of the other sign
    sound = torch.arange(24, device="cuda") != 4
    assert (db[0][sound] == float("inf")).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [20, 90])
def test_hidden_values_near_the_smallest_floats(rows, dtype):
    """hidden of 2^-120 and about: of the parts that such a number is taken apart into the second and third are subnormal."""
    s = Set(rows, 48, 40, 16, 2, dtype, dtype, seed=930)
    s.x.mul_(2.0 ** -60)
    s.a.mul_(2.0 ** -60)
    s.base.zero_()
    y, hidden = s.adapters.forward(s.x, s.index, return_hidden=True)
    values, bounds = s.reference()                       # y is of the order of hidden
    assert 2.0 ** -124 < values[1].abs().max() < 2.0 ** -112
    close(hidden, values[1], bounds[1])
    # The parts of scale * hidden are cut to multiples of the smallest bf16 number, 2^-133, so that together they are less than that short of
    # it: on top of the sums' bound y may be off by 2^-133 for every rank, times its weight.
    cut = 2.0 ** -133 * s.b.double().abs().sum(2).amax(0).cpu() if dtype == BF16 else 0.0
    close(y, values[0], bounds[0] + cut)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("cols", [5, 64, 785])
def test_dropout_of_nothing_is_the_input_bit_by_bit(cols, dtype):
    """At p = 0 nothing is drawn and every element kept, whatever it holds; a probability that rounds to no limit at all drops as little."""
    x = rand(950, 70, cols, dtype=dtype)
    x[3], x[4], x[5] = -0.0, float("inf"), torch.finfo(dtype).smallest_normal / 2
    bits = {2: torch.int16, 4: torch.int32}[dtype.itemsize]
    count = torch.tensor([7], device="cuda")
    for p, call in ((0.0, 3), (0.0, count), (2.0 ** -34, 3)):
        assert torch.equal(digital.dropout(x, p, 9, call).view(bits), x.view(bits))
    x[6] = float("nan")
    assert torch.equal(torch.isnan(digital.dropout(x, 0.0, 9)), torch.isnan(x))


@pytest.mark.parametrize("rows", [30, 100])
@pytest.mark.parametrize("rank", [12, 16, 64])
@pytest.mark.parametrize("level", [30, 0, -34])
def test_three_levels_of_hidden_values(level, rank, rows):
    """Half precision: ranks of 2^30, 1 and 2^-34, each of which alone makes a share of the columns.  The scale brings those of one level into
    the type's range."""
    s = Set(rows, 48, 45, rank, 2, F16, F16, seed=960)
    s.a.zero_()
    s.b.zero_()
    for k, exponent in enumerate((30, 0, -34)):
        x, r, d = slice(16 * k, 16 * k + 16), slice(k, None, 3), slice(k, None, 3)
        s.x[:, x] = rand(961 + k, rows, 16, dtype=F16, std=2.0 ** (exponent // 2 - 1))
        s.a[:, r, x] = rand(964 + k, *s.a[:, r, x].shape, dtype=F16, std=2.0 ** (exponent // 2 - 1))
        s.b[:, d, r] = rand(967 + k, *s.b[:, d, r].shape, dtype=F16)
    s.scale.fill_(2.0 ** -level)
    s.base.zero_()
    y, few = s.adapters.forward(s.x, digital.AdapterRows(s.index, 2), base=s.base), s.forward()
    values, bounds = s.reference()
    some = s.index.cpu() >= 0
    part = values[0][:, {30: 0, 0: 1, -34: 2}[level]::3][some].abs()
    assert 2.0 ** -4 < part.median() < 2.0 ** 8
    for got in (y, few):
        close(got, values[0], bounds[0])
