"""Dense products with their epilogue, and their gradients, against the definition in 64 bits."""
import pytest
import torch

from mintccl_amd.dense import activation_grad, input_grad, product, weight_grad
from tests.block_oracle import DT, EVALUATED, STEEPEST, UNIT, activated64, close, product64, slope64, sum_units
from tests.expert_oracle import HALF_ULP, randn

pytestmark = pytest.mark.gpu

#: rows, cols, depth: one of everything, ends inside tiles and blocks of the depth, odd strides, every tile
SHAPES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (16, 33, 65), (17, 64, 128), (32, 100, 1000), (33, 70, 72), (64, 64, 64), (65, 130, 200), (100, 257, 8),
          (128, 128, 192), (50, 501, 250), (129, 1000, 1001), (300, 520, 136), (1, 2000, 4096), (20, 4096, 520), (40, 96, 8192), (1300, 1290, 264),
          (1408, 2560, 136), (3333, 4100, 72), (3584, 4096, 128)]


def operands(rows, cols, depth, dt, dev, seed=1):
    return randn(rows, depth, seed=seed, dtype=DT[dt], dev=dev), randn(cols, depth, seed=seed + 1, dtype=DT[dt], dev=dev)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols,depth", SHAPES)
def test_product(dev, rows, cols, depth, dt):
    x, w = operands(rows, cols, depth, dt, dev)
    want, size = product64(x, w)
    close(product(x, w), want, size, DT[dt], sum_units(depth, dt))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols,depth", SHAPES)
def test_gradients_of_a_product(dev, rows, cols, depth, dt):
    """(depth of the input's gradient: the columns; of the weight's: the rows)"""
    d, w = randn(rows, cols, seed=3, dtype=DT[dt], dev=dev), randn(cols, depth, seed=4, dtype=DT[dt], dev=dev)
    want, size = product64(d, w.t())
    close(input_grad(d, w), want, size, DT[dt], sum_units(cols, dt))
    x = randn(rows, depth, seed=5, dtype=DT[dt], dev=dev)
    want, size = product64(d.t(), x.t())
    close(weight_grad(d, x), want, size, DT[dt], sum_units(rows, dt))
    close(weight_grad(d, x, dtype=torch.float32), want, size, torch.float32, sum_units(rows, dt))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols,depth", [(192, 200, 4000), (1096, 1032, 1000), (2000, 2000, 136), (904, 2200, 1528), (1304, 3000, 1000), (3584, 4096, 128),
                                             (1704, 600, 2000), (20, 12304, 72), (7, 12304, 72)])
def test_every_tile(dev, rows, cols, depth, dt):
    """The result's rows and columns and the sums' length decide about the tiles: each kind of them in each of the three forms."""
    x, w = operands(rows, cols, depth, dt, dev)
    want, size = product64(x, w)
    units = sum_units(depth, dt)
    close(product(x, w), want, size, DT[dt], units)
    close(input_grad(x, w.t().contiguous()), want, size, DT[dt], units)
    close(weight_grad(x.t().contiguous(), w.t().contiguous()), want, size, DT[dt], units)


@pytest.mark.parametrize("activation", [None, "relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt,wide", [("bf16", False), ("bf16", True), ("f16", False), ("f32", False)])
@pytest.mark.parametrize("rows,cols,depth", [(1, 70, 100), (20, 333, 129), (70, 130, 64), (90, 77, 4000), (140, 1700, 96), (300, 2100, 41)])
def test_epilogue(dev, rows, cols, depth, dt, wide, activation):
    x, w = operands(rows, cols, depth, dt, dev)
    w = w * depth ** -0.5
    out = torch.float32 if wide else DT[dt]
    bias, residual = randn(cols, seed=7, dtype=DT[dt], dev=dev), randn(rows, cols, seed=8, dtype=out, dev=dev)
    z64, size = product64(x, w)
    z64, size = z64 + bias.cpu().double(), size + bias.cpu().double().abs()
    a64 = activated64(z64, activation)
    units = sum_units(depth, dt)
    of_a = STEEPEST * size + a64.abs() + (z64.abs() + 1) * (EVALUATED / units)
    got, z = product(x, w, bias=bias, activation=activation, residual=residual, keep=True, dtype=out)
    close(z, z64, size, DT[dt], units)
    close(got, a64 + residual.cpu().double(), of_a + residual.cpu().double().abs(), out, units)
    assert torch.equal(got, product(x, w, bias=bias, activation=activation, residual=residual, dtype=out))
    # into the residual itself, and into rows of a wider matrix
    own = residual.clone()
    assert product(x, w, bias=bias, activation=activation, residual=own, out=own) is own and torch.equal(own, got)
    room = torch.full((rows, cols + 9), 3.0, dtype=out, device=dev)
    product(x, w, bias=bias, activation=activation, residual=residual, out=room[:, 5:5 + cols])
    assert torch.equal(room[:, 5:5 + cols], got) and bool((room[:, :5] == 3).all()) and bool((room[:, 5 + cols:] == 3).all())


@pytest.mark.parametrize("activation", [None, "relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dt,wide", [("bf16", False), ("bf16", True), ("f16", True), ("f16", False), ("f32", False)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 513), (300, 70), (3000, 8)])
def test_activation_grad(dev, rows, cols, dt, wide, activation):
    z = randn(rows, cols, seed=2, dtype=DT[dt], dev=dev) * 3
    d = randn(rows, cols, seed=3, dtype=torch.float32 if wide else DT[dt], dev=dev)
    slope = slope64(z, activation)
    want = d.cpu().double() * slope
    d_z, d_bias = activation_grad(d, z, activation)
    # (a slope: at most 1.13, of terms of magnitude 1 + |z|; a sum over rows: its magnitudes, roundings as many as rows at most)
    size = d.cpu().double().abs() * (2 + z.cpu().double().abs())
    close(d_z, want, size, DT[dt], EVALUATED)
    close(d_bias, want.sum(0), size.sum(0), DT[dt], EVALUATED + rows * UNIT)
    assert torch.equal(activation_grad(d, z, activation, bias=False)[0], d_z)
    if activation is None:
        again, same = activation_grad(d, None, dtype=DT[dt])
        assert torch.equal(again, d_z) and torch.equal(same, d_bias)
        assert (again is d) == (not wide)


def test_activations_far_out(dev):
    """Numbers where exponentials leave the range: the activations and their slopes go to what they go to."""
    z = torch.tensor([[-1e4, -200.0, -89.0, -30.0, 0.0, 30.0, 89.0, 200.0, 1e4]], device=dev)
    one = torch.eye(9, device=dev)
    for name in ("relu", "silu", "sigmoid", "tanh", "gelu", "gelu_tanh"):
        got = product(z, one, activation=name)
        want, slope = activated64(z.cpu(), name), slope64(z, name)
        assert torch.allclose(got.cpu().double(), want, rtol=1e-6, atol=1e-30 if name != "gelu" else 1e-6), name
        assert torch.allclose(activation_grad(torch.ones_like(z), z, name)[0].cpu().double(), slope, rtol=1e-5, atol=1e-6), name


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols,depth", [(1, 40, 70), (20, 40, 70), (70, 90, 130), (200, 1500, 520)])
def test_rows_any_distance_apart(dev, rows, cols, depth, dt):
    """What lies between and behind the rows is not used: it is NaN."""
    x, w = operands(rows, cols, depth, dt, dev)
    want = product(x, w)
    d = randn(rows, cols, seed=9, dtype=DT[dt], dev=dev)
    of_x, of_w = input_grad(d, w), weight_grad(d, x)

    def spread(t, start, more):
        room = torch.full((t.shape[0] * (t.shape[1] + more) + start,), float("nan"), dtype=t.dtype, device=dev)
        v = room[start:].view(t.shape[0], t.shape[1] + more)[:, :t.shape[1]]
        v.copy_(t)
        return v

    for start, more in ((0, 1), (3, 8), (1, 5), (0, 8 - depth % 8 if depth % 8 else 8), (8, 64)):
        same = (lambda a, b: torch.equal(a, b))
        xs, ws, ds = (spread(t, start, more) for t in (x, w, d))
        for got, ref, units, size in ((product(xs, ws), want, depth, product64(x, w)[1]), (input_grad(ds, ws), of_x, cols, product64(d, w.t())[1]),
                                      (weight_grad(ds, xs), of_w, rows, product64(d.t(), x.t())[1])):
            # (another path may add in another order)
            assert same(got, ref) or bool(((got.double() - ref.double()).abs().cpu() <= 2 * (HALF_ULP[DT[dt]] * ref.double().abs().cpu() + sum_units(units, dt) * size)).all())


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("off_x,off_w", [(0, 1), (1, 0), (1, 1), (3, 8)])
@pytest.mark.parametrize("rows,cols,depth", [(700, 1001, 2051), (1030, 2000, 1992)])
def test_operands_that_are_copied(dev, rows, cols, depth, off_x, off_w, dt):
    """Rows that begin at any number of a wider matrix, both operands or one of them, whose surroundings are not read into the result."""
    def rows_at(t, off):
        room = torch.full((t.shape[0] + 1, t.shape[1] + 24), float("nan"), dtype=t.dtype, device=dev)
        room[:-1, off:off + t.shape[1]] = t
        return room[:-1, off:off + t.shape[1]]
    x, w = operands(rows, cols, depth, dt, dev)
    want, size = product64(x, w)
    close(product(rows_at(x, off_x), rows_at(w, off_w)), want, size, DT[dt], sum_units(depth, dt))
    d = randn(rows, cols, seed=3, dtype=DT[dt], dev=dev)
    want, size = product64(d, w.t())
    close(input_grad(rows_at(d, off_x), rows_at(w, off_w)), want, size, DT[dt], sum_units(cols, dt))
    want, size = product64(d.t(), x.t())
    close(weight_grad(rows_at(d, off_x), rows_at(x, off_w)), want, size, DT[dt], sum_units(rows, dt))


def test_nothing_to_do(dev):
    z = torch.zeros
    for dt in DT.values():
        x, w = z(0, 8, dtype=dt, device=dev), z(5, 8, dtype=dt, device=dev)
        assert product(x, w).shape == (0, 5) and product(w, x).shape == (5, 0)
        bias, residual = randn(5, seed=1, dtype=dt, dev=dev), randn(3, 5, seed=2, dtype=dt, dev=dev)
        got = product(z(3, 0, dtype=dt, device=dev), z(5, 0, dtype=dt, device=dev), bias=bias, residual=residual, activation="relu")
        assert torch.equal(got, (bias.float().relu() + residual.float()).to(dt))
        got = product(z(40, 0, dtype=dt, device=dev), z(5, 0, dtype=dt, device=dev), bias=bias)
        assert torch.equal(got, bias.expand(40, 5))
        assert torch.equal(weight_grad(z(0, 5, dtype=dt, device=dev), x), z(5, 8, dtype=dt, device=dev))
        assert torch.equal(input_grad(z(3, 0, dtype=dt, device=dev), z(0, 8, dtype=dt, device=dev)), z(3, 8, dtype=dt, device=dev))
        d_z, d_bias = activation_grad(z(0, 5, dtype=dt, device=dev), z(0, 5, dtype=dt, device=dev), "silu")
        assert d_z.shape == (0, 5) and torch.equal(d_bias, z(5, dtype=dt, device=dev))


def test_nan_and_infinity_show(dev):
    for rows in (3, 70, 300):
        x, w = operands(rows, 300, 200, "bf16", dev)
        x[1, 150], x[2, 7] = float("nan"), float("inf")
        got = product(x, w).float()
        assert bool(got[1].isnan().all()) and not bool(got[2].isfinite().any()) and bool(got[0].isfinite().all()) and (rows == 3 or bool(got[3:].isfinite().all()))


def test_gradients_against_differences(dev):
    """The loss <d, out> by x, w and bias in 32 bits: the gradient along a direction is the difference of the loss a step along it, over the step."""
    rows, cols, depth, step = 33, 50, 70, 2.0 ** -7
    x, w, b = randn(rows, depth, seed=1, dev=dev), randn(cols, depth, seed=2, dev=dev) * depth ** -0.5, randn(cols, seed=3, dev=dev)
    d = randn(rows, cols, seed=4, dev=dev)
    for name in (None, "silu", "gelu", "gelu_tanh", "tanh", "sigmoid"):
        _, z = product(x, w, bias=b, activation=name, keep=True)
        d_z, d_b = activation_grad(d, z, name)
        loss = lambda x, w, b: float((product(x, w, bias=b, activation=name).double() * d.double()).sum())  # noqa: E731
        for i, grad in enumerate((input_grad(d_z, w), weight_grad(d_z, x), d_b)):
            args = [x, w, b]
            v = torch.sign(randn(*args[i].shape, seed=20 + i, dev=dev)) * (1 if i == 0 else 0.25)
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + step * v, args[i] - step * v
            want = (loss(*up) - loss(*down)) / (2 * step)
            got, size = float((grad.double() * v.double()).sum()), float((grad.double() * v.double()).norm())
            # the third derivatives' part: step^2 / 6 of it, in a loss of rows * cols terms that are independent; and the outputs' rounding
            assert abs(got - want) <= 4 * step ** 2 * size * 4 + 1e-2 * size, (name, i, got, want, size)


def test_the_same_bits_every_time_and_on_another_stream(dev):
    side = torch.cuda.Stream()
    for rows, cols, depth in ((5, 300, 1000), (40, 96, 8192), (600, 1290, 264)):
        x, w = operands(rows, cols, depth, "bf16", dev)
        d = randn(rows, cols, seed=3, dtype=torch.bfloat16, dev=dev)
        calls = (lambda: product(x, w, activation="silu"), lambda: input_grad(d, w), lambda: weight_grad(d, x), lambda: activation_grad(d, d, "gelu")[1])
        first = [f() for f in calls]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            again = [f() for f in calls]
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again)) and all(torch.equal(a, f()) for a, f in zip(first, calls))


def test_refusals(dev):
    x, w = operands(4, 6, 8, "bf16", dev)
    cases = [
        (TypeError, "type of x", lambda: product(x, w.float())), (ValueError, "rows of 8", lambda: product(x, w[:, :7])),
        (ValueError, "one piece", lambda: product(x.t().contiguous().t(), w)), (TypeError, "bias", lambda: product(x, w, bias=torch.zeros(6, device=dev))),
        (ValueError, "bias", lambda: product(x, w, bias=torch.zeros(5, dtype=x.dtype, device=dev))),
        (ValueError, "residual", lambda: product(x, w, residual=torch.zeros(4, 5, dtype=x.dtype, device=dev))),
        (TypeError, "residual", lambda: product(x, w, residual=torch.zeros(4, 6, device=dev))),
        (TypeError, "operands' type", lambda: product(x, w, dtype=torch.float16)), (TypeError, "come in", lambda: product(x, w, dtype=torch.float64)),
        (TypeError, "another type", lambda: product(x, w, dtype=torch.float32, out=torch.zeros(4, 6, dtype=x.dtype, device=dev))),
        (ValueError, "out must be", lambda: product(x, w, out=torch.zeros(4, 7, dtype=x.dtype, device=dev))),
        (ValueError, "overlap", lambda: product(x, w, out=torch.zeros(6, dtype=x.dtype, device=dev).expand(4, 6))),
        (ValueError, "activation", lambda: product(x, w, activation="swish")), (TypeError, "device tensor", lambda: product(x, w.cpu())),
        (TypeError, "float16, bfloat16", lambda: product(x.double(), w.double())),
        (ValueError, "rows of 4", lambda: input_grad(x[:, :4].contiguous(), w)), (ValueError, "different numbers", lambda: weight_grad(x[:3], w)),
        (ValueError, "z is wanted", lambda: activation_grad(x, None, "silu")), (ValueError, "like grad", lambda: activation_grad(x, w, "silu")),
        (TypeError, "operands' type", lambda: activation_grad(x, x.to(torch.float16), "silu")),
    ]
    for error, text, call in cases:
        with pytest.raises(error, match=text):
            call()
    leaf = x.float().requires_grad_()
    for call in (lambda: product(leaf, w.float()), lambda: input_grad(leaf[:, :6], w.float()), lambda: weight_grad(leaf, x.float()),
                 lambda: activation_grad(leaf, None)):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
    with torch.no_grad():
        product(leaf, w.float())
