"""Norms, the residual stream's join and their gradients against the definition in 64 bits."""
import pytest
import torch

from mintccl_amd.norms import Norm, join, join_grad, norm, norm_grad
from tests.block_oracle import DT, ROW, close, gate64, join_grad64, norm64, norm_grad64, norm_parts
from tests.expert_oracle import HALF_ULP, randn

pytestmark = pytest.mark.gpu

#: every kernel: a wavefront to a row, thread blocks of 256 to 1024, rows that do not fit registers; ends inside a lane's numbers
WIDTHS = [1, 7, 64, 65, 512, 520, 1023, 1024, 1500, 2048, 2501, 4096, 5000, 8192, 9001, 16384, 20011]
EPS = 1e-5
GATES = [(None, None), ("channel", None), ("row", "tanh"), ("all", "sigmoid"), ("all", "silu"), ("channel", "tanh"), ("row", None)]


def rows_for(width):
    return 37 if width <= 2048 else 5


def cpu(t):
    return None if t is None else t.cpu()


def parts(n):
    return None if n is None else (cpu(n.weight), cpu(n.bias), n.kind, n.eps)


def a_norm(width, kind, bias, dt, dev, seed):
    return Norm((1 + 0.2 * randn(width, seed=seed)).to(dt).to(dev), randn(width, seed=seed + 1, dtype=dt, dev=dev) if bias else None, kind, EPS)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("kind,bias", [("rms", False), ("layer", True), ("rms", True), ("layer", False)])
@pytest.mark.parametrize("x_dt,dt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")])
def test_norm_and_its_gradient(dev, width, kind, bias, x_dt, dt):
    rows = rows_for(width)
    x = randn(rows, width, seed=1, dtype=DT[x_dt], dev=dev) * 3 + 0.5
    n = a_norm(width, kind, bias, DT[x_dt], dev, 2)
    want = norm64(x.cpu(), cpu(n.weight), cpu(n.bias), kind, EPS)
    size = norm_parts(x.cpu(), kind, EPS)[2] * n.weight.cpu().double().abs() + (n.bias.cpu().double().abs() if bias else 0)
    close(norm(x, n, dtype=DT[dt]), want, size, DT[dt])
    d = randn(rows, width, seed=5, dtype=DT[dt], dev=dev)
    got = norm_grad(d, x, n)
    wants, sizes = norm_grad64(d.cpu(), x.cpu(), n.weight.cpu(), kind, EPS)
    close(got.x, wants[0], sizes[0], DT[x_dt])
    close(got.weight, wants[1], sizes[1], DT[x_dt])
    assert (got.bias is not None) == bias
    if bias:
        close(got.bias, wants[2], sizes[2], DT[x_dt])


def check_join(dev, rows, width, kind, bias, s_dt, dt, after, before, gate, gate_by, d_stream=True, d_next=True, seed=1):
    stream, y = randn(rows, width, seed=seed, dtype=DT[s_dt], dev=dev) * 2, randn(rows, width, seed=seed + 1, dtype=DT[dt], dev=dev) * 3
    after = a_norm(width, kind, bias, DT[s_dt], dev, seed + 2) if after else None
    before = a_norm(width, kind, bias, DT[s_dt], dev, seed + 4) if before else None
    shape = {None: None, "channel": (width,), "row": (rows, 1), "all": (rows, width)}[gate]
    g = randn(*shape, seed=seed + 6, dtype=DT[dt], dev=dev) if shape else None
    options = {"after": after, "gate": g, "gate_by": gate_by, "scale": 0.75, "carry": 1.125, "before": before}
    r, h = join(stream, y, **options)
    y64 = y.cpu().double()
    u, size = y64, y64.abs()
    if after:
        u = norm64(y.cpu(), *parts(after))
        size = norm_parts(y.cpu(), kind, EPS)[2] * after.weight.cpu().double().abs() + (after.bias.cpu().double().abs() if bias else 0)
    if g is not None:
        a = gate64(g.cpu(), gate_by)[0]
        u, size = u * a, size * a.abs()
    s64 = stream.cpu().double()
    close(r, 1.125 * s64 + 0.75 * u, 1.125 * s64.abs() + 0.75 * size, DT[s_dt])
    assert (h is not None) == (before is not None)
    if before:
        # the norm is of the stream as it is stored: norm() of it, to the last bit
        assert torch.equal(h, norm(r, before, dtype=DT[dt]))
    ds = randn(rows, width, seed=seed + 7, dtype=DT[s_dt], dev=dev) if d_stream or not before else None
    dn = randn(rows, width, seed=seed + 8, dtype=DT[dt], dev=dev) if d_next and before else None
    got = join_grad(ds, dn, r, y, **options)
    want = join_grad64(cpu(ds), cpu(dn), r.cpu(), y.cpu(), after=parts(after), gate=cpu(g), gate_by=gate_by, scale=0.75, carry=1.125, before=parts(before))
    types = {"stream": DT[s_dt], "y": DT[dt], "gate": DT[dt]}
    for name, value in got._asdict().items():
        absent = name == "gate" and g is None or name.startswith("after") and not after or name.startswith("before") and not before or name.endswith("bias") and not bias
        assert (value is None) == absent, name
        if value is not None:
            # (sums of up to 37 rows, of values that the row's sums have gone into twice: the block's and the stream's)
            close(value, *want[name], types.get(name, DT[s_dt]), 2 * ROW)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("s_dt,dt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")])
def test_join_and_its_gradient(dev, width, s_dt, dt):
    for i, (gate, by) in enumerate(GATES[:5]):
        check_join(dev, rows_for(width), width, ("rms", "layer")[i % 2], i % 2 == 1, s_dt, dt, True, True, gate, by)


@pytest.mark.parametrize("width", [64, 70, 1024, 1023, 2048, 2047, 4096, 4095, 8192, 8191])
@pytest.mark.parametrize("s_dt,dt", [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")])
def test_every_gate_with_and_without_biases(dev, width, s_dt, dt):
    """All kernels of the gradients: a gate's kind, biases or none, whole lanes or not, each number of lanes."""
    for gate in ("channel", "row", "all"):
        for bias in (False, True):
            check_join(dev, 5, width, "layer", bias, s_dt, dt, True, True, gate, "tanh")


@pytest.mark.parametrize("gate,by", GATES)
@pytest.mark.parametrize("after,before", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("width", [130, 1500, 9001])
def test_join_with_and_without(dev, width, after, before, gate, by):
    for kind, bias in (("rms", False), ("layer", True), ("rms", True)):
        for d_stream, d_next in ((True, True), (True, False), (False, True)):
            check_join(dev, 6, width, kind, bias, "f32", "bf16", after, before, gate, by, d_stream, d_next)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 255, 1030, 2100, 4500])
@pytest.mark.parametrize("width", [33, 700, 2050])
def test_sums_over_many_rows(dev, rows, width):
    x, d, n = randn(rows, width, seed=1, dev=dev), randn(rows, width, seed=2, dev=dev), a_norm(width, "layer", True, torch.float32, dev, 3)
    got = norm_grad(d, x, n)
    wants, sizes = norm_grad64(d.cpu(), x.cpu(), n.weight.cpu(), "layer", EPS)
    # (a group adds up to five rows one behind the other, and a column has 2048 groups, added up by 16 wavefronts, in eights)
    for value, want, size in zip(got, wants, sizes):
        close(value, want, size, torch.float32, 2 * ROW)


def test_norms_without_weights(dev):
    x, d = randn(9, 300, seed=1, dev=dev), randn(9, 300, seed=2, dev=dev)
    for kind in ("rms", "layer"):
        n = Norm(None, None, kind, EPS)
        close(norm(x, n), norm64(x.cpu(), None, None, kind, EPS), norm_parts(x.cpu(), kind, EPS)[2], torch.float32)
        got = norm_grad(d, x, n)
        wants, sizes = norm_grad64(d.cpu(), x.cpu(), None, kind, EPS)
        close(got.x, wants[0], sizes[0], torch.float32)
        assert got.weight is None and got.bias is None
    bias = randn(300, seed=3, dev=dev)
    got = norm_grad(d, x, Norm(None, bias, "layer", EPS))
    assert got.weight is None
    close(got.bias, d.cpu().double().sum(0), d.cpu().double().abs().sum(0), torch.float32)


def test_special_rows(dev):
    """Rows of zeros, of one number, of numbers that all are alike and far from zero, of the largest and smallest ones; a NaN and an
    infinity stay in their row."""
    n = Norm(torch.ones(64, device=dev), None, "rms", 1e-6)
    x = torch.zeros(7, 64, device=dev)
    x[1] = 1000.0
    x[2, 5] = 3.0
    x[3] = 1e-20
    x[4, 0], x[5, 1] = float("nan"), float("inf")
    x[6] = 1e18
    got = norm(x, n)
    assert bool((got[0] == 0).all()) and torch.allclose(got[1], torch.ones(64, device=dev)) and torch.allclose(got[2, 5], torch.tensor(8.0, device=dev))
    assert torch.allclose(got[3], torch.full((64,), 1e-17, device=dev)) and bool(got[4].isnan().all()) and bool(got[5, 1].isnan()) and bool((got[5, 2:] == 0).all())
    assert torch.allclose(got[6], torch.ones(64, device=dev))
    like = torch.full((3, 2048), 4096.0, device=dev)
    like[1, 0] = 4097.0
    centred = norm(like, Norm(None, None, "layer", 1e-5))
    assert bool((centred[0] == 0).all()) and torch.allclose(centred.cpu().double(), norm64(like.cpu(), None, None, "layer", 1e-5), rtol=1e-3, atol=1e-4)


def test_rows_any_distance_apart_and_in_place(dev):
    for rows, width, dt in ((5, 70, "bf16"), (3, 2501, "f16"), (4, 1024, "f32"), (2, 9001, "bf16")):
        t = DT[dt]
        stream, y, g = (randn(rows, width, seed=i, dtype=t, dev=dev) for i in (1, 2, 3))
        n, m = a_norm(width, "rms", False, t, dev, 4), a_norm(width, "rms", False, t, dev, 6)
        options = {"after": n, "gate": g, "gate_by": "sigmoid", "before": m}
        r, h = join(stream, y, **options)
        d = join_grad(h, r, r, y, **options)

        def spread(v):
            room = torch.full((rows, width + 13), float("nan"), dtype=v.dtype, device=dev)
            room[:, 3:3 + width] = v
            return room[:, 3:3 + width]

        wide = {**options, "gate": spread(g)}
        r2, h2 = join(spread(stream), spread(y), **wide)
        assert torch.equal(r, r2) and torch.equal(h, h2)
        for a, b in zip(d, join_grad(spread(h), spread(r), spread(r), spread(y), **wide)):
            assert a is None and b is None or torch.equal(a, b)
        own = stream.clone()
        same, h3 = join(own, y, **options, out=own)
        assert same is own and torch.equal(own, r) and torch.equal(h3, h)
        room = torch.full((rows, width + 13), 7.0, dtype=t, device=dev)
        join(stream, y, **options, out=room[:, 3:3 + width])
        assert torch.equal(room[:, 3:3 + width], r) and bool((room[:, :3] == 7).all()) and bool((room[:, 3 + width:] == 7).all())
        x = stream.clone()
        assert norm(x, n, out=x) is x and torch.equal(x, norm(stream, n))
        # a gate of which all rows are one: its gradient is that of every number, not their sum
        shared = g[:1].expand(rows, width)
        full = {**options, "gate": shared.contiguous()}
        for a, b in zip(join_grad(h, r, r, y, **full), join_grad(h, r, r, y, **{**options, "gate": shared})):
            assert a is None and b is None or torch.equal(a, b)


def test_no_rows(dev):
    x = torch.zeros(0, 33, device=dev)
    n = Norm(torch.ones(33, device=dev), torch.ones(33, device=dev), "layer", EPS)
    assert norm(x, n).shape == (0, 33)
    d = norm_grad(x, x, n)
    assert d.x.shape == (0, 33) and torch.equal(d.weight, torch.zeros(33, device=dev)) and torch.equal(d.bias, torch.zeros(33, device=dev))
    for gate in (torch.ones(33, device=dev), torch.ones(0, 1, device=dev), x):
        options = {"after": n, "before": n, "gate": gate}
        r, h = join(x, x, **options)
        d = join_grad(r, h, r, x, **options)
        assert r.shape == h.shape == d.y.shape == (0, 33) and d.gate.shape == gate.shape
        for t in (d.after_weight, d.after_bias, d.before_weight, d.before_bias) + ((d.gate,) if gate.dim() == 1 else ()):
            assert torch.equal(t, torch.zeros(33, device=dev))
    empty = torch.zeros(3, 0, device=dev)
    assert norm(empty, Norm(None)).shape == (3, 0) and norm_grad(empty, empty, Norm(None)).x.shape == (3, 0)


def test_gradients_against_differences(dev):
    rows, width, step = 7, 90, 2.0 ** -8
    leaf = {"stream": randn(rows, width, seed=1, dev=dev), "y": randn(rows, width, seed=2, dev=dev), "aw": 1 + 0.2 * randn(width, seed=3, dev=dev),
            "ab": randn(width, seed=4, dev=dev), "bw": 1 + 0.2 * randn(width, seed=5, dev=dev), "bb": randn(width, seed=6, dev=dev)}
    d, e = randn(rows, width, seed=7, dev=dev), randn(rows, width, seed=8, dev=dev)
    for kind in ("rms", "layer"):
        for by, shape in ((None, (width,)), ("sigmoid", (rows, width)), ("tanh", (rows, 1)), ("silu", (width,))):
            v = {**leaf, "gate": randn(*shape, seed=9, dev=dev)}
            options = lambda v: {"after": Norm(v["aw"], v["ab"], kind, EPS), "before": Norm(v["bw"], v["bb"], kind, EPS), "gate": v["gate"],  # noqa: E731
                                 "gate_by": by, "scale": 0.5, "carry": 1.25}
            def loss(v):
                r, h = join(v["stream"], v["y"], **options(v))
                return float((r.double() * d.double()).sum() + (h.double() * e.double()).sum())
            r, _ = join(v["stream"], v["y"], **options(v))
            g = join_grad(d, e, r, v["y"], **options(v))
            for name, grad in (("stream", g.stream), ("y", g.y), ("gate", g.gate), ("aw", g.after_weight), ("ab", g.after_bias), ("bw", g.before_weight),
                               ("bb", g.before_bias)):
                way = torch.sign(randn(*v[name].shape, seed=30, dev=dev))
                want = (loss({**v, name: v[name] + step * way}) - loss({**v, name: v[name] - step * way})) / (2 * step)
                got, size = float((grad.double() * way.double()).sum()), float(grad.double().norm())
                # the third derivatives' part (step^2 / 6 of them, each at most some tens of the first) and the losses' rounding in 32 bits
                assert abs(got - want) <= 1e-2 * size, (kind, by, name, got, want, size)


def test_the_same_bits_every_time_and_on_another_stream(dev):
    side = torch.cuda.Stream()
    for rows, width in ((3, 60), (1000, 1500), (300, 8192), (40, 9001)):
        s, y = randn(rows, width, seed=1, dev=dev), randn(rows, width, seed=2, dtype=torch.bfloat16, dev=dev)
        n = a_norm(width, "rms", False, torch.float32, dev, 3)
        options = {"after": n, "gate": y[0].contiguous(), "before": n}

        def both():
            r, h = join(s, y, **options)
            return [r, h, *(t for t in join_grad(r, h, r, y, **options) if t is not None)]

        first = both()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            again = both()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again)) and all(torch.equal(a, b) for a, b in zip(first, both()))


def test_offsets_beyond_32_bits(dev):
    """Rows whose first numbers are more than 2**32 bytes apart."""
    width, rows = 70, 3
    room = torch.zeros(2 * (1 << 31) + 4096, dtype=torch.bfloat16, device=dev)
    x = room.as_strided((rows, width), (1 << 31, 1))
    x.copy_(randn(rows, width, seed=1, dtype=torch.bfloat16, dev=dev))
    n = a_norm(width, "rms", False, torch.bfloat16, dev, 2)
    assert torch.equal(norm(x, n), norm(x.contiguous(), n))
    d = norm_grad(x, x, n)
    assert torch.equal(d.x, norm_grad(x.contiguous(), x.contiguous(), n).x)
    del room, x
    torch.cuda.empty_cache()


def test_refusals(dev):
    s, y = torch.zeros(4, 6, device=dev), torch.zeros(4, 6, dtype=torch.bfloat16, device=dev)
    n = Norm(torch.ones(6, device=dev))
    for error, text, call in [
        (ValueError, "kind", lambda: norm(s, n._replace(kind="batch"))), (TypeError, "must be a Norm", lambda: norm(s, None)),
        (ValueError, "6 channels", lambda: norm(s, Norm(torch.ones(5, device=dev)))), (TypeError, "one type", lambda: norm(s, Norm(n.weight, y[0]))),
        (ValueError, "contiguous", lambda: norm(s, Norm(torch.ones(12, device=dev)[::2]))), (TypeError, "dtype", lambda: norm(y, n, dtype=torch.float32)),
        (TypeError, "come in", lambda: norm(s, n, dtype=torch.float64)), (ValueError, "one piece", lambda: norm(torch.zeros(6, 4, device=dev).t(), n)),
        (ValueError, "like stream", lambda: join(s, y[:3])), (TypeError, "y's type or float32", lambda: join(y, s)),
        (TypeError, "y's type or float32", lambda: join(y.half(), y)), (ValueError, "gate must be", lambda: join(s, y, gate=torch.ones(5, device=dev))),
        (ValueError, "gate must be", lambda: join(s, y, gate=torch.ones(4, 2, device=dev))), (ValueError, "gate_by", lambda: join(s, y, gate=s, gate_by="relu")),
        (TypeError, "another type", lambda: join(s, y, out=y)), (ValueError, "overlap", lambda: join(s, y, out=s[:1].expand(4, 6))),
        (ValueError, "no gradient", lambda: join_grad(None, None, s, y)), (ValueError, "no norm", lambda: join_grad(s, y, s, y)),
        (TypeError, "stream's type", lambda: join_grad(y, None, s, y)), (TypeError, "result's type", lambda: join_grad(s, s, s, y, before=n)),
        (TypeError, "y must be", lambda: join_grad(s, None, s, None)),
        (TypeError, "device tensor", lambda: norm(s.cpu(), n)), (TypeError, "float16, bfloat16", lambda: norm(s.double(), n)),
    ]:
        with pytest.raises(error, match=text):
            call()
    leaf = s.clone().requires_grad_()
    for call in (lambda: norm(leaf, n), lambda: norm(s, Norm(leaf[0].detach().requires_grad_())), lambda: join(leaf, y), lambda: norm_grad(leaf, s, n)):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            call()
