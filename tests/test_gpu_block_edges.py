"""Calls of the operators around an expert layer at the ends of what they take: offsets that descend, infinities, numbers that leave
the range of 32 bits, rows of no numbers and very many of them, norms with biases and without weights, tensors with tangents."""
import pytest
import torch

from mintccl_amd import _lib, block8, combine, dense, experts, routing
from mintccl_amd.common import DTYPE_CODE
from mintccl_amd.dense import activation_grad, input_grad, product, weight_grad
from mintccl_amd.norms import Norm, join, join_grad, norm, norm_grad
from mintccl_amd.routing import balance, balance_grad
from tests.block_oracle import DT, EVALUATED, UNIT, balance64, close, norm64
from tests.expert_oracle import randn
from tests.test_gpu_balance import SHARE, inputs, offsets_of, tokens_units
from tests.test_gpu_norms import a_norm, parts

pytestmark = pytest.mark.gpu


def gradient_by_the_c_abi(x, experts, offsets, found, add=None, z=0.0):
    """balance_grad into the middle of memory that is NaN, with the logits in the middle of such memory: (the gradient, whether all around it is as it was)."""
    (t, e), dev = x.shape, x.device
    def room(v):
        all_ = torch.full((t + 6, e + 5), float("nan"), dtype=x.dtype, device=dev)
        inside = all_[3:3 + t, 2:2 + e]
        if v is not None:
            inside.copy_(v)
        return all_, inside
    (_, logits), (around, out) = room(x), room(None)
    more = None if add is None else room(add)[1]
    op = _lib.BalanceOp(logits=logits.data_ptr(), chosen=experts.data_ptr(), offsets=offsets.data_ptr(), row_stride=logits.stride(0), tokens=t,
                        sequences=offsets.numel() - 1, experts=e, topk=experts.shape[1], dtype=DTYPE_CODE[x.dtype], z=z)
    one = torch.ones((), device=dev)
    _lib.check(_lib.lib().mint_balance_grad(op, one.data_ptr(), found.counts.data_ptr(), found.there.data_ptr(), 0 if more is None else more.data_ptr(),
                                            0 if more is None else more.stride(0), out.data_ptr(), out.stride(0), torch.cuda.current_stream().cuda_stream), "mint_balance_grad")
    got = out.clone()
    out.fill_(float("nan"))
    return got, bool(around.isnan().all())


ANYTHING = [[90, 10, 60], [2 ** 31 - 1, -2 ** 31, 7], [-5, 20, 2000], [0, 100, 0, 100, 0, 100], [100, 0], [60, 60, 20, 20, 80], [-1, -1, -1], "random"]


@pytest.mark.parametrize("t", [1, 5, 100, 3000, 40000])
@pytest.mark.parametrize("list_", ANYTHING, ids=str)
def test_every_row_of_the_gradient_is_written_whatever_the_offsets_say(dev, t, list_):
    """Offsets are numbers in device memory: where they descend, are negative or beyond the tokens, every row of the gradient is still some number (and
    with another gradient added, no less), and nothing around it is written."""
    x, experts = inputs(t, 9, 2, "f32", dev, masks=False)
    if list_ == "random":
        offsets = torch.randint(-t // 8, t + t // 8 + 1, (300,), generator=torch.Generator().manual_seed(t))
    else:
        offsets = torch.tensor([v if abs(v) > 2000 else v * t // 100 for v in list_])
    offsets = offsets.to(torch.int32).to(dev)
    found = balance(x, experts, offsets=offsets, z=1e-3)
    assert bool(found.loss.isfinite()) and bool(found.shares.isfinite().all())
    got, kept = gradient_by_the_c_abi(x, experts, offsets, found, z=1e-3)
    assert kept and bool(got.isfinite().all())
    more = randn(t, 9, seed=4, dev=dev)
    both, kept = gradient_by_the_c_abi(x, experts, offsets, found, more, z=1e-3)
    # (the same gradient, before the sum with the other one is rounded)
    assert kept and bool(((both.double() - more.double() - got.double()).abs() <= UNIT * (2 * got.double().abs() + more.double().abs())).all())


@pytest.mark.parametrize("world", [1, 4])
@pytest.mark.parametrize("norms", [{"kind": "layer", "biases": True}, {"kind": "rms", "biases": True}, {"kind": "layer", "weights": False},
                                   {"kind": "rms", "weights": False, "biases": True}])
def test_a_blocks_norms_with_biases_and_without_weights(dev, world, norms):
    """Each norm's weight and bias that there is has its gradient, and one that is not there has none."""
    found = experts.block_distances(world, dev, **norms)
    for name in ("before", "after"):
        for rank in range(world):
            assert (f"{name} of rank {rank}" in found) == norms.get("weights", True)
            assert (f"{name}_bias of rank {rank}" in found) == norms.get("biases", False)
    for name, off in found.items():
        assert off < (1e-4 if name == "loss" else experts.FAR), (name, off)


#: The slopes' limits at -inf and at +inf.
LIMITS = {"relu": (0.0, 1.0), "silu": (0.0, 1.0), "sigmoid": (0.0, 0.0), "tanh": (0.0, 0.0), "gelu": (0.0, 1.0), "gelu_tanh": (0.0, 1.0)}


@pytest.mark.parametrize("activation", list(LIMITS))
@pytest.mark.parametrize("dt", list(DT))
def test_slopes_at_infinities(dev, dt, activation):
    """What the activation was applied to is kept as an infinity where it leaves its type's range: the slope there is its limit."""
    inf = float("inf")
    z = torch.tensor([[-inf, inf, 1.0, -inf, inf, -2.0, 0.5, inf, -inf]], dtype=DT[dt], device=dev)
    d = torch.full_like(z, 0.5)
    d_z, d_bias = activation_grad(d, z, activation)
    low, high = LIMITS[activation]
    want = torch.where(z == -inf, low / 2, torch.where(z == inf, high / 2, d_z))
    assert torch.equal(d_z, want) and bool(d_z.isfinite().all()) and bool(d_bias.isfinite().all())
    nan = torch.full_like(z, float("nan"))
    assert bool(activation_grad(d, nan, activation)[0].isnan().all())


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_gradients_where_what_is_kept_leaves_its_range(dev, activation):
    """f16 operands whose products are below -65504: the result is near zero, and so are its gradients."""
    rows, cols, depth = 40, 24, 64
    x, w = torch.full((rows, depth), 128.0, dtype=torch.float16, device=dev), torch.full((cols, depth), 0.25, dtype=torch.float16, device=dev)
    w[3], w[5] = -32.0, 32.0
    out, z = product(x, w, activation=activation, keep=True, dtype=torch.float32)
    assert bool((z[:, 3] == -float("inf")).all()) and bool((z[:, 5] == float("inf")).all()) and bool((out[:, 3] == 0).all()) and bool((out[:, 5] == 2.0 ** 18).all())
    d_z, d_bias = activation_grad(torch.ones_like(out), z, activation)
    assert bool((d_z[:, 3] == 0).all()) and bool((d_z[:, 5] == 1).all()) and float(d_bias[3]) == 0 and float(d_bias[5]) == rows
    d_x, d_w = input_grad(d_z, w), weight_grad(d_z, x)
    assert bool(d_x.isfinite().all()) and bool(d_w.isfinite().all()) and bool((d_w[3] == 0).all())


@pytest.mark.parametrize("shape", ["channel", "row", "all"])
@pytest.mark.parametrize("width", [16, 1500, 4104, 9001])
def test_gates_by_silu_at_infinities(dev, width, shape):
    """silu goes to 0 at -inf, and its slope to 0 and, at inf, to 1: a gate of -inf shuts its numbers out, with finite gradients."""
    rows, inf = 5, float("inf")
    size = {"channel": (width,), "row": (rows, 1), "all": (rows, width)}[shape]
    g = randn(*size, seed=1, dev=dev)
    shut = torch.arange(g.numel(), device=dev).view(size) % 3 == 0
    g = torch.where(shut, -inf, g)
    s, y = randn(rows, width, seed=2, dev=dev), randn(rows, width, seed=3, dev=dev)
    r, _ = join(s, y, gate=g, gate_by="silu")
    where = shut.expand(rows, width)
    assert torch.equal(r[where], s[where]) and bool(r.isfinite().all())
    d = join_grad(s, None, r, y, gate=g, gate_by="silu")
    assert bool(d.gate.isfinite().all()) and bool((d.gate[shut] == 0).all()) and bool((d.y[where] == 0).all()) and bool(d.y.isfinite().all())
    # open without end: the gradient is that of the gate's own value (whole numbers, whose sums are exact)
    ones_ = torch.ones(rows, width, device=dev)
    wide = join_grad(ones_, None, ones_, 2 * ones_, gate=torch.full(size, inf, device=dev), gate_by="silu").gate
    assert bool((wide == 2 * {"channel": rows, "row": width, "all": 1}[shape]).all())


@pytest.mark.parametrize("bias", [None, False, True])
@pytest.mark.parametrize("width", [16, 70, 1500, 2501, 4096, 8192, 9001])
def test_infinite_gates_by_channel(dev, width, bias):
    """An infinite gate makes infinities of its channel, whether the block's output is normed (with a bias or none) or not, in rows of every length."""
    rows, inf = 6, float("inf")
    s, y = randn(rows, width, seed=1, dev=dev), randn(rows, width, seed=2, dev=dev)
    after = None if bias is None else a_norm(width, "rms", bias, torch.float32, dev, 3)
    u = y.cpu().double() if after is None else norm64(y.cpu(), *parts(after))
    g = randn(width, seed=5, dev=dev)
    at = torch.arange(width, device=dev)
    g[at % 5 == 1], g[at % 5 == 3] = inf, -inf
    r, _ = join(s, y, after=after, gate=g, scale=0.5)
    want = s.cpu().double() + 0.5 * u * g.cpu().double()
    ends = want.isinf() & (u.abs() > 1e-4)                    # (u is off by less than that: its sign is known)
    assert int(ends.sum()) > width and torch.equal(r.cpu().double()[ends], want[ends]) and bool(r.cpu()[~want.isinf()].isfinite().all())


def test_long_rows_beyond_a_launchs_thread_blocks(dev):
    """Rows too long for registers, more of them than one launch takes: each is what it is alone."""
    rows, width = (1 << 18) + 1037, 8200
    g = torch.Generator(dev).manual_seed(3)
    s, y = (torch.empty(rows, width, dtype=torch.bfloat16, device=dev).normal_(generator=g) for _ in range(2))
    n = a_norm(width, "layer", True, torch.bfloat16, dev, 3)
    row = torch.randn(rows, 1, generator=g, device=dev)
    for gate in (torch.sigmoid(n.weight), row, y):
        new, h = join(s, y, after=n, before=n, gate=gate)
        for part in (slice(0, 5), slice(1030, 1045), slice((1 << 18) - 3, (1 << 18) + 4), slice(rows - 5, rows)):
            alone = join(s[part].clone(), y[part].clone(), after=n, before=n, gate=gate if gate.dim() == 1 else gate[part].clone())
            assert torch.equal(new[part], alone[0]) and torch.equal(h[part], alone[1])
    again = join(s, y, after=n, before=n, gate=y, out=s)
    assert torch.equal(again[0], new) and torch.equal(again[1], h)
    del s, y, new, h, again
    torch.cuda.empty_cache()


def test_more_long_rows_than_a_launch_has_threads_for(dev):
    """2^22 rows of 8200 numbers, all of them one: the results are 69 GB."""
    rows, width = 1 << 22, 8200
    x = randn(1, width, seed=1, dtype=torch.bfloat16, dev=dev)
    n = a_norm(width, "rms", False, torch.bfloat16, dev, 3)
    want, got = norm(x, n), norm(x.expand(rows, width), n)
    for i in range(0, rows, 1 << 18):
        assert bool((got[i:i + (1 << 18)] == want).all())
    del got
    torch.cuda.empty_cache()


def test_tensors_with_a_tangent_are_refused(dev):
    """Results carry no tangent of forward-mode differentiation, so an operand that has one is refused, by each of the operators."""
    from torch.autograd import forward_ad
    x, w, d = (torch.randn(8, 128, generator=torch.Generator().manual_seed(i)).to(dev) for i in range(3))
    n, one = Norm(w[0].contiguous()), torch.ones((), device=dev)
    weights, chosen = routing.route(x, 2)
    plan = routing.assign(chosen, 128)
    found = balance(x, chosen)
    eight = block8.quantise_weight(w)
    rows = torch.randn(16, 128, generator=torch.Generator().manual_seed(5)).to(dev)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        of = lambda call, *at: [lambda i=i: call(*(dual(t) if k == i else t for k, t in enumerate(at))) for i in range(len(at))]  # noqa: E731
        calls = [*of(lambda a: norm(a, n), x), *of(lambda a: norm(x, Norm(a)), n.weight), *of(join, x, w), *of(lambda a: join(x, w, gate=a), d),
                 *of(lambda a, b: norm_grad(a, b, n), d, x), *of(lambda a, b, c, e: join_grad(a, b, c, e, before=n), d, d, x, w),
                 *of(dense.product, x, w), *of(lambda a, b: dense.product(x, w, bias=a, residual=b), w[:, 0].contiguous(), d[:, :8].contiguous()),
                 *of(lambda a, b: dense.activation_grad(a, b, "silu"), d, x), *of(dense.input_grad, d[:, :8].contiguous(), w), *of(dense.weight_grad, d, x),
                 *of(lambda a: balance(a, chosen), x), *of(lambda a, b: balance_grad(a, b, chosen, found, add=d), one, x), *of(lambda a: balance_grad(one, x, chosen, found, add=a), d),
                 *of(lambda a: routing.route(a, 2), x), *of(lambda a, b: routing.route_grad(a, b, chosen), weights, x),
                 *of(lambda a: block8.quantise(a), x), *of(lambda a: block8.quantise_weight(a), w), *of(lambda a: block8.product(a, eight), x),
                 *of(lambda a, b: combine.combine(a, plan, b), rows, weights), *of(lambda a, b, c: combine.combine_grad(a, b, plan, c), d, rows, weights)]
        for call in calls:
            with pytest.raises(RuntimeError, match="tangent"):
                call()
        # what it was made from is taken, also under no_grad, which leaves tangents alone
        want = norm(x, n)
        assert torch.equal(norm(forward_ad.unpack_dual(dual(x)).primal, n), want)
        with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
            norm(dual(x), n)
        x_dual = dual(x)
        with torch.inference_mode():
            assert torch.equal(norm(x_dual, n), want)
    assert torch.equal(norm(x, n), want)


def test_gates_by_row_of_rows_without_numbers(dev):
    """Rows of no numbers have a gate each all the same: its gradient is a sum of nothing."""
    s, gate = torch.zeros(5, 0, device=dev), randn(5, 1, seed=1, dev=dev)
    for options in ({"gate": gate}, {"after": Norm(None)}, {"before": Norm(None)}, {"gate": s, "after": Norm(s[0])}, {"gate": s[0]}):
        assert join(s, s, **options)[0].shape == join_grad(s, None, s, s, **options).y.shape == (5, 0)
    assert torch.equal(join_grad(s, None, s, s, gate=gate, gate_by="silu").gate, torch.zeros(5, 1, device=dev))
    for dt in DT.values():
        room = torch.full((700 * 3,), float("nan"), dtype=dt, device=dev)
        op = _lib.JoinGradOp(to_gate=room.data_ptr(), to_gate_stride=3, d_stream=gate.data_ptr())
        op.join = _lib.JoinOp(stream=gate.data_ptr(), y=gate.data_ptr(), gate=gate.data_ptr(), rows=699, width=0, stream_dtype=_lib.F32, dtype=_lib.F32,
                              gate_dtype=DTYPE_CODE[dt], gate_form=2, scale=1.0, carry=1.0)
        _lib.check(_lib.lib().mint_join_grad(op, torch.cuda.current_stream().cuda_stream), "mint_join_grad")
        room = room.view(700, 3)
        assert bool((room[:699, 0] == 0).all()) and bool(room[:, 1:].isnan().all()) and bool(room[699].isnan().all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("t,e,lengths", [(40, 24, None), (700, 200, None), (900, 40, [11] * 81), (1200, 12, [1, 0, 3, 7] * 100), (300, 600, [150, 150])])
def test_sigmoids_that_are_all_too_small_for_32_bits(dev, t, e, lengths, dt):
    """Tokens whose logits are all far below zero still have shares: their sigmoids' quotients, which no power of e leaves the range of."""
    x, experts = inputs(t, e, 3, dt, dev)
    offsets = offsets_of(lengths, dev, 2 if lengths and sum(lengths) + 2 < t else 0)
    far = torch.arange(t, device=dev) // 3 % 4
    x = (x.float() - torch.tensor([0.0, 90.0, 140.0, 400.0], device=dev)[far][:, None]).to(DT[dt])
    got = balance(x, experts, score="sigmoid", offsets=offsets, z=1e-3)
    leaf = x.cpu().double().requires_grad_()
    loss, counts, shares, there = balance64(leaf, experts.cpu(), "sigmoid", None if offsets is None else offsets.cpu(), 1e-3)
    assert torch.equal(got.counts.cpu(), counts) and torch.equal(got.there.cpu(), there)
    units = tokens_units(t)
    close(got.shares, shares, shares, torch.float32, units)
    close(got.loss, loss.detach(), loss.detach(), torch.float32, 2 * units + (64 + 16 + len(lengths or []) / 64) * UNIT)
    grad = balance_grad(torch.ones((), device=dev), x, experts, got, score="sigmoid", offsets=offsets, z=1e-3)
    want = torch.autograd.grad(loss, leaf)[0].masked_fill(torch.isneginf(leaf), 0)
    v, some, every = leaf.detach(), max(int((there > 0).sum()), 1), max(int(there.sum()), 1)
    p = (torch.sigmoid(v) / torch.sigmoid(v).sum(1, keepdim=True)).nan_to_num(0)
    # (the sums' log is rounded at the magnitude of the logits: that is in the first factor of z's part)
    size = 2e-3 / every * (torch.logsumexp(v, 1, keepdim=True).abs() + 16).nan_to_num(0, 0, 0) * torch.softmax(v, 1).nan_to_num(0)
    ends = [0, t] if offsets is None else offsets.tolist()
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        load = e * counts[i].double() / (3 * max(int(there[i]), 1)) / (some * max(int(there[i]), 1))
        size[a:b] += p[a:b] * (load + (p[a:b] * load).sum(1, keepdim=True))
    close(grad, want, size, DT[dt], 4 * SHARE)


@pytest.mark.parametrize("e", [24, 100, 200, 400, 1000])
def test_a_tokens_gradient_does_not_depend_on_the_tokens_beside_it(dev, e):
    """... not even where those are done again: to the last bit."""
    x, experts = inputs(300, e, 3, "f32", dev, masks=False)
    x = x - torch.tensor([0.0, 38.0, 41.0, 43.0, 60.0], device=dev)[torch.arange(300, device=dev) % 5][:, None]
    other = x.clone()
    other[::3] -= 300.0
    one = torch.ones((), device=dev)
    for offsets in (None, torch.tensor([0, 7, 7, 100, 300], dtype=torch.int32, device=dev)):
        found = balance(x, experts, score="sigmoid", offsets=offsets)
        a, b = (balance_grad(one, v, experts, found, score="sigmoid", offsets=offsets) for v in (x, other))
        same = torch.arange(300, device=dev) % 3 != 0
        assert torch.equal(a[same], b[same]) and bool(a.isfinite().all()) and bool(b.isfinite().all())


def test_slopes_of_the_hyperbolic_tangent_far_out(dev):
    """1 / cosh^2, relative to itself: its exponential is a few roundings off, two reciprocals and three products are one each or two."""
    z = torch.linspace(-40, 40, 4001, device=dev)[None]
    want = 1 / torch.cosh(z.cpu().double()) ** 2
    close(activation_grad(torch.ones_like(z), z, "tanh")[0], want, want, torch.float32, EVALUATED)


@pytest.mark.parametrize("shape", ["channel", "row", "all"])
@pytest.mark.parametrize("width", [200, 4104, 9001])
def test_slopes_of_gates_by_a_hyperbolic_tangent_far_out(dev, width, shape):
    """A gate's gradient by tanh, relative to itself: 1 / cosh^2 has no difference that cancels."""
    rows = 3
    size = {"channel": (width,), "row": (rows, 1), "all": (rows, width)}[shape]
    n = torch.Size(size).numel()
    g = (torch.arange(n, device=dev) * (40.0 / max(n - 1, 1)) - (20 if shape != "row" else 9)).view(size)
    ones_ = torch.ones(rows, width, device=dev)
    got = join_grad(ones_, None, ones_, ones_, gate=g, gate_by="tanh").gate
    want = (width if shape == "row" else rows if shape == "channel" else 1) / torch.cosh(g.cpu().double()) ** 2
    # (the sums are of whole numbers; one product and its rounding beside the slope's own 16)
    close(got, want, want, torch.float32, 18 * UNIT)


def test_sums_over_rows_of_very_many_columns(dev):
    """More columns than a grid's first dimension has threads for: 2^28 of a bias, 2^26 of a norm's weight."""
    cols = (1 << 28) + 77
    d = torch.empty(2, cols, dtype=torch.float16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    d_bias = activation_grad(d, None)[1]
    # (two numbers, added in 32 bits and rounded once)
    assert torch.equal(d_bias, (d[0].float() + d[1].float()).half())
    del d, d_bias
    width = (1 << 26) + 24
    x = torch.ones(2, width, dtype=torch.bfloat16, device=dev)
    x[1] = -1
    d = (torch.arange(width, device=dev) % 64).bfloat16().expand(2, width).clone()
    d[1] *= 3
    n = Norm(torch.ones(width, dtype=torch.bfloat16, device=dev), torch.zeros(width, dtype=torch.bfloat16, device=dev), "rms", 0.0)
    got = norm_grad(d, x, n)
    # (the rows' mean squares are 1: the weight's gradient is d0 - 3 d0, the bias's d0 + 3 d0, whole numbers)
    assert torch.equal(got.weight, -2 * d[0]) and torch.equal(got.bias, 4 * d[0])
    del d, x, n, got
    torch.cuda.empty_cache()
