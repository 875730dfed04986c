"""The expert layer's operators against plain implementations in 64 bits: routing,
assignment, 8-bit block products, combination, and their gradients."""
import math

import numpy as np
import pytest
import torch

from mintccl_amd.block8 import Blocks, product, quantise, quantise_weight, transposed, weight_grad
from mintccl_amd.combine import combine, combine_grad
from mintccl_amd.routing import Assignment, assign, route, route_grad

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
#: relative distance of neighbouring numbers of a type, halved: what one rounding does
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in DT.values()}
#: what a number below the type's normal range may be off
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def randn(*shape, seed, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def rounded_within(got, want, dtype, extra=0.0):
    """`got` is `want` (64 bits) up to `extra`, rounded once to `dtype`."""
    got, want = got.double().cpu(), want.cpu()
    return bool(((got - want).abs() <= (want.abs() + extra) * HALF_ULP[dtype] * 1.001 + TINY[dtype] + extra).all())


# ---- routing ---------------------------------------------------------------------
def keys64(x, score, bias):
    x = x.double().cpu()
    key = (torch.sigmoid(x) if score == "sigmoid" else x) + (0 if bias is None else bias.double().cpu())
    return key.masked_fill(x == -math.inf, -math.inf)


def check_choice(x, experts, k, score="softmax", bias=None, groups=1, kept=1, group_top=1, slack=0.0):
    """The experts are k of the largest keys in order, within `slack` (0: exactly, and the lowest
    expert first among equals)."""
    key, experts = keys64(x, score, bias), experts.cpu().long()
    t, e = key.shape
    for row in range(t):
        own = key[row].clone()
        if groups > 1:
            best = own.view(groups, -1).sort(dim=-1, descending=True).values[:, :group_top]
            of = torch.where(best == -math.inf, 0, best).sum(-1).where(best[:, 0] > -math.inf, torch.tensor(-math.inf))
            order = of.sort(descending=True, stable=True).indices
            keep = order[:kept].tolist()
            used = {int(i) // (e // groups) for i in experts[row] if i >= 0}
            extra = used - set(keep)
            for g in extra:            # a group within the slack of one that was kept stands for it
                assert slack and of[g] >= of[order[kept - 1]] - slack, (row, used, keep)
            live = set(keep) if not extra else used
            for g in range(groups):
                if g not in live:
                    own.view(groups, -1)[g] = -math.inf
        for j in range(k):
            left = own.max()
            i = int(experts[row, j])
            if left == -math.inf:
                assert i == -1, (row, j)
                continue
            assert 0 <= i < e, (row, j, i)
            if slack:
                assert own[i] >= left - slack, (row, j)
            else:
                assert i == int((own == left).nonzero()[0, 0]), (row, j)
            own[i] = -math.inf


def weights64(x, experts, score, renormalise, scale):
    x = x.double()
    valid = experts >= 0
    s = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, -1).nan_to_num(0.0)
    w = s.gather(1, experts.clamp_min(0).long()) * valid
    if renormalise:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    return w * scale


ROUTES = [(1, 8, 2, "softmax", False, 1, 1, 1, True, "f32"), (5, 64, 6, "softmax", False, 1, 1, 1, False, "bf16"),
          (67, 65, 8, "softmax", True, 1, 1, 1, True, "f32"), (33, 127, 8, "sigmoid", True, 1, 1, 1, True, "f32"),
          (130, 256, 8, "sigmoid", True, 8, 4, 2, True, "f32"), (9, 256, 8, "sigmoid", True, 8, 4, 2, False, "bf16"),
          (17, 96, 4, "softmax", False, 4, 2, 1, False, "f16"), (6, 1024, 64, "softmax", False, 1, 1, 1, True, "f32"),
          (4, 1000, 16, "sigmoid", False, 4, 1, 2, True, "f16"), (3, 1, 1, "softmax", False, 1, 1, 1, False, "f32"),
          (8, 513, 3, "softmax", True, 1, 1, 1, False, "f16"), (7, 64, 64, "sigmoid", False, 64, 64, 2, True, "bf16")]


@pytest.mark.parametrize("t,e,k,score,biased,groups,kept,top,renorm,dt", ROUTES)
def test_route_and_its_gradient(dev, t, e, k, score, biased, groups, kept, top, renorm, dt):
    x = randn(t, e, seed=t * e, scale=2.0, dtype=DT[dt])
    bias = randn(e, seed=e, scale=0.1) if biased else None
    w, chosen = route(x.to(dev), k, score=score, bias=None if bias is None else bias.to(dev), groups=groups, kept=kept,
                      group_top=top, renormalise=renorm, scale=1.5)
    # a softmax without a bias goes by the logits themselves; other keys carry a few roundings of numbers below 16
    check_choice(x, chosen, k, score, bias, groups, kept, top, slack=0.0 if score == "softmax" and not biased and top == 1 else 1e-5)
    chosen = chosen.cpu()
    x64 = x.double().requires_grad_()
    want = weights64(x64, chosen, score, renorm, 1.5)
    # exp of a difference of up to 16 (half an ulp of it, 2^-21) and its own few ulps, a sum of up to 1024
    # terms over a tree of depth 16, divisions: 2^-17 in all
    assert torch.allclose(w.double().cpu(), want.detach(), rtol=2.0 ** -17, atol=1e-30)
    d = randn(t, k, seed=7)
    (want * d.double()).sum().backward()
    got = route_grad(d.to(dev), x.to(dev), chosen.to(dev), score=score, renormalise=renorm, scale=1.5)
    assert got.dtype == x.dtype and got.shape == x.shape
    # the weights' errors times d, and a cancelling difference: by the largest d and weight
    slack = 2.0 ** -16 * 1.5 * float(d.abs().max()) * max(1.0, float(want.detach().max()))
    assert rounded_within(got, x64.grad, x.dtype, extra=slack)
    # and the formula against differences of the forward pass in 64 bits
    h, probe = 1e-5, randn(t, e, seed=8).double()
    f = lambda y: float((weights64(y, chosen, score, renorm, 1.5) * d.double()).sum())  # noqa: E731
    numeric = (f(x.double() + h * probe) - f(x.double() - h * probe)) / (2 * h)
    analytic = float((got.double().cpu() * probe).sum())
    room = float((got.double().cpu().abs() * probe.abs()).sum()) * (HALF_ULP[x.dtype] * 2 + 1e-5) + 1e-4 + slack * t * k * 8
    assert abs(numeric - analytic) <= room


def test_route_masks_and_special_logits(dev):
    inf, nan = math.inf, math.nan
    rows = {
        "all masked": [-inf] * 8,
        "fewer than k": [-inf, 1.0, -inf, -inf, 2.0, -inf, -inf, -inf],
        "one": [-inf] * 7 + [0.0],
        "equal": [1.0] * 8,
        "zeros of both signs": [-1.0, -0.0, 0.0, -0.0, -2.0, 0.0, -1.0, -1.0],
        "lowest finite": [-3.0e38] * 4 + [-inf] * 4,
        "far apart": [100.0, -100.0, 90.0, 0.0, -3e38, 1.0, 2.0, 3.0],
    }
    x = torch.tensor(list(rows.values()))
    w, chosen = (v.cpu() for v in route(x.to(dev), 3))
    want = [[-1, -1, -1], [4, 1, -1], [7, -1, -1], [0, 1, 2], [1, 2, 3], [0, 1, 2], [0, 2, 7]]
    assert chosen.tolist() == want
    assert torch.allclose(w.double(), weights64(x, chosen, "softmax", True, 1.0).nan_to_num(0.0), rtol=1e-6, atol=1e-30)
    d = torch.ones(len(rows), 3)
    d[:, 1] = 2.0
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            g = route_grad(d.to(dev), x.to(dev), chosen.to(dev), score=score, renormalise=renorm).cpu()
            assert torch.isfinite(g).all()
            assert (g[0] == 0).all() and (g[x == -inf] == 0).all()
    # NaN: ranked first, shown in the weights, and the experts exist; sigmoid of infinity is 1
    y = torch.tensor([[0.0, nan, 1.0, -nan, 2.0, 3.0, -inf, 0.0], [0.0, inf, 1.0, inf, 2.0, 3.0, -inf, 0.0]])
    w, chosen = (v.cpu() for v in route(y.to(dev), 3))
    assert chosen.tolist() == [[1, 3, 5], [1, 3, 5]] and torch.isnan(w[0]).all()
    w, chosen = (v.cpu() for v in route(y.to(dev), 3, score="sigmoid", renormalise=False))
    assert chosen.tolist() == [[1, 3, 5], [1, 3, 5]] and w[1, :2].tolist() == [1.0, 1.0]
    # a bias of -inf masks too, and biased keys below zero still count
    bias = torch.tensor([-5.0, -inf, -5.0, -inf, -4.0, -6.0, -inf, -inf])
    _, chosen = route(torch.zeros(1, 8).to(dev), 6, score="sigmoid", bias=bias.to(dev))
    assert chosen.cpu().tolist() == [[4, 0, 2, 5, -1, -1]]
    # groups without an expert left, and with one
    z = torch.tensor([[-inf, -inf, 1.0, -inf, 0.5, 0.5, -inf, -inf]])
    _, chosen = route(z.to(dev), 4, groups=4, kept=3, group_top=2)
    assert chosen.cpu().tolist() == [[2, 4, 5, -1]]


def test_route_takes_rows_any_distance_apart(dev):
    wide = randn(11, 300, seed=3, dtype=torch.bfloat16).to(dev)
    for view in (wide[:, 1:257], wide[::2, :256], wide[:, :77], wide[:1].expand(5, -1)[:, :256]):
        a, b = route(view, 8), route(view.contiguous(), 8)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        d = randn(*a[0].shape, seed=4).to(dev)
        assert torch.equal(route_grad(d, view, a[1]), route_grad(d, view.contiguous(), a[1]))
    w, chosen = route(wide[:0], 4)
    assert w.shape == chosen.shape == (0, 4) and route_grad(w, wide[:0], chosen).shape == (0, 300)


# ---- assignment --------------------------------------------------------------------
def assigned(chosen, count, first=0):
    """The same on the host."""
    flat = chosen.reshape(-1).astype(np.int64) - first
    bucket = np.where((flat >= 0) & (flat < count), flat, count)
    order = np.argsort(bucket, kind="stable")
    offsets = np.concatenate([[0], np.cumsum(np.bincount(bucket, minlength=count + 1)[:count])])
    place = np.empty_like(order)
    place[order] = np.arange(len(order))
    slots = np.where(bucket < count, place, -1).reshape(chosen.shape)
    tokens = np.where(np.arange(len(order)) < offsets[-1], order // chosen.shape[1], -1)
    return offsets, tokens, slots


@pytest.mark.parametrize("t,k,e,count,first", [
    (0, 2, 4, 4, 0), (1, 1, 1, 1, 0), (1, 8, 128, 128, 0), (63, 1, 5, 5, 0), (65, 3, 7, 7, 0), (500, 6, 64, 16, 16),
    (2048, 8, 256, 256, 0), (2049, 8, 300, 37, 100), (16384, 8, 256, 256, 0), (9001, 3, 1024, 1024, 0), (20011, 4, 2, 1, 1),
    (30000, 1, 1000, 1000, 0)])
def test_assign(dev, t, k, e, count, first):
    rng = np.random.default_rng(t + k)
    chosen = rng.integers(0, e, (t, k)).astype(np.int32)
    chosen[rng.random((t, k)) < 0.1] = -1
    if t > 4:
        chosen[t // 2] = 2 ** 31 - 1                   # no expert of anybody's
        chosen[t // 3:t // 3 + 70 // k] = e - 1         # many of one expert in a row
    got = assign(torch.from_numpy(chosen).to(dev), count, first)
    for mine, want in zip(got, assigned(chosen, count, first)):
        assert mine.dtype == torch.int32 and np.array_equal(mine.cpu().numpy(), want)


# ---- rounding to 8 bits ----------------------------------------------------------------
def plain8(x, dim):
    """(values as floats before scaling, scales) by the definition, in 32 bits on the CPU."""
    x = x.float().movedim(dim, -1)
    n = x.shape[-1]
    full = torch.zeros(*x.shape[:-1], -(-n // 128) * 128)
    full[..., :n] = x
    full = full.unflatten(-1, (-1, 128))
    most = full.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -96)
    r = torch.full_like(most, 448.0) / most
    q = (full * r).to(torch.float8_e4m3fn).float().flatten(-2)[..., :n].movedim(-1, dim)
    return q, (most / torch.full_like(most, 448.0)).squeeze(-1).movedim(-1, dim)


def values(x, dim):
    q, s = plain8(x, dim)
    return q.double() * s.double().repeat_interleave(128, dim).narrow(dim, 0, x.shape[dim])


def same_floats(a, b):
    return np.array_equal(a.detach().cpu().numpy(), b.detach().cpu().numpy(), equal_nan=True)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,depth", [(1, 1), (3, 127), (2, 128), (5, 129), (70, 1000), (1, 4096), (33, 2500)])
def test_quantise_is_the_definition_bit_for_bit(dev, rows, depth, dt):
    x = randn(rows, depth, seed=rows + depth, dtype=DT[dt])
    x[:, ::17] *= 30
    q, s = quantise(x.to(dev))
    want, scale = plain8(x, 1)
    assert q.shape == x.shape and same_floats(q.float(), want) and same_floats(s, scale)


def test_quantise_special_blocks(dev):
    x = torch.zeros(8, 256)
    x[1, :128] = 2.0 ** -120                     # below what a block is scaled to
    x[2, 3], x[2, 4] = math.inf, 1.0
    x[3, 5] = math.nan
    x[4, :4] = torch.tensor([448.0, 17.0, 18.0, -19.0])       # between two 8-bit numbers: to the even one
    x[5, 7] = 3.0e38
    x[6] = randn(256, seed=1) * 1e-30
    x[7, 200] = -0.0
    for dt in (torch.float32, torch.bfloat16):
        q, s = quantise(x.to(dt).to(dev))
        want, scale = plain8(x.to(dt), 1)
        assert same_floats(s[[0, 1, 2, 4, 5, 6, 7]], scale[[0, 1, 2, 4, 5, 6, 7]])
        assert same_floats(q.float()[[0, 1, 2, 4, 5, 6, 7]], want[[0, 1, 2, 4, 5, 6, 7]])
        # a NaN shows in everything that is made from its block
        assert torch.isnan(s[3, 0]) and torch.isnan(q.float()[3, :128]).all() and (q.float()[3, 128:] == 0).all()
    strided = randn(9, 400, seed=2).to(dev)
    for view in (strided[:, 1:300], strided[::3, 8:264], strided[:1].expand(4, -1)):
        a, b = quantise(view), quantise(view.contiguous())
        assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)


def square_values(w):
    q, s = [], []
    w = w.float()
    n, k = w.shape
    full = torch.zeros(-(-n // 128) * 128, -(-k // 128) * 128)
    full[:n, :k] = w
    tiles = full.view(full.shape[0] // 128, 128, -1, 128)
    most = tiles.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -96)
    q = (tiles * (torch.full_like(most, 448.0) / most)).to(torch.float8_e4m3fn).float()
    return q.reshape(full.shape)[:n, :k], (most / torch.full_like(most, 448.0))[:, 0, :, 0]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape", [(1, 1), (127, 130), (128, 128), (300, 1000), (3, 129, 257)])
def test_quantise_weight(dev, shape, dt):
    w = randn(*shape, seed=sum(shape), dtype=DT[dt])
    got = quantise_weight(w.to(dev))
    back = transposed(got)
    for i, m in enumerate(w.reshape(-1, *shape[-2:])):
        q, s = square_values(m)
        mine = Blocks(*(v.reshape(-1, *v.shape[-2:])[i] for v in got))
        assert same_floats(mine.q.float(), q) and same_floats(mine.scale, s)
        turned = Blocks(*(v.reshape(-1, *v.shape[-2:])[i] for v in back))
        assert same_floats(turned.q.float(), q.t()) and same_floats(turned.scale, s.t())


# ---- products ------------------------------------------------------------------------
def weight64(w: Blocks):
    q, s = w.q.float().double().cpu(), w.scale.double().cpu()
    return q * s.repeat_interleave(128, -2)[..., :q.shape[-2], :].repeat_interleave(128, -1)[..., :q.shape[-1]]


def near_product(got, x, w, dtype):
    """Sums of 128 products in 32 bits, then of the blocks' (each at most 2^-23 of the sum of magnitudes,
    also where an addition cuts off), the scales' two products, and one rounding to the result's type."""
    want, size = x @ w.transpose(-1, -2), x.abs() @ w.abs().transpose(-1, -2)
    blocks = -(-x.shape[-1] // 128)
    extra = size * (128 + blocks + 4) * 2.0 ** -23
    off = (got.double().cpu() - want).abs()
    return bool((off <= extra + (want.abs() + extra) * HALF_ULP[dtype] * 1.001 + TINY[dtype]).all())


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,depth", [
    (1, 1, 1), (1, 128, 128), (1, 1000, 1000), (2, 16, 127), (7, 65, 129), (16, 4096, 512), (17, 100, 2500), (33, 257, 384),
    (50, 500, 250), (64, 64, 64), (100, 48, 4096), (129, 300, 640), (300, 130, 1000), (700, 600, 300)])
def test_product(dev, rows, cols, depth, dt):
    x = randn(rows, depth, seed=rows, dtype=DT[dt])
    w = quantise_weight(randn(cols, depth, seed=cols).to(dev))
    got = product(x.to(dev), w, dtype=DT[dt])
    assert got.dtype == DT[dt] and got.shape == (rows, cols)
    assert near_product(got, values(x, 1), weight64(w), DT[dt])
    # the same from activations rounded beforehand, and into a view of the caller's
    room = torch.full((rows, cols + 24), 7.0, dtype=DT[dt], device=dev)
    out = room[:, 3:3 + cols]
    assert product(quantise(x.to(dev)), w, out=out) is out
    assert torch.equal(out, got) and (room[:, :3] == 7).all() and (room[:, 3 + cols:] == 7).all()


@pytest.mark.parametrize("dt", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,cols,depth", [(33, 70, 4100), (64, 130, 9001), (130, 1000, 5000), (65, 4096, 2600), (40, 20, 33000)])
def test_product_of_few_tiles_and_a_long_depth(dev, rows, cols, depth, dt):
    """Thread blocks that share a tile: every call adds the same parts in the same order, whatever the workspace held."""
    x = randn(rows, depth, seed=depth, dtype=DT[dt]).to(dev)
    w = quantise_weight(randn(cols, depth, seed=cols).to(dev))
    got = product(x, w, dtype=DT[dt])
    assert near_product(got, values(x.cpu(), 1), weight64(w), DT[dt])
    rounded = quantise(x)
    for fill in (0, 1, 255):
        room = torch.full((64 << 20,), fill, dtype=torch.uint8, device=dev)
        del room                                                     # (what the next workspace is made of)
        assert torch.equal(product(x, w, dtype=DT[dt]), got)
        assert torch.equal(product(rounded, w, dtype=DT[dt]), got)


def test_product_of_few_tiles_in_a_graph(dev):
    x = randn(50, 6000, seed=1, dtype=torch.bfloat16).to(dev)
    w = quantise_weight(randn(300, 6000, seed=2).to(dev))
    out = torch.empty(50, 300, dtype=torch.bfloat16, device=dev)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        product(x, w, out=out)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            product(x, w, out=out)
    for seed in range(4):
        x.copy_(randn(50, 6000, seed=10 + seed, dtype=torch.bfloat16))
        want = product(x, w)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)



def test_product_reads_nothing_behind_a_row(dev):
    """8-bit rows in a wider buffer whose rest is NaN."""
    for rows, cols, depth in ((5, 70, 200), (130, 140, 1000), (40, 33, 17)):
        x, w = quantise(randn(rows, depth, seed=1).to(dev)), quantise_weight(randn(cols, depth, seed=2).to(dev))

        def among_nan(b):
            wide = torch.full((b.q.shape[0], 1040), 0x7F, dtype=torch.uint8, device=dev)
            wide[:, 16:16 + depth] = b.q.view(torch.uint8)
            return Blocks(wide[:, 16:16 + depth].view(b.q.dtype), b.scale)
        assert torch.equal(product(among_nan(x), among_nan(w), dtype=torch.float32), product(x, w, dtype=torch.float32))


def test_product_shows_nan_and_infinity(dev):
    x = randn(20, 300, seed=1)
    x[3, 200], x[5, 10] = math.nan, math.inf
    w = quantise_weight(randn(50, 300, seed=2).to(dev))
    got = product(x.to(dev), w, dtype=torch.float32).cpu()
    bad = torch.isnan(got).all(1)
    assert bad[3] and bad[5] and bad.sum() == 2 and torch.isfinite(got[~bad]).all()


def test_product_scales_in_any_layout(dev):
    x, w = randn(40, 500, seed=1).to(dev), quantise_weight(randn(200, 500, seed=2).to(dev))
    q, s = quantise(x)
    want = product(x, w)
    assert torch.equal(product(Blocks(q, s.contiguous()), w), want)
    assert torch.equal(product(Blocks(q, s.t().contiguous().t()), w), want)
    far = torch.zeros(2, 4, 3, device=dev)
    far[..., 0] = w.scale
    assert torch.equal(product(x, Blocks(w.q, far[..., 0])), want)


def test_product_of_nothing(dev):
    w = quantise_weight(randn(40, 256, seed=1).to(dev))
    assert product(torch.zeros(0, 256, device=dev), w).shape == (0, 40)
    assert product(torch.zeros(3, 256, device=dev), quantise_weight(torch.zeros(0, 256, device=dev))).shape == (3, 0)
    none = product(torch.zeros(3, 0, device=dev), quantise_weight(torch.zeros(5, 0, device=dev)))
    assert none.shape == (3, 5) and (none == 0).all()
    assert (weight_grad(torch.zeros(0, 5, device=dev), torch.zeros(0, 9, device=dev)) == 0).all()


def make_plan(dev, counts, t, k, seed):
    """An assignment with `counts` places for its experts, the rest of t * k pairs without."""
    rng = np.random.default_rng(seed)
    flat = np.full(t * k, -1, np.int32)
    flat[:sum(counts)] = np.repeat(np.arange(len(counts)), counts)
    return assign(torch.from_numpy(rng.permutation(flat).reshape(t, k)).to(dev), len(counts))


PLANS = [([3], 3, 1), ([0, 1, 0], 1, 1), ([1, 1, 1, 1], 2, 2), ([0, 0, 0], 2, 3), ([5, 0, 16, 17, 1, 33], 40, 2),
         ([128, 129, 0, 127, 1], 100, 4), ([300, 2, 260], 200, 3), ([1] * 70, 12, 6)]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts,t,k", PLANS)
def test_product_by_expert(dev, counts, t, k, gather):
    plan, e = make_plan(dev, counts, t, k, seed=t), len(counts)
    for cols, depth, dt in ((192, 256, torch.bfloat16), (70, 300, torch.float32)):
        x = randn(t if gather else t * k, depth, seed=depth, dtype=dt)
        w = quantise_weight(randn(e, cols, depth, seed=cols).to(dev))
        got = product(x.to(dev), w, plan, gather=gather, dtype=dt)
        offsets, tokens = plan.offsets.tolist(), plan.tokens.cpu().long()
        x64, w64 = values(x, 1), weight64(w)
        for i in range(e):
            a, b = offsets[i], offsets[i + 1]
            assert near_product(got[a:b], x64[tokens[a:b]] if gather else x64[a:b], w64[i], dt), i
        assert (got[offsets[-1]:] == 0).all()
        assert torch.equal(product(quantise(x.to(dev)), w, plan, gather=gather, dtype=dt), got)


@pytest.mark.parametrize("rows,cols,depth", [(1, 1, 1), (5, 7, 9), (128, 64, 128), (129, 130, 70), (1000, 300, 200)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_weight_grad(dev, rows, cols, depth, dt):
    d, x = randn(rows, cols, seed=1, dtype=DT[dt], scale=1e-3), randn(rows, depth, seed=2, dtype=DT[dt])
    for out in (torch.float32, torch.bfloat16):
        got = weight_grad(d.to(dev), x.to(dev), dtype=out)
        assert got.shape == (cols, depth) and got.dtype == out
        assert near_product(got, values(d, 0).t(), values(x, 0).t(), out)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts,t,k", PLANS)
def test_weight_grad_by_expert(dev, counts, t, k, gather):
    plan, e, cols, depth = make_plan(dev, counts, t, k, seed=t), len(counts), 70, 136
    d, x = randn(t * k, cols, seed=1), randn(t if gather else t * k, depth, seed=2, dtype=torch.bfloat16)
    got = weight_grad(d.to(dev), x.to(dev), plan, gather=gather)
    offsets, tokens = plan.offsets.tolist(), plan.tokens.cpu().long()
    for i in range(e):
        a, b = offsets[i], offsets[i + 1]
        if a == b:
            assert (got[i] == 0).all()
        else:
            own = x[tokens[a:b]] if gather else x[a:b]
            assert near_product(got[i], values(d[a:b], 0).t(), values(own, 0).t(), torch.float32), i


def test_gradients_of_a_product_against_differences(dev):
    """Small whole numbers and a 448 in each block are 8-bit numbers as they are: products are exact, so
    differences of them are the derivatives."""
    g = torch.Generator().manual_seed(5)
    whole = lambda *s: torch.randint(-8, 9, s, generator=g).float()  # noqa: E731
    rows, cols, depth = 130, 20, 256
    x, wf, d = whole(rows, depth), whole(cols, depth), whole(rows, cols)
    x[:, ::128] = x[::128, :] = 448.0
    wf[0, ::128] = 448.0
    d[:, 0] = d[::128, :] = 448.0
    w = quantise_weight(wf.to(dev))
    assert torch.equal(w.q.float().cpu(), wf) and (w.scale == 1).all()
    f = lambda xx: float((product(xx.to(dev), w, dtype=torch.float32).double().cpu() * d.double()).sum())  # noqa: E731
    dx = product(d.to(dev), transposed(w), dtype=torch.float32).cpu()
    dw = weight_grad(d.to(dev), x.to(dev)).cpu()
    for i, j in ((1, 1), (64, 200), (129, 130), (77, 5)):
        near = x.clone()
        near[i, j] += 1 if x[i, j] < 8 else -1
        assert f(near) - f(x) == float(dx[i, j]) * float(near[i, j] - x[i, j])
    for n, j in ((1, 1), (19, 255), (7, 130)):
        near = wf.clone()
        near[n, j] += 1 if wf[n, j] < 8 else -1
        other = product(x.to(dev), quantise_weight(near.to(dev)), dtype=torch.float32).double().cpu()
        base = product(x.to(dev), w, dtype=torch.float32).double().cpu()
        assert float(((other - base) * d.double()).sum()) == float(dw[n, j]) * float(near[n, j] - wf[n, j])


# ---- combination -----------------------------------------------------------------------
@pytest.mark.parametrize("t,k,width,dt", [(1, 1, 1, "f32"), (1, 6, 2048, "bf16"), (3, 2, 7, "f16"), (40, 8, 513, "bf16"), (130, 5, 1000, "f32"),
                                          (257, 4, 4096, "bf16"), (9, 9, 72, "f16"), (2, 64, 64, "bf16")])
def test_combine_and_its_gradients(dev, t, k, width, dt):
    rng = np.random.default_rng(t * k)
    chosen = rng.integers(0, 2 * k, (t, k)).astype(np.int32)
    chosen[rng.random((t, k)) < 0.2] = -1
    chosen[t // 2] = -1 if t > 1 else chosen[0]                   # a token of no expert
    plan = assign(torch.from_numpy(chosen).to(dev), 2 * k)
    slots, used = plan.slots.cpu().long(), int(plan.offsets[-1])
    rows, d = randn(t * k, width, seed=1, dtype=DT[dt]), randn(t, width, seed=2, dtype=DT[dt])
    rows[used:] = math.nan                                        # nobody's
    weights = randn(t, k, seed=3)
    there = (slots >= 0)[..., None]
    own = torch.where(there, rows.double()[slots.clamp_min(0)], 0.0)
    for w in (weights, None):
        w64 = torch.ones(t, k).double() if w is None else w.double()
        want = (own * w64[..., None]).sum(1)
        size = (own.abs() * w64.abs()[..., None]).sum(1)
        got = combine(rows.to(dev), plan, None if w is None else w.to(dev))
        extra = size * (k + 1) * 2.0 ** -24                       # k roundings of fused additions
        off = (got.double().cpu() - want).abs()
        assert (off <= extra + (want.abs() + extra) * HALF_ULP[DT[dt]] * 1.001 + TINY[DT[dt]]).all()
        d_rows, d_weights = combine_grad(d.to(dev), rows.to(dev), plan, None if w is None else w.to(dev))
        expected = torch.zeros(t * k, width).double()
        expected[slots[slots >= 0]] = (w64[..., None] * d.double()[:, None])[slots >= 0]
        assert rounded_within(d_rows, (expected.float().double() if w is not None else expected), DT[dt], extra=2.0 ** -24 * float(expected.abs().max()))
        assert (d_rows[used:] == 0).all()
        if w is None:
            assert d_weights is None
        else:
            dot, bound = (own * d.double()[:, None]).sum(-1), (own.abs() * d.double().abs()[:, None]).sum(-1)
            assert ((d_weights.double().cpu() - dot).abs() <= bound * (width + 8) * 2.0 ** -24 + 1e-40).all()
    # the formula against differences (the sum is linear in the rows and in the weights)
    h, dw, dr = 0.5, randn(t, k, seed=6).double(), torch.where(torch.arange(t * k)[:, None] < used, randn(t * k, width, seed=7).double(), 0.0)
    f = lambda r, w: float(((torch.where(there, r[slots.clamp_min(0)], 0.0) * w[..., None]).sum(1) * d.double()).sum())  # noqa: E731
    d_rows, d_weights = (v.double().cpu() for v in combine_grad(d.to(dev), rows.to(dev), plan, weights.to(dev)))
    r64, w64 = rows.double(), weights.double()
    numeric = (f(r64, w64 + h * dw) - f(r64, w64 - h * dw)) / (2 * h)
    room = float((own.abs() * d.double().abs()[:, None]).sum(-1).mul(dw.abs()).sum()) * (width + 8) * 2.0 ** -24 + 1e-9
    assert abs(numeric - float((d_weights * dw).sum())) <= room
    numeric = (f(r64 + h * dr, w64) - f(r64 - h * dr, w64)) / (2 * h)
    room = float((d_rows.abs() * dr.abs()).sum()) * HALF_ULP[DT[dt]] * 2.01 + 1e-3 * HALF_ULP[DT[dt]] + 1e-9
    assert abs(numeric - float((d_rows * dr).sum())) <= room


def test_combine_of_strided_rows_into_the_callers(dev):
    plan = make_plan(dev, [3, 4, 2], 5, 2, seed=1)
    wide = randn(10, 300, seed=1, dtype=torch.bfloat16).to(dev)
    for view in (wide[:, 1:200], wide[:, 8:264]):
        want = combine(view.contiguous(), plan)
        room = torch.full((5, 310), 7.0, dtype=torch.bfloat16, device=dev)
        out = room[:, 5:5 + view.shape[1]]
        assert combine(view, plan, out=out) is out and torch.equal(out, want)
        assert (room[:, :5] == 7).all() and (room[:, 5 + view.shape[1]:] == 7).all()
        d = wide[:5].flip(0)[:, 1:1 + view.shape[1]]
        w = randn(5, 2, seed=2).to(dev)
        a, b = combine_grad(d, view, plan, w), combine_grad(d.contiguous(), view.contiguous(), plan, w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- all of them -------------------------------------------------------------------------
def test_the_same_bits_every_time_and_on_another_stream(dev):
    x = randn(500, 64, seed=1).to(dev)
    tokens, w = randn(500, 320, seed=2, dtype=torch.bfloat16).to(dev), quantise_weight(randn(64, 100, 320, seed=3).to(dev))

    def all_of_them():
        weights, chosen = route(x, 4)
        plan = assign(chosen, 64)
        y = product(tokens, w, plan, gather=True)
        out = combine(y, plan, weights)
        d_rows, d_weights = combine_grad(out, y, plan, weights)
        return [weights, chosen, *plan, y, out, d_rows, d_weights, weight_grad(d_rows, tokens, plan, gather=True),
                route_grad(d_weights, x, chosen)]
    first = all_of_them()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = all_of_them()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, all_of_them()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals(dev):
    x, w = randn(4, 256, seed=1).to(dev), quantise_weight(randn(8, 256, seed=2).to(dev))
    plan = make_plan(dev, [2, 2], 4, 1, seed=1)
    logits, chosen = x[:, :16], torch.zeros(4, 2, dtype=torch.int32, device=dev)
    with pytest.raises(TypeError, match="device tensor"):
        route(x.cpu(), 2)
    with pytest.raises(TypeError, match="float16"):
        route(x.double(), 2)
    with pytest.raises(ValueError, match="1..16"):
        route(logits, 17)
    with pytest.raises(ValueError, match="divide"):
        route(logits, 2, groups=3)
    with pytest.raises(ValueError, match="kept"):
        route(logits, 2, groups=4, kept=5)
    with pytest.raises(ValueError, match="score"):
        route(logits, 2, score="tanh")
    with pytest.raises(ValueError, match="bias"):
        route(logits, 2, bias=torch.zeros(15, device=dev))
    with pytest.raises(ValueError, match="one piece"):
        route(x.t(), 2)
    with pytest.raises(ValueError, match="experts"):
        route(torch.zeros(1, 1025, device=dev), 2)
    with pytest.raises(TypeError, match="int32"):
        assign(chosen.long(), 4)
    with pytest.raises(ValueError, match="count"):
        assign(chosen, 1025)
    with pytest.raises(ValueError, match="each choice"):
        route_grad(torch.zeros(4, 3, device=dev), logits, chosen)
    with pytest.raises(ValueError, match="rows of 255"):
        product(x[:, :255], w)
    with pytest.raises(ValueError, match="16 bytes"):
        product(x[:, :255], Blocks(w.q[:, 1:], w.scale))
    with pytest.raises(ValueError, match="block of 128"):
        product(x, Blocks(w.q, w.scale[:, :1]))
    with pytest.raises(TypeError, match="float8"):
        product(x, Blocks(w.q.float(), w.scale))
    with pytest.raises(ValueError, match="3 dimensions"):
        product(x, w, plan)
    with pytest.raises(ValueError, match="gather"):
        product(x, w, gather=True)
    with pytest.raises(ValueError, match="overlap"):
        product(x, w, out=torch.zeros(8, device=dev).expand(4, 8))
    with pytest.raises(TypeError, match="float16, bfloat16"):
        product(x, w, dtype=torch.float64)
    with pytest.raises(TypeError, match="another type"):
        product(x, w, dtype=torch.float16, out=torch.zeros(4, 8, device=dev))
    three = Blocks(w.q[None].expand(3, -1, -1), w.scale[None].expand(3, -1, -1))
    with pytest.raises(ValueError, match="2 experts"):
        product(x, three, plan)
    with pytest.raises(ValueError, match="different numbers"):
        weight_grad(x, x[:3])
    with pytest.raises(ValueError, match="each place"):
        combine_grad(x, x[:3], plan)
    with pytest.raises(ValueError, match="must be"):
        combine(x, plan, out=torch.zeros(4, 255, device=dev))
    with pytest.raises(TypeError, match="int32"):
        combine(x, Assignment(plan.offsets, plan.tokens, plan.slots.long()))


@pytest.mark.parametrize("world,options", [(1, {}), (4, {"score": "sigmoid", "renormalise": True}), (8, {"renormalise": False})])
def test_a_layer_of_experts_over_ranks(dev, world, options):
    """Forward and backward over virtual ranks, through the collectives, against the plain layer."""
    from mintccl_amd import experts
    for name, off in experts.distances(world, dev, **options).items():
        assert off < experts.FAR, (name, off)


def test_offsets_beyond_32_bits(dev):
    """Results and inputs of more than 2^31 elements (more than 4 GiB): the last rows are what they are alone."""
    rows, cols = 600_001, 4096
    x = randn(rows, 130, seed=1, dtype=torch.bfloat16).to(dev)
    w = quantise_weight(randn(cols, 130, seed=2).to(dev))
    y = product(x, w)
    for at in (slice(0, 64), slice(rows // 2, rows // 2 + 64), slice(rows - 64, rows)):
        assert torch.equal(y[at], product(x[at], w))
    q, s = quantise(y)                                   # its input lies beyond 4 GiB
    want = quantise(y[-3:].clone())
    assert torch.equal(q[-3:].view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(s[-3:], want.scale)
    del q, s
    slots = torch.tensor([[rows - 1, 0], [rows // 2, rows - 2]], dtype=torch.int32, device=dev)
    plan = Assignment(torch.tensor([rows], dtype=torch.int32, device=dev), slots.view(-1), slots)
    got = combine(y, plan)
    assert torch.equal(got, (y[slots[:, 0].long()].float() + y[slots[:, 1].long()].float()).bfloat16())
    torch.cuda.empty_cache()


def test_in_a_graph(dev):
    """Captured once and replayed with other inputs, eager work between the replays."""
    logits, tokens = randn(300, 32, seed=1).to(dev), randn(300, 256, seed=2, dtype=torch.bfloat16).to(dev)
    w = quantise_weight(randn(32, 128, 256, seed=3).to(dev))

    def layer():
        weights, chosen = route(logits, 4)
        plan = assign(chosen, 32)
        y = product(tokens, w, plan, gather=True)
        out = combine(y, plan, weights)
        d_rows, d_weights = combine_grad(out, y, plan, weights)
        return [weights, chosen, *plan, y, out, d_rows, weight_grad(d_rows, tokens, plan, gather=True), route_grad(d_weights, logits, chosen)]
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer()
    for i in range(4):
        logits.copy_(randn(300, 32, seed=10 + i))
        tokens.copy_(randn(300, 256, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, layer()):
            assert torch.equal(a, b), i
