"""Products in 8 bits against their definition in 64 bits where sums, rows and kernels can go wrong."""
import pytest
import torch

from mintccl_amd.block8 import product, quantise, quantise_weight, weight_grad
from mintccl_amd.routing import Assignment, assign
from tests.expert_oracle import off_by, randn, rounded8, unlike, weight64

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- sums ------------------------------------------------------------------------
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols,depth", [(1, 70, 384), (5, 300, 256), (20, 130, 384), (50, 200, 384), (100, 1000, 128), (64, 96, 256), (700, 1999, 384)])
def test_sums_of_products_that_are_unlike(dev, rows, cols, depth, dt):
    """Large products that cancel among small ones: the sums are whole numbers that results in 16-bit floats and in 32 bits have exactly."""
    x, weights = unlike(rows, depth)
    x, wf = x.to(dev), weights(cols).to(dev)
    w = quantise_weight(wf)
    assert torch.equal(w.q.float(), wf) and (w.scale == 1).all()
    want = x.double() @ wf.double().t()
    assert torch.equal(want.half().double(), want)
    for given in (x, x.to(DT[dt]), quantise(x)):
        got = product(given, w, dtype=DT[dt])
        if dt == "bf16":
            assert off_by(got, x.double(), wf.double()) <= 0
        else:
            assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dt", list(DT))
def test_sums_of_weights_gradients_that_are_unlike(dev, dt):
    for rows, cols, depth in ((128, 40, 70), (384, 130, 300), (256, 700, 1100)):
        x, weights = unlike(depth, rows)
        x, d = x.t().contiguous().to(dev), weights(cols).t().contiguous().to(dev)
        want = d.double().t() @ x.double()
        got = weight_grad(d, x, dtype=DT[dt])
        if dt == "bf16":
            assert off_by(got, d.double().t(), x.double().t()) <= 0
        else:
            assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,cols,depth", [(3, 200, 1000), (40, 130, 1000), (200, 300, 2048), (1000, 2000, 512)])
def test_sums_with_large_channels(dev, rows, cols, depth, dt):
    """One channel in eight 60 times larger than the others, as layers' outputs have them."""
    x = randn(rows, depth, seed=rows, dev=dev)
    x[:, ::8] *= 60
    x = x.to(DT[dt])
    w = quantise_weight(randn(cols, depth, seed=cols, dev=dev))
    assert off_by(product(x, w, dtype=DT[dt]), rounded8(x, 1), weight64(w)) <= 0
    assert off_by(product(x, w, dtype=torch.float32), rounded8(x, 1), weight64(w)) <= 0
    d = randn(rows, 90, seed=3, dev=dev)
    d[::8] *= 60
    got = weight_grad(d, x, dtype=DT[dt])
    assert off_by(got, rounded8(d, 0).t(), rounded8(x, 0).t()) <= 0


def test_sums_by_expert_that_are_unlike(dev):
    x, weights = unlike(300, 256)
    wf = torch.stack([weights(130), -weights(130), weights(130).flip(0)]).to(dev)
    counts = torch.tensor([0] * 200 + [1] * 3 + [2] * 90 + [-1] * 7, dtype=torch.int32)
    plan = assign(counts[torch.randperm(300, generator=torch.Generator().manual_seed(1))][:, None].contiguous().to(dev), 3)
    x = x.to(dev)
    got = product(x, quantise_weight(wf), plan, gather=True, dtype=torch.float16)
    at = plan.offsets.tolist()
    for e in range(3):
        rows = x[plan.tokens[at[e]:at[e + 1]].long()]
        assert torch.equal(got[at[e]:at[e + 1]].double(), rows.double() @ wf[e].double().t())


# ---- rows -------------------------------------------------------------------------
def planned(dev, counts, tokens, k, seed):
    """An assignment with `counts` places for its experts, the rest of tokens * k pairs without."""
    flat = torch.full((tokens * k,), -1, dtype=torch.int32)
    flat[:sum(counts)] = torch.repeat_interleave(torch.arange(len(counts), dtype=torch.int32), torch.tensor(counts))
    return assign(flat[torch.randperm(tokens * k, generator=torch.Generator().manual_seed(seed))].view(tokens, k).to(dev), len(counts))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("counts,tokens,k,cols,depth", [
    ([3, 0, 5], 8, 1, 70, 300), ([20, 30, 22], 40, 2, 130, 256), ([200, 1, 99, 300], 300, 2, 200, 384), ([1500, 0, 600], 1100, 2, 2000, 200),
    ([2100, 1900], 2000, 2, 3700, 130)])
def test_gathered_rows_that_are_not_there_are_zeros(dev, counts, tokens, k, cols, depth, dt):
    """Token numbers outside x among an expert's rows: forward, and as the weights' gradient has them."""
    plan, e = planned(dev, counts, tokens, k, seed=tokens), len(counts)
    x = randn(tokens, depth, seed=1, dtype=DT[dt], dev=dev)
    x[-1] = float("nan")                                     # (nothing of a row that stands in for another)
    w = quantise_weight(randn(e, cols, depth, seed=2, dev=dev))
    lost = torch.randperm(sum(counts), generator=torch.Generator().manual_seed(3))[:1 + sum(counts) // 7].to(dev)
    named = plan.tokens.clone()
    named[lost] = torch.tensor([-1, tokens, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)[torch.arange(len(lost), device=dev) % 4]
    missing = torch.zeros(tokens * k, dtype=torch.bool, device=dev)
    missing[lost] = True
    broken = Assignment(plan.offsets, named, plan.slots)
    for given in (x, quantise(x)):
        want = torch.where(missing[:, None], 0, product(given, w, plan, gather=True, dtype=DT[dt]))
        got = product(given, w, broken, gather=True, dtype=DT[dt])
        assert torch.equal(got[missing], want[missing])
        there = ~missing & (plan.tokens != tokens - 1)
        assert torch.equal(got[there], want[there]) and torch.isfinite(got[there]).all()
    x[-1] = 1.0
    d = randn(tokens * k, 90, seed=4, dtype=DT[dt], dev=dev)
    at = plan.offsets.tolist()
    got = weight_grad(d, x, broken, gather=True, dtype=DT[dt])
    for i in range(e):
        own = torch.where(missing[at[i]:at[i + 1], None], 0, x[plan.tokens[at[i]:at[i + 1]].long()])
        assert off_by(got[i], rounded8(d[at[i]:at[i + 1]], 0).t(), rounded8(own, 0).t()) <= 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("offsets,rows,cols,depth", [
    ([2, 2, 5], 6, 70, 300), ([1, 9, 9, 17], 40, 130, 256), ([17, 17, 30, 60], 64, 40, 200), ([70, 100, 300], 300, 200, 384),
    ([300, 900, 900, 1500], 2100, 2000, 200), ([600, 600], 600, 100, 128), ([5] * 71, 80, 64, 100), ([513, 2500, 3600], 4000, 3700, 130)])
def test_rows_that_are_no_experts_are_zeros(dev, offsets, rows, cols, depth, dt):
    """Rows before the first expert's too, whatever the result's memory held."""
    at, e = torch.tensor(offsets, dtype=torch.int32, device=dev), len(offsets) - 1
    x, w = randn(rows, depth, seed=1, dtype=DT[dt], dev=dev), quantise_weight(randn(e, cols, depth, seed=2, dev=dev))
    tokens = torch.arange(rows, dtype=torch.int32, device=dev)
    plan = Assignment(at, tokens, tokens[:, None])
    for given in (x, quantise(x)):
        got = product(given, w, plan, out=torch.full((rows, cols), float("nan"), dtype=DT[dt], device=dev))
        assert (got[:offsets[0]] == 0).all() and (got[offsets[-1]:] == 0).all()
        for i in range(e):
            own = slice(offsets[i], offsets[i + 1])
            assert off_by(got[own], rounded8(x[own], 1), weight64(type(w)(w.q[i], w.scale[i]))) <= 0


def test_an_assignment_of_more_tokens_than_rows_is_refused(dev):
    plan = planned(dev, [4, 3], 6, 2, seed=1)
    x, w, d = randn(5, 128, seed=1, dev=dev), quantise_weight(randn(2, 64, 128, seed=2, dev=dev)), randn(12, 64, seed=3, dev=dev)
    for call in (lambda: product(x, w, plan, gather=True), lambda: product(quantise(x), w, plan, gather=True),
                 lambda: weight_grad(d, x, plan, gather=True)):
        with pytest.raises(ValueError, match="x has 5 rows, the assignment 6 tokens"):
            call()
    more = randn(9, 128, seed=1, dev=dev)                       # (rows behind the tokens' are nobody's)
    assert torch.equal(product(more, w, plan, gather=True), product(more[:6], w, plan, gather=True))
    for call in (lambda: product(x, w, gather=True), lambda: weight_grad(d, d, gather=True)):
        with pytest.raises(ValueError, match="gather needs"):
            call()


# ---- kernels ------------------------------------------------------------------------
def ran(call):
    """What `call` returns, and the names of the kernels that it launched, without blanks."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        got = call()
        torch.cuda.synchronize()
    return got, [e.name.replace(" ", "").replace("mint::(anonymousnamespace)::", "").removeprefix("void") for e in prof.events() if "_kernel<" in e.name]


CODE = {"f16": 0, "bf16": 1, "f32": 2, "bytes": 3}
#: Tiles by their template arguments: rows, columns, wavefronts down, blocks of the depth in LDS, sets of wavefronts.  For each the
#: results that take it, and (rows, columns) and depths with which it is chosen: fewer blocks of the depth than are under way, as
#: many, more, and a last one that is not whole.
DENSE = [
    ("64,64,4,2,1", ("bf16", "f16", "f32"), (100, 300), (1, 100, 128, 130, 256, 300, 1000)),
    ("64,64,4,4,2", ("bf16",), (130, 900), (1100, 1152, 1280, 2500)),
    ("64,64,4,2,2", ("f16", "f32"), (130, 900), (1100, 1152, 2400)),
    ("64,64,4,2,2", ("bf16",), (1000, 2000), (1100, 1152)),
    ("128,128,4,3,1", ("bf16",), (1500, 2000), (1, 100, 128, 130, 256, 384, 400, 512, 1000)),
    ("128,128,4,2,1", ("bf16",), (38401, 128), (100, 128, 130, 256, 300, 640)),
    ("128,256,2,3,1", ("bf16", "f16", "f32"), (2000, 4000), (1, 100, 128, 130, 256, 384, 400, 512, 1000)),
    ("256,256,2,2,1", ("bf16",), (4000, 4000), (1, 100, 128, 130, 256, 300, 384, 1000)),
]


def for_each_type(cases):
    return [(tile, dt, *rest) for tile, types, *rest in cases for dt in types]


def kernel(tile, dt, along=False, joined=False):
    return f"product_kernel<{CODE[dt]},{tile},{str(along).lower()},{str(along).lower()},{str(joined).lower()}>"


@pytest.mark.parametrize("tile,dt,shape,depths", for_each_type(DENSE))
def test_every_tile(dev, tile, dt, shape, depths):
    rows, cols = shape
    for depth in depths:
        x, w = randn(rows, depth, seed=depth, dtype=DT[dt], dev=dev), quantise_weight(randn(cols, depth, seed=1, dev=dev))
        got, names = ran(lambda: product(x, w, dtype=DT[dt]))
        assert any(n.startswith(kernel(tile, dt)) for n in names), names
        assert off_by(got, rounded8(x, 1), weight64(w)) <= 0, depth


@pytest.mark.parametrize("dt,tile,depths", [("bf16", "64,64,4,4,2", (4096, 4100, 9001)), ("f16", "64,64,4,2,2", (2560, 2600, 9001)),
                                            ("f32", "64,64,4,2,2", (2560, 2600, 9001))])
def test_every_shared_tile(dev, dt, tile, depths):
    for (rows, cols), depth in zip(((50, 300), (33, 64), (128, 4000)), depths):
        x, w = randn(rows, depth, seed=depth, dtype=DT[dt], dev=dev), quantise_weight(randn(cols, depth, seed=1, dev=dev))
        got, names = ran(lambda: product(quantise(x), w, dtype=DT[dt]))
        assert any(n.startswith(kernel(tile, dt, joined=True)) for n in names), names
        assert off_by(got, rounded8(x, 1), weight64(w)) <= 0, depth


THIN = [((5, 300), "given", "1,8"), ((16, 50), "given", "1,8"), ((3, 12400), "given", "1,2"), ((5, 300), "bytes", "1,8"), ((3, 12400), "bytes", "1,2"),
        ((20, 300), "bytes", "2,8"), ((32, 12400), "bytes", "2,2")]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("shape,given,variant", THIN)
def test_every_kernel_of_few_rows(dev, shape, given, variant, dt):
    rows, cols = shape
    for depth in (1, 100, 128, 130, 1000, 1024) + ((4100, 6500) if cols < 1000 and rows < 6 else ()):
        x, w = randn(rows, depth, seed=depth, dtype=DT[dt], dev=dev), quantise_weight(randn(cols, depth, seed=1, dev=dev))
        operand = quantise(x) if given == "bytes" else x
        got, names = ran(lambda: product(operand, w, dtype=DT[dt]))
        assert any(n.startswith(f"thin_kernel<{CODE[dt]},{CODE[dt if given == 'given' else 'bytes']},{variant}>") for n in names), names
        assert off_by(got, rounded8(x, 1), weight64(w)) <= 0, depth


BY_EXPERT = [
    ("64,64,4,2,1", ("bf16", "f32"), [60, 0, 71], 900, (1, 128, 300, 1000)),
    ("64,64,4,4,2", ("bf16",), [60, 70], 900, (1100, 1152)),
    ("64,64,4,2,2", ("f16", "f32"), [60, 70], 900, (1100, 1152)),
    ("64,64,4,2,2", ("bf16",), [900, 100], 1850, (1100,)),
    ("128,128,4,3,1", ("bf16",), [1400, 100], 2000, (1, 100, 256, 384, 400, 1000)),
    ("128,128,4,2,1", ("bf16",), [10000, 9000], 384, (100, 130, 384)),
    ("128,256,2,3,1", ("bf16", "f16", "f32"), [1200, 800], 3700, (1, 100, 256, 384, 400, 1000)),
    ("256,256,2,2,1", ("bf16",), [3000, 0, 1000], 3700, (1, 100, 256, 300, 1000)),
]


@pytest.mark.parametrize("tile,dt,counts,cols,depths", for_each_type(BY_EXPERT))
def test_every_tile_by_expert(dev, tile, dt, counts, cols, depths):
    tokens, e = (sum(counts) + 1) // 2, len(counts)
    plan = planned(dev, counts, tokens, 2, seed=tokens)
    at = plan.offsets.tolist()
    for depth in depths:
        x, w = randn(tokens, depth, seed=depth, dtype=DT[dt], dev=dev), quantise_weight(randn(e, cols, depth, seed=1, dev=dev))
        got, names = ran(lambda: product(x, w, plan, gather=True, dtype=DT[dt]))
        assert any(n.startswith(kernel(tile, dt)) for n in names), names
        for i in range(e):
            rows = slice(at[i], at[i + 1])
            assert off_by(got[rows], rounded8(x[plan.tokens[rows].long()], 1), weight64(type(w)(w.q[i], w.scale[i]))) <= 0, (depth, i)
        assert (got[at[-1]:] == 0).all()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("counts,given,variant", [([3, 0, 20, 1], "given", "1,8"), ([3, 0, 70, 1], "bytes", "2,8"), ([1] * 40 + [30, 0], "given", "1,2"),
                                                  ([20] * 40, "bytes", "2,2")])
def test_every_kernel_of_few_rows_by_expert(dev, counts, given, variant, dt):
    e, cols = len(counts), 70 if len(counts) < 10 else 500
    tokens = sum(counts)
    plan = planned(dev, counts, tokens, 1, seed=tokens)
    at = plan.offsets.tolist()
    for depth in (1, 128, 300, 1000):
        x, w = randn(tokens, depth, seed=depth, dtype=DT[dt], dev=dev), quantise_weight(randn(e, cols, depth, seed=1, dev=dev))
        operand = quantise(x) if given == "bytes" else x
        got, names = ran(lambda: product(operand, w, plan, gather=True, dtype=DT[dt]))
        assert any(n.startswith(f"thin_kernel<{CODE[dt]},{CODE[dt if given == 'given' else 'bytes']},{variant}>") for n in names), names
        for i in range(e):
            rows = slice(at[i], at[i + 1])
            assert off_by(got[rows], rounded8(x[plan.tokens[rows].long()], 1), weight64(type(w)(w.q[i], w.scale[i]))) <= 0, (depth, i)


GRADIENTS = [
    ("64,64,4,2,1", ("bf16", "f16", "f32"), (100, 300), (1, 128, 130, 300, 1000)),
    ("64,64,4,4,2", ("bf16",), (130, 900), (1100, 2500)),
    ("64,64,4,2,2", ("f16", "f32"), (130, 900), (1100, 2500)),
    ("64,64,4,2,2", ("bf16",), (1000, 2000), (1100,)),
    ("128,128,4,3,1", ("bf16",), (1500, 2000), (1, 130, 300, 512, 1000)),
    ("128,128,4,2,1", ("bf16",), (38401, 128), (100, 300, 512)),
    ("128,256,2,3,1", ("bf16", "f16", "f32"), (2000, 4000), (1, 130, 300, 512, 1000)),
    ("256,256,2,2,1", ("bf16",), (4000, 4000), (1, 130, 300, 512, 1000)),
]


@pytest.mark.parametrize("tile,dt,shape,rows", for_each_type(GRADIENTS))
def test_every_tile_of_a_gradient(dev, tile, dt, shape, rows):
    cols, depth = shape
    for n in rows:
        d, x = randn(n, cols, seed=n, dtype=DT[dt], dev=dev), randn(n, depth, seed=1, dtype=DT[dt], dev=dev)
        got, names = ran(lambda: weight_grad(d, x, dtype=DT[dt]))
        assert any(n_.startswith(kernel(tile, dt, along=True)) for n_ in names), names
        assert off_by(got, rounded8(d, 0).t(), rounded8(x, 0).t()) <= 0, n


GRADIENTS_BY_EXPERT = [
    ("64,64,4,2,1", ("bf16", "f32"), [300, 0, 129], (100, 200)),
    ("64,64,4,4,2", ("bf16",), [2000, 700], (100, 200)),
    ("64,64,4,2,2", ("f16", "f32"), [2000, 700], (100, 200)),
    ("128,128,4,3,1", ("bf16",), [300, 129], (700, 2000)),
    ("128,128,4,2,1", ("bf16",), [300, 129], (19200, 128)),
    ("128,256,2,3,1", ("bf16", "f16", "f32"), [300, 129], (1300, 2000)),
    ("256,256,2,2,1", ("bf16",), [700, 0, 129], (2000, 2500)),
]


@pytest.mark.parametrize("tile,dt,counts,shape", for_each_type(GRADIENTS_BY_EXPERT))
def test_every_tile_of_a_gradient_by_expert(dev, tile, dt, counts, shape):
    (cols, depth), e, tokens = shape, len(counts), sum(counts) // 2 + 5
    plan = planned(dev, counts, tokens, 2, seed=tokens)
    at = plan.offsets.tolist()
    d, x = randn(tokens * 2, cols, seed=2, dtype=DT[dt], dev=dev), randn(tokens, depth, seed=1, dtype=DT[dt], dev=dev)
    got, names = ran(lambda: weight_grad(d, x, plan, gather=True, dtype=DT[dt]))
    assert any(n.startswith(kernel(tile, dt, along=True)) for n in names), names
    for i in range(e):
        rows = slice(at[i], at[i + 1])
        if at[i] == at[i + 1]:
            assert (got[i] == 0).all()
        else:
            assert off_by(got[i], rounded8(d[rows], 0).t(), rounded8(x[plan.tokens[rows].long()], 0).t()) <= 0, i
