"""The loss that balances experts, its counts and its gradient against the definition in 64 bits."""
import pytest
import torch

from mintccl_amd.routing import Balance, balance, balance_grad, route, route_grad
from tests.block_oracle import DT, UNIT, balance64, close
from tests.expert_oracle import HALF_ULP, randn

pytestmark = pytest.mark.gpu

#: A share: an exponential (of a difference that is rounded: |x| < 16 makes 16 more), a sum over at most 1024 experts (16 numbers of a lane, six
#: steps) and a quotient; then a sum over tokens, of which a wavefront has at most 64 of a tile, and tiles.
SHARE = 64 * UNIT


def tokens_units(t):
    return SHARE + (64 + 4 + t / 256 / 8 + 16) * UNIT


CASES = [  # tokens, experts, k, score, lengths of sequences, z, dtype
    (1, 1, 1, "softmax", None, 0.0, "f32"), (1, 128, 8, "sigmoid", None, 1e-3, "f32"), (8, 64, 6, "softmax", None, 0.0, "bf16"),
    (17, 5, 2, "softmax", [3, 0, 9, 5], 0.5, "f32"), (300, 64, 6, "sigmoid", [100, 100, 90], 1e-3, "bf16"), (300, 65, 4, "softmax", None, 1e-2, "f16"),
    (1000, 130, 8, "softmax", [1, 1, 500, 0, 0, 400], 0.0, "f16"), (4099, 256, 8, "sigmoid", None, 0.0, "f32"), (2500, 512, 3, "softmax", [2500], 0.0, "bf16"),
    (700, 1024, 16, "sigmoid", [350, 350], 1e-3, "f32"), (70, 300, 40, "softmax", [1] * 70, 1e-3, "f32"), (20000, 8, 2, "softmax", [7] * 2000, 0.1, "f32"),
]


def inputs(t, e, k, dt, dev, masks=True, seed=1):
    x = randn(t, e, seed=seed) * 2
    if masks and t > 4:
        x[t // 3] = -float("inf")                            # a token with no expert left
        x[:, e // 2] = torch.where(torch.arange(t) % 3 == 0, -float("inf"), x[:, e // 2]) if e > 1 else x[:, e // 2]
        x[t // 2, 1:] = -float("inf")                        # ... with one
    x = x.to(DT[dt])
    chosen = x.float().sort(dim=-1, descending=True, stable=True)
    experts = torch.where(chosen.values[:, :k] == -float("inf"), -1, chosen.indices[:, :k]).to(torch.int32).contiguous()
    return x.to(dev), experts.to(dev)


def offsets_of(lengths, dev, start=0):
    return None if lengths is None else torch.tensor([start + sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=dev)


#: each number of experts of a lane in each type, alone and in tiles
CASES += [(t, e, 4, ("softmax", "sigmoid")[i % 2], None, 1e-3, dt) for i, e in enumerate((60, 100, 250, 500, 1000)) for t in (50, 90) for dt in ("f32", "bf16", "f16")]


@pytest.mark.parametrize("t,e,k,score,lengths,z,dt", CASES)
def test_balance_and_its_gradient(dev, t, e, k, score, lengths, z, dt):
    x, experts = inputs(t, e, k, dt, dev)
    offsets = offsets_of(lengths, dev, 2 if lengths and sum(lengths) + 2 < t else 0)
    got = balance(x, experts, score=score, offsets=offsets, z=z)
    leaf = x.cpu().double().requires_grad_()
    loss, counts, shares, there = balance64(leaf, experts.cpu(), score, None if offsets is None else offsets.cpu(), z)
    assert torch.equal(got.counts.cpu(), counts) and torch.equal(got.there.cpu(), there)
    units = tokens_units(t)
    close(got.shares, shares, shares, torch.float32, units)
    # (terms are not negative; the sums over experts and sequences: six steps each, and a lane's own)
    close(got.loss, loss.detach(), loss.detach().abs() + 1e-30, torch.float32, 2 * units + (64 + 16 + len(lengths or []) / 64) * UNIT)
    d = torch.tensor(0.75, device=dev)
    grad = balance_grad(d, x, experts, got, score=score, offsets=offsets, z=z)
    want = torch.autograd.grad(loss * 0.75, leaf)[0].masked_fill(torch.isneginf(leaf), 0)
    # the magnitude: a token's p (a + <p, a>), and z's
    ends = [0, t] if offsets is None else offsets.tolist()
    size = torch.zeros(t, e, dtype=torch.float64)
    some, every = max(int((there > 0).sum()), 1), max(int(there.sum()), 1)
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        v = leaf.detach()[a:b]
        p = torch.softmax(v, 1).nan_to_num(0) if score == "softmax" else torch.sigmoid(v) / torch.sigmoid(v).sum(1, keepdim=True).clamp_min(1e-300)
        n = max(int(there[i]), 1)
        load = 0.75 * e * counts[i].double() / (k * n) / (some * n)
        size[a:b] = p * (load + (p * load).sum(1, keepdim=True))
        size[a:b] += 2 * z * 0.75 / every * (torch.logsumexp(v, 1, keepdim=True).abs() + 16).nan_to_num(0, 0, 0) * torch.softmax(v, 1).nan_to_num(0)
    close(grad, want, size, DT[dt], 4 * SHARE)
    # added to another gradient, and rounded once; also into its place
    more = randn(t, e, seed=9, dtype=DT[dt], dev=dev)
    close(balance_grad(d, x, experts, got, score=score, offsets=offsets, z=z, add=more), want + more.cpu().double(), size + more.cpu().double().abs(), DT[dt], 4 * SHARE)


def test_even_and_one_sided(dev):
    """1 where all is even; as many as there are experts where one has everything."""
    e, t = 16, 64
    x = torch.zeros(t, e, device=dev)
    even = (torch.arange(t * 2, dtype=torch.int32, device=dev) % e).view(t, 2)
    assert abs(float(balance(x, even).loss) - 1) < 1e-6
    x[:, 3] = 60.0
    assert abs(float(balance(x, torch.full((t, 1), 3, dtype=torch.int32, device=dev)).loss) - e) < 1e-5


def test_tokens_outside_the_sequences(dev):
    x, experts = inputs(50, 12, 2, "f32", dev, masks=False)
    alone = balance(x[10:40].contiguous(), experts[10:40].contiguous())
    offsets = torch.tensor([10, 40], dtype=torch.int32, device=dev)
    x[:10] = float("nan")
    found = balance(x, experts, offsets=offsets)
    assert torch.equal(found.counts, alone.counts) and torch.allclose(found.loss, alone.loss) and torch.allclose(found.shares, alone.shares)
    one = torch.ones((), device=dev)
    grad = balance_grad(one, x, experts, found, offsets=offsets)
    assert bool((grad[:10] == 0).all()) and bool((grad[40:] == 0).all()) and bool((grad[10:40] != 0).any())
    more = randn(50, 12, seed=4, dev=dev)
    added = balance_grad(one, x, experts, found, offsets=offsets, add=more)
    assert torch.equal(added[:10], more[:10]) and torch.equal(added[40:], more[40:])
    nowhere = balance(x, experts, offsets=torch.tensor([50, 50, 50], dtype=torch.int32, device=dev))
    assert float(nowhere.loss) == 0 and int(nowhere.counts.sum()) == 0 and int(nowhere.there.sum()) == 0


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_as_many_sequences_as_there_may_be(dev, score):
    """65535 sequences of one token, of none and of two, tokens before them and behind them: each has a term of its own."""
    t, e, s, before = 66000, 20, 65535, 311
    x, _ = inputs(t, e, 1, "f32", dev, masks=False)
    experts = torch.randint(0, e, (t, 1), generator=torch.Generator().manual_seed(3)).int().to(dev)
    lengths = torch.ones(s, dtype=torch.int64)
    lengths[5::64], lengths[6::64] = 0, 2
    ends = before + torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)])
    got = balance(x, experts, score=score, offsets=ends.int().to(dev), z=0.0)
    leaf = x.cpu().double().requires_grad_()
    p = torch.softmax(leaf, 1) if score == "softmax" else torch.sigmoid(leaf) / torch.sigmoid(leaf).sum(1, keepdim=True)
    of = torch.repeat_interleave(torch.arange(s), lengths)
    inside = slice(before, before + len(of))
    n = lengths.clamp_min(1).double()[:, None]
    shares = torch.zeros(s, e, dtype=torch.float64).index_add(0, of, p[inside]) / n
    counts = torch.zeros(s, e, dtype=torch.float64).index_add(0, of, torch.nn.functional.one_hot(experts.cpu()[inside, 0].long(), e).double())
    loss = (counts * e / n * shares).sum() / (lengths > 0).sum()
    assert torch.equal(got.counts.cpu().double(), counts) and torch.equal(got.there.cpu().long(), lengths)
    close(got.shares, shares.detach(), shares.detach(), torch.float32, SHARE + 4 * UNIT)
    # (a sequence's terms in two blocks of 16 experts, 64 sequences to a thread, lanes and wavefronts)
    close(got.loss, loss.detach(), loss.detach(), torch.float32, SHARE + (4 + 8 + 64 + 6 + 16) * UNIT)
    grad = balance_grad(torch.tensor(1e4, device=dev), x, experts, got, score=score, offsets=ends.int().to(dev))
    want = torch.autograd.grad(loss * 1e4, leaf)[0]
    load = torch.zeros(t, e, dtype=torch.float64)
    load[inside] = (counts * e / n / n / (lengths > 0).sum() * 1e4)[of]
    size = p.detach() * (load + (p.detach() * load).sum(1, keepdim=True))
    close(grad, want, size, torch.float32, 4 * SHARE)
    assert not grad[:before].any() and not grad[before + len(of):].any()


def test_offsets_that_say_anything(dev):
    """Offsets that descend, are negative or beyond the tokens: nothing outside is read or written, whatever comes out."""
    x, experts = inputs(100, 9, 2, "f32", dev, masks=False)
    for list_ in ([90, 10, 60], [-5, 20, 2000], [0, 100, 0, 100, 0, 100], [2 ** 31 - 1, -2 ** 31, 7]):
        offsets = torch.tensor(list_, dtype=torch.int32, device=dev)
        found = balance(x, experts, offsets=offsets)
        grad = balance_grad(torch.ones((), device=dev), x, experts, found, offsets=offsets)
        torch.cuda.synchronize()
        assert grad.shape == x.shape and bool((found.counts >= 0).all())


def test_special_logits(dev):
    x, experts = inputs(6, 8, 2, "f32", dev, masks=False)
    x[1] = -float("inf")
    x[2, 3:] = torch.finfo(torch.float32).min
    x[3, 0] = 3e4
    for score in ("softmax", "sigmoid"):
        found = balance(x, experts, score=score, z=1e-6)
        grad = balance_grad(torch.ones((), device=dev), x, experts, found, score=score, z=1e-6)
        assert int(found.there) == 5 and bool(found.loss.isfinite()) and bool(found.shares.isfinite().all()) and bool(grad.isfinite().all())
        assert bool((grad[1] == 0).all())
    everything = torch.full((3, 4), -float("inf"), device=dev)
    none = torch.full((3, 2), -1, dtype=torch.int32, device=dev)
    found = balance(everything, none, z=1.0)
    assert float(found.loss) == 0 and int(found.there) == 0
    assert bool((balance_grad(torch.ones((), device=dev), everything, none, found, z=1.0) == 0).all())
    x[4, 2] = float("nan")
    assert bool(balance(x, experts).loss.isnan())
    # experts that do not exist, and one named twice
    odd = torch.tensor([[0, 0], [8, -1], [100, 3], [-7, 2 ** 31 - 1], [1, 1], [2, 3]], dtype=torch.int32, device=dev)
    assert balance(torch.zeros(6, 8, device=dev), odd).counts.tolist() == [[2, 2, 1, 2, 0, 0, 0, 0]]


def test_no_tokens(dev):
    x, experts = torch.zeros(0, 7, device=dev), torch.zeros(0, 2, dtype=torch.int32, device=dev)
    for offsets in (None, torch.zeros(4, dtype=torch.int32, device=dev)):
        found = balance(x, experts, offsets=offsets, z=1.0)
        assert float(found.loss) == 0 and bool((found.counts == 0).all()) and bool((found.shares == 0).all())
        assert balance_grad(torch.ones((), device=dev), x, experts, found, offsets=offsets).shape == (0, 7)


def test_logits_any_distance_apart_and_gradients_against_differences(dev):
    t, e = 40, 12
    room = torch.full((t, e + 5), float("nan"), device=dev)
    x, experts = inputs(t, e, 3, "f32", dev)
    room[:, 2:2 + e] = x
    offsets = offsets_of([15, 25], dev)
    step = 2.0 ** -7
    for score in ("softmax", "sigmoid"):
        options = {"score": score, "offsets": offsets, "z": 0.25}
        a, b = balance(x, experts, **options), balance(room[:, 2:2 + e], experts, **options)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        one = torch.ones((), device=dev)
        grad = balance_grad(one, x, experts, a, **options)
        assert torch.equal(grad, balance_grad(one, room[:, 2:2 + e], experts, b, **options))
        way = torch.sign(randn(t, e, seed=5, dev=dev))
        want = (float(balance(x + step * way, experts, **options).loss) - float(balance(x - step * way, experts, **options).loss)) / (2 * step)
        got = float((grad.double() * way.double()).sum())
        # the loss is rounded to 2^-24 of about 4, over 2 steps: 3e-5; its third derivative's part: step^2 of the gradient's size
        assert abs(got - want) <= 1e-4 + 4 * step ** 2 * float(grad.double().abs().sum()), (score, got, want)


def test_counts_of_all_ranks(dev):
    """Two ranks' counts and tokens summed: each one's gradient is its part of that of the tokens together."""
    x, experts = inputs(90, 16, 2, "f32", dev)
    whole = balance(x, experts)
    one = torch.ones((), device=dev)
    want = balance_grad(one, x, experts, whole)
    halves = [(x[:50].contiguous(), experts[:50].contiguous()), (x[50:].contiguous(), experts[50:].contiguous())]
    found = [balance(*h) for h in halves]
    both = Balance(whole.loss, found[0].counts + found[1].counts, whole.shares, found[0].there + found[1].there)
    assert torch.equal(both.counts, whole.counts) and torch.equal(both.there, whole.there)
    assert torch.equal(torch.cat([balance_grad(one, *h, both) for h in halves]), want)


def test_with_the_router(dev):
    x = randn(500, 64, seed=3, dtype=torch.bfloat16, dev=dev)
    weights, experts = route(x, 6, score="sigmoid")
    found = balance(x, experts, score="sigmoid")
    assert int(found.counts.sum()) == 500 * 6
    by_route = route_grad(torch.ones_like(weights), x, experts, score="sigmoid", renormalise=False)
    one = torch.ones((), device=dev)
    alone = balance_grad(one, x, experts, found, score="sigmoid")
    both = balance_grad(one, x, experts, found, score="sigmoid", add=by_route)
    want = by_route.double() + alone.double()
    # (the part alone is rounded too)
    assert bool(((both.double() - want).abs() <= HALF_ULP[torch.bfloat16] * (want.abs() + alone.double().abs()) * 1.01 + 1e-30).all())


def test_the_same_bits_every_time_and_on_another_stream(dev):
    side = torch.cuda.Stream()
    x, experts = inputs(5000, 100, 4, "bf16", dev)
    offsets = offsets_of([1200, 1300, 2400], dev)
    def both():
        f = balance(x, experts, offsets=offsets, z=1e-3)
        return [*f, balance_grad(f.loss, x, experts, f, offsets=offsets, z=1e-3)]
    first = both()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        again = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again)) and all(torch.equal(a, b) for a, b in zip(first, both()))


def test_refusals(dev):
    x, experts = inputs(6, 8, 2, "f32", dev)
    found = balance(x, experts)
    one = torch.ones((), device=dev)
    for error, text, call in [
        (ValueError, "score", lambda: balance(x, experts, score="top")), (TypeError, "int32", lambda: balance(x, experts.long())),
        (ValueError, "chosen by these", lambda: balance(x, experts[:5])), (ValueError, "1..1024", lambda: balance(torch.zeros(6, 1025, device=dev), experts)),
        (TypeError, "int32", lambda: balance(x, experts, offsets=torch.zeros(2, dtype=torch.int64, device=dev))),
        (ValueError, "two numbers", lambda: balance(x, experts, offsets=torch.zeros(1, dtype=torch.int32, device=dev))),
        (TypeError, "float32", lambda: balance_grad(one.double(), x, experts, found)), (ValueError, "one number", lambda: balance_grad(x[0], x, experts, found)),
        (ValueError, "sequences and experts", lambda: balance_grad(one, x, experts, found._replace(counts=found.counts[:, :7].contiguous()))),
        (TypeError, "logits' type", lambda: balance_grad(one, x, experts, found, add=x.half())), (ValueError, "like logits", lambda: balance_grad(one, x, experts, found, add=x[:5])),
        (TypeError, "device tensor", lambda: balance(x.cpu(), experts)), (TypeError, "float16, bfloat16", lambda: balance(x.double(), experts)),
    ]:
        with pytest.raises(error, match=text):
            call()
    with pytest.raises(RuntimeError, match="requires a gradient"):
        balance(x.clone().requires_grad_(), experts)
