"""Routing, assignment and combination at the ends of their ranges."""
import math

import pytest
import torch

from mintccl_amd.combine import combine, combine_grad
from mintccl_amd.routing import assign, route, route_grad
from tests.expert_oracle import randn

pytestmark = pytest.mark.gpu


def test_gradients_of_no_tokens(dev):
    """Every result is there, and empty."""
    plan = assign(torch.zeros(0, 3, dtype=torch.int32, device=dev), 4)
    rows, weights = torch.zeros(0, 64, device=dev), torch.zeros(0, 3, device=dev)
    assert combine(rows, plan, weights).shape == (0, 64)
    d_rows, d_weights = combine_grad(rows, rows, plan, weights)
    assert d_rows.shape == (0, 64) and d_weights.shape == (0, 3) and d_weights.dtype == torch.float32
    assert combine_grad(rows, rows, plan)[1] is None
    logits = torch.zeros(0, 8, device=dev)
    assert route_grad(d_weights, logits, plan.slots).shape == (0, 8)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("experts,groups", [(16, 4), (12, 4), (256, 8), (320, 8), (18, 3)])
def test_groups_masked_by_the_lowest_number(dev, experts, groups, dt):
    """Groups whose two best keys are the type's lowest number: their sum is beyond 32 bits' range, and their experts are there all the same, behind all
    others and in order."""
    per, low = experts // groups, torch.finfo(dt).min
    x = torch.full((4, experts), low)
    x[1, per * (groups - 1):] = torch.arange(per).flip(0).float()       # the last group counts
    x[2, per:2 * per] = -math.inf                                       # the second one is masked altogether
    x[3] = -math.inf
    x[3, 2 * per + 1:2 * per + 3] = low                                 # (two experts of the third group)
    x = x.to(dt).to(dev)
    w, chosen = (v.cpu() for v in route(x, 4, groups=groups, kept=2, group_top=2))
    first = list(range(min(4, per))) + list(range(per, per + 4))
    assert chosen[0].tolist() == first[:4]
    last = [per * (groups - 1) + i for i in range(per)]
    assert chosen[1].tolist() == (last + first)[:4]
    assert chosen[2].tolist() == (list(range(min(4, per))) + [2 * per + i for i in range(4)])[:4]
    assert chosen[3].tolist() == [2 * per + 1, 2 * per + 2, -1, -1]
    assert torch.allclose(w[0], torch.full((4,), 0.25)) and w[3].tolist() == [0.5, 0.5, 0.0, 0.0]


def test_gradient_of_scores_that_almost_vanish(dev):
    """Sigmoids near the end of 32 bits' range, divided by their sum: the quotients are ordinary numbers, and so are the gradients."""
    x = torch.tensor([[-88.0, -88.5, -87.5, -95.0], [-80.0, -85.0, -88.0, -70.0], [-86.0, -86.0, -86.0, -86.0], [-20.0, 3.0, -60.0, 0.0]], device=dev)
    d = torch.tensor([[4.0, -7.0, 100.0], [1.0, 2.0, -3.0], [1.0, 0.0, 0.0], [1.0, -1.0, 2.0]], device=dev)
    w, chosen = route(x, 3, score="sigmoid")
    assert chosen.tolist() == [[2, 0, 1], [3, 0, 1], [0, 1, 2], [1, 3, 0]]
    x64 = x.double().requires_grad_()
    s = torch.sigmoid(x64).gather(1, chosen.long())
    want = s / s.sum(-1, keepdim=True)
    # a score of 2^-126 and less has 22 bits here at -88.5: 2^-21 of it, three scores, a sum and quotients
    assert torch.allclose(w.double(), want, rtol=2.0 ** -17, atol=0)
    (want * d.double()).sum().backward()
    got = route_grad(d, x, chosen, score="sigmoid")
    assert torch.isfinite(got).all()
    assert ((got.double() - x64.grad).abs() <= 2.0 ** -15 * d.abs().max(1, keepdim=True).values.double()).all()


def test_more_tokens_than_a_launch_has_threads_for(dev):
    """2^26 tokens and some, 64 threads each in the gradient: the same as alone at the ends and where launches meet."""
    n, k = (1 << 26) + 77, 2
    some = randn(1 << 16, 8, seed=1, dtype=torch.bfloat16, dev=dev)
    x = torch.empty(n, 8, dtype=torch.bfloat16, device=dev)
    for at in range(0, n, 1 << 16):                  # (no two parts alike)
        x[at:at + (1 << 16)] = some[:n - at].roll(at >> 16, 0)
    d = torch.ones(n, k, device=dev)
    d[1::3, 1] = -2.0
    w, chosen = route(x, k)
    got = route_grad(d, x, chosen)
    for at in (0, (1 << 25) - 50, (1 << 26) - 50, n - 100):
        own = slice(at, at + 100)
        alone = route(x[own], k)
        assert torch.equal(w[own], alone[0]) and torch.equal(chosen[own], alone[1])
        assert torch.equal(got[own], route_grad(d[own], x[own], alone[1]))
    assert (chosen >= 0).all() and torch.isfinite(w.view(-1)).all()
    del x, w, chosen, got, d
    torch.cuda.empty_cache()


def test_slots_behind_the_experts_places_have_no_gradient(dev):
    """Places that the offsets do not count: their rows are cleared, by the same blocks every time, whatever the slots say."""
    plan = assign(torch.arange(4096, dtype=torch.int32, device=dev).view(1024, 4) % 8, 8)
    some = plan._replace(offsets=plan.offsets[:5])                # four of the eight experts
    used = int(some.offsets[-1])
    rows, d, w = randn(4096, 520, seed=1, dev=dev), randn(1024, 520, seed=2, dev=dev), randn(1024, 4, seed=3, dev=dev)
    whole, there = combine_grad(d, rows, plan, w), plan.slots < used
    for _ in range(5):
        d_rows, d_weights = combine_grad(d, rows, some, w)
        assert torch.equal(d_rows[:used], whole[0][:used]) and (d_rows[used:] == 0).all()
        assert torch.equal(d_weights[there], whole[1][there]) and (d_weights[~there] == 0).all()
