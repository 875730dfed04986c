"""The layer of experts over virtual ranks."""
import weakref

import pytest
import torch

from mintccl_amd.common import VirtualComm
from mintccl_amd.experts import ExpertLayer, small_layer
from tests.expert_oracle import randn

pytestmark = pytest.mark.gpu


def small(world, dev, **options):
    s = small_layer(world, dev)
    return ExpertLayer(VirtualComm(world_size=world, device=dev), s["router"], s["up"], s["down"], 4, **options), s


def test_passes_keep_apart_what_their_gradients_need(dev):
    """Two batches forward and then their backward passes: each one's gradients are what they are alone."""
    layer, s = small(2, dev)
    other = {n: [randn(*t.shape, seed=50 + i, dtype=t.dtype, dev=dev) for i, t in enumerate(s[n])] for n in ("tokens", "grads")}

    def gradients(kept, batch):
        d_tokens, found = layer.backward(batch["grads"], kept)
        return [*d_tokens, *(f[n] for f in found for n in ("up", "down", "router"))]

    alone = []
    for batch in (s, other):
        kept = []
        layer.forward(batch["tokens"], kept)
        alone.append(gradients(kept, batch))
    first, second = [], []
    layer.forward(s["tokens"], first)
    layer.forward(other["tokens"], second)
    for got, want in ((gradients(first, s), alone[0]), (gradients(second, other), alone[1])):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="another pass"):
        layer.forward(s["tokens"], first)
    with pytest.raises(ValueError, match="forward pass"):
        layer.backward(s["grads"], [])


def test_a_layer_that_only_answers_keeps_nothing(dev):
    layer, s = small(2, dev)
    kept = []
    want = layer.forward(s["tokens"], kept)
    there = [weakref.ref(t) for t in kept[0] if isinstance(t, torch.Tensor)]
    assert there and all(t() is not None for t in there)
    kept.clear()
    assert all(t() is None for t in there)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    got = layer.forward(s["tokens"])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated(dev) == before
