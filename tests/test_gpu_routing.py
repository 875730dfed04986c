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
