"""Prediction-head operators at the ends of their ranges, against their definitions in 64 bits (heads_reference)."""
import math

import pytest
import torch

import heads_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _inputs(n, v, d, dt, bias, seed=0):
    g = _gen(seed + 1000 * n + v)
    h = torch.randn(n, d, generator=g, device="cuda").to(dt)
    w = (torch.randn(v, d, generator=g, device="cuda") * (1.5 / math.sqrt(d))).to(dt)
    b = (0.5 * torch.randn(v, generator=g, device="cuda")).to(dt) if bias else None
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    up = torch.rand(n, generator=g, device="cuda") / max(n, 1)
    return h, w, b, y, up


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_rows_and_one_gradient_wanted(dt, reduction):
    from yolact_amd import heads
    h, w, b, y, _ = _inputs(0, 12, 32, dt, True)
    for which in range(3):
        leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((h, w, b))]
        loss = heads.ClassLoss.apply(*leaves, y, -1, reduction)
        grad, = torch.autograd.grad(loss.sum(), [leaves[which]])
        assert grad.shape == leaves[which].shape and not grad.any()
