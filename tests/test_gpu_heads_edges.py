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


@pytest.mark.parametrize("dt,n,v,d,bias", [(t, 300, 333, 64, True) for t in TYPES] + [(t, 2048, 8192, 130, bias) for t in TYPES for bias in (True, False)])
def test_lse_of_every_row(dt, n, v, d, bias):
    """lse is the logits' own, whatever the label: of ignored rows, of rows whose label is outside the vocabulary, and of rows
    2^40 apart in magnitude (f16: 2^8).  A NaN stays in its row."""
    from yolact_amd import heads
    h, w, b, y, _ = _inputs(n, v, d, dt, bias)
    span = 4 if dt == torch.float16 else 20
    h *= torch.exp2(torch.randint(-span, span + 1, (n, 1), generator=_gen(1), device="cuda").float()).to(dt)
    y[::3], y[1::7], y[2::7] = -1, v, -7
    want = ref.class_loss(h, w, b, torch.zeros_like(y), None)["lse"]
    losses, lse = heads.class_loss(h, w, y, bias=b)
    ref.within(lse, *want, "lse")
    ref.within(losses, *ref.class_loss(h, w, b, y, None)["losses"], "losses")
    h[0, 3] = math.nan
    again = heads.class_loss(h, w, y, bias=b)[1]
    assert again[0].isnan() and torch.equal(again[1:], lse[1:])
