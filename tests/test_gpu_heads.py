"""Prediction-head operators on the device against their definitions in 64 bits (heads_reference states the bounds)."""
import math

import numpy as np
import pytest
import torch

import heads_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
NAN = float("nan")


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _loss_inputs(n, v, d, dt, bias, ignored, seed=0, scale=1.5):
    g = _gen(seed + 1000 * n + v)
    h = torch.randn(n, d, generator=g, device="cuda").to(dt)
    w = (torch.randn(v, d, generator=g, device="cuda") * (scale / math.sqrt(d))).to(dt)
    b = (0.5 * torch.randn(v, generator=g, device="cuda")).to(dt) if bias else None
    y = torch.randint(0, v, (n,), generator=g, device="cuda")
    y[torch.rand(n, generator=g, device="cuda") < ignored] = -1
    up = torch.rand(n, generator=g, device="cuda") / max(n, 1)
    return h, w, b, y, up


def _check_loss(h, w, b, y, up, ignore=-1):
    from yolact_amd import heads
    losses, lse = heads.class_loss(h, w, y, bias=b, ignore_index=ignore)
    gh, gw, gb = heads.class_loss_backward(h, w, y, lse, up, bias=b, ignore_index=ignore)
    want = ref.class_loss(h, w, b, y, up, ignore)
    kept = y != ignore                                    # the lse of a row that takes no part is not promised
    ref.within(losses, *want["losses"], "losses")
    ref.within(lse[kept], want["lse"][0][kept], want["lse"][1][kept], "lse")
    ref.within(gh, *want["grad_h"], "grad_features")
    ref.within(gw, *want["grad_w"], "grad_weight")
    if b is not None:
        ref.within(gb, *want["grad_b"], "grad_bias")
    else:
        assert gb is None
    return losses, lse, gh, gw, gb


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 2, 3), (5, 81, 256), (33, 129, 100), (100, 81, 256), (64, 1000, 64), (257, 130, 31),
                                   (31, 4099, 130), (1, 3001, 64), (130, 2, 96), (700, 300, 257)])
def test_class_loss_sizes(n, v, d, dt):
    _check_loss(*_loss_inputs(n, v, d, dt, bias=(n + v) % 2 == 0, ignored=0.25 if n > 4 else 0.0))


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d,bias", [(2050, 20011, 72, True), (1411, 3331, 513, True), (4111, 3331, 128, False), (40, 70001, 96, False), (20000, 81, 64, True)])
def test_class_loss_large_tiles_and_pieces(n, v, d, bias, dt):
    """Enough tiles for the large tile shape, more than one piece of the vocabulary, a split k axis."""
    _check_loss(*_loss_inputs(n, v, d, dt, bias=bias, ignored=0.1))


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(9000, 18011, 68), (9001, 18011, 1031), (500, 140001, 41), (257, 150000, 1024)])
def test_class_loss_over_pieces_of_the_backward_pass(n, v, d, dt):
    """The gradient of the features adds up over pieces of the vocabulary, with and without a split of that axis."""
    _check_loss(*_loss_inputs(n, v, d, dt, True, 0.1))


@pytest.mark.parametrize("n,v,d,dt,bias", [(1 << 18, 3, 8, torch.bfloat16, True), (1 << 18, 40, 16, torch.float32, False), (2, 1 << 21, 8, torch.float16, True),
                                           (1, 1 << 21, 4, torch.float32, False), (3, 5, 65536, torch.bfloat16, True), (70, 90, 65536, torch.float32, True),
                                           (100000, 513, 40, torch.float16, True), (513, 4000, 2048, torch.bfloat16, True)])
def test_class_loss_long_axes(n, v, d, dt, bias):
    _check_loss(*_loss_inputs(n, v, d, dt, bias, 0.1))


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(200, 333, 64), (1500, 2900, 500)])
def test_class_loss_ignored_rows_and_masked_classes_may_hold_anything(n, v, d, dt):
    h, w, b, y, up = _loss_inputs(n, v, d, dt, True, 0.3)
    b[torch.arange(0, v, 5, device="cuda")] = -math.inf
    y = torch.where((y >= 0) & (y % 5 == 0), (y + 1) % v, y)
    plain = [t.clone() if t is not None else None for t in _check_loss(h, w, b, y, up)]
    h[y == -1] = NAN
    h[torch.nonzero(y == -1)[0]] = math.inf
    w[b == -math.inf] = NAN
    got = _check_loss(h, w, b, y, up)
    for a, c, kept in zip(plain, got, (None, y != -1, None, None, None)):
        a, c = (a, c) if kept is None else (a[kept], c[kept])
        assert torch.equal(a, c)
    assert not got[2][y == -1].any() and not got[3][b == -math.inf].any() and not got[4][b == -math.inf].any()


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(100, 333, 64), (2048, 8192, 128)])
@pytest.mark.parametrize("what", [1e30, -math.inf, NAN], ids=str)
def test_class_loss_gradients_of_ignored_rows_may_hold_anything(n, v, d, dt, what):
    h, w, b, y, up = _loss_inputs(n, v, d, dt, True, 0.3)
    up[y == -1] = what
    _check_loss(h, w, b, y, up)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(100, 333, 64), (2048, 8192, 128)])
@pytest.mark.parametrize("what", [math.inf, NAN], ids=str)
def test_class_loss_a_gradient_that_is_not_finite_stays_with_its_row(n, v, d, dt, what):
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(n, v, d, dt, True, 0.0)
    up *= 2.0 ** -30
    _, lse = heads.class_loss(h, w, y, bias=b)
    bad = up.clone()
    bad[5] = what
    gh, gw, _ = heads.class_loss_backward(h, w, y, lse, bad, bias=b)
    up[5] = 0.0
    value, bound = ref.class_loss(h, w, b, y, up)["grad_h"]
    rest = torch.arange(n, device="cuda") != 5
    ref.within(gh[rest], value[rest], bound[rest], "grad_features")
    assert not torch.isfinite(gh[5]).any() and not torch.isfinite(gw).any()


@pytest.mark.parametrize("n,v,d", [(100, 333, 64), (2048, 8192, 130)])
@pytest.mark.parametrize("what", [math.inf, NAN], ids=str)
def test_class_loss_features_that_are_not_finite_stay_with_their_row(n, v, d, what):
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(n, v, d, torch.float32, True, 0.0)
    h, w = h * 2.0 ** 30, w * 2.0 ** -30
    bad = h.clone()
    bad[7, 3] = what
    losses, lse = heads.class_loss(bad, w, y, bias=b)
    gh, gw, _ = heads.class_loss_backward(bad, w, y, lse, up, bias=b)
    want = ref.class_loss(h, w, b, y, up)
    rest = torch.arange(n, device="cuda") != 7
    for got, name in ((losses, "losses"), (lse, "lse"), (gh, "grad_h")):
        ref.within(got[rest], want[name][0][rest], want[name][1][rest], name)
        assert not torch.isfinite(got[7]).any()


@pytest.mark.parametrize("far", [2.0 ** 16, 2.0 ** 24, 2.0 ** 36], ids=str)
def test_class_loss_large_float32_beside_far_larger_values(far):
    """Every value is off by at most 2^-22 of itself or 2^-39 of the largest of its tensor, dz by 2^-38 of the largest g: one
    row of features and one class are `far` times the others.  A logit is then off by sum_d (eh |w| + |h| ew) more, eh and ew
    being those errors, and what follows from it by the same part."""
    from yolact_amd import heads
    n, v, d = 2048, 8192, 128
    h, w, b, y, up = _loss_inputs(n, v, d, torch.float32, True, 0.1)
    h[17] *= far
    y[17] = -1 if far > 2.0 ** 30 else y[17]        # (a row that takes no part sets no scale)
    w[99] *= min(far, 2.0 ** 24)
    losses, lse = heads.class_loss(h, w, y, bias=b)
    gh, gw, gb = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    want = ref.class_loss(h, w, b, y, up)
    kept = y >= 0
    ah, aw = h.double().abs() * kept[:, None], w.double().abs()
    eh, ew = torch.maximum(ah * 2.0 ** -22, ah.max() * 2.0 ** -39 * kept[:, None]), torch.maximum(aw * 2.0 ** -22, aw.max() * 2.0 ** -39 + 0 * aw)
    ez = (eh @ (aw + ew).t() + ah @ ew.t()).amax(dim=1)                                  # [n]
    ref.within(losses[kept], want["losses"][0][kept], (want["losses"][1] + 2 * ez)[kept], "losses")
    ref.within(lse[kept], want["lse"][0][kept], (want["lse"][1] + ez)[kept], "lse")
    g = up.double() * kept
    z = torch.where(kept[:, None], h, 0 * h).double() @ w.double().t() + b.double()
    p = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    dz = p.clone()
    dz[torch.arange(n, device="cuda")[kept], y[kept]] -= 1.0
    dz = dz.abs() * g[:, None]
    ep = torch.nan_to_num(p * torch.expm1(2 * ez)[:, None], nan=1.0, posinf=1.0).clamp(max=1.0)     # (both are in [0, 1])
    edz = g[:, None] * ep + torch.maximum(dz * 2.0 ** -22, g.max() * 2.0 ** -38 * (g > 0)[:, None])
    ref.within(gh, want["grad_h"][0], want["grad_h"][1] + edz @ (aw + ew) + dz @ ew, "grad_features")
    ref.within(gw, want["grad_w"][0], want["grad_w"][1] + edz.t() @ (ah + eh) + dz.t() @ eh, "grad_weight")


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(200, 333, 64), (2048, 8192, 130)])
def test_class_loss_masks_of_the_lowest_value(n, v, d, dt):
    """A bias of the type's lowest value masks as one of -inf does: its exponentials are zero.  Where it is every class's, and
    beyond what lse can tell apart, results stay finite."""
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(n, v, d, dt, True, 0.2)
    y = torch.where((y >= 0) & (y % 5 == 0), (y + 1) % v, y)
    out = []
    for low in (-math.inf, torch.finfo(dt).min):
        b[::5] = low
        losses, lse = heads.class_loss(h, w, y, bias=b)
        out.append((losses, lse, *heads.class_loss_backward(h, w, y, lse, up, bias=b)))
    off = y % 5 == 0                                          # (the wrap round v may have put a label on a masked class)
    assert not bool(off[y >= 0].any())
    for a, c, name in zip(*out, ("losses", "lse", "grad_features", "grad_weight", "grad_bias")):
        assert torch.equal(a, c), name
    b[:] = torch.finfo(dt).min
    losses, lse = heads.class_loss(h, w, y, bias=b)
    for t in (losses, lse, *heads.class_loss_backward(h, w, y, lse, up, bias=b)):
        assert torch.isfinite(t).all()


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,d", [(200, 333, 64), (2048, 8192, 130)])
def test_class_loss_one_class_of_the_highest_value(n, v, d, dt):
    """It has all of the probability: its rows have loss 0, the others pull from it to their label.  The sum of exponentials
    and a probability exp(z - lse) take log2 e times the largest logit, or lse, rounded: factors of 1 +- 2^-24 |lse| each,
    lse's own rounding another.  f16's 65504 is small enough for that to show, as 2^-7 of g and 2^-7 in the loss; the other
    types' 3.4e38 is not: there the sum is 1, and p, which would be above 1 or 0, the one or the other."""
    from_p = 2.0 ** -7 if dt == torch.float16 else 0.0
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(n, v, d, dt, True, 0.2)
    b[7] = torch.finfo(dt).max
    h /= 4 if dt == torch.float16 else 1                      # (the sum with the bias stays finite in float32 in any case)
    y[::3] = 7
    losses, lse = heads.class_loss(h, w, y, bias=b)
    gh, gw, gb = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    assert bool((losses[y == 7].abs() <= from_p).all()) and (from_p or not gh[y == 7].any())
    rest = (y >= 0) & (y != 7)
    assert torch.isfinite(losses).all() and bool((losses[rest] > 6e4).all())
    onehot = torch.zeros(n, v, dtype=torch.float64, device="cuda")
    onehot[rest, y[rest]] = -1.0
    onehot[rest, 7] = 1.0
    dz = onehot * up.double()[:, None]
    most = dz.abs()
    most[y >= 0, 7] = up.double()[y >= 0]                     # (where p enters)
    for got, want, size in ((gh, dz @ w.double(), most @ w.double().abs()), (gw, dz.t() @ h.double(), most.t() @ h.double().abs()), (gb, dz.sum(0), most.sum(0))):
        ref.within(got, want, (from_p + 4 * ref.HALF[dt] + (n + 8) * ref.F) * size + 2.0 ** -24, "gradient")


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_class_loss_labels_that_cannot_be(dt):
    """A masked class as label: +inf.  A label outside the vocabulary: NaN, no gradient, nothing else touched."""
    h, w, b, y, up = _loss_inputs(50, 40, 32, dt, True, 0.2)
    b[7] = -math.inf
    y[3], y[4], y[5], y[6] = 7, 40, -2, 1 << 40
    losses, lse, gh, gw, gb = _check_loss(h, w, b, y, up)
    assert losses[3] == math.inf and losses[4:7].isnan().all()
    assert not gh[4:7].any() and torch.isfinite(gh).all() and torch.isfinite(gw).all()


def test_class_loss_nothing_left():
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(9, 12, 32, torch.float32, True, 0.0)
    # no class takes part
    b.fill_(-math.inf)
    losses, lse = heads.class_loss(h, w, y, bias=b)
    assert (losses == math.inf).all() and (lse == -math.inf).all()
    for g in heads.class_loss_backward(h, w, y, lse, up, bias=b):
        assert not g.any()
    # no row takes part
    y.fill_(-100)
    b.zero_()
    hh, ww, bb = (t.clone().requires_grad_() for t in (h, w, b))
    for reduction in ("mean", "sum", "none"):
        loss = heads.ClassLoss.apply(hh, ww, bb, y, -100, reduction)
        assert not loss.any()
        for g in torch.autograd.grad(loss.sum(), (hh, ww, bb)):
            assert not g.any()
    # no row at all
    h0, y0 = h[:0].clone().requires_grad_(), y[:0]
    loss = heads.ClassLoss.apply(h0, ww, bb, y0, -1, "mean")
    assert float(loss.detach()) == 0.0
    gs = torch.autograd.grad(loss, (h0, ww, bb))
    assert gs[0].shape == (0, 32) and not gs[1].any() and not gs[2].any()


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_class_loss_logits_beyond_the_precision_of_their_exponentials(dt):
    """z = +-c beside zeros, c about 2^20 to 2^40 (f16: 2^30): z log2 e is off by 2^-24 of itself, which is more than any
    exponent for the larger ones.  lse is c to a few half steps; the gradient lies between 0 and g w, whatever p came to."""
    from yolact_amd import heads
    for c in range(20, 41 if dt != torch.float16 else 31):
        h = torch.zeros(40, 8, dtype=dt, device="cuda")
        w = torch.zeros(300, 8, dtype=dt, device="cuda")
        h[:20, 0], h[20:, 0] = 1.3 * 2.0 ** (c // 2), -1.3 * 2.0 ** (c // 2)
        w[7, 0] = 1.2 * 2.0 ** (c - c // 2)
        z = float(h[0, 0].double() * w[7, 0].double())
        y = torch.tensor([7, 9, 7, 9], device="cuda").repeat_interleave(10)
        up = torch.full((40,), 2.0 ** -12, device="cuda")
        losses, lse = heads.class_loss(h, w, y)
        gh, gw, _ = heads.class_loss_backward(h, w, y, lse, up)
        low = math.log(299)
        rows = lambda *v: torch.tensor(v, dtype=torch.float64, device="cuda").repeat_interleave(10)
        ref.within(lse, rows(z, z, low, low), rows(z, z, 0, 0) * 2.0 ** -22 + 2e-6, "lse")
        ref.within(losses, rows(0, z, z + low, low), rows(z, z, z, 0) * 2.0 ** -22 + 2e-6, "losses")
        assert torch.isfinite(gh).all() and torch.isfinite(gw).all()
        top = float(w[7, 0]) * 2.0 ** -12 * (1 + ref.HALF[dt])
        assert float(gh[:, 0].double().abs().max()) <= top and not gh[30:].any() and not gh[:, 1:].any()
        assert bool((gh[:10, 0] <= 0).all()) and bool((gh[10:20, 0] >= 0).all())


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_class_loss_extreme_logits(dt):
    """Rows whose softmax is one class, rows of large equal logits; gradients far below the type's smallest normal."""
    h, w, b, y, up = _loss_inputs(96, 500, 64, dt, False, 0.1, scale=40.0)
    _check_loss(h, w, b, y, up)
    _check_loss(torch.zeros_like(h), w, b, y, up)
    if dt != torch.float16:
        _check_loss(h / 64, w, b, y, up * 1e-12)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_class_loss_autograd(dt, reduction):
    """Reductions, leading dimensions, int32 labels, labels of another ignored value, non-contiguous inputs, an
    upstream gradient; a gradient that nobody asks for."""
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(60, 130, 40, dt, True, 0.2)
    y = torch.where(y == -1, torch.full_like(y, 1000), y)
    ht = h.view(4, 15, 40).transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()      # same values, other strides
    wt, bt = w.clone().requires_grad_(), b.clone().requires_grad_()
    yt = y.to(torch.int32).view(4, 15)
    loss = heads.ClassLoss.apply(ht, wt, bt, yt, 1000, reduction)
    want = ref.class_loss(h, w, b, y, None, 1000)
    counted = int((y != 1000).sum())
    if reduction == "none":
        assert loss.shape == (4, 15)
        g, gl = up, up.view(4, 15)
    else:
        per = 1.0 / counted if reduction == "mean" else 1.0
        val, err = want["losses"][0].sum() * per, want["losses"][1].sum() * per
        ref.within(loss, val, err + 2 * ref.F * val.abs(), "loss")
        gl = torch.tensor(0.75, device="cuda")
        g = torch.full((60,), 0.75 * per, dtype=torch.float64, device="cuda")
    grads = torch.autograd.grad(loss, (ht, wt, bt), gl, retain_graph=True)
    want = ref.class_loss(h, w, b, y, g, 1000)
    ref.within(grads[0].reshape(60, 40), *want["grad_h"], "grad_features")
    ref.within(grads[1], *want["grad_w"], "grad_weight")
    ref.within(grads[2], *want["grad_b"], "grad_bias")
    loss += 1.0                                                # the result is the caller's to change
    again = torch.autograd.grad(loss, (ht, wt, bt), gl)
    assert all(torch.equal(a, c) for a, c in zip(grads, again))                                # same call, same bits


@pytest.mark.parametrize("n,v,d", [(60, 130, 40), (20, 9000, 64), (700, 90, 300)])
def test_class_loss_gradients_that_nobody_needs(n, v, d):
    from yolact_amd import heads
    for dt in TYPES:
        h, w, b, y, up = _loss_inputs(n, v, d, dt, True, 0.2)
        _, lse = heads.class_loss(h, w, y, bias=b)
        full = heads.class_loss_backward(h, w, y, lse, up, bias=b)
        for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (1, 0, 1)):
            leaves = [t.clone().requires_grad_(bool(k)) for t, k in zip((h, w, b), need)]
            loss = heads.ClassLoss.apply(*leaves, y, -1, "none")
            got = torch.autograd.grad(loss, [t for t in leaves if t.requires_grad], up)
            assert all(torch.equal(a, c) for a, c in zip(got, [g for g, k in zip(full, need) if k]))


def test_class_loss_gradients_against_differences():
    """Directional differences of the 64-bit definition; the bound on the derivative is the sum of the elements' bounds
    times the direction, plus the difference's own 1e-7."""
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(20, 90, 24, torch.float32, True, 0.2)
    _, lse = heads.class_loss(h, w, y, bias=b)
    grads = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    want = ref.class_loss(h, w, b, y, up)
    total = lambda hh, ww, bb: float((ref.class_loss_value(hh, ww, bb, y) * up.double()).sum())
    args = [t.double() for t in (h, w, b)]
    for i, name in enumerate(("grad_h", "grad_w", "grad_b")):
        dirn = torch.randn(args[i].shape, generator=_gen(i), device="cuda", dtype=torch.float64)
        plus, minus = list(args), list(args)
        plus[i], minus[i] = args[i] + 1e-4 * dirn, args[i] - 1e-4 * dirn
        diff = (total(*plus) - total(*minus)) / 2e-4
        assert abs(diff - float((grads[i].double() * dirn).sum())) <= float((want[name][1] * dirn.abs()).sum()) + 1e-7


def test_class_loss_unaligned_inputs():
    """Tensors that begin at an odd element: contiguous, but not on 16 bytes."""
    for dt in TYPES:
        h, w, b, y, up = _loss_inputs(70, 100, 64, dt, True, 0.1)
        def shift(t):
            s = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            s[1:] = t.reshape(-1)
            return s[1:].view(t.shape)
        a = _check_loss(h, w, b, y, up)
        c = _check_loss(shift(h), shift(w), shift(b), y, up)
        assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_python_refusals():
    from yolact_amd import heads
    h, w, b, y, up = _loss_inputs(6, 10, 8, torch.float32, True, 0.0)
    for bad in (dict(features=h.to(torch.bfloat16)), dict(features=h.t().contiguous().t()), dict(features=h[:, :4].contiguous()),
                dict(labels=y[:5]), dict(labels=y.float()), dict(bias=b[:9]), dict(bias=b.to(torch.float16)), dict(weight=w.double()),
                dict(labels=y.cpu())):
        args = dict(features=h, weight=w, labels=y, bias=b)
        args.update(bad)
        with pytest.raises(ValueError):
            heads.class_loss(**args)
    _, lse = heads.class_loss(h, w, y)
    with pytest.raises(ValueError):
        heads.class_loss_backward(h, w, y, lse[:5], up)
    with pytest.raises(ValueError):
        heads.class_loss_backward(h, w, y, lse, up.double())
    wq = heads.quantize_rows(w)
    for x, kw in ((h[:, :4].contiguous(), {}), (h.double(), {}), (h, dict(bias=b[:3])), (h, dict(bias=b.to(torch.bfloat16))),
                  (h, dict(out_dtype=torch.int32)), (heads.quantize_rows(h[:, :4].contiguous()), {})):
        with pytest.raises(ValueError):
            heads.quantized_linear(x, wq, **kw)
    with pytest.raises(ValueError):
        heads.quantize_rows(h.t())
    for index in (1 << 63, (1 << 64) - 1, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="ignore_index"):
            heads.class_loss(h, w, y, ignore_index=index)
        with pytest.raises(ValueError, match="ignore_index"):
            heads.ClassLoss.apply(h, w, b, y, index)
    state = torch.zeros(2, dtype=torch.int64, device="cuda")
    for x, p, s in ((h, 1.5, state), (h, 0.5, state[:1]), (h, 0.5, state.int()), (h.t(), 0.5, state), (y, 0.5, state)):
        with pytest.raises(ValueError):
            heads.dropout(x, p, s)


def test_sizes_past_32_bits_are_refused():
    """2^32 + 5 is not 5 (the tensors are large, nothing touches them)."""
    from yolact_amd import heads
    many = (1 << 32) + 5
    long = torch.empty(many, dtype=torch.bfloat16, device="cuda")
    labels = torch.empty(many, dtype=torch.int32, device="cuda")
    small, one = torch.zeros(5, 1, dtype=torch.bfloat16, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    wq = heads.quantize_rows(small)
    for call in (lambda: heads.class_loss(long[:, None], small, labels), lambda: heads.class_loss(small, long[:, None], one),
                 lambda: heads.class_loss(long[None], long[None], one[:1]), lambda: heads.class_loss_backward(long[:, None], small, labels, labels, labels),
                 lambda: heads.ClassLoss.apply(long[:, None], small, None, labels), lambda: heads.quantize_rows(long[None]),
                 lambda: heads.quantize_rows(long[:, None]), lambda: heads.quantized_linear(long[:, None], wq)):
        with pytest.raises(ValueError, match="too large"):
            call()


# ---- quantized linear ------------------------------------------------------------------------------------------------
def _check_quantized(x, w, b, out_dtype):
    from yolact_amd import heads
    wq = heads.quantize_rows(w)
    qw, sw = ref.quantize(w)
    assert torch.equal(wq.q[:, :w.shape[1]].long(), qw) and not wq.q[:, w.shape[1]:].any()
    assert torch.equal(wq.scale.view(torch.int32), sw.view(torch.int32))
    y = heads.quantized_linear(x, wq, bias=b, out_dtype=out_dtype)
    qx, sx = ref.quantize(x)
    ref.within(y, *ref.quantized_linear(qx, sx, qw, sw, b, out_dtype), "quantized_linear")
    xq = heads.quantize_rows(x)
    assert torch.equal(xq.q[:, :x.shape[1]].long(), qx) and torch.equal(xq.scale, sx)
    assert torch.equal(heads.quantized_linear(xq, wq, bias=b, out_dtype=out_dtype), y)
    return y


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n,v,k", [(1, 1, 1), (1, 4, 128), (1, 1003, 257), (2, 81, 256), (7, 130, 33), (17, 515, 64), (33, 4, 300), (100, 81, 256),
                                   (300, 257, 129), (5, 20000, 512), (1, 5000, 4096), (3, 300, 5001), (2500, 5200, 96), (8, 77, 7000), (1, 1000, 50000), (1, 70, 70000), (1, 20001, 640),
                                   (5000, 81, 256), (4099, 4, 100), (4111, 33, 511), (9001, 130, 128), (70000, 32, 64)])
def test_quantized_linear_sizes(n, v, k, dt):
    g = _gen(n + v + k)
    x = (torch.randn(n, k, generator=g, device="cuda") * 3).to(dt)
    w = (torch.randn(v, k, generator=g, device="cuda") / math.sqrt(k)).to(dt)
    b = torch.randn(v, generator=g, device="cuda") if n % 2 else None
    for out_dtype in (torch.float32, dt):
        _check_quantized(x, w, b, out_dtype)


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_quantize_rows_ties_zeros_and_extremes(dt):
    """Quotients that are exactly a half, rows of zeros, rows of the type's largest and smallest values."""
    top = torch.finfo(dt).max
    small = 2.0 ** -24 if dt == torch.float16 else 2.0 ** -133 if dt == torch.bfloat16 else 2.0 ** -149
    rows = [torch.arange(-127, 128, device="cuda") / 2.0, torch.zeros(255, device="cuda"), torch.linspace(-1, 1, 255, device="cuda") * top,
            torch.arange(-127, 128, device="cuda").double() * small, (torch.arange(-127, 128, device="cuda") % 2) * small * 127.0,
            torch.linspace(0, 1e-30, 255, device="cuda"), torch.randint(-254, 255, (255,), generator=_gen(5), device="cuda") / 2.0]
    rows[0][0], rows[-1][0] = 127.0, 127.0
    x = torch.stack([r.double() for r in rows]).to(dt)
    w = torch.randn(9, 255, generator=_gen(1), device="cuda").to(dt)
    from yolact_amd import heads
    q, s = ref.quantize(x)
    got = heads.quantize_rows(x)
    assert torch.equal(got.scale.view(torch.int32), s.view(torch.int32))
    assert torch.equal(got.q[:, :255].long(), q)
    deq = got.dequantize().double()
    assert torch.equal(deq, (q.double() * s.double()[:, None]).float().double())
    assert float((got.q[1].abs().max())) == 0 and float(heads.quantized_linear(x, heads.quantize_rows(w))[1].abs().max()) == 0.0


def test_quantized_rows_that_are_not_finite():
    from yolact_amd import heads
    x = torch.randn(6, 200, generator=_gen(2), device="cuda")
    x[1, 3], x[2, 199], x[4, 0] = NAN, math.inf, -math.inf
    w = torch.randn(50, 200, generator=_gen(3), device="cuda")
    w[7, 7] = NAN
    q = heads.quantize_rows(x)
    bad = torch.tensor([False, True, True, False, True, False], device="cuda")
    assert torch.equal(q.scale.isnan(), bad)
    y = heads.quantized_linear(x, heads.quantize_rows(w))
    want = bad[:, None] | (torch.arange(50, device="cuda") == 7)
    assert torch.equal(y.isnan(), want)
    z = heads.quantized_linear(q, heads.quantize_rows(w))
    assert torch.equal(z.isnan(), want) and torch.equal(z[~want], y[~want])


def test_quantized_linear_largest_sums():
    """k = 131072 of all 127s: the integer sum is 2 114 060 288, just inside 32 bits."""
    k = 131072
    x, w = torch.ones(3, k, device="cuda"), torch.ones(5, k, device="cuda")
    w[1] = -1
    y = _check_quantized(x, w, None, torch.float32)
    assert float(y[0, 0]) > 0 and float(y[0, 1]) < 0
    assert abs(float(y[0, 0]) - k) < 1


def test_dropout_past_32_bits_of_elements():
    """2^32 + 5 elements: the mask of the last ones."""
    from yolact_amd import heads
    n = (1 << 32) + 5
    y = heads.dropout(torch.ones(n, dtype=torch.bfloat16, device="cuda"), 0.5, _state(5, 7))
    tail = (y[-4101:] != 0).cpu().numpy()
    first = n - 4101
    assert np.array_equal(tail, ref.keep_mask(4104, 0.5, 5, 7 + first // 4)[first % 4:][:4101])


def test_quantized_linear_empty_and_unaligned():
    from yolact_amd import heads
    w = torch.randn(5, 48, generator=_gen(1), device="cuda")
    wq = heads.quantize_rows(w)
    assert heads.quantized_linear(torch.empty(0, 48, device="cuda"), wq).shape == (0, 5)
    assert heads.quantized_linear(torch.empty(2, 0, 48, device="cuda"), wq).shape == (2, 0, 5)
    assert heads.quantize_rows(torch.empty(0, 48, device="cuda")).q.shape[0] == 0
    s = torch.randn(7 * 48 + 1, generator=_gen(2), device="cuda")
    x = s[1:].view(7, 48)
    assert torch.equal(heads.quantized_linear(x, wq), heads.quantized_linear(x.clone(), wq))
    assert torch.equal(heads.quantized_linear(x[0], wq), heads.quantized_linear(x, wq)[0])


def test_quantized_rows_made_by_hand():
    from yolact_amd import heads
    x = torch.randn(2, 3, 200, generator=_gen(4), device="cuda")
    w = heads.quantize_rows(torch.randn(9, 200, generator=_gen(5), device="cuda"))
    a = heads.quantize_rows(x)
    kept = heads.QuantizedRows(a.q.cpu().cuda(), a.scale.clone(), 200, (2, 3))
    assert torch.equal(heads.quantized_linear(kept, w), heads.quantized_linear(x, w))
    for q, scale, k, lead in ((a.q.cpu(), a.scale, 200, (2, 3)), (a.q, a.scale.cpu(), 200, (2, 3)), (a.q[:, :200].contiguous(), a.scale, 200, (2, 3)),
                              (a.q, a.scale[:5], 200, (2, 3)), (a.q, a.scale, 200, (7,)), (a.q, a.scale, 300, (2, 3)), (a.q, a.scale, 0, (2, 3)),
                              (a.q.int(), a.scale, 200, (2, 3)), (a.q, a.scale.double(), 200, (2, 3)), (a.q.t().contiguous().t(), a.scale, 200, (2, 3))):
        with pytest.raises((ValueError, RuntimeError)):
            heads.QuantizedRows(q, scale, k, lead)


# ---- dropout ---------------------------------------------------------------------------------------------------------
def _state(key, first):
    return torch.tensor([key, first], dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 3, 4, 5, 255, 1024, 4099, 300001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout(n, p, dt):
    from yolact_amd import heads
    key, first = 0x123456789ABCDEF, (1 << 32) - 7
    x = torch.randn(n, generator=_gen(n), device="cuda").to(dt)
    y = heads.dropout(x, p, _state(key, first))
    keep = torch.from_numpy(ref.keep_mask(n, p, key, first)).cuda()
    want = torch.where(keep, x.double() / (1.0 - p) if p < 1 else x.double(), torch.zeros_like(x, dtype=torch.float64))
    # the factor and the product round once each in float32, the result once to the type
    half = ref.HALF[dt] if dt != torch.float32 else 0.0
    ref.within(y, want, (2.01 * ref.F + half * (1 + 3 * ref.F)) * want.abs() + (2.0 ** -25 if dt == torch.float16 else 0.0), "dropout")
    assert torch.equal(y != 0, keep & (x != 0))


def test_dropout_any_counter_unaligned_in_place_and_not_finite():
    from yolact_amd import heads
    for key, first in ((0, 0), (-1, -1), (-5, -3), (1 << 62, 1 << 62)):
        x = torch.ones(1003, device="cuda")
        keep = torch.from_numpy(ref.keep_mask(1003, 0.3, key % (1 << 64), first % (1 << 64))).cuda()
        assert torch.equal(heads.dropout(x, 0.3, _state(key, first)) != 0, keep)
    for dt in TYPES:
        s = torch.randn(1000, generator=_gen(4), device="cuda").to(dt)
        whole = heads.dropout(s[1:].clone(), 0.4, _state(9, 9))
        assert torch.equal(heads.dropout(s[1:], 0.4, _state(9, 9)), whole)
        buf = s[1:].clone()
        assert heads.dropout(buf, 0.4, _state(9, 9), out=buf) is buf and torch.equal(buf, whole)
    x = torch.full((4096,), NAN, device="cuda")
    x[::2] = math.inf
    y = heads.dropout(x, 0.5, _state(1, 2))
    keep = torch.from_numpy(ref.keep_mask(4096, 0.5, 1, 2)).cuda()
    assert not y[~keep].any() and torch.equal(y[keep].isnan(), x[keep].isnan())
    assert heads.dropout(torch.empty(0, 5, device="cuda"), 0.5, _state(1, 2)).shape == (0, 5)


def test_dropout_into_a_tensor_that_a_graph_has_kept_is_seen():
    from yolact_amd import heads
    state = torch.tensor([3, 0], device="cuda")
    x = torch.randn(64, device="cuda", requires_grad=True)
    y = x * 2.0
    z = y * y
    heads.dropout(y.detach(), 0.5, state, out=y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    with pytest.raises(RuntimeError, match="overlap"):
        heads.dropout(x.detach()[:32], 0.5, state, out=x.detach()[8:40])
    with torch.inference_mode():
        a = torch.ones(10, device="cuda")
        assert heads.dropout(a, 1.0, state, out=a) is a and not a.any()


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_dropout_autograd(dt):
    from yolact_amd import heads
    x = torch.randn(37, 65, generator=_gen(6), device="cuda").to(dt).requires_grad_()
    g = torch.randn(37, 65, generator=_gen(7), device="cuda").to(dt)
    st = _state(77, 5)
    y = heads.Dropout.apply(x.t(), 0.25, st)                # not contiguous: the mask follows the values' own order
    gx, = torch.autograd.grad(y, x, g.t())
    assert torch.equal(gx.t(), heads.dropout(g.t().contiguous(), 0.25, st))
    y = heads.Dropout.apply(x, 0.25, st)
    st[1] += 10
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, x, g)


# ---- together --------------------------------------------------------------------------------------------------------
def test_streams_and_graphs():
    """The whole training step and the whole answer captured into one graph each on a side stream, replayed on changed
    inputs with eager work in between: every replay is the eager result, bit for bit."""
    from yolact_amd import heads
    for dt in TYPES:
        h, w, b, y, up = _loss_inputs(150, 700, 96, dt, True, 0.2)
        st = _state(3, 0)
        wq = heads.quantize_rows(w)
        b32 = b.float()

        def step():
            x = heads.dropout(h, 0.2, st)
            losses, lse = heads.class_loss(x, w, y, bias=b)
            gx, gw, gb = heads.class_loss_backward(x, w, y, lse, up, bias=b)
            return [losses, heads.dropout(gx, 0.2, st), gw, gb, heads.quantized_linear(h, wq, bias=b32)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other, pool=graph.pool()):
            outs2 = step()
        for r in range(4):
            h.copy_(torch.randn(h.shape, generator=_gen(100 + r), device="cuda").to(dt))
            st[1] += 4096
            want = [t.clone() for t in step()]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs, want)), (dt, r)
            other.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(outs2, want)), (dt, r)


def test_first_call_in_a_graph():
    """Shapes that no eager call has launched before: the many-row kernel with a large LDS, the few-row one, a split f32 step."""
    from yolact_amd import heads
    x, w = torch.randn(5000, 250, generator=_gen(1), device="cuda"), torch.randn(141, 250, generator=_gen(2), device="cuda")
    wq = heads.quantize_rows(w)
    h, ww, b, y, up = _loss_inputs(1300, 3001, 600, torch.float32, True, 0.1)

    def step():
        losses, lse = heads.class_loss(h, ww, y, bias=b)
        return [heads.quantized_linear(x, wq), heads.quantized_linear(x[:3], wq), losses] + list(heads.class_loss_backward(h, ww, y, lse, up, bias=b))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(3):
        x.mul_(1.1)
        h.mul_(0.9)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want))


def test_autograd_step_in_a_graph():
    from yolact_amd import heads
    h, w, b, y, _ = _loss_inputs(64, 300, 64, torch.bfloat16, True, 0.2)
    st = _state(3, 0)

    def step():
        leaves = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = heads.class_head_loss(leaves[0], leaves[1], leaves[2], y, dropout_p=0.1, state=st)
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(3):
        w.add_(0.01)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want))


def test_train_then_answer_through_detect():
    """The head as it is used: a few steps of class_head_loss on the features, then its weights in 8 bits feeding Detect -
    whose detections on the 8-bit logits are those on the same logits made in plain torch."""
    from yolact_amd import Detect, heads
    g = _gen(11)
    B, A, D, C, ph = 2, 240, 64, 5, 12
    feats = torch.randn(B, A, D, generator=g, device="cuda")
    y = torch.randint(0, C, (B, A), generator=g, device="cuda")
    proj = torch.randn(C, D, generator=g, device="cuda")
    feats += 0.5 * proj[y]
    y[:, ::3] = -1
    w, b = (0.01 * torch.randn(C, D, generator=g, device="cuda")).requires_grad_(), torch.zeros(C, device="cuda", requires_grad=True)
    st = _state(1, 0)
    for _ in range(3):
        loss = heads.class_head_loss(feats, w, b, y, dropout_p=0.1, state=st)
        gw, gb = torch.autograd.grad(loss, (w, b))
        assert torch.isfinite(loss) and torch.isfinite(gw).all()
        with torch.no_grad():
            w -= gw
            b -= gb
        st[1] += feats.numel() // 4
    w, b = w.detach(), b.detach()
    wo, wm = 0.1 * torch.randn(4, D, generator=g, device="cuda"), 0.1 * torch.randn(32, D, generator=g, device="cuda")
    net = heads.QuantizedHeads((w, b), wo, wm)(feats)
    assert net["pred_cls"].shape == (B, A, C) and net["pred_offset"].shape == (B, A, 4) and net["pred_mask_coef"].shape == (B, A, 32)
    plain = {}
    for name, ww, bb in (("pred_cls", w, b), ("pred_offset", wo, None), ("pred_mask_coef", wm, None)):
        q, s = ref.quantize(feats.reshape(B * A, D))
        qw, sw = ref.quantize(ww)
        value, bound = ref.quantized_linear(q, s, qw, sw, bb, torch.float32)
        ref.within(net[name].reshape(B * A, -1), value, bound, name)
        plain[name] = value.float().reshape(net[name].shape)
    c = torch.rand(A, 2, generator=g, device="cuda") * 40 + 12
    priors = torch.cat([c - 8, c + 8], dim=1).contiguous()
    rest = dict(priors=priors, proto_out=torch.randn(B, ph, ph, 32, generator=g, device="cuda").relu())
    det = Detect(C, 300, 100, 0.05, 0.5)
    a, p = det({**net, **rest}, [B, 64, 64, 3]), det({**plain, **rest}, [B, 64, 64, 3])
    assert (a["num_detections"] > 0).all() and torch.equal(a["num_detections"], p["num_detections"])
    assert float((a["detection_scores"] - p["detection_scores"]).abs().max()) < 1e-5
