"""Prediction-head operators at the ends of their ranges, against their definitions in 64 bits (heads_reference)."""
import math

import pytest
import torch

import heads_precision as precision
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


def _large_float32_bounds(h, w, b, y, up):
    """What large float32 calls are allowed beyond the reference's bounds.  Logits: each value is off by 2^-22 of itself - three
    such errors a product, 12 F, are within the reference's (D + 2) F - or by 2^-39 of its row's largest, which is less than that
    beside the row's largest product.  Gradients: the softmax's difference d by 2^-22 of itself or 2^-38 (half a step
    of f16's subnormals, of d times 2^13), the weight by 2^-39 of the largest, gradient times features by 2^-39 of theirs."""
    want = ref.class_loss(h, w, b, y, up)
    kept = (y >= 0) & (y < w.shape[0])
    hk = torch.where(kept[:, None], h, 0 * h).double().nan_to_num(0.0)
    gh = hk * torch.where(kept, up, 0 * up).double()[:, None]
    g = torch.where(kept, up, 0 * up).double().abs()
    wd = w.double()
    z = hk @ wd.t() + (b.double() if b is not None else 0.0)
    dd = torch.exp(z - torch.logsumexp(z, dim=1, keepdim=True))
    dd[torch.arange(len(y), device="cuda")[kept], y[kept]] -= 1.0
    dd = dd.abs() * kept[:, None]
    off = 2.0 ** -38 * kept[:, None] + 0 * dd
    more_h = g[:, None] * (off @ wd.abs() + dd.sum(dim=1, keepdim=True) * wd.abs().max() * 2.0 ** -39)
    more_w = off.t() @ gh.abs() + dd.t().sum(dim=1, keepdim=True) * gh.abs().max() * 2.0 ** -39
    want["grad_h"] = (want["grad_h"][0], want["grad_h"][1] + 1.01 * more_h)
    want["grad_w"] = (want["grad_w"][0], want["grad_w"][1] + 1.01 * more_w)
    return want


def _check_large_float32(h, w, b, y, up, wild=()):
    """wild: rows whose own results are not finite; if one of them takes part, neither is the weight's gradient."""
    from yolact_amd import heads
    losses, lse = heads.class_loss(h, w, y, bias=b)
    grads = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    rest = torch.ones_like(y, dtype=torch.bool)
    rest[list(wild)] = False
    tame = h.clone()
    tame[~rest] = 0.0
    want = _large_float32_bounds(tame, w, b, y, up)
    for got, name in ((losses, "losses"), (lse, "lse"), (grads[0], "grad_h")):
        ref.within(got[rest], want[name][0][rest], want[name][1][rest], name)
    if all(int(y[i]) < 0 for i in wild):
        for got, name in zip(grads[1:], ("grad_w", "grad_b") if b is not None else ("grad_w",)):
            ref.within(got, *want[name], name)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("row,features,weight", [(2.0 ** 120, 1.0, 2.0 ** -116), (1.0, 2.0 ** 112, 2.0 ** -112), (1.0, 2.0 ** 118, 2.0 ** -119),
                                                 (2.0 ** -100, 2.0 ** -110, 2.0 ** 112), (1.0, 1.0, 2.0 ** -125)])
def test_large_float32_values_at_the_ends_of_the_type(row, features, weight, bias):
    """Values of 2^116 and more, and tensors whose largest value is 2^-110 and less, with logits of ordinary size."""
    h, w, b, y, up = _inputs(2048, 8192, 130, torch.float32, bias)
    h, w = h * features, w * weight
    h[5] *= row
    _check_large_float32(h, w, b, y, up * 2048)


def test_large_float32_rows_of_zeros_beside_very_large_ones():
    """One row of 2^100 against a class of 2^60: its logit is infinite.  Rows of zeros have the bias as logits."""
    h, w, b, y, up = _inputs(2048, 8192, 130, torch.float32, True)
    h[0] *= 2.0 ** 100
    h[1:9] = 0.0
    w[3] *= 2.0 ** 60
    _check_large_float32(h, w, b, y, up, wild=(0,))
    y[0] = -1
    _check_large_float32(h, w, b, y, up, wild=(0,))


def test_large_float32_rows_of_far_smaller_gradients():
    h, w, b, y, up = _inputs(2048, 8192, 130, torch.float32, True)
    up[::2] *= 2.0 ** -30
    _check_large_float32(h, w, b, y, up)


@pytest.mark.parametrize("dt,n,v,d", [(torch.float32, 2048, 8192, 130), (torch.bfloat16, 2048, 8192, 130), (torch.bfloat16, 100, 333, 64), (torch.float32, 100, 333, 64)])
def test_gradients_below_the_smallest_normal_ones(dt, n, v, d):
    """Upstream gradients of 2^-118 and less, features of 2^40: the weight's gradient is of ordinary size."""
    from yolact_amd import heads
    h, w, b, y, up = _inputs(n, v, d, dt, True)
    h, w = h * 2.0 ** 40, w * 2.0 ** -40
    up *= 2.0 ** -118
    bounds = _large_float32_bounds if n == 2048 and dt == torch.float32 else ref.class_loss
    _, lse = heads.class_loss(h, w, y, bias=b)
    gh, gw, gb = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    want = bounds(h, w, b, y, up)
    for got, name in ((gh, "grad_h"), (gw, "grad_w"), (gb, "grad_b")):
        ref.within(got, *want[name], name)
    # one gradient for all rows, itself no normal number
    one = torch.tensor(1.37 * 2.0 ** -130, device="cuda")
    leaf = w.clone().requires_grad_()
    gw, = torch.autograd.grad(heads.ClassLoss.apply(h, leaf, b, y, -1, "sum"), [leaf], one)
    ref.within(gw, *bounds(h, w, b, y, torch.full_like(up, 1.0) * one)["grad_w"], "grad_w")


@pytest.mark.parametrize("rows,v", [((1 << 28) + 3, 20), ((1 << 23) + 3, 600)])
def test_quantized_linear_past_32_bits_of_results(rows, v):
    """A row's results depend on that row alone: those at the ends of a call of 2^32 results are a small call's."""
    from yolact_amd import heads
    x = torch.randint(-100, 100, (rows, 1), generator=_gen(rows), device="cuda", dtype=torch.int8).to(torch.bfloat16)
    w = heads.quantize_rows(torch.randn(v, 1, generator=_gen(v), device="cuda"))
    b = torch.randn(v, generator=_gen(v + 1), device="cuda")
    y = heads.quantized_linear(x, w, bias=b, out_dtype=torch.bfloat16)
    assert y.numel() > 1 << 32
    for at in (0, (1 << 32) // v - 50, rows - 100):
        part = x[at:at + 100].contiguous()
        few = heads.quantized_linear(part, w, bias=b, out_dtype=torch.bfloat16)
        assert torch.equal(y[at:at + 100], few)
        ref.within(few, *ref.quantized_linear(*ref.quantize(part), w.q[:, :1].long(), w.scale, b, torch.bfloat16), "quantized_linear")


@pytest.mark.parametrize("dt", TYPES[1:], ids=str)
@pytest.mark.parametrize("n,v,d", [(200, 333, 64), (512, 4099, 130), (700, 300, 257), (100, 81, 256)])
def test_precision_of_two_planes_of_dz(n, v, d, dt):
    """Up to 512 rows, or 2^30 multiplications, the gradients of 16-bit calls are off by their own rounding and little more."""
    from yolact_amd import heads
    h, w, b, y, up = _inputs(n, v, d, dt, True)
    up *= n
    y[::5] = -1
    _, lse = heads.class_loss(h, w, y, bias=b)
    got = dict(zip(("grad_h", "grad_w"), heads.class_loss_backward(h, w, y, lse, up, bias=b)))
    for name, (value, bound) in precision.two_planes(h, w, b, y, up).items():
        ref.within(got[name], value, bound, name)
        assert precision.relative(got[name], value) <= precision.ROUNDED * ref.HALF[dt], name


@pytest.mark.parametrize("dt", TYPES[1:], ids=str)
def test_precision_of_one_plane_of_dz(dt):
    """Beyond that dz is rounded once, like the gradients."""
    from yolact_amd import heads
    h, w, b, y, up = _inputs(1300, 1290, 1290, dt, True)
    up *= 1300
    _, lse = heads.class_loss(h, w, y, bias=b)
    got = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    dz, _, _ = precision.softmax_difference(h, w, b, y, up)
    for have, value in zip(got, (dz @ w.double(), dz.t() @ h.double())):
        assert precision.relative(have, value) <= precision.ROUNDED_TWICE * ref.HALF[dt]


def test_precision_of_large_float32():
    """2.16e9 multiplications: two f16 planes.  Losses: a logit's error (the terms of one have a root mean square of 1.5 over
    sqrt d, so 1.5 in all), and four roundings to float32 of numbers between 8 and 16 - lse, its logarithm's two units,
    the difference -, half a step of which is two of 2^-22, again a third of the square in the mean; a third more allowed."""
    from yolact_amd import heads
    n, v, d = 1300, 1290, 1290
    h, w, b, y, up = _inputs(n, v, d, torch.float32, False)
    losses, lse = heads.class_loss(h, w, y)
    gh, gw, _ = heads.class_loss_backward(h, w, y, lse, up)
    dz, z, _ = precision.softmax_difference(h, w, None, y, up)
    assert precision.relative(gh, dz @ w.double()) <= precision.rms_of_planes(v)
    assert precision.relative(gw, dz.t() @ h.double()) <= precision.rms_of_planes(n)
    off = losses.double() - (torch.logsumexp(z, dim=1) - z.gather(1, y[:, None])[:, 0])
    allowed = math.hypot(1.5 * precision.rms_of_planes(d), 4.0 / 3.0 * math.sqrt(4 * 4 / 3.0) * precision.STEP)
    assert float(off.square().mean().sqrt()) <= allowed


def test_quantized_heads_of_a_convolution():
    """A head whose last layer is a 3 x 3 convolution with all anchors of a place in its channels: on unfolded neighbourhoods."""
    from yolact_amd import heads
    B, ch, H, W, A, classes, k = 2, 24, 7, 9, 3, 5, 3
    fmap = torch.randn(B, ch, H, W, generator=_gen(1), device="cuda")
    kernels = [torch.randn(A * n, ch, k, k, generator=_gen(n), device="cuda") / math.sqrt(ch * k * k) for n in (classes, 4, 32)]
    bias = torch.randn(A * classes, generator=_gen(9), device="cuda")
    rows = torch.nn.functional.unfold(fmap, k, padding=1).transpose(1, 2).contiguous()
    net = heads.QuantizedHeads((kernels[0].flatten(1), bias), kernels[1].flatten(1), kernels[2].flatten(1))(rows)
    q, s = ref.quantize(rows.reshape(B * H * W, -1))
    for (name, got), kernel, b in zip(net.items(), kernels, (bias, None, None)):
        qw, sw = ref.quantize(kernel.flatten(1))
        ref.within(got.reshape(B * H * W, -1), *ref.quantized_linear(q, s, qw, sw, b, torch.float32), name)
        # and near the convolution itself: each of the products is off by half a step of either operand at most
        conv = torch.nn.functional.conv2d(fmap.cpu().double(), kernel.cpu().double(), b.cpu().double() if b is not None else None, padding=1)
        conv = conv.permute(0, 2, 3, 1).reshape(B * H * W, -1).cuda()
        x, w = rows.reshape(B * H * W, -1).double().abs(), kernel.flatten(1).double().abs()
        half_x, half_w = 0.5 * s.double()[:, None] + 0 * x, 0.5 * sw.double()[:, None] + 0 * w
        ref.within(got.reshape(B * H * W, -1), conv, 1.0001 * (half_x @ (w + half_w).t() + x @ half_w.t()) + 1e-5, name)
        assert got.reshape(B, H * W * A, -1).shape[2] == got.shape[2] // A


def test_large_float32_nothing_left():
    """No row takes part, no class does, or all values are zeros: in the size that runs through planes."""
    from yolact_amd import heads
    h, w, b, y, up = _inputs(2048, 8192, 130, torch.float32, True)
    none = torch.full_like(y, -1)
    for reduction in ("mean", "sum", "none"):
        leaves = [t.clone().requires_grad_() for t in (h, w, b)]
        loss = heads.ClassLoss.apply(*leaves, none, -1, reduction)
        assert not loss.any() and not any(g.any() for g in torch.autograd.grad(loss.sum(), leaves))
    off = torch.full_like(b, -math.inf)
    losses, lse = heads.class_loss(h, w, y, bias=off)
    assert bool((losses == math.inf).all()) and bool((lse == -math.inf).all())
    assert not any(g.any() for g in heads.class_loss_backward(h, w, y, lse, up, bias=off))
    _check_large_float32(0 * h, 0 * w, b, y, up)
    _check_large_float32(0 * h, w, b, y, up)
    _check_large_float32(h, 0 * w, b, y, 0 * up)


def test_large_float32_gradients_that_nobody_needs_and_replays():
    """Each gradient alone is the same as beside the others; a captured step with a gradient a row follows its inputs."""
    from yolact_amd import heads
    h, w, b, y, up = _inputs(1300, 3001, 600, torch.float32, True)
    y[::4] = -1
    _, lse = heads.class_loss(h, w, y, bias=b)
    full = heads.class_loss_backward(h, w, y, lse, up, bias=b)
    for i in range(3):
        leaves = [t.clone().requires_grad_(k == i) for k, t in enumerate((h, w, b))]
        got, = torch.autograd.grad(heads.ClassLoss.apply(*leaves, y, -1, "none"), [leaves[i]], up)
        assert torch.equal(got, full[i])

    def step():
        losses, lse = heads.class_loss(h, w, y, bias=b)
        return [losses, lse, *heads.class_loss_backward(h, w, y, lse, up, bias=b)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for r in range(3):
        h.mul_(3.0)
        w.mul_(0.2)
        up.mul_(2.0 ** -20)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want))
