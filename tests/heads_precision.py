"""Bounds on the class loss's gradients that tell its precisions apart: tighter than heads_reference's, which allow a rounding
of dz to the type at every size."""
from __future__ import annotations

import math

import torch

import heads_reference as ref

STEP = 2.0 ** -22        # two f16 planes of a float32


def softmax_difference(h, w, b, y, up):
    """(p - onehot) g in 64 bits, the sums of products' absolute values, and g."""
    z = h.double() @ w.double().t()
    if b is not None:
        z = z + b.double()
    d = torch.softmax(z, dim=1)
    kept = y >= 0
    d[torch.arange(len(y), device=y.device)[kept], y[kept]] -= 1.0
    g = torch.where(kept, up, torch.zeros_like(up)).double()
    return d * g[:, None], z, g


def two_planes(h, w, b, y, up):
    """{name: (value, bound)} of grad_h and grad_w where dz has two planes of a 16-bit type: dz is off by u^2 of itself, u half
    a step of the type (the second plane rounds what the first left, which is at most u of it), f16's also by half a step of
    its subnormals, 2^-38 of the largest g.  The rest is as in heads_reference: sums of D, N and V terms in float32, the
    probabilities' error from the logits', one rounding of the result."""
    dt, F = h.dtype, ref.F
    u = ref.HALF[dt]
    dz, z, g = softmax_difference(h, w, b, y, up)
    hd, wd = h.double(), w.double()
    n, v, d = len(y), w.shape[0], h.shape[1]
    size = hd.abs() @ wd.abs().t() + (b.double().abs() if b is not None else 0.0)
    off_z = ((d + 2) * F * size).amax(dim=1, keepdim=True)
    top = z.abs().amax(dim=1, keepdim=True)
    p = torch.softmax(z, dim=1)
    rel = 2 * off_z + (76 + v / 64 + 9 * top) * F
    off = g.abs()[:, None] * p * rel * 1.01 + 3 * F * dz.abs() + u * u * dz.abs()
    if dt == torch.float16:
        off = off + 2.0 ** -38 * g.abs().max()
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -133
    out = {}
    for name, a, m, e, k in (("grad_h", dz, wd, off, v), ("grad_w", dz.t().contiguous(), hd, off.t().contiguous(), n)):
        value = a @ m
        err = e @ m.abs() + (k + 4) * F * ((a.abs() + e) @ m.abs())
        out[name] = (value, err + u * (value.abs() + err) + tiny)
    return out


def rms_of_planes(k):
    """Float32 as two f16 planes, root mean square error of a sum of k products relative to that of its terms, in steps of
    2^-22, where signs are random.  What a plane leaves is at most a step: a third of its square in the mean, for either factor; the
    product of the two second planes, which is left out, is at most a step too, a ninth.  Every 32 terms of each of the three
    products the sum is rounded to float32, a quarter of a step at most, again a third of its square.  A third more allowed."""
    return 4.0 / 3.0 * math.sqrt(7.0 / 9.0 + 3.0 * k / 32.0 / 16.0 / 3.0) * STEP


# Root mean square error of values rounded to a type, in half steps of it: 1 / sqrt 3 where all of them are just above a power
# of two, half of that just below the next, 0.38 to 0.43 for values spread over binades.  dz in one plane adds as much again.
ROUNDED, ROUNDED_TWICE = 0.5, 0.5 * math.sqrt(2.0)


def relative(got, value):
    return float((got.double() - value).norm() / value.norm())
