"""The prediction-head operators in 64 bits, with the bounds that their tests allow (plain torch, any device)."""
from __future__ import annotations

import math

import numpy as np
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative: eps / 2
F = 2.0 ** -24


def class_loss(h, w, b, labels, grad, ignore=-1):
    """Definition and error bounds.  h [N,D], w [V,D], b [V] or None, labels [N], grad [N] float64 dL/dloss.
    Returns {name: (value, bound)} for losses, lse, grad_h, grad_w, grad_b.

    Bounds, with u = half a step of the type and F = 2^-24 that of float32: a logit is D products summed in float32 and
    a bias added, |dz| <= (D + 2) F (|h||w| + |b|) =: e, per row the largest over the classes that take part.  exp and
    log of the hardware are taken as 4 F relative, their arguments' roundings as 2 F |argument| <= 2 F * 2 max|z|; a sum
    of V positive terms in any order as V F, in the kernel's (lanes, tiles, joins) as far less, so (64 + V / 64) F.
    So lse is off by e + (4 + 64 + V/64) F + 4 F max|z| + F |lse| and a probability, relatively, by e + lse's error +
    (4 + 4 max|z|) F.  dz = g (p - onehot): g is off by 2 F (a division and a factor), the difference by F, and dz is
    rounded to the type (u; f16: or to the step of its subnormals, 2^-38 of the largest g).  A product of K such terms
    adds K F, its rounding u.
    (Large float32 products run as three products of f16 planes: 3 K sums and 2^-24 more per product at worst, each a third
    of them far smaller than the first; the bound of the direct product is kept for them too.)"""
    dt = h.dtype
    u = HALF[dt]
    N, D = h.shape
    V = w.shape[0]
    h, w = h.double(), w.double()
    bias = b.double() if b is not None else torch.zeros(V, dtype=torch.float64, device=h.device)
    off = bias == -math.inf
    w = torch.where(off[:, None], torch.zeros_like(w), w)
    counted = (labels != ignore) & (labels >= 0) & (labels < V)
    hz = torch.where((labels != ignore)[:, None], h, torch.zeros_like(h))
    z = hz @ w.t() + bias
    fin = torch.where(off, torch.zeros_like(bias), bias)
    e = ((D + 2) * F * (hz.abs() @ w.abs().t() + fin.abs())).amax(dim=1)
    zmax = torch.where(off, torch.zeros_like(z), z).abs().amax(dim=1)
    lse = torch.logsumexp(z, dim=1)
    e_lse = e + (68 + V / 64) * F + 4 * F * zmax + F * torch.where(lse.isinf(), torch.zeros_like(lse), lse).abs()
    at = torch.where(counted, labels, torch.zeros_like(labels)).long()
    picked = z.gather(1, at[:, None])[:, 0]
    losses = torch.where(picked == -math.inf, torch.full_like(lse, math.inf), lse - picked)
    losses = torch.where(counted, losses, torch.where(labels == ignore, torch.zeros_like(lse), torch.full_like(lse, math.nan)))
    e_loss = e_lse + e + F * (lse.abs() + zmax)
    out = {"losses": (losses, torch.where(labels == ignore, torch.zeros_like(e_loss), e_loss)), "lse": (lse, e_lse)}
    if grad is None:
        return out
    g = torch.where(counted, grad.double(), torch.zeros_like(lse))
    p = torch.where((lse == -math.inf)[:, None], torch.zeros_like(z), torch.exp(z - lse[:, None]))
    d = p.clone()
    d[torch.arange(N, device=h.device)[counted], at[counted]] -= 1.0
    d = torch.where(off[None, :], torch.zeros_like(d), d)
    dz = d * g[:, None]
    rel = (e + e_lse + (4 + 4 * zmax) * F)[:, None]
    e32 = g.abs()[:, None] * (p * rel * 1.01 + F * d.abs()) + 2 * F * dz.abs()
    e_dz = e32 + u * (dz.abs() + e32)
    if dt == torch.float16 and N:
        e_dz = e_dz + 2.0 ** -38 * g.abs().max() * (dz != 0)
    tiny = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -133      # half a step of the result's subnormals
    for name, a, m, k in (("grad_h", dz, w, V), ("grad_w", dz.t().contiguous(), hz, N)):
        v = a @ m
        ea = e_dz if name == "grad_h" else e_dz.t().contiguous()
        err = ea @ m.abs() + (k + 4) * F * ((a.abs() + ea) @ m.abs())
        out[name] = (v, err + u * (v.abs() + err) + tiny)
    if b is not None:
        v = dz.sum(dim=0)
        err = e32.sum(dim=0) + (N + 4) * F * (dz.abs() + e32).sum(dim=0)
        out["grad_b"] = (v, err + u * (v.abs() + err) + tiny)
    return out


def class_loss_value(h, w, b, labels, ignore=-1):
    """The rows' losses alone, of 64-bit inputs."""
    z = h @ w.t() + (b if b is not None else 0.0)
    kept = labels != ignore
    picked = z.gather(1, torch.where(kept, labels, torch.zeros_like(labels))[:, None])[:, 0]
    return torch.where(kept, torch.logsumexp(z, dim=1) - picked, torch.zeros_like(picked))


def within(got, value, bound, what):
    got = got.double()
    same = (got == value) | (got.isnan() & value.isnan())
    far = torch.where(same, torch.zeros_like(got), (got - value).abs() - bound)
    bad = ~(far <= 0)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(far[bad].max())} over its bound, " \
                                f"first at {torch.nonzero(bad)[0].tolist()}"


def quantize(x):
    """(q int64, scale float32) of the rows of x, in 64 bits."""
    d = x.double()
    bad = ~torch.isfinite(d).all(dim=1)
    d = torch.where(bad[:, None], torch.zeros_like(d), d)
    scale = (d.abs().amax(dim=1) / 127.0).float()
    s = scale.double()[:, None]
    q = torch.where(s > 0, d / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(d)).round().clamp(-127, 127)
    return q.long(), torch.where(bad, torch.full_like(scale, math.nan), scale)


def quantized_linear(q, sx, wq, sw, b, out_dtype):
    """(value, bound): the integer sum is exact, its conversion, the product with a scale and the fused multiply-add with
    the other round once each in float32, the output type once more."""
    acc = (q.double() @ wq.double().t()) * sx.double()[:, None] * sw.double()[None, :]
    add = b.double() if b is not None else torch.zeros(wq.shape[0], dtype=torch.float64, device=q.device)
    y = acc + add
    err = 3.01 * F * acc.abs() + F * (acc.abs() + add.abs())
    tiny = 2.0 ** -149 if out_dtype != torch.float16 else 2.0 ** -25
    return y, err + (HALF[out_dtype] if out_dtype != torch.float32 else 0.0) * (y.abs() + err) + tiny


def philox(key: int, first: int, blocks: int) -> np.ndarray:
    """Philox4x32-10: [blocks, 4] uint32 of the 64-bit counters first .. first + blocks - 1 (upper 64 bits 0)."""
    c = [int(first) + i for i in range(blocks)] if blocks < 64 else None
    ctr = (np.uint64(first % (1 << 64)) + np.arange(blocks, dtype=np.uint64)) if c is None else np.array([v % (1 << 64) for v in c], dtype=np.uint64)
    lo32, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    c0, c1, c2, c3 = ctr & lo32, ctr >> s32, np.zeros(blocks, np.uint64), np.zeros(blocks, np.uint64)
    k0, k1 = key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = c0 * np.uint64(0xD2511F53), c2 * np.uint64(0xCD9E8D57)
        c0, c1, c2, c3 = (b >> s32) ^ c1 ^ np.uint64(k0), b & lo32, (a >> s32) ^ c3 ^ np.uint64(k1), a & lo32
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([c0, c1, c2, c3], axis=1).astype(np.uint32)


def keep_mask(n: int, p: float, key: int, first: int) -> np.ndarray:
    words = philox(key, first, (n + 3) // 4).reshape(-1)[:n].astype(np.uint64)
    return words >= np.uint64(math.floor(p * 2.0 ** 32))
