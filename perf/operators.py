"""Timing cases of the prediction-head operators (yolact_amd.heads) and their plain forms.

Three operators that sit at the two ends of a detector's class head:

class loss        softmax cross entropy of features [N,D] against a class matrix [V,D], logits never kept, with the
                  gradients of features, matrix and bias
quantized linear  y = x W^T + b with W and x as 8-bit integers, one scale per row of W and one per row of x: the head's
                  product when it only answers
dropout           on the features, its mask computed again from a counter in the backward pass

`own = False` computes them from elementary torch operations in 32 bits (64 where 32 lose what matters),
`own = True` calls the package.  `exact` is the operators' definition in 64 bits, written apart from the plain form.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# The class and anchor counts 81 and 19248 and the 256 features are the ones of the 550 x 550 configuration; the
# other sizes are generic.
LARGEST_FLOPS = 6.0 * 4096 * 4096 * 128000


def listed():
    return [
        # the positives of one image against the 81 classes: the smallest training call, latency counts
        dict(name="loss_positives", op="loss", mode="mean", n=100, v=81, d=256, dtype="f32", bias=True, ignored=0.0),
        # every anchor of an image, most of them neutral (ignored)
        dict(name="loss_anchors", op="loss", mode="mean", n=19248, v=81, d=256, dtype="bf16", bias=True, ignored=0.75),
        # a class matrix of ordinary vocabulary size
        dict(name="loss_vocab", op="loss", mode="mean", n=8192, v=32000, d=2048, dtype="bf16", bias=False, ignored=0.1),
        # the largest: wide features, large vocabulary
        dict(name="loss_vocab_large", op="loss", mode="mean", n=4096, v=128000, d=4096, dtype="bf16", bias=False, ignored=0.0),
        # odd and ragged in every size, a weight for every row's loss
        dict(name="loss_ragged", op="loss", mode="rows", n=1537, v=30011, d=1000, dtype="f16", bias=True, ignored=0.3),
        # full precision training
        dict(name="loss_full", op="loss", mode="mean", n=2048, v=8192, d=1024, dtype="f32", bias=True, ignored=0.1),
        # scoring a handful of rows, forward only: one pass over the class matrix
        dict(name="loss_score", op="loss", mode="score", n=5, v=50021, d=1024, dtype="bf16", bias=False, ignored=0.0),
        # one row against a large matrix: reading the matrix is all there is
        dict(name="int8_single", op="int8", n=1, v=32000, k=4096, dtype="bf16", out="f32", bias=True),
        # the class head over all anchors of four images, float32 out as Detect takes it
        dict(name="int8_anchors", op="int8", n=76992, v=81, k=256, dtype="f32", out="f32", bias=True),
        # many rows against a large matrix
        dict(name="int8_large", op="int8", n=8192, v=16384, k=4096, dtype="bf16", out="bf16", bias=False),
        # dropout on the positives' features, and on a large batch of them
        dict(name="dropout_positives", op="dropout", n=100, d=256, dtype="f32", p=0.1),
        dict(name="dropout_large", op="dropout", n=16389, d=4096, dtype="bf16", p=0.25),
    ]


def _spread(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]; now and then a multiple of 64, mostly odd sizes."""
    x = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if x >= 128 and rng.random() < 0.4:
        x = x // 64 * 64
    return max(lo, min(hi, x))


def draw(rng):
    op = rng.choice(["loss", "loss", "loss", "int8", "int8", "dropout"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "dropout":
        d = _spread(rng, 32, 4096)
        n = _spread(rng, 1, max(2, 67000000 // d))
        return dict(op=op, n=n, d=d, dtype=dtype, p=rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]))
    if op == "int8":
        k, v = _spread(rng, 32, 4096), _spread(rng, 4, 32000)
        n = _spread(rng, 1, 77000)
        while float(n) * v * k > 8192.0 * 16384 * 4096 or n * v > 1 << 28:
            n = n // 2
        return dict(op=op, n=max(n, 1), v=v, k=k, dtype=dtype, out=rng.choice(["f32", "f32", "bf16", "f16"]),
                    bias=rng.random() < 0.5)
    mode = rng.choice(["mean", "mean", "rows", "score"])
    d, v = _spread(rng, 32, 4096), _spread(rng, 2, 128000)
    n = _spread(rng, 1, 20000)
    while 6.0 * n * v * d > (LARGEST_FLOPS if dtype != "f32" else LARGEST_FLOPS / 16) or n * v > 1 << 29:
        n = n // 2
    return dict(op=op, mode=mode, n=max(n, 1), v=v, d=d, dtype=dtype, bias=rng.random() < 0.5,
                ignored=rng.choice([0.0, 0.1, 0.5]))


def _inputs(case, seed):
    """The inputs proper, from the seed alone, as a program holds them: tensors on the GPU."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 17)
    dt = DTYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if case["op"] == "dropout":
        state = torch.randint(0, 1 << 62, (2,), generator=g, device="cuda", dtype=torch.int64)
        return dict(x=rnd(case["n"], case["d"]).to(dt), grad=rnd(case["n"], case["d"]).to(dt), state=state)
    if case["op"] == "int8":
        # features with a few strong channels, a class matrix of the usual initialisation
        x = rnd(case["n"], case["k"]) * (1.0 + 4.0 * (torch.rand(case["k"], generator=g, device="cuda") < 0.02))
        w = rnd(case["v"], case["k"]) / math.sqrt(case["k"])
        b = rnd(case["v"]) if case["bias"] else None
        return dict(x=x.to(dt), w=w.to(dt), b=b)
    n, v, d = case["n"], case["v"], case["d"]
    h = rnd(n, d).to(dt)
    w = rnd(v, d)
    w *= 1.5 / math.sqrt(d)
    w = w.to(dt)
    b = (0.5 * rnd(v)).to(dt) if case["bias"] else None
    # low classes far more frequent than high ones, as words and object classes are
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    labels = torch.clamp((torch.exp(u * math.log(v + 1.0)) - 1.0).long(), 0, v - 1)
    labels[torch.rand(n, generator=g, device="cuda") < case["ignored"]] = -1
    grad = torch.rand(n, generator=g, device="cuda") / n if case["mode"] == "rows" else None
    return dict(h=h, w=w, b=b, labels=labels, grad=grad)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] == "int8":
        # a program that answers keeps its class matrix in 8 bits
        if own:
            from yolact_amd import heads
            state["wq"] = heads.quantize_rows(state["w"])
        else:
            q, s = _plain_quantize(state["w"])
            state["wq"] = (q.to(torch.int8), s)
        del state["w"]
    elif case["op"] == "loss" and case["mode"] != "score":
        for k in ("h", "w", "b"):
            if state[k] is not None:
                state[k].requires_grad_()
    elif case["op"] == "dropout":
        state["x"].requires_grad_()
    return state


def run(state):
    case = state["case"]
    if case["op"] == "loss":
        return _own_loss(case, state) if own else _plain_loss(case, state)
    if case["op"] == "int8":
        return _own_int8(case, state) if own else _plain_int8(case, state)
    return _own_dropout(case, state) if own else _plain_dropout(case, state)


# ---- the package's calls --------------------------------------------------------------------------------------------
def _own_loss(case, s):
    from yolact_amd import heads
    if case["mode"] == "score":
        losses, lse = heads.class_loss(s["h"], s["w"], s["labels"], bias=s["b"])
        return {"losses": losses, "lse": lse}
    reduction = "mean" if case["mode"] == "mean" else "none"
    loss = heads.ClassLoss.apply(s["h"], s["w"], s["b"], s["labels"], -1, reduction)
    leaves = [s["h"], s["w"]] + ([s["b"]] if s["b"] is not None else [])
    grads = torch.autograd.grad(loss, leaves, s["grad"])
    out = {"loss": loss.detach(), "grad_h": grads[0], "grad_w": grads[1]}
    if s["b"] is not None:
        out["grad_b"] = grads[2]
    return out


def _own_int8(case, s):
    from yolact_amd import heads
    return {"y": heads.quantized_linear(s["x"], s["wq"], bias=s["b"], out_dtype=DTYPES[case["out"]])}


def _own_dropout(case, s):
    from yolact_amd import heads
    y = heads.Dropout.apply(s["x"], case["p"], s["state"])
    gx, = torch.autograd.grad(y, [s["x"]], s["grad"])
    return {"y": y.detach(), "grad_x": gx}


# ---- plain forms ----------------------------------------------------------------------------------------------------
@torch.no_grad()
def _plain_loss(case, s):
    h, w = s["h"].float(), s["w"].float()
    labels = s["labels"]
    valid = labels >= 0
    at = labels.clamp(min=0)[:, None]
    logits = h @ w.t()
    if s["b"] is not None:
        logits += s["b"].float()
    top = logits.max(dim=1, keepdim=True).values
    picked = logits.gather(1, at)
    e = logits.sub_(top).exp_()
    total = e.sum(dim=1, keepdim=True)
    lse = top + total.log()
    losses = torch.where(valid, (lse - picked)[:, 0], torch.zeros_like(lse[:, 0]))
    if case["mode"] == "score":
        return {"losses": losses, "lse": lse[:, 0].contiguous()}
    if case["mode"] == "mean":
        count = valid.sum().clamp(min=1).float()
        loss = losses.sum() / count
        g = valid.float() / count
    else:
        loss = losses
        g = torch.where(valid, s["grad"], torch.zeros_like(s["grad"]))
    d = e.div_(total)
    d.scatter_add_(1, at, torch.full_like(picked, -1.0))
    d.mul_(g[:, None])
    dt = s["h"].dtype
    out = {"loss": loss, "grad_h": (d @ w).to(dt), "grad_w": (d.t() @ h).to(dt)}
    if s["b"] is not None:
        out["grad_b"] = d.sum(dim=0).to(dt)
    return out


def _plain_quantize(x):
    """Rows as whole numbers of [-127, 127] and a scale: scale = max|x| / 127, q = x / scale to the nearest, ties to
    even.  In 64 bits, where no quotient of two 32-bit numbers comes to lie on the wrong side of a half."""
    x = x.double()
    scale = (x.abs().amax(dim=1) / 127.0).float()
    s = scale.double()[:, None]
    q = torch.where(s > 0, x / s, torch.zeros_like(x)).round().clamp(-127, 127)
    return q.float(), scale


@torch.no_grad()
def _plain_int8(case, s):
    q, sx = _plain_quantize(s["x"])
    wq, sw = s["wq"]
    y = q @ wq.float().t()
    y = y * sx[:, None] * sw
    if s["b"] is not None:
        y = y + s["b"]
    return {"y": y.to(DTYPES[case["out"]])}


def _plain_philox(state, blocks, device):
    """Philox 4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011) of the counters
    state[1] + 0 .. blocks-1 under the key state[0]: int64 [blocks, 4], each word in [0, 2^32)."""
    mask = 0xFFFFFFFF
    c = torch.arange(blocks, device=device, dtype=torch.int64) + state[1]
    c0, c1 = c & mask, (c >> 32) & mask
    c2, c3 = torch.zeros_like(c), torch.zeros_like(c)
    k0, k1 = state[0] & mask, (state[0] >> 32) & mask
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # (the low 64 bits of the products: all there are)
        c0, c1, c2, c3 = ((p1 >> 32) & mask) ^ c1 ^ k0, p1 & mask, ((p0 >> 32) & mask) ^ c3 ^ k1, p0 & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([c0, c1, c2, c3], dim=1)


@torch.no_grad()
def _plain_dropout(case, s):
    x, grad = s["x"], s["grad"]
    n = x.numel()
    words = _plain_philox(s["state"], (n + 3) // 4, x.device).reshape(-1)[:n].reshape(x.shape)
    keep = words >= math.floor(case["p"] * 4294967296.0)
    factor = 1.0 / (1.0 - case["p"])
    zero = torch.zeros((), device=x.device)
    return {"y": torch.where(keep, x.float() * factor, zero).to(x.dtype),
            "grad_x": torch.where(keep, grad.float() * factor, zero).to(x.dtype)}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    b = BYTES[case["dtype"]]
    n = case["n"]
    if case["op"] == "dropout":
        return {"bytes": 4.0 * n * case["d"] * b + 16, "flops": 2.0 * n * case["d"]}
    if case["op"] == "int8":
        v, k = case["v"], case["k"]
        return {"bytes": float(n) * k * b + float(v) * k + 4.0 * v + (4.0 * v if case["bias"] else 0.0)
                + float(n) * v * BYTES[case["out"]], "flops": 2.0 * n * v * k}
    v, d = case["v"], case["d"]
    read = (float(n) + v) * d * b + 8.0 * n + (v * b if case["bias"] else 0.0)
    if case["mode"] == "score":
        return {"bytes": read + 8.0 * n, "flops": 2.0 * n * v * d}
    rows = 8.0 * n if case["mode"] == "rows" else 4.0
    return {"bytes": read + (float(n) + v) * d * b + (v * b if case["bias"] else 0.0) + rows, "flops": 6.0 * n * v * d}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s = _inputs(case, seed)
    return {"loss": _exact_loss, "int8": _exact_int8, "dropout": _exact_dropout}[case["op"]](case, s)


def _exact_loss(case, s):
    """Row block by row block: log_softmax's definition and the chain rule."""
    n, v = case["n"], case["v"]
    w = s["w"].double()
    b = s["b"].double() if s["b"] is not None else torch.zeros(v, dtype=torch.float64, device="cuda")
    counted = s["labels"] != -1
    if case["mode"] == "rows":
        up = s["grad"].double() * counted
    else:
        up = counted.double() / max(int(counted.sum()), 1)
    losses = torch.zeros(n, dtype=torch.float64, device="cuda")
    lses = torch.zeros(n, dtype=torch.float64, device="cuda")
    train = case["mode"] != "score"
    if train:
        gh = torch.empty(n, case["d"], dtype=torch.float64, device="cuda")
        gw = torch.zeros_like(w)
        gb = torch.zeros_like(b)
    step = max(1, min(n, (1 << 27) // v))
    for i in range(0, n, step):
        h = s["h"][i:i + step].double()
        z = torch.addmm(b, h, w.t())
        lse = torch.logsumexp(z, dim=1)
        lses[i:i + step] = lse
        rows = torch.nonzero(counted[i:i + step])[:, 0]
        cols = s["labels"][i:i + step][rows]
        losses[i + rows] = lse[rows] - z[rows, cols]
        if train:
            prob = torch.exp(z - lse[:, None])
            prob[rows, cols] -= 1.0
            prob *= up[i:i + step, None]
            gh[i:i + step] = prob @ w
            gw += prob.t().contiguous() @ h
            gb += prob.sum(dim=0)
    if not train:
        return {"losses": losses, "lse": lses}
    out = {"loss": losses if case["mode"] == "rows" else losses.sum() / max(int(counted.sum()), 1), "grad_h": gh, "grad_w": gw}
    if s["b"] is not None:
        out["grad_b"] = gb
    return out


def _exact_int8(case, s):
    def whole(t):
        t = t.to(torch.float64)
        step = t.abs().max(dim=1, keepdim=True)[0].div(torch.full((1, 1), 127.0, dtype=torch.float64, device=t.device))
        step = step.to(torch.float32).to(torch.float64)          # the scale is a 32-bit number by definition
        safe = torch.where(step == 0, torch.ones_like(step), step)
        return torch.clip(torch.round(t / safe), -127.0, 127.0), step
    w, sw = whole(s["w"])
    y = torch.empty(case["n"], case["v"], dtype=torch.float64, device="cuda")
    block = max(1, (1 << 26) // max(case["v"], case["k"]))
    for i in range(0, case["n"], block):
        q, sx = whole(s["x"][i:i + block])
        y[i:i + block] = (q @ w.t()) * sx * sw.t()
    if s["b"] is not None:
        y += s["b"].double()
    return {"y": y}


def _exact_dropout(case, s):
    """The counter-based generator in unsigned whole numbers on the host."""
    import numpy as np
    n = case["n"] * case["d"]
    if n > 1 << 27:
        return None
    key, first = (int(t) for t in s["state"].cpu())
    c = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(first)
    word = lambda t: (t & np.uint64(0xFFFFFFFF)).astype(np.uint32)
    x = [word(c), word(c >> np.uint64(32)), np.zeros(c.shape, np.uint32), np.zeros(c.shape, np.uint32)]
    k = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    for r in range(10):
        a = x[0].astype(np.uint64) * np.uint64(0xD2511F53)
        m = x[2].astype(np.uint64) * np.uint64(0xCD9E8D57)
        x = [word(m >> np.uint64(32)) ^ x[1] ^ np.uint32(k[0]), word(m), word(a >> np.uint64(32)) ^ x[3] ^ np.uint32(k[1]), word(a)]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    r = np.stack(x, axis=1).reshape(-1)[:n]
    keep = torch.from_numpy(r >= np.uint32(math.floor(case["p"] * 2.0 ** 32))).to("cuda").reshape(case["n"], case["d"])
    scale = 1.0 / (1.0 - case["p"])
    return {"y": s["x"].double() * scale * keep, "grad_x": s["grad"].double() * scale * keep}
