"""Operators of the prediction head, on the device: what trains the class head and what runs it in 8 bits.

* ``class_loss`` / ``class_loss_backward`` / ``ClassLoss`` - softmax cross entropy of features against a class matrix,
  for vocabularies of any size: the logits are never stored (``csrc/class_loss.hip``).  It stands beside the mask part
  of the training loss (``consumer.LossMaskAssembly``).
* ``quantize_rows`` / ``quantized_linear`` - the head's products in 8-bit integers with one scale per row of either
  operand, float32 out as ``Detect`` takes it (``csrc/quantized.hip``); ``QuantizedHeads`` puts the three of them together.
* ``dropout`` / ``Dropout`` - a mask that is computed again instead of stored (``csrc/dropout.hip``);
  ``class_head_loss`` applies it to the features on their way into the class loss.

torch is plumbing (device memory, current stream, autograd); there is no CPU fallback.  Tensors live on one CUDA device,
are contiguous, and results are stream-ordered on torch's current stream of that device.  Workspaces are torch tensors of
the call itself, so calls on different streams or captured graphs share nothing.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_TYPES = {torch.float32: _lib.YP_F32, torch.bfloat16: _lib.YP_BF16, torch.float16: _lib.YP_F16}
_REDUCTIONS = ("none", "sum", "mean")


def _check(name, t, dtypes, shape=None, device=None):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in dtypes and t.is_contiguous() and \
            (shape is None or t.shape == shape) and (device is None or t.device == device):
        return t.data_ptr()
    if not isinstance(t, torch.Tensor) or not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be a CUDA tensor" + (f" on {device}" if device is not None else ""))
    want = " or ".join(str(d) for d in dtypes)
    raise ValueError(f"{name} must be contiguous {want}" + (f" of shape {tuple(shape)}" if shape is not None else "") +
                     f", got {t.dtype} {tuple(t.shape)}")


def _fits(name, *sizes):
    for n in sizes:
        if n > 0x7FFFFFFF:                       # (what the C entries take; a larger one would arrive as another number)
            raise ValueError(f"{name} of {n} is too large")


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)      # (torch.cuda.current_stream makes an object: 1.9 us of 4)


def _workspace(nbytes, device):
    if nbytes < 0:
        _lib.check(int(nbytes))
    return torch.empty((int(nbytes),), dtype=torch.uint8, device=device) if nbytes > 0 else None


def _ptr(t):
    return t.data_ptr() if t is not None else None


# ---- class loss ------------------------------------------------------------------------------------------------------
def _class_loss_args(features, weight, labels, bias):
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be a CUDA tensor [classes, features]")
    V, D = weight.shape
    if not isinstance(features, torch.Tensor) or features.dim() < 1 or features.shape[-1] != D:
        raise ValueError(f"features must be a CUDA tensor [..., {D}]")
    dev, lead = weight.device, features.shape[:-1]
    p_w = _check("weight", weight, _TYPES)
    p_h = _check("features", features, (weight.dtype,), device=dev)
    p_y = _check("labels", labels, (torch.int64, torch.int32), lead, dev)
    p_b = _check("bias", bias, (weight.dtype,), (V,), dev) if bias is not None else None
    _fits("rows, classes or features", labels.numel(), V, D)
    return p_h, p_w, p_b, p_y, labels.numel(), V, D, lead, dev


def _label(ignore_index):
    ignore_index = int(ignore_index)
    if not -1 << 63 <= ignore_index < 1 << 63:
        raise ValueError("ignore_index must fit an int64")
    return ignore_index


def _class_loss_forward(args, label_bytes, type_, ignore_index, p_losses, p_lse, p_sum=None, p_mean=None, p_count=None):
    p_h, p_w, p_b, p_y, N, V, D, _, dev = args
    L = _lib.load()
    ws = _workspace(L.yp_class_loss_workspace(N, V, D, type_, p_b is not None, 0), dev)
    _lib.check(L.yp_class_loss(dev.index, N, V, D, type_, p_h, p_w, p_b, p_y, label_bytes, ignore_index, _ptr(ws),
                               p_losses, p_lse, p_sum, p_mean, p_count, _stream(dev)))


def class_loss(features, weight, labels, bias=None, ignore_index: int = -1):
    """Softmax cross entropy of ``features`` [..., D] against the class matrix ``weight`` [V, D] (and ``bias`` [V]), all of
    one type (float32, bfloat16, float16): returns ``(losses, lse)``, float32 of the shape of ``labels`` [...] (int64 or
    int32), with ``lse = log sum exp`` of the logits and ``losses = lse - logit[label]``.

    A row labelled ``ignore_index`` takes no part (loss 0) whatever its features hold; any other label outside [0, V) has
    loss NaN.  ``lse`` is the logits' own in these rows too.  A class whose bias is -inf takes no part, whatever its weights hold; as a label its loss is +inf.
    Large float32 calls (2^31 multiplications and more) take each value to 2^-22 of itself or 2^-39 of the largest in its row.
    No gradient is recorded here: ``ClassLoss`` is the differentiable form."""
    args = _class_loss_args(features, weight, labels, bias)
    lead, dev = args[-2:]
    losses = torch.empty(lead, dtype=torch.float32, device=dev)
    lse = torch.empty(lead, dtype=torch.float32, device=dev)
    _class_loss_forward(args, labels.element_size(), _TYPES[weight.dtype], _label(ignore_index), losses.data_ptr(), lse.data_ptr())
    return losses, lse


def _class_loss_backward(features, weight, labels, bias, ignore_index, p_lse, p_grad, per_row, p_count, wanted=(True, True, True)):
    """The call itself, on checked tensors; gradients that are not wanted are None."""
    V, D = weight.shape
    N, dev = labels.numel(), weight.device
    L, dt = _lib.load(), _TYPES[weight.dtype]
    ws = _workspace(L.yp_class_loss_workspace(N, V, D, dt, bias is not None, 1), dev)
    gh = torch.empty_like(features) if wanted[0] else None
    gw = torch.empty_like(weight) if wanted[1] else None
    gb = torch.empty_like(bias) if bias is not None and wanted[2] else None
    _lib.check(L.yp_class_loss_backward(dev.index, N, V, D, dt, features.data_ptr(), weight.data_ptr(), _ptr(bias), labels.data_ptr(),
                                        labels.element_size(), ignore_index, p_lse, p_grad, per_row, p_count, _ptr(ws),
                                        _ptr(gh), _ptr(gw), _ptr(gb), _stream(dev)))
    return gh, gw, gb


def class_loss_backward(features, weight, labels, lse, grad_losses, bias=None, ignore_index: int = -1):
    """Gradients of ``class_loss``'s losses: ``(grad_features, grad_weight, grad_bias or None)`` given ``lse`` as the forward
    returned it for the same inputs and ``grad_losses`` (float32, the shape of ``labels``).  The logits are computed again,
    in pieces of the vocabulary; sums run in float32 in a fixed order.  16-bit gradients are rounded twice beyond 512 rows
    and 2^30 multiplications: the logits' gradients to the type, relative to the largest of ``grad_losses``, and the results;
    up to there the first is held twice as precise.  Large float32 calls: as ``class_loss``, the weight's gradient
    to 2^-39 of the largest feature times its row's gradient, the features' to 2^-39 of the largest weight."""
    lead, dev = _class_loss_args(features, weight, labels, bias)[-2:]
    _check("lse", lse, (torch.float32,), lead, dev)
    p_grad = _check("grad_losses", grad_losses, (torch.float32,), lead, dev)
    return _class_loss_backward(features, weight, labels, bias, _label(ignore_index), lse.data_ptr(), p_grad, 1, None)


class ClassLoss(torch.autograd.Function):
    """Differentiable class loss: ``ClassLoss.apply(features, weight, bias, labels, ignore_index=-1, reduction="mean")``.
    ``reduction`` "none" gives the rows' losses, "sum" and "mean" one value, "mean" over the rows that are not ignored (0 if
    there are none).  Gradients flow to features, weight and bias (which may be None); those nobody needs are not computed.
    The three are of one type, under autocast too: cast a master weight of another (``weight.to(features.dtype)``).
    When forward and backward are captured into a graph, capture both, on leaves whose eager graphs are gone."""

    @staticmethod
    def forward(ctx, features, weight, bias, labels, ignore_index=-1, reduction="mean"):
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction must be one of {_REDUCTIONS}")
        features, weight, labels = features.contiguous(), weight.contiguous(), labels.contiguous()
        bias = bias.contiguous() if bias is not None else None
        ignore_index = _label(ignore_index)
        args = _class_loss_args(features, weight, labels, bias)
        N, lead, dev = args[4], args[-2], args[-1]
        kept = torch.empty((N + 1,), dtype=torch.float32, device=dev)          # lse of the rows, and how many count
        p_lse = kept.data_ptr()
        loss = torch.empty(lead if reduction == "none" else (), dtype=torch.float32, device=dev)
        p_loss = loss.data_ptr()
        _class_loss_forward(args, labels.element_size(), _TYPES[weight.dtype], ignore_index, p_loss if reduction == "none" else None, p_lse,
                            p_loss if reduction == "sum" else None, p_loss if reduction == "mean" else None, p_lse + 4 * N)
        ctx.save_for_backward(features, weight, bias, labels, kept)
        ctx.cfg = (ignore_index, reduction)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        features, weight, bias, labels, kept = ctx.saved_tensors
        ignore_index, reduction = ctx.cfg
        grad = grad.contiguous()             # (float32 and of the result's shape: autograd has seen to it)
        p_lse = kept.data_ptr()
        gh, gw, gb = _class_loss_backward(features, weight, labels, bias, ignore_index, p_lse, grad.data_ptr(), int(reduction == "none"),
                                          p_lse + 4 * (kept.shape[0] - 1) if reduction == "mean" else None, ctx.needs_input_grad)
        return gh, gw, gb, None, None, None


# ---- dropout ---------------------------------------------------------------------------------------------------------
def dropout(x, p: float, state, out=None):
    """``x`` (float32, bfloat16, float16, any shape) with every element kept with probability 1 - p, then divided by it, else
    0 (also where x is not finite).  ``state`` is an int64 CUDA tensor [2]: the key and the first counter; element i uses
    word i % 4 of Philox4x32-10 at counter ``state[1] + i // 4``.  The same state gives the same mask - which is how the
    backward pass has it - so advance ``state[1]`` by ``(x.numel() + 3) // 4`` before the next use, and not before the
    backward of this one.  It is read on the device: a captured call follows it on every replay.  ``out`` may be x, but not
    overlap it otherwise; torch sees it change, as by an operation in place.
    No gradient is recorded here: ``Dropout`` is the differentiable form."""
    p_x = _check("x", x, _TYPES)
    dev = x.device
    p_s = _check("state", state, (torch.int64,), (2,), dev)
    if not 0.0 <= float(p) <= 1.0:
        raise ValueError("p must be in [0, 1]")
    made = out is None
    if made:
        out = torch.empty_like(x)
    p_o = _check("out", out, (x.dtype,), x.shape, dev)
    _lib.check(_lib.load().yp_dropout(dev.index, x.numel(), _TYPES[x.dtype], float(p), p_s, p_x, p_o, _stream(dev)))
    if not (made or out.is_inference()):
        torch.autograd.graph.increment_version(out)
    return out


class Dropout(torch.autograd.Function):
    """Differentiable dropout: ``Dropout.apply(x, p, state)``.  Only ``state`` is kept for the backward pass, which computes
    the mask again; changing ``state`` in between is an error that torch reports."""

    @staticmethod
    def forward(ctx, x, p, state):
        y = dropout(x.contiguous(), p, state)
        ctx.save_for_backward(state)
        ctx.p = float(p)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        state, = ctx.saved_tensors
        return dropout(grad.contiguous(), ctx.p, state), None, None


def class_head_loss(features, weight, bias, labels, dropout_p: float = 0.0, state=None, ignore_index: int = -1, reduction: str = "mean"):
    """The class head's training step: dropout on the features (``dropout_p`` > 0 needs ``state``), then ``ClassLoss``."""
    if dropout_p:
        if state is None:
            raise ValueError("dropout needs its state")
        features = Dropout.apply(features, dropout_p, state)
    return ClassLoss.apply(features, weight, bias, labels, ignore_index, reduction)


# ---- quantized linear ------------------------------------------------------------------------------------------------
class QuantizedRows:
    """Rows in 8 bits: ``q`` int8 [rows, padded k] (k up to the next multiple of 128, the padding zero), ``scale`` float32
    [rows], ``k``, and the shape ``lead`` that the rows had; row r stands for ``q[r, :k] * scale[r]``.  ``quantize_rows`` makes
    them; so may a caller who has kept ``q`` and ``scale``."""

    def __init__(self, q, scale, k, lead):
        kp = int(_lib.load().yp_quantized_row_bytes(k))
        if kp < 0:
            _lib.check(kp)
        rows = math.prod(lead)
        _check("q", q, (torch.int8,), (rows, kp))
        _check("scale", scale, (torch.float32,), (rows,), q.device)
        self._set(q, scale, k, lead)

    def _set(self, q, scale, k, lead):
        self.q, self.scale, self.k, self.lead = q, scale, int(k), tuple(lead)
        return self

    @property
    def device(self):
        return self.q.device

    def dequantize(self):
        """The values the rows stand for, float32 [..., k]."""
        return (self.q[:, :self.k].float() * self.scale[:, None]).reshape(*self.lead, self.k)


def quantize_rows(x) -> QuantizedRows:
    """``x`` [..., k] (float32, bfloat16, float16) in 8 bits, one scale per row: scale = max|x| / 127, q = x / scale to the
    nearest, ties to even.  A row that holds an infinity or NaN has scale NaN.  k <= 131072."""
    p_x = _check("x", x, _TYPES)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have at least one element per row")
    dev, k, lead = x.device, x.shape[-1], x.shape[:-1]
    rows = x.numel() // k
    _fits("rows or k", rows, k)
    L = _lib.load()
    kp = int(L.yp_quantized_row_bytes(k))
    if kp < 0:
        _lib.check(kp)
    q = torch.empty((rows, kp), dtype=torch.int8, device=dev)
    scale = torch.empty((rows,), dtype=torch.float32, device=dev)
    _lib.check(L.yp_quantize_rows(dev.index, rows, k, _TYPES[x.dtype], p_x, q.data_ptr(), scale.data_ptr(), _stream(dev)))
    return QuantizedRows.__new__(QuantizedRows)._set(q, scale, k, lead)      # (nothing to check)


def quantized_linear(x, weight: QuantizedRows, bias=None, out_dtype=torch.float32):
    """``x @ weight^T + bias`` with 8-bit integer products: ``x`` [..., k] float32 / bfloat16 / float16 (quantized row by row
    on the way) or ``QuantizedRows``; ``weight`` = ``quantize_rows`` of a [v, k] matrix; ``bias`` float32 [v].  Returns
    [..., v] of ``out_dtype``: integer sums are exact, scales and bias are applied in float32, one rounding to the type.
    For answering: no gradient is recorded."""
    if not isinstance(weight, QuantizedRows) or len(weight.lead) != 1 or weight.lead[0] < 1:
        raise ValueError("weight must be quantize_rows of a [v, k] matrix")
    if out_dtype not in _TYPES:
        raise ValueError("out_dtype must be float32, bfloat16 or float16")
    dev, v, k = weight.device, weight.lead[0], weight.k
    L = _lib.load()
    p_b = _check("bias", bias, (torch.float32,), (v,), dev) if bias is not None else None
    ws = None
    if isinstance(x, QuantizedRows):
        if x.k != k or x.device != dev:
            raise ValueError(f"x must hold rows of {k} on {dev}")
        lead, rows, dt, p_x, p_s = x.lead, x.scale.shape[0], _lib.YP_INT8, x.q.data_ptr(), x.scale.data_ptr()
    else:
        p_x, p_s = _check("x", x, _TYPES, device=dev), None
        if x.dim() < 1 or x.shape[-1] != k:
            raise ValueError(f"x must have rows of {k}")
        lead, rows, dt = x.shape[:-1], x.numel() // k, _TYPES[x.dtype]
        _fits("rows", rows)
        ws = _workspace(L.yp_quantized_linear_workspace(rows, k), dev)
    out = torch.empty((*lead, v), dtype=out_dtype, device=dev)
    _lib.check(L.yp_quantized_linear(dev.index, rows, v, k, dt, p_x, p_s, weight.q.data_ptr(), weight.scale.data_ptr(), p_b, _ptr(ws),
                                     out.data_ptr(), _TYPES[out_dtype], _stream(dev)))
    return out


class QuantizedHeads:
    """Three products on the same rows of features in 8 bits: class logits, box offsets and mask coefficients, in the type
    ``Detect`` takes.  Each head is a float weight [out, D], or a pair of it and a float32 bias [out].  With a row of features per
    anchor the shapes are ``Detect``'s.  The reference's last layers (layers/head.py) are convolutions whose channels hold all
    anchors of a place: there a row is a place's unfolded neighbourhood, D its k * k * channels values, a head's
    weight the kernel as [anchors * values, D], and the results are reshaped from [B, places, anchors * values] to
    [B, places * anchors, values]."""

    def __init__(self, cls, offset, mask_coef):
        def keep(h):
            w, b = h if isinstance(h, (tuple, list)) else (h, None)
            return quantize_rows(w), b
        self.heads = {"pred_cls": keep(cls), "pred_offset": keep(offset), "pred_mask_coef": keep(mask_coef)}

    def __call__(self, features):
        """features [..., D] -> {"pred_cls": [..., C], "pred_offset": [..., 4], "pred_mask_coef": [..., K]} float32 (as many
        values as the heads' weights have rows), the features quantized once.  The coefficients are what the product gives: the reference's tanh (layers/head.py:81) is
        the caller's, who may want it in place."""
        x = quantize_rows(features)
        return {name: quantized_linear(x, w, bias=b) for name, (w, b) in self.heads.items()}
