"""Prediction-head operators without a GPU: the 64-bit references themselves, sizes of workspaces, refusals at the C ABI
and in Python."""
import ctypes
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from yolact_amd import _lib, heads

import heads_precision as precision
import heads_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = ctypes.c_void_p(4096)      # a non-null, aligned address that is never read: every call below is refused first


def test_philox_known_answer():
    """The published test vector of Philox4x32-10 for an all-zero key and counter, and a counter past 32 bits."""
    assert [hex(v) for v in ref.philox(0, 0, 1)[0]] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    a, b = ref.philox(7, (1 << 32) - 2, 100), ref.philox(7, 1 << 32, 4)
    assert np.array_equal(a[2:6], b)


def test_class_loss_reference_against_autograd_and_differences():
    g = torch.Generator().manual_seed(3)
    h, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((7, 5), (11, 5), (11,)))
    y = torch.tensor([0, 3, -1, 10, 3, -1, 7])
    up = torch.rand(7, generator=g, dtype=torch.float64)
    leaves = [t.clone().requires_grad_() for t in (h, w, b)]
    loss = torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].t() + leaves[2], y, ignore_index=-1, reduction="none")
    want = torch.autograd.grad((loss * up).sum(), leaves)
    ref.HALF[torch.float64] = 0.0
    try:
        got = ref.class_loss(h, w, b, y, up)
        def total(hh, ww, bb):
            r = ref.class_loss(hh, ww, bb, y, None)["losses"][0]
            return float((r * up).sum())
        for name, a, t, i in (("grad_h", want[0], h, 0), ("grad_w", want[1], w, 1), ("grad_b", want[2], b, 2)):
            assert torch.allclose(got[name][0], a, rtol=1e-12, atol=1e-14)
            dirn = torch.randn(t.shape, generator=g, dtype=torch.float64)
            args = [h, w, b]
            plus, minus = list(args), list(args)
            plus[i], minus[i] = t + 1e-5 * dirn, t - 1e-5 * dirn
            assert abs((total(*plus) - total(*minus)) / 2e-5 - float((got[name][0] * dirn).sum())) < 1e-8
    finally:
        del ref.HALF[torch.float64]


def test_declared_argument_counts_match_the_header():
    """ctypes passes what the prototypes in _lib.py say: they have to have as many arguments as the header's."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "yolact_post.h")).read(), flags=re.S)
    L = _lib.load()
    for name in ("yp_class_loss", "yp_class_loss_backward", "yp_class_loss_workspace", "yp_quantized_row_bytes",
                 "yp_quantized_linear_workspace", "yp_quantize_rows", "yp_quantized_linear", "yp_dropout"):
        args = re.search(r"\b%s\s*\(([^;]*)\)\s*;" % name, text).group(1)
        assert len(args.split(",")) == len(getattr(L, name).argtypes), name


def _refused(rc, needle):
    assert rc == -1
    assert needle in _lib.load().yp_last_error().decode(), _lib.load().yp_last_error()


@pytest.mark.parametrize("change,needle", [
    (dict(n=-1), "n must"), (dict(n=(1 << 20) + 1), "n must"), (dict(v=0), "v must"), (dict(v=(1 << 24) + 1), "v must"),
    (dict(d=0), "d must"), (dict(d=65537), "d must"), (dict(dtype=3), "dtype"), (dict(label_bytes=2), "label_bytes"),
    (dict(features=None), "null"), (dict(weight=None), "null"), (dict(labels=None), "null"), (dict(ws=None), "null"),
    (dict(lse=None), "null"), (dict(losses=ctypes.c_void_p(4097)), "aligned"), (dict(features=ctypes.c_void_p(4097)), "aligned"),
    (dict(bias=ctypes.c_void_p(4097)), "aligned"), (dict(labels=ctypes.c_void_p(4100)), "aligned"),
    (dict(ws=ctypes.c_void_p(4096 + 16)), "256-byte"),
])
def test_class_loss_refuses(change, needle):
    a = dict(n=4, v=9, d=8, dtype=1, features=P, weight=P, bias=None, labels=P, label_bytes=8, ws=P, losses=P, lse=P)
    a.update(change)
    _refused(_lib.load().yp_class_loss(0, a["n"], a["v"], a["d"], a["dtype"], a["features"], a["weight"], a["bias"], a["labels"],
                                       a["label_bytes"], -1, a["ws"], a["losses"], a["lse"], None, None, None, None), needle)


@pytest.mark.parametrize("change,needle", [
    (dict(n=-1), "n must"), (dict(dtype=9), "dtype"), (dict(lse=None), "null"), (dict(grad=None), "null"), (dict(stride=2), "grad_stride"),
    (dict(gh=None, gw=None), "null"), (dict(gb=P), "grad_bias"),
    (dict(gw=ctypes.c_void_p(4097)), "aligned"), (dict(count=ctypes.c_void_p(4098)), "aligned"), (dict(ws=ctypes.c_void_p(4097)), "256-byte"),
])
def test_class_loss_backward_refuses(change, needle):
    a = dict(n=4, v=9, d=8, dtype=0, bias=None, lse=P, grad=P, stride=1, count=None, ws=P, gh=P, gw=P, gb=None)
    a.update(change)
    _refused(_lib.load().yp_class_loss_backward(0, a["n"], a["v"], a["d"], a["dtype"], P, P, a["bias"], P, 8, -1, a["lse"], a["grad"], a["stride"],
                                                a["count"], a["ws"], a["gh"], a["gw"], a["gb"], None), needle)


def test_class_loss_backward_of_no_rows_needs_no_gradient_pointer():
    """The gradient of features that have no row is an empty tensor, whose address is null."""
    L = _lib.load()
    for bias in (None, P):
        assert L.yp_class_loss_backward(0, 0, 9, 8, 0, None, P, bias, None, 8, -1, None, None, 1, None, None, None, None, None, None) == 0


@pytest.mark.parametrize("change,needle", [
    (dict(rows=-1), "rows"), (dict(k=0), "k must"), (dict(k=131073), "k must"), (dict(dtype=4), "dtype"), (dict(out_dtype=3), "out_dtype"),
    (dict(v=0), "v must"), (dict(x=None), "null"), (dict(ws=None), "null"), (dict(dtype=3), "null"), (dict(out=None), "null"),
    (dict(wq=ctypes.c_void_p(4104)), "aligned"), (dict(bias=ctypes.c_void_p(4098)), "aligned"), (dict(ws=ctypes.c_void_p(4096 + 64)), "256-byte"),
    (dict(rows=(1 << 31) - 1, v=1 << 24), "too large"),
])
def test_quantized_linear_refuses(change, needle):
    a = dict(rows=4, v=9, k=8, dtype=0, x=P, xs=None, wq=P, ws_=P, bias=None, ws=P, out=P, out_dtype=0)
    a.update(change)
    _refused(_lib.load().yp_quantized_linear(0, a["rows"], a["v"], a["k"], a["dtype"], a["x"], a["xs"], a["wq"], a["ws_"], a["bias"], a["ws"],
                                             a["out"], a["out_dtype"], None), needle)


def test_quantize_rows_and_dropout_refuse():
    L = _lib.load()
    _refused(L.yp_quantize_rows(0, 4, 0, 0, P, P, P, None), "k must")
    _refused(L.yp_quantize_rows(0, 4, 8, 3, P, P, P, None), "dtype")
    _refused(L.yp_quantize_rows(0, 4, 8, 0, P, ctypes.c_void_p(4100), P, None), "16 bytes")
    _refused(L.yp_quantize_rows(0, 4, 8, 0, None, P, P, None), "null")
    assert L.yp_quantize_rows(0, 0, 8, 0, None, None, None, None) == 0
    for p in (-0.1, 1.1, float("nan")):
        _refused(L.yp_dropout(0, 4, 0, p, P, P, P, None), "p must")
    _refused(L.yp_dropout(0, -1, 0, 0.5, P, P, P, None), "count")
    _refused(L.yp_dropout(0, 4, 3, 0.5, P, P, P, None), "dtype")
    _refused(L.yp_dropout(0, 4, 0, 0.5, None, P, P, None), "null")
    _refused(L.yp_dropout(0, 4, 0, 0.5, ctypes.c_void_p(4100), P, P, None), "aligned")
    _refused(L.yp_dropout(0, 4, 0, 0.5, P, ctypes.c_void_p(4097), P, None), "aligned")
    assert L.yp_dropout(0, 0, 0, 0.5, None, None, None, None) == 0


def test_dropout_refuses_tensors_that_overlap_in_part():
    L = _lib.load()
    for dtype, apart in ((0, 12), (0, -12), (1, 6), (2, -2)):
        _refused(L.yp_dropout(0, 4, dtype, 0.5, P, ctypes.c_void_p(8192), ctypes.c_void_p(8192 + apart), None), "overlap")


def test_workspace_sizes():
    L = _lib.load()
    assert L.yp_quantized_row_bytes(1) == 128 and L.yp_quantized_row_bytes(129) == 256
    assert L.yp_quantized_linear_workspace(3, 256) == 3 * 256 + 3 * 4
    assert L.yp_class_loss_workspace(0, 9, 8, 0, 0, 1) == 0
    # a training step over a large vocabulary holds a small part of the logits
    n, v, d = 8192, 128000, 1024
    assert L.yp_class_loss_workspace(n, v, d, 1, 0, 1) < n * v * 2 / 3
    assert L.yp_class_loss_workspace(n, v, d, 1, 0, 0) < n * v * 2 / 8 + v * d * 2 + n * d * 2
    assert L.yp_class_loss_workspace(4, 9, 8, 7, 0, 0) == -1


def test_python_refuses_what_is_not_on_the_device():
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        heads.class_loss(x, torch.zeros(9, 8), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match=r"\[classes, features\]"):
        heads.class_loss(x, torch.zeros(9), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        heads.quantize_rows(x)
    with pytest.raises(ValueError, match="CUDA"):
        heads.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="quantize_rows"):
        heads.quantized_linear(x, torch.zeros(9, 8))
    with pytest.raises(ValueError, match="reduction"):
        heads.ClassLoss.apply(x, torch.zeros(9, 8), None, torch.zeros(3, dtype=torch.int64), -1, "all")
    with pytest.raises(ValueError, match="state"):
        heads.class_head_loss(x, torch.zeros(9, 8), None, torch.zeros(3, dtype=torch.int64), dropout_p=0.5)


def test_assembly_names_the_registers_it_writes():
    """A register that an asm block writes by name is in its clobber list: the compiler may keep something there."""
    csrc = os.path.join(ROOT, "yolact_amd", "csrc")
    seen = 0
    for name in sorted(os.listdir(csrc)):
        for block in re.findall(r"asm\s+volatile\s*\((.*?)\);", open(os.path.join(csrc, name)).read(), flags=re.S):
            code, *rest = re.split(r"(?<!:):(?!:)|::", block)
            for reg in re.findall(r"\b[sv]_\w+\s+(m0|vcc|exec|scc|[sv]\d+)\b", code):
                seen += 1
                assert f'"{reg}"' in rest[-1], (name, block)
    assert seen > 0


def test_quantized_linear_takes_every_size_that_is_stated():
    """rows v <= 2^37 and v <= 2^24, narrow weights too (refused here for the workspace's alignment, after the sizes)."""
    bad = ctypes.c_void_p(4096 + 64)
    for rows, v, needle in (((1 << 31) - 1, 4, "256-byte"), ((1 << 31) - 1, 64, "256-byte"), ((1 << 31) - 1, 65, "too large"), (1 << 30, 128, "256-byte"),
                            (1 << 13, 1 << 24, "256-byte"), ((1 << 13) + 1, 1 << 24, "too large"), (1 << 13, (1 << 24) + 1, "v must")):
        _refused(_lib.load().yp_quantized_linear(0, rows, v, 8, 0, P, None, P, P, None, bad, P, 0, None), needle)


_PLANS = r"""
#include "gemm_launch.hpp"
#include <cstdio>
int main() {
  long long bad = 0;
  auto see = [&](const char* what, long long wgs, long long i, long long j, long long steps) {
    if (wgs < YP_MAX_WORKGROUPS) return;
    if (bad++ < 5) printf("%s %lld %lld %lld\n", what, i, j, steps);
  };
  for (long long steps : {1, 2, 5, 40, 1024})
    for (long long v = 1; v <= (1 << 24); v += 1 + v / 40) {
      const long long rows = (1ll << 37) / v < 2147483647ll ? (1ll << 37) / v : 2147483647ll, n = (1ll << 38) / v < (1 << 20) ? (1ll << 38) / v : (1 << 20);
      for (long long j : {rows, rows - rows / 40, rows / 2}) see("quantized", yp_plan_workgroups(yp_plan_tiles(v, j, steps, YP_TILE_L)), v, j, steps);
      for (long long j : {n, n - n / 40, n / 2}) if (j > 0) see("loss", yp_plan_workgroups(yp_plan_tiles(v, j, steps, YP_TILE_L)), v, j, steps);
    }
  for (long long d : {1, 64, 4096, 65536})
    for (long long n = 1; n <= (1 << 20); n += 1 + n / 10)
      for (long long piece : {1, 256, 4096, 1 << 17})
        for (int largest : {YP_TILE_L, YP_TILE_M}) {
          yp_tile_plan a = {}, b = {};
          yp_plan_two(d, piece, (n + 31) / 32, d, n, (piece + 31) / 32, largest, &a, &b);
          see("gradients", yp_plan_workgroups(a) + yp_plan_workgroups(b) + (piece + 31) / 32, d, n, piece);
        }
  return bad != 0;
}
"""


def test_plans_fit_a_launch(tmp_path):
    """Every size that the entries take gets a plan whose workgroups one launch can hold (host code only)."""
    src, exe = tmp_path / "plans.hip", tmp_path / "plans"
    src.write_text(_PLANS)
    subprocess.check_call([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-host-only", "-O1", "-std=c++17", "-x", "hip",
                           "-I" + os.path.join(ROOT, "yolact_amd", "csrc"), str(src), "-o", str(exe)])
    run = subprocess.run([str(exe)], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
def test_precision_bounds_tell_one_plane_of_dz_from_two(dt):
    """The gradients as the kernels compute them, in 64 bits but for dz's planes and the result's rounding: two planes are
    within the bounds, one is not."""
    g = torch.Generator().manual_seed(1)
    n, v, d = 200, 333, 64
    h = torch.randn(n, d, generator=g).to(dt)
    w = (torch.randn(v, d, generator=g) * (1.5 / math.sqrt(d))).to(dt)
    y = torch.randint(-1, v, (n,), generator=g)
    up = torch.rand(n, generator=g)
    dz, _, gg = precision.softmax_difference(h, w, None, y, up)
    by = (2.0 ** 13 if dt == torch.float16 else 1.0) / gg.max()
    want = precision.two_planes(h, w, None, y, up)
    for planes in (1, 2):
        first = (dz * by).to(dt).double()
        q = (first + ((dz * by - first).to(dt).double() if planes == 2 else 0.0)) / by
        for name, got in (("grad_h", (q @ w.double()).to(dt)), ("grad_w", (q.t() @ h.double()).to(dt))):
            value, bound = want[name]
            inside = bool(((got.double() - value).abs() <= bound).all())
            near = precision.relative(got, value) <= precision.ROUNDED * ref.HALF[dt]
            assert inside == near == (planes == 2), (planes, name)
