"""Losses over many classes without a GPU: the oracle against torch, and what the entry points refuse."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from na1d_amd import _lib, losses, models
from oracle import losses_oracle as O


def _inputs(N=17, D=24, V=31, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(N, D, generator=g, dtype=torch.float64), torch.randn(V, D, generator=g, dtype=torch.float64) * 0.3,
            torch.randint(0, V, (N,), generator=g))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_oracle_cross_entropy_is_torchs(reduction):
    x, w, t = _inputs()
    t[3] = t[9] = -100
    x.requires_grad_(True), w.requires_grad_(True)
    want = F.cross_entropy(1.7 * x @ w.t(), t, reduction=reduction)
    rows, ok, e = O.softmax_targets(x.detach(), w.detach(), t, 1.7)
    assert torch.allclose(O.reduced(rows, ok, reduction), want.detach(), atol=1e-12)
    up = torch.rand(17, dtype=torch.float64) if reduction == "none" else torch.tensor(0.7, dtype=torch.float64)
    dx, dw = torch.autograd.grad(want, [x, w], up)
    gx, gw, _ = O.linear_gradients(x.detach(), w.detach(), e, O.shares(ok, reduction, up))
    assert torch.allclose(gx, dx, atol=1e-12) and torch.allclose(gw, dw, atol=1e-12)


@pytest.mark.parametrize("subs", [1, 3])
def test_oracle_margin_is_the_models_head(subs):
    x, w, t = _inputs(V=31 * subs)
    t = t // subs
    head = models.ArcMarginSubCenters(24, 31, m=0.2, s=32.0, subcenters=subs).double()
    with torch.no_grad():
        head.W.copy_(w.view(31, subs, 24))
        x[2] = -3 * w.view(31, subs, 24)[t[2], 0] + 0.01 * x[2]          # past the margin's end (with one centre)
        x[5] += 4 * w.view(31, subs, 24)[t[5], 0]
    x.requires_grad_(True)
    want, _ = head(x, t)
    dx, dw = torch.autograd.grad(want, [x, head.W])
    rows, ok, e, _ = O.margin(x.detach(), head.W.detach(), t)
    assert torch.allclose(O.reduced(rows, ok, "mean"), want.detach(), atol=1e-10)
    gx, gw, _ = O.margin_gradients(x.detach(), head.W.detach(), e, O.shares(ok, "mean", 1.0))
    assert torch.allclose(gx, dx, atol=1e-10) and torch.allclose(gw.view_as(dw), dw, atol=1e-10)


def test_oracle_teacher_is_torchs_divergence():
    x, w, t = _inputs()
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(17, 4, generator=g, dtype=torch.float64)
    ids = torch.stack([torch.randperm(31, generator=g)[:4] for _ in range(17)])
    x.requires_grad_(True), w.requires_grad_(True)
    T = 2.5
    dense = torch.full((17, 31), -torch.inf, dtype=torch.float64).scatter_(1, ids, logits)
    q = torch.softmax(dense / T, 1)
    want = T * T * F.kl_div(F.log_softmax(x @ w.t() / T, 1), q, reduction="batchmean")
    rows, ok, e = O.teacher(x.detach(), w.detach(), logits, ids, T)
    assert torch.allclose(O.reduced(rows, ok, "mean"), want.detach(), atol=1e-12)
    gx, gw, _ = O.linear_gradients(x.detach(), w.detach(), e, O.shares(ok, "mean", 1.0))
    dx, dw = torch.autograd.grad(want, [x, w])
    assert torch.allclose(gx, dx, atol=1e-12) and torch.allclose(gw, dw, atol=1e-12)
    # absent entries, and one class twice is the sum of its shares
    ids[0], ids[1, 2:] = -1, -3
    ids[2, 1] = ids[2, 0]
    rows, ok, e = O.teacher(x.detach(), w.detach(), logits, ids, T)
    assert not ok[0] and rows[0] == 0 and not e[0].any()
    q = torch.softmax(logits[2] / T, 0)
    assert math.isclose(float(e[2, ids[2, 0]]), T * float(torch.softmax(x[2].detach() @ w.detach().t() / T, 0)[ids[2, 0]] - q[0] - q[1]), abs_tol=1e-12)


def _head(**kw):
    h = losses._Head(dtype=0, kind=0, reduction=1, subcenters=1, top=0, teacher_type=0, ids_64=1, scale=1.0, margin=0.0,
                     ignore_index=-100, N=4, V=100, D=64, x_stride=64, w_stride=64)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


@pytest.mark.parametrize("status,change", [
    (-2, {"dtype": 2}), (-2, {"kind": 2, "top": 4, "teacher_type": 3}), (-5, {"kind": 3}), (-5, {"reduction": 3}), (-5, {"N": 0}), (-5, {"V": 0}),
    (-3, {"D": 60}), (-3, {"D": 0}), (-5, {"x_stride": 56}), (-6, {"w_stride": 68}), (-11, {"scale": 0.0}), (-11, {"scale": math.nan}),
    (-11, {"scale": math.inf}), (-11, {"kind": 1, "margin": -0.1}), (-11, {"kind": 1, "margin": 1.6}), (-11, {"kind": 1, "margin": math.nan}),
    (-8, {"subcenters": 2}), (-8, {"kind": 1, "subcenters": 256}), (-5, {"kind": 2, "top": 0}), (-8, {"kind": 2, "top": 257}), (-5, {"subcenters": 0}),
    (-8, {"N": (1 << 20) + 1}), (-8, {"V": (1 << 24) + 1}), (-8, {"N": 1 << 20, "V": (1 << 16) + 1}), (-8, {"x_stride": (1 << 20) + 8}),
    (-8, {"V": 1 << 22, "D": 1 << 16, "x_stride": 1 << 16, "w_stride": 1 << 16}),
], ids=str)
def test_sizes_that_the_native_call_refuses(status, change):
    lib, h = _lib.load(), _head(**change)
    ref, fake = ctypes.byref(h), ctypes.c_void_p(0x1000)
    assert lib.na1d_head_saved_bytes(ref) == status and lib.na1d_head_workspace_bytes(ref, 1) == status
    assert lib.na1d_head_forward(ref, fake, None, fake, fake, fake, fake, fake, 1 << 40, fake, 1 << 40, None) == status
    assert lib.na1d_head_backward(ref, fake, fake, fake, fake, fake, fake, fake, 1 << 40, fake, 1 << 40, None) == status


def test_pointers_and_workspaces_that_the_native_call_refuses():
    lib, h = _lib.load(), _head()
    ref, ok, odd, big = ctypes.byref(h), ctypes.c_void_p(0x1000), ctypes.c_void_p(0x1008), 1 << 40
    saved, ws, back = lib.na1d_head_saved_bytes(ref), lib.na1d_head_workspace_bytes(ref, 0), lib.na1d_head_workspace_bytes(ref, 1)
    assert min(saved, ws, back) > 0
    f = lambda loss, *a: lib.na1d_head_forward(ref, loss, None, *a, None)
    for i in (0, 1, 2, 3, 5):
        a = [ok, ok, ok, ok, None, ok]
        a[i] = None
        assert f(*a, big, ok, big) == -1
    assert f(ok, odd, ok, ok, None, ok, big, ok, big) == -6 and f(ok, ok, ok, ok, None, odd, big, ok, big) == -6
    assert f(ok, ok, ok, ok, None, ok, saved - 1, ok, big) == -10 and f(ok, ok, ok, ok, None, ok, big, ok, ws - 1) == -10
    b = lambda *a: lib.na1d_head_backward(ref, *a, None)
    assert b(ok, ok, None, ok, ok, ok, ok, big, ok, big) == -1 and b(ok, ok, ok, ok, ok, None, ok, big, ok, big) == -1
    assert b(odd, ok, ok, ok, ok, ok, ok, big, ok, big) == -6 and b(ok, odd, ok, ok, ok, ok, ok, big, ok, big) == -6
    assert b(ok, ok, ok, ok, ok, ok, ok, saved - 1, ok, big) == -10 and b(ok, ok, ok, ok, ok, ok, ok, big, ok, back - 1) == -10
    assert b(None, None, ok, ok, ok, ok, ok, big, ok, big) == 0                     # nothing asked for
    teacher = _head(kind=2, top=4)
    assert lib.na1d_head_forward(ctypes.byref(teacher), ok, None, ok, ok, ok, None, ok, big, ok, big, None) == -1


def test_arguments_that_the_functions_refuse():
    x, w, t = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(9, 16, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    ids, logits = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)
    ce, mg, kd = losses.linear_cross_entropy, losses.margin_cross_entropy, losses.linear_distillation
    with pytest.raises(_lib.NA1DError, match="GPU"):
        ce(x, w, t)
    for call, error in ((lambda: ce(x, w, t, reduction="max"), ValueError), (lambda: ce(x, w[:, :8], t), ValueError), (lambda: ce(x, w, t[:3]), ValueError),
                        (lambda: ce(x, w.view(3, 3, 16), t), ValueError), (lambda: mg(x, w.view(1, 3, 3, 16), t), ValueError),
                        (lambda: ce(x, w, t.float()), TypeError), (lambda: ce(x.float(), w.float(), t), TypeError), (lambda: ce(x, w.half(), t), TypeError),
                        (lambda: kd(x, w, logits[:, :2], ids), ValueError), (lambda: kd(x, w, logits.double(), ids), TypeError),
                        (lambda: kd(x, w, logits[:, :0], ids[:, :0]), ValueError), (lambda: kd(x, w, logits.repeat(1, 100), ids.repeat(1, 100)), ValueError),
                        (lambda: kd(x, w, logits[:3], ids[:3]), ValueError)):
        with pytest.raises(error):
            call()
