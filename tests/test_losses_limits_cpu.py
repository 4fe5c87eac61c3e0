"""What the losses over many classes ask for and refuse at the ends of their range, without a GPU."""
import ctypes
import random

import pytest
import torch

from na1d_amd import _lib, losses, ops


def _head(**kw):
    h = losses._Head(dtype=0, kind=0, reduction=1, subcenters=1, top=0, teacher_type=0, ids_64=1, scale=1.0, margin=0.0,
                     ignore_index=-100, N=4, V=100, D=64, x_stride=64, w_stride=64)
    for k, v in kw.items():
        setattr(h, k, v)
    h.x_stride = h.w_stride = h.D
    return h


def _most(N, D, K):
    """512 MB, or 1.25 GB from 2^19 rows (times sub-centres) on, dx in fp32, and 256 classes' weight rows in fp32 where rows come in batches."""
    return (5 << 28 if N * K > 1 << 19 else 1 << 29) + 4 * N * D + (1024 * K * D if N * K > 1 << 21 else 0)


@pytest.mark.parametrize("N,V,K,D", [
    (65536, 131072, 1, 1024), (131072, 262144, 1, 512), (262144, 262144, 1, 512), (65536, 128256, 1, 4096), (131072, 128256, 1, 4096), (131072, 65536, 1, 1024),
    (1 << 14, 1 << 22, 4, 8), (1 << 15, 1 << 21, 8, 8), (1 << 16, 1 << 20, 16, 8), (1 << 20, 1 << 16, 1, 8), (1 << 20, 65536, 200, 64), (1 << 20, 65536, 255, 64),
    (1 << 20, 65793, 255, 4112)])
def test_a_backwards_workspace_does_not_grow_with_the_classes(N, V, K, D):
    h = _head(N=N, V=min(V, (1 << 36) // N), subcenters=K, kind=int(K > 1), D=D)
    nbytes = _lib.load().na1d_head_workspace_bytes(ctypes.byref(h), 1)
    assert 0 < nbytes <= _most(N, D, K)


def test_a_backwards_workspace_of_any_size():
    rng, lib, taken = random.Random(0), _lib.load(), 0
    for _ in range(400):
        kind = rng.randrange(3)
        K = int(2 ** rng.uniform(0, 8)) if kind == 1 else 1
        N, V, D = int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 24)), 8 * int(2 ** rng.uniform(0, 10))
        nbytes = lib.na1d_head_workspace_bytes(ctypes.byref(_head(kind=kind, N=N, V=V, D=D, subcenters=K, top=9, dtype=rng.randrange(2))), 1)
        assert nbytes == _lib.UNSUPPORTED or 0 < nbytes <= _most(N, D, K), (kind, N, V, D, K)
        taken += nbytes > 0
    assert taken > 200


def _on_meta(N=5, D=16, V=30, dtype=torch.bfloat16):
    return (torch.empty(N, D, dtype=dtype, device="meta"), torch.empty(V, D, dtype=dtype, device="meta"), torch.empty(N, dtype=torch.int64, device="meta"))


def test_a_second_derivative_of_the_op_is_refused():
    """Also where a gradient is a part of a larger loss, which would be differentiated without it."""
    x, w, target = _on_meta()
    x.requires_grad_(True), w.requires_grad_(True)
    for wanted in ([x], [w], [x, w]):
        loss, _ = torch.ops.na_cuda.class_loss_forward(x, w, target, None, 0, 1.0, 0.0, -100, 1)
        grads = torch.autograd.grad(loss, wanted, torch.empty((), device="meta"), create_graph=True)
        penalty = sum(g.float().square().sum() for g in grads)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(loss + penalty, wanted, torch.empty((), device="meta"))
        loss, _ = torch.ops.na_cuda.class_loss_forward(x, w, target, None, 0, 1.0, 0.0, -100, 1)
        assert [g.shape for g in torch.autograd.grad(loss, wanted, torch.empty((), device="meta"))] == [t.shape for t in wanted]


def test_arguments_that_the_ops_refuse():
    """Called by themselves they check what the losses check: the kernels read as many rows and ids as x and the sizes say."""
    x, w, target = _on_meta()
    ids, logits = torch.empty(5, 3, dtype=torch.int64, device="meta"), torch.empty(5, 3, device="meta")
    f, b = torch.ops.na_cuda.class_loss_forward, torch.ops.na_cuda.class_loss_backward
    rest = (1.0, 0.0, -100)
    loss, saved = f(x, w, target, None, 0, *rest, 0)
    assert loss.shape == (5,) and saved.numel() > 0
    mean, _ = f(x, w, ids, logits, 2, *rest, 1)
    assert mean.shape == ()
    for call in (lambda: f(x, w, target[:4], None, 0, *rest, 1), lambda: f(x, w, ids, None, 0, *rest, 1), lambda: f(x, w, target.float(), None, 0, *rest, 1),
                 lambda: f(x, w[:, :8], target, None, 0, *rest, 1), lambda: f(x, w.half(), target, None, 0, *rest, 1), lambda: f(x.float(), w.float(), target, None, 0, *rest, 1),
                 lambda: f(x, w.view(10, 3, 16), target, None, 0, *rest, 1), lambda: f(x, w, target, None, 3, *rest, 1), lambda: f(x, w, target, None, 0, *rest, 3),
                 lambda: f(x, w, target, logits, 0, *rest, 1), lambda: f(x, w, target, None, 2, *rest, 1), lambda: f(x, w, ids[:4], logits[:4], 2, *rest, 1),
                 lambda: f(x, w, ids, logits[:, :2], 2, *rest, 1), lambda: f(x, w, ids, logits.double(), 2, *rest, 1),
                 lambda: f(x, w[:0], target, None, 0, *rest, 1),
                 lambda: b(loss[:4], x, w, target, None, saved, 0, *rest, 0, True, True), lambda: b(loss, x, w, target, None, saved, 0, *rest, 1, True, True),
                 lambda: b(loss.double(), x, w, target, None, saved, 0, *rest, 0, True, True), lambda: b(loss, x, w, target[:4], None, saved, 0, *rest, 0, True, True),
                 lambda: b(loss, x, w, target, None, saved.float(), 0, *rest, 0, True, True), lambda: b(loss, x, w, target, None, saved[::2], 0, *rest, 0, True, True)):
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()
    assert [g.shape for g in b(loss, x, w, target, None, saved, 0, *rest, 0, True, False)] == [(5, 16), (0,)]


@pytest.mark.parametrize("kind,scale,fine", [(0, 2.9e38, False), (1, 2.9e38, False), (0, 1.9e38, True), (2, 1e-23, False), (2, 2e19, False), (2, 1e-18, True), (2, 1e18, True)])
def test_scales_that_fp32_cannot_work_with(kind, scale, fine):
    """The kernels work with scale * log2(e), and with a temperature's reciprocal and square: each has to be a number."""
    ref = ctypes.byref(_head(kind=kind, scale=scale, top=3))
    for nbytes in (_lib.load().na1d_head_saved_bytes(ref), _lib.load().na1d_head_workspace_bytes(ref, 1)):
        assert nbytes > 0 if fine else nbytes == -11
