"""Losses over a large number of classes without the logits in memory (``na1d_head_*`` of the C ABI): what stands behind a speaker
model's embeddings in training, and the same for the vocabulary of a language model.

:func:`linear_cross_entropy` is softmax cross entropy of ``x @ weight.t()``, :func:`margin_cross_entropy` the additive angular margin
of models/SoftMaxLoss.py:99-138 with its sub-centres, :func:`linear_distillation` the divergence from a teacher of which the
largest logits are kept.  The ``[rows, classes]`` logits are never whole in memory: the forward keeps a sum of exponentials to a row,
the backward works the logits out again, a range of classes at a time.

All take ``x [..., D]`` and ``weight`` in bfloat16 or float16 on the GPU, D a multiple of 8, and give fp32 losses and
gradients in the types of x and weight (fp16: scale the loss as ever).  Rows may lie apart (any stride that is a multiple of 8
elements, a class's rows together up to 2^20 of them); what is laid out otherwise is packed first.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}
_TARGETS, _MARGIN, _TEACHER = range(3)
MAX_TOP = 256                                        # NA1D_HEAD_MAX_TOP
_MAX_STRIDE = 1 << 20                                # elements from one row, or from one class's rows to the next, that the native call takes
_FP32 = 2
_IDS = (torch.int32, torch.int64)


class _Head(ctypes.Structure):                       # na1d_head
    _fields_ = ([(n, ctypes.c_int32) for n in "dtype kind reduction subcenters top teacher_type ids_64".split()]
                + [(n, ctypes.c_float) for n in ("scale", "margin")]
                + [(n, ctypes.c_int64) for n in "ignore_index N V D x_stride w_stride".split()])


def _rows(t, to_class=1):
    """``t [..., D]`` as rows, ``to_class`` of them to a class: their number apart, contiguous and 16-byte aligned."""
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 or (t.shape[0] > 1 and (t.stride(0) % 8 or not t.shape[1] <= t.stride(0) <= _MAX_STRIDE // to_class)):
        t = t.contiguous()
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _head(x, weight, ids, teacher, kind, scale, margin, ignore_index, reduction):
    return _Head(_lib.dtype_tag(x.dtype), kind, reduction, weight.shape[1] if weight.dim() == 3 else 1,
                 0 if teacher is None else teacher.shape[-1],
                 0 if teacher is None else _FP32 if teacher.dtype == torch.float32 else _lib.dtype_tag(teacher.dtype),
                 int(ids.dtype == torch.int64), scale, margin, ignore_index, x[..., 0].numel(), weight.shape[0], x.shape[-1], 0, 0)


def _sizes(h, backward):
    lib, ref = _lib.load(), ctypes.byref(h)
    saved, ws = lib.na1d_head_saved_bytes(ref), lib.na1d_head_workspace_bytes(ref, backward)
    _lib.check(int(min(saved, ws, 0)), "na1d_head_workspace_bytes")
    return saved, ws


def head_forward(x, weight, ids, teacher, hits, kind, scale, margin, ignore_index, reduction):
    """Loss, and what the backward needs of the forward; `hits` (bool, a value to a row, or None) is written to.  Arguments as checked
    by the functions below."""
    shape = x.shape[:-1] if reduction == 0 else ()
    loss = torch.empty(shape, dtype=torch.float32, device=x.device)
    if x.numel() == 0:
        if hits is not None:
            hits.zero_()
        return loss.zero_(), torch.empty(0, dtype=torch.uint8, device=x.device)
    h = _head(x, weight, ids, teacher, kind, scale, margin, ignore_index, reduction)
    xr, wr, ids = _rows(x), _rows(weight, h.subcenters), ids.contiguous()
    teacher = None if teacher is None else teacher.contiguous()
    h.x_stride, h.w_stride = _stride(xr), _stride(wr)
    nsaved, nws = _sizes(h, 0)
    saved, ws = (torch.empty(n, dtype=torch.uint8, device=x.device) for n in (nsaved, nws))
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().na1d_head_forward(ctypes.byref(h), _lib._p(loss), _lib._p(hits), _lib._p(xr), _lib._p(wr), _lib._p(ids),
                                                 _lib._p(teacher), _lib._p(saved), nsaved, _lib._p(ws), nws, _lib._stream(x)), "na1d_head_forward")
    return loss, saved


def head_backward(dloss, x, weight, ids, teacher, saved, kind, scale, margin, ignore_index, reduction, want_x, want_weight):
    """Gradients of x and weight (an empty tensor for one that is not wanted)."""
    dx = torch.empty(x.shape if want_x else (0,), dtype=x.dtype, device=x.device)
    dw = torch.empty(weight.shape if want_weight else (0,), dtype=weight.dtype, device=x.device)
    if x.numel() == 0:
        return dx.zero_(), dw.zero_()
    h = _head(x, weight, ids, teacher, kind, scale, margin, ignore_index, reduction)
    xr, wr, ids, dloss = _rows(x), _rows(weight, h.subcenters), ids.contiguous(), dloss.contiguous()
    h.x_stride, h.w_stride = _stride(xr), _stride(wr)
    _, nws = _sizes(h, 1)
    ws = torch.empty(nws, dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().na1d_head_backward(ctypes.byref(h), _lib._p(dx) if want_x else None, _lib._p(dw) if want_weight else None,
                                                  _lib._p(dloss), _lib._p(xr), _lib._p(wr), _lib._p(ids), _lib._p(saved), saved.numel(),
                                                  _lib._p(ws), nws, _lib._stream(x)), "na1d_head_backward")
    return dx, dw


_AGAIN = "the gradients of na1d_amd's losses cannot be differentiated again"


def _final(grad):
    """A gradient that has none of its own: whoever asks for one is told, also where it is a part of a larger sum."""
    if grad is None or not torch.is_grad_enabled():
        return grad
    return torch._C._functions.DelayedError(_AGAIN.encode(), 1)(grad.requires_grad_(True))


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, ids, teacher, hits, *args):
        loss, saved = head_forward(x, weight, ids, teacher, hits, *args)
        ctx.save_for_backward(x, weight, ids, teacher, saved)
        ctx.args = args
        return loss

    @staticmethod
    def backward(ctx, dloss):
        x, weight, ids, teacher, saved = ctx.saved_tensors
        want = ctx.needs_input_grad[:2]
        with torch.no_grad():
            dx, dw = head_backward(dloss, x, weight, ids, teacher, saved, *ctx.args, *want)
        return (_final(dx if want[0] else None), _final(dw if want[1] else None)) + (None,) * 8


def _loss(x, weight, ids, teacher, return_hits, *args):
    nodes = _lib.nodes()
    hits = torch.empty(x.shape[:-1], dtype=torch.bool, device=x.device) if return_hits else None
    out = None if nodes is None else nodes.head(x, weight, ids, teacher, hits, *args)
    if out is None:
        out = _HeadLoss.apply(x, weight, ids, teacher, hits, *args)
    return (out, hits) if return_hits else out


def check_operands(x, weight, ids, ids_shape, weight_dims=(2,), what="target"):
    """What the losses and the registered ops ask of their tensors; the sizes' limits are the native call's."""
    if x.dim() < 1 or weight.dim() not in weight_dims or x.shape[-1] != weight.shape[-1]:
        raise ValueError("x must be [..., D] and weight %s, got %s and %s" % (
            " or ".join("[V, K, D]" if d == 3 else "[V, D]" for d in weight_dims), list(x.shape), list(weight.shape)))
    if ids.shape != ids_shape:
        raise ValueError("%s must be %s, got %s" % (what, list(ids_shape), list(ids.shape)))
    if ids.dtype not in _IDS:
        raise TypeError("%s must be int32 or int64, got %s" % (what, ids.dtype))
    _lib.dtype_tag(x.dtype)
    if x.dtype != weight.dtype:
        raise TypeError("x and weight must have one dtype, got %s and %s" % (x.dtype, weight.dtype))
    if x.device != weight.device or x.device != ids.device:
        raise _lib.NA1DError("x, weight and %s must be on one device" % what)
    if x.shape[-1] % 8 or x.shape[-1] == 0:
        raise _lib.NA1DError("the last dimension must be a positive multiple of 8, got %d" % x.shape[-1])
    if weight.numel() == 0:
        raise _lib.NA1DError("weight must have at least one class")


def check_arguments(x, weight, ids, reduction, ids_shape, weight_dims=(2,), what="target"):
    if reduction not in _REDUCTIONS:
        raise ValueError("reduction must be one of %s, got %r" % (", ".join(_REDUCTIONS), reduction))
    check_operands(x, weight, ids, ids_shape, weight_dims, what)
    if x.device.type != "cuda":
        raise _lib.NA1DError("NA1D tensors must live on the GPU (got device %s); there is no CPU path" % x.device)


def check_entries(x, teacher_logits, teacher_ids):
    if teacher_logits.shape != teacher_ids.shape or teacher_logits.dim() < 1 or not 0 < teacher_logits.shape[-1] <= MAX_TOP:
        raise ValueError("teacher_logits must be like teacher_ids, with 1 to %d entries to a row; got %s" % (MAX_TOP, list(teacher_logits.shape)))
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("teacher_logits must be float32, bfloat16 or float16, got %s" % teacher_logits.dtype)
    if teacher_logits.device != x.device:
        raise _lib.NA1DError("x and teacher_logits must be on one device")


def check_teacher(x, weight, teacher_logits, teacher_ids, reduction):
    check_entries(x, teacher_logits, teacher_ids)
    check_arguments(x, weight, teacher_ids, reduction, x.shape[:-1] + teacher_logits.shape[-1:], what="teacher_ids")


def linear_cross_entropy(x, weight, target, scale=1.0, ignore_index=-100, reduction="mean", return_hits=False):
    """Softmax cross entropy of the logits ``scale * x @ weight.t()``.

    ``x [..., D]``, ``weight [V, D]``, ``target [...]`` (int32 or int64).  Rows whose target is ``ignore_index`` have loss 0 and no
    gradient and do not count in the mean (0 if no row counts); any other target outside ``[0, V)`` makes its row's loss NaN
    and has no gradient.  ``reduction``: "mean", "sum" or "none" (a loss to a row).  The rows themselves have to be finite, ignored
    ones too: they take part in the weight's gradient with a factor of zero.  ``return_hits``: also a bool to a row that says whether
    no class has a larger logit than the target (a row without a target is none).
    """
    check_arguments(x, weight, target, reduction, x.shape[:-1])
    return _loss(x, weight, target, None, return_hits, _TARGETS, float(scale), 0.0, int(ignore_index), _REDUCTIONS[reduction])


def margin_cross_entropy(x, weight, target, margin=0.2, scale=32.0, ignore_index=-100, reduction="mean", return_hits=False):
    """Additive angular margin softmax (models/SoftMaxLoss.py:99-138) on the cosines of ``x [..., D]`` and ``weight [V, D]`` or
    ``[V, K, D]``, where a class's cosine is that of the nearest of its K rows (the lowest of equals).

    The target's cosine cos(theta) becomes cos(theta + margin) where theta + margin < pi, else cos(theta) - margin sin(pi - margin);
    the derivative takes the squared sine of theta as 1e-6 at least.  ``0 <= margin < pi / 2``.  A row of zeros (no longer
    than 1e-12) has cosine 0 with everything and no gradient; one whose squares' sum is beyond fp32 (bfloat16, 1.8e19 and longer)
    has none, and what depends on it is NaN.  Hits are by the cosines, without the margin.  Other arguments as in
    :func:`linear_cross_entropy`.
    """
    check_arguments(x, weight, target, reduction, x.shape[:-1], weight_dims=(2, 3))
    return _loss(x, weight, target, None, return_hits, _MARGIN, float(scale), float(margin), int(ignore_index), _REDUCTIONS[reduction])


def linear_distillation(x, weight, teacher_logits, teacher_ids, temperature=1.0, reduction="mean"):
    """Divergence of the student's softmax over all classes, ``p = softmax(x @ weight.t() / temperature)``, from a teacher of which
    each row has the largest logits: ``temperature^2 * sum over the entries of q (log q - log p[id])`` with
    ``q = softmax(teacher_logits / temperature)`` over the row's entries.

    ``teacher_logits [..., top]`` (bfloat16, float16 or float32; no gradient goes there), ``teacher_ids [..., top]`` (int32 or int64),
    ``top`` up to 256.  Entries with an id below 0 are not there, nor are those with a logit of -inf; a row without any has loss 0
    and no gradient and does not count in the mean (0 if no row counts).  An id of V or more makes its row's loss NaN, without a
    gradient.  A class that is there twice has both entries' shares.
    """
    check_teacher(x, weight, teacher_logits, teacher_ids, reduction)
    return _loss(x, weight, teacher_ids, teacher_logits.detach(), False, _TEACHER, float(temperature), 0.0, 0, _REDUCTIONS[reduction])
