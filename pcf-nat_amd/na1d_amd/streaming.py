"""Attention of unbounded streams (``na1d_sink_*`` of the C ABI): a causal window of any length behind each token, and a few first
tokens, the sinks, that stay visible for good.  Token t sees token u where ``u <= t`` and (``t - u < win_size`` or ``u < sinks``).

:func:`sink_attention` is a layer over whole sequences, in training or over a prompt.

Queries may have more heads than keys and values (a multiple: head h goes with key head ``h // (heads // kv_heads)``).  All tensors
are token-major, ``[N, T, heads, head_dim]``, in bfloat16 or float16 on the GPU, head_dim a multiple of 8 up to 128.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_MAX_ROW = 1 << 20                                   # elements from one token to the next that the native call takes
_LONGEST = 1 << 24


class _Sink(ctypes.Structure):                       # na1d_sink
    _fields_ = ([(n, ctypes.c_int32) for n in "dtype heads kv_heads head_dim".split()] + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_int64) for n in "N T window sinks".split()]
                + [(n, ctypes.c_int64 * 3) for n in ("q_strides", "k_strides", "v_strides")])


def _rows(t):
    """``t [N, T, heads, C]`` as the native call takes it: channels contiguous, the other strides multiples of 8 within its limits."""
    N, T, H, C = t.shape
    s = t.stride()
    if (s[3] != 1 or (N > 1 and s[0] % 8) or (T > 1 and (s[1] % 8 or not C <= s[1] <= _MAX_ROW)) or (H > 1 and s[2] % 8)
            or min(s) < 0 or max(s[0], s[2]) > 1 << 40):
        t = t.contiguous()
    return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 else t


def _strides(t):
    """{sample, head, row} element strides; those of dimensions of one entry do not matter."""
    N, T, H, C = t.shape
    s = t.stride()
    return (ctypes.c_int64 * 3)(s[0] if N > 1 else 0, s[2] if H > 1 else 0, s[1] if T > 1 else C)


def _window(win_size, sinks):
    if int(win_size) != win_size or int(sinks) != sinks or win_size < 1 or sinks < 0:
        raise _lib.NA1DError("win_size must be an integer of at least 1 and sinks one of at least 0, got %r and %r" % (win_size, sinks))
    return min(int(win_size), 1 << 40), min(int(sinks), 1 << 40)


def _scale(scale, C):
    return float(C ** -0.5 if scale is None else scale)


def check_operands(q, k, v, t_valid=None):
    """What the operator asks of its tensors; the sizes' limits are the native call's."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("q must be [N, T, heads, C] and k, v [N, T, kv_heads, C], got %s, %s and %s" % (list(q.shape), list(k.shape), list(v.shape)))
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError("the heads of q must be a multiple of those of k and v, got %d and %d" % (q.shape[2], k.shape[2]))
    _lib.dtype_tag(q.dtype)
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError("q, k and v must have one dtype, got %s, %s and %s" % (q.dtype, k.dtype, v.dtype))
    if not q.device == k.device == v.device:
        raise _lib.NA1DError("q, k and v must be on one device")
    if q.shape[3] % 8 or not 0 < q.shape[3] <= 128:
        raise _lib.NA1DError("head_dim must be a multiple of 8 up to 128, got %d" % q.shape[3])
    check_lengths(t_valid, q, "t_valid")


def check_lengths(lengths, q, what):
    if lengths is None:
        return
    if lengths.dtype != torch.int32 or lengths.shape != q.shape[:1]:
        raise ValueError("%s must be int32 [%d], got %s %s" % (what, q.shape[0], lengths.dtype, list(lengths.shape)))
    if lengths.device != q.device:
        raise _lib.NA1DError("%s must be on the device of the other operands" % what)


def _check_gpu(q):
    if q.device.type != "cuda":
        raise _lib.NA1DError("NA1D tensors must live on the GPU (got device %s); there is no CPU path" % q.device)


def _sink(q, k, v, win_size, sinks, scale):
    return _Sink(_lib.dtype_tag(q.dtype), q.shape[2], k.shape[2], q.shape[3], scale, q.shape[0], q.shape[1], win_size, sinks,
                 _strides(q), _strides(k), _strides(v))


def _bytes(name, h):
    n = getattr(_lib.load(), name)(ctypes.byref(h))
    _lib.check(int(min(n, 0)), name)
    return n


def sink_forward(q, k, v, t_valid, win_size, sinks, scale, want_saved):
    """Output and what a backward needs (nothing, if it is not wanted).  Arguments as checked by the functions below."""
    q, k, v = _rows(q), _rows(k), _rows(v)
    t_valid = None if t_valid is None else t_valid.contiguous()
    h = _sink(q, k, v, win_size, sinks, scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    nsaved = _bytes("na1d_sink_saved_bytes", h) if want_saved else 0
    saved = torch.empty(nsaved, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().na1d_sink_forward(ctypes.byref(h), _lib._p(out), _lib._p(saved) if want_saved else None, nsaved, _lib._p(q), _lib._p(k), _lib._p(v),
                                                 _lib._p(t_valid), _lib._stream(q)), "na1d_sink_forward")
    return out, saved


def sink_backward(dout, q, k, v, t_valid, out, saved, win_size, sinks, scale):
    """Gradients of q, k and v."""
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    q, k, v = _rows(q), _rows(k), _rows(v)
    t_valid = None if t_valid is None else t_valid.contiguous()
    dout, out = (t.clone() if t.data_ptr() % 16 else t for t in (dout.contiguous(), out.contiguous()))
    h = _sink(q, k, v, win_size, sinks, scale)
    nbytes = _bytes("na1d_sink_backward_workspace_bytes", h)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().na1d_sink_backward(ctypes.byref(h), _lib._p(dq), _lib._p(dk), _lib._p(dv), _lib._p(q), _lib._p(k), _lib._p(v), _lib._p(out),
                                                  _lib._p(dout), _lib._p(saved), saved.numel(), _lib._p(t_valid), _lib._p(ws), nbytes, _lib._stream(q)),
                   "na1d_sink_backward")
    return dq, dk, dv


_AGAIN = "the gradients of na1d_amd's sink_attention cannot be differentiated again"


def _final(grad):
    """A gradient that has none of its own: whoever asks for one is told, also where it is a part of a larger sum."""
    if not torch.is_grad_enabled():
        return grad
    return torch._C._functions.DelayedError(_AGAIN.encode(), 1)(grad.requires_grad_(True))


class _SinkAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, t_valid, win_size, sinks, scale):
        out, saved = sink_forward(q, k, v, t_valid, win_size, sinks, scale, True)
        ctx.save_for_backward(q, k, v, t_valid, out, saved)
        ctx.args = (win_size, sinks, scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        tensors = ctx.saved_tensors
        with torch.no_grad():
            grads = sink_backward(dout, *tensors, *ctx.args)
        return tuple(_final(g) if want else None for g, want in zip(grads, ctx.needs_input_grad)) + (None,) * 4


def sink_attention(q, k, v, win_size, sinks=0, t_valid=None, scale=None):
    """``softmax(q k^T * scale) v`` over the tokens that each token sees: the ``win_size`` newest ones, itself among them, and the first ``sinks``.

    q ``[N, T, heads, C]``, k and v ``[N, T, kv_heads, C]``, which may be views of one projection's output (any strides that are
    multiples of 8 with contiguous channels; others are packed first).  ``t_valid`` int32 ``[N]``: tokens from there on do not exist; they
    may hold anything, and their outputs and gradients are 0.  The tokens before have to be finite.  ``scale`` (finite and above
    0) defaults to ``C ** -0.5``.  Returns ``[N, T, heads, C]``.  The gradients cannot be differentiated again (asking for it raises).
    """
    check_operands(q, k, v, t_valid)
    _check_gpu(q)
    win_size, sinks = _window(win_size, sinks)
    scale = _scale(scale, q.shape[3])
    nodes = _lib.nodes()
    if nodes is not None and hasattr(nodes, "sink"):
        out = nodes.sink(q, k, v, t_valid, win_size, sinks, scale)
        if out is not None:
            return out
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _SinkAttention.apply(q, k, v, t_valid, win_size, sinks, scale)
    return sink_forward(q, k, v, t_valid, win_size, sinks, scale, False)[0]
