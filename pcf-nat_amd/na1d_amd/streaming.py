"""Attention of unbounded streams (``na1d_sink_*`` of the C ABI): a causal window of any length behind each token, and a few first
tokens, the sinks, that stay visible for good.  Token t sees token u where ``u <= t`` and (``t - u < win_size`` or ``u < sinks``).

:func:`sink_attention` is a layer over whole sequences, in training or over a prompt.  Where a stream goes on, its keys and values are in
caches (:func:`new_cache`) that hold what can still be seen and never grow: :func:`cache_append` puts a prompt there,
:func:`cache_step` takes the next token or a few, :func:`cache_attend` is a step whose tokens are in the caches already.  A cache has its
rows in 16 bits or, as :class:`Rows4`, in 4.  None of them has forward-mode derivatives or goes through ``torch.func``'s transforms, and calls over caches
are not traced by ``torch.jit.trace``: they raise.

Position p of a stream is in row p of its cache where ``p < sinks``, else in row ``sinks + (p - sinks) % (capacity - sinks)``.  ``lengths`` (int32
``[N]``, on the GPU) says how many tokens the streams have seen; one whose entry is negative (or above 2^30) is idle: its rows stay as they
are and its output is 0.  The caches of all layers go with one ``lengths``, which the caller counts up behind the last of them.

Queries may have more heads than keys and values (a multiple: head h goes with key head ``h // (heads // kv_heads)``).  All tensors
are token-major, ``[N, T, heads, head_dim]``, in bfloat16 or float16 on the GPU, head_dim a multiple of 8 up to 128.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _lib

_MAX_ROW = 1 << 20                                   # elements from one token to the next that the native call takes
_LONGEST = 1 << 24


class _Sink(ctypes.Structure):                       # na1d_sink
    _fields_ = ([(n, ctypes.c_int32) for n in "dtype heads kv_heads head_dim".split()] + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_int64) for n in "N T window sinks".split()]
                + [(n, ctypes.c_int64 * 3) for n in ("q_strides", "k_strides", "v_strides")])


class _Cache(ctypes.Structure):                      # na1d_sink_cache
    _fields_ = ([(n, ctypes.c_int32) for n in "dtype bits kv_heads head_dim".split()] + [(n, ctypes.c_int64) for n in "N capacity sinks".split()]
                + [(n, ctypes.c_void_p) for n in "k v k_ranges v_ranges".split()])


class Rows4(NamedTuple):
    """Rows held in 4 bits: ``low + code * step``, 15 steps over the row's range.

    ``codes`` uint8 ``[N, kv_heads, capacity, C // 2]``: byte i of a row has channel 2 i in its low four bits, channel 2 i + 1 in its high
    ones.  ``ranges`` ``[N, kv_heads, capacity, 2]`` in the type of the rows: step, ``(largest - least) / 15`` rounded to that type, and least value.  A code is
    ``(x - least) / step`` in fp32, rounded to the nearest (even of equals) of 0 .. 15; 0 where the step is.  C is 32, 64, 96 or 128."""
    codes: torch.Tensor
    ranges: torch.Tensor


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


def _nodes(win_size, sinks):
    """The native path, where what it is given are numbers that it takes as they are."""
    return _lib.nodes() if type(win_size) is type(sinks) is int and 0 < win_size < 1 << 40 and 0 <= sinks < 1 << 40 else None


def _written(*caches):
    for c in caches:
        for t in c if isinstance(c, Rows4) else (c,):
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)


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


def saved_bytes(q):
    """na1d_sink_saved_bytes of a call on ``q``, in arithmetic that symbolic sizes go through too."""
    N, T, H, C = q.shape
    wide = next(w for w in (16, 32, 64, 96, 128) if C <= w)
    return 16 * ((N * H * T + 3) // 4) + N * H * ((T + 15) // 16) * 16 * wide


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
    """Every call goes through it, one without gradients too: forward-mode derivatives and transforms are refused by it, and a tracer sees it."""
    @staticmethod
    def forward(ctx, q, k, v, t_valid, win_size, sinks, scale, grad):
        want = grad and any(ctx.needs_input_grad)
        out, saved = sink_forward(q, k, v, t_valid, win_size, sinks, scale, want)
        if want:
            ctx.save_for_backward(q, k, v, t_valid, out, saved)
            ctx.args = (win_size, sinks, scale)
        return out

    @staticmethod
    def backward(ctx, dout):
        tensors = ctx.saved_tensors
        with torch.no_grad():
            grads = sink_backward(dout, *tensors, *ctx.args)
        return tuple(_final(g) if want else None for g, want in zip(grads, ctx.needs_input_grad)) + (None,) * 5


def sink_attention(q, k, v, win_size, sinks=0, t_valid=None, scale=None):
    """``softmax(q k^T * scale) v`` over the tokens that each token sees: the ``win_size`` newest ones, itself among them, and the first ``sinks``.

    q ``[N, T, heads, C]``, k and v ``[N, T, kv_heads, C]``, which may be views of one projection's output (any strides that are
    multiples of 8 with contiguous channels; others are packed first).  ``t_valid`` int32 ``[N]``: tokens from there on do not exist; they
    may hold anything, and their outputs and gradients are 0.  The tokens before have to be finite.  ``scale`` (above 0,
    up to 2.3e38) defaults to ``C ** -0.5``.  Returns ``[N, T, heads, C]``.  The gradients cannot be differentiated again (asking for it raises).
    """
    nodes = _nodes(win_size, sinks)
    out = None if nodes is None else nodes.sink(q, k, v, win_size, sinks, t_valid, scale)
    if out is not None:
        return out
    check_operands(q, k, v, t_valid)
    _check_gpu(q)
    win_size, sinks = _window(win_size, sinks)
    scale = _scale(scale, q.shape[3])
    return _SinkAttention.apply(q, k, v, t_valid, win_size, sinks, scale, torch.is_grad_enabled() or torch.jit.is_tracing())


# ------------------------------------------------------------------------------------------------ caches
def new_cache(batch, kv_heads, capacity, head_dim, bits=16, dtype=torch.bfloat16, device="cuda"):
    """A pair of caches, for keys and for values, of ``capacity`` rows to a head: a window of ``win_size`` with ``sinks`` takes
    ``sinks + win_size``, and one more for every token more than one that a step has.  ``bits``: 16, or 4 (:class:`Rows4`)."""
    _lib.dtype_tag(dtype)
    if bits == 16:
        return tuple(torch.zeros(batch, kv_heads, capacity, head_dim, dtype=dtype, device=device) for _ in "kv")
    if bits != 4 or head_dim not in (32, 64, 96, 128):
        raise _lib.NA1DError("bits must be 16, or 4 with a head_dim of 32, 64, 96 or 128; got %r and %r" % (bits, head_dim))
    return tuple(Rows4(torch.zeros(batch, kv_heads, capacity, head_dim // 2, dtype=torch.uint8, device=device),
                       torch.zeros(batch, kv_heads, capacity, 2, dtype=dtype, device=device)) for _ in "kv")


def _check_untraced():
    if torch.jit.is_tracing():
        raise _lib.NA1DError("calls over a cache cannot be traced: a trace would not hold what they write to it and read from it")


def _has_tangent(t):
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None


def check_tangents(*tensors):
    if any(_has_tangent(t) for t in tensors):
        raise _lib.NA1DError("sink_attention has no forward-mode derivative")


def _check_cache(cache, what):
    """Shape of the rows that a cache stands for and their type; its memory has to be as the native call takes it, since it is written to."""
    if isinstance(cache, Rows4):
        codes, ranges = cache
        if codes.dim() != 4 or codes.dtype != torch.uint8 or ranges.shape != codes.shape[:3] + (2,):
            raise ValueError("%s must have codes uint8 [N, kv_heads, capacity, C / 2] and ranges [N, kv_heads, capacity, 2], got %s %s and %s" % (
                what, codes.dtype, list(codes.shape), list(ranges.shape)))
        if codes.shape[3] not in (16, 32, 48, 64):
            raise _lib.NA1DError("a cache in 4 bits has a head_dim of 32, 64, 96 or 128, got %d" % (2 * codes.shape[3]))
        if codes.device != ranges.device:
            raise _lib.NA1DError("codes and ranges of %s must be on one device" % what)
        shape, dtype = codes.shape[:3] + (2 * codes.shape[3],), ranges.dtype
    else:
        if cache.dim() != 4:
            raise ValueError("%s must be [N, kv_heads, capacity, C], got %s" % (what, list(cache.shape)))
        shape, dtype = cache.shape, cache.dtype
    _lib.dtype_tag(dtype)
    for t in cache if isinstance(cache, Rows4) else (cache,):
        if not t.is_contiguous() or (t.numel() and not t.is_meta and t.data_ptr() % 16):
            raise _lib.NA1DError("%s must be contiguous and 16-byte aligned" % what)
        if t.requires_grad or _has_tangent(t):
            raise _lib.NA1DError("%s is written to without a gradient: it must not require one" % what)
    return tuple(shape), dtype


def _device(cache):
    return cache[0].device if isinstance(cache, Rows4) else cache.device


def _parts(k_cache, v_cache):
    """Codes or rows of both, and their ranges (None: rows in 16 bits)."""
    k, v = (c if isinstance(c, Rows4) else (c, None) for c in (k_cache, v_cache))
    return k[0], v[0], k[1], v[1]


def _check_caches(k_cache, v_cache, sinks):
    (shape, dtype), other = _check_cache(k_cache, "k_cache"), _check_cache(v_cache, "v_cache")
    if (shape, dtype) != other or isinstance(k_cache, Rows4) != isinstance(v_cache, Rows4):
        raise ValueError("k_cache and v_cache must be alike, got %s %s and %s %s" % ((list(shape), dtype) + (list(other[0]), other[1])))
    if _device(k_cache) != _device(v_cache):
        raise _lib.NA1DError("k_cache and v_cache must be on one device")
    if shape[1] == 0 or shape[3] % 8 or not 0 < shape[3] <= 128:
        raise _lib.NA1DError("a cache has at least one head, and a head_dim that is a multiple of 8 up to 128, got %s" % list(shape))
    if not sinks < shape[2]:
        raise _lib.NA1DError("a cache of %d rows has no room behind %d sinks" % (shape[2], sinks))
    return shape, dtype


def _check_apart(k_cache, v_cache, *read):
    """What a call writes to shares no memory with what it reads or writes besides."""
    def extent(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
    there = [extent(t) for t in _parts(k_cache, v_cache) if t is not None and t.numel() and not t.is_meta]
    rest = there + [extent(t) for t in read if t.numel() and not t.is_meta]
    for i, (a, b) in enumerate(there):
        if any(a < d and c < b for c, d in rest[i + 1:]):
            raise _lib.NA1DError("k_cache and v_cache are written to: they must not share memory with each other or with q, k and v")


def _check_tokens(t, shape, dtype, device, heads, what):
    N, K, _, C = shape
    if t.dim() != 4 or t.shape[0] != N or t.shape[3] != C or (t.shape[2] != K if heads == "kv_heads" else t.shape[2] == 0 or t.shape[2] % K):
        raise ValueError("%s must be [%d, tokens, %s, %d] with the caches' %d kv_heads, got %s" % (what, N, heads, C, K, list(t.shape)))
    if t.dtype != dtype:
        raise TypeError("%s must have the caches' dtype, got %s and %s" % (what, t.dtype, dtype))
    if t.device != device:
        raise _lib.NA1DError("%s must be on the device of the caches" % what)


def _check_room(shape, window, sinks, fresh):
    if window > shape[2] - sinks - max(fresh - 1, 0):
        raise _lib.NA1DError("a cache of %d rows is too small for %d sinks, a window of %d and %d tokens at a time: that takes %d" % (
            shape[2], sinks, window, fresh, sinks + window + max(fresh - 1, 0)))


def _cache(k_cache, v_cache, shape, dtype, sinks):
    four = isinstance(k_cache, Rows4)
    N, K, S, C = shape
    pointers = (k_cache.codes, v_cache.codes, k_cache.ranges, v_cache.ranges) if four else (k_cache, v_cache, None, None)
    return _Cache(_lib.dtype_tag(dtype), 4 if four else 16, K, C, N, S, sinks, *(_lib._p(t) for t in pointers))


def cache_append(k, v, k_cache, v_cache, lengths=None, sinks=0, t_valid=None):
    """Tokens ``k, v [N, T, kv_heads, C]`` become positions ``lengths[n]`` and following of their streams (``lengths`` None: from 0 on).

    ``t_valid`` int32 ``[N]``: only so many of a stream's tokens are there.  What a later token cannot see is not kept: of the tokens behind the
    sinks the last ``capacity - sinks`` are.  The caches are written to in place (they share no memory with each other or with the tokens), and nothing is
    returned; no gradient goes through them."""
    nodes = _nodes(1, sinks)
    if nodes is not None and nodes.sink_append(k, v, *_parts(k_cache, v_cache), lengths, sinks, t_valid):
        return
    _check_untraced()
    _, sinks = _window(1, sinks)
    shape, dtype = _check_caches(k_cache, v_cache, sinks)
    device = _device(k_cache)
    _check_tokens(k, shape, dtype, device, "kv_heads", "k")
    _check_tokens(v, shape, dtype, device, "kv_heads", "v")
    if k.shape[1] != v.shape[1]:
        raise ValueError("k and v must have equally many tokens, got %d and %d" % (k.shape[1], v.shape[1]))
    check_lengths(lengths, k, "lengths")
    check_lengths(t_valid, k, "t_valid")
    _check_apart(k_cache, v_cache, k, v)
    _check_gpu(k)
    k, v = _rows(k.detach()), _rows(v.detach())
    lengths, t_valid = (None if t is None else t.contiguous() for t in (lengths, t_valid))
    c = _cache(k_cache, v_cache, shape, dtype, sinks)
    with torch.cuda.device(device):
        _lib.check(_lib.load().na1d_sink_append(ctypes.byref(c), _lib._p(k), _lib._p(v), _strides(k), _strides(v), _lib._p(lengths), _lib._p(t_valid), k.shape[1],
                                                _lib._stream(k)), "na1d_sink_append")
    _written(k_cache, v_cache)


def _over_cache(q, k, v, k_cache, v_cache, lengths, win_size, sinks, scale):
    nodes = None if lengths is None else _nodes(win_size, sinks)
    out = None if nodes is None else nodes.sink_over(q, k, v, *_parts(k_cache, v_cache), lengths, win_size, sinks, scale)
    if out is not None:
        return out
    _check_untraced()
    win_size, sinks = _window(win_size, sinks)
    shape, dtype = _check_caches(k_cache, v_cache, sinks)
    device = _device(k_cache)
    _check_tokens(q, shape, dtype, device, "heads", "q")
    for t, what in ((k, "k"), (v, "v")) if k is not None else ():
        _check_tokens(t, shape, dtype, device, "kv_heads", what)
        if t.shape[1] != q.shape[1]:
            raise ValueError("%s must have as many tokens as q, got %d and %d" % (what, t.shape[1], q.shape[1]))
    if k is not None:
        _check_apart(k_cache, v_cache, q, k, v)
    if lengths is None:
        raise ValueError("lengths must be int32 [%d]" % shape[0])
    check_lengths(lengths, q, "lengths")
    _check_room(shape, win_size, sinks, q.shape[1])
    if any(t is not None and (torch.is_grad_enabled() and t.requires_grad or _has_tangent(t)) for t in (q, k, v)):
        raise _lib.NA1DError("attention over a cache has no gradient: call it under torch.no_grad(), or sink_attention")
    _check_gpu(q)
    scale = _scale(scale, shape[3])
    q, k, v = (None if t is None else _rows(t) for t in (q, k, v))
    lengths = lengths.contiguous()
    fresh, heads = q.shape[1], q.shape[2]
    out = torch.empty(q.shape, dtype=dtype, device=device)
    c = _cache(k_cache, v_cache, shape, dtype, sinks)
    lib = _lib.load()
    nbytes = lib.na1d_sink_attend_workspace_bytes(ctypes.byref(c), fresh, heads, win_size)
    _lib.check(int(min(nbytes, 0)), "na1d_sink_attend_workspace_bytes")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    with torch.cuda.device(device):
        tail = (_lib._p(lengths), fresh, heads, win_size, scale, _lib._p(ws), nbytes, _lib._stream(q))
        if k is None:
            _lib.check(lib.na1d_sink_attend(ctypes.byref(c), _lib._p(out), _lib._p(q), _strides(q), *tail), "na1d_sink_attend")
        else:
            _lib.check(lib.na1d_sink_step(ctypes.byref(c), _lib._p(out), _lib._p(q), _lib._p(k), _lib._p(v), _strides(q), _strides(k), _strides(v), *tail),
                       "na1d_sink_step")
            _written(k_cache, v_cache)
    return out


def cache_step(q, k, v, k_cache, v_cache, lengths, win_size, sinks=0, scale=None):
    """The next tokens of each stream, ``q [N, fresh, heads, C]``, ``k, v [N, fresh, kv_heads, C]``: they are put into the caches at positions ``lengths[n]``
    and following, and attend to what each of them sees, as the caches hold it.  Returns ``[N, fresh, heads, C]``.

    ``capacity - sinks >= win_size + fresh - 1``.  ``lengths`` stays as it is: the caller adds ``fresh``.  The rows have to be finite.  There is no gradient."""
    if k is None or v is None:
        raise ValueError("cache_step takes k and v; tokens that are in the caches already go through cache_attend")
    return _over_cache(q, k, v, k_cache, v_cache, lengths, win_size, sinks, scale)


def cache_attend(q, k_cache, v_cache, lengths, win_size, sinks=0, scale=None):
    """:func:`cache_step` for tokens that :func:`cache_append` has put into the caches: ``q`` has the last ``fresh`` of the ``lengths[n]`` tokens (the
    output of one that would lie before position 0 is 0)."""
    return _over_cache(q, None, None, k_cache, v_cache, lengths, win_size, sinks, scale)


def cache_rows(cache):
    """What the rows of a cache stand for, ``[N, kv_heads, capacity, C]``: a new tensor for :class:`Rows4`, a 16-bit cache itself.

    Where a step was rounded up its last code may stand for more than the type's largest number: that number then."""
    nodes = _lib.nodes() if isinstance(cache, Rows4) else None
    out = None if nodes is None else nodes.sink_rows(*cache)
    if out is not None:
        return out
    if isinstance(cache, Rows4):
        _check_untraced()
    shape, dtype = _check_cache(cache, "cache")
    if not isinstance(cache, Rows4):
        return cache
    _check_gpu(cache.codes)
    out = torch.empty(shape, dtype=dtype, device=cache.codes.device)
    with torch.cuda.device(out.device):
        _lib.check(_lib.load().na1d_sink_rows(_lib._p(out), _lib._p(cache.codes), _lib._p(cache.ranges), shape[0] * shape[1] * shape[2], shape[3],
                                              _lib.dtype_tag(dtype), _lib._stream(out)), "na1d_sink_rows")
    return out
