"""What the attention of streams asks for and refuses, and its oracle, without a GPU."""
import ctypes

import pytest
import torch

from na1d_amd import _lib, streaming
from oracle import streaming_oracle as O


def _on(device, N=2, T=9, H=4, K=2, C=16, dtype=torch.bfloat16):
    return [torch.empty(N, T, h, C, dtype=dtype, device=device) for h in (H, K, K)]


@pytest.mark.parametrize("change,error", [
    (lambda q, k, v: (q[0], k, v), ValueError), (lambda q, k, v: (q, k[:, :5], v[:, :5]), ValueError), (lambda q, k, v: (q, k, v[:, :, :1]), ValueError),
    (lambda q, k, v: (q[:, :, :3], k, v), ValueError), (lambda q, k, v: (q[..., :8], k, v), ValueError), (lambda q, k, v: (q, k[:, :, :0], v[:, :, :0]), ValueError),
    (lambda q, k, v: (q.half(), k, v), TypeError), (lambda q, k, v: (q.float(), k.float(), v.float()), TypeError),
    (lambda q, k, v: (q[..., :12], k[..., :12], v[..., :12]), _lib.NA1DError), (lambda q, k, v: (q, k, torch.empty(v.shape, dtype=v.dtype)), _lib.NA1DError)])
def test_operands_that_do_not_fit(change, error):
    with pytest.raises(error):
        streaming.sink_attention(*change(*_on("meta")), 4)


@pytest.mark.parametrize("window,sinks", [(0, 0), (-1, 0), (4, -1), (2.5, 0), (4, 0.5)])
def test_windows_that_are_none(window, sinks):
    with pytest.raises(_lib.NA1DError):
        streaming._window(window, sinks)


def test_heads_too_wide_and_lengths_of_another_kind():
    with pytest.raises(_lib.NA1DError, match="head_dim"):
        streaming.sink_attention(*_on("meta", C=136), 4)
    for lengths in (torch.zeros(2), torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="t_valid"):
            streaming.sink_attention(*_on("meta"), 4, t_valid=lengths.to("meta"))
    with pytest.raises(_lib.NA1DError, match="device"):
        streaming.sink_attention(*_on("meta"), 4, t_valid=torch.zeros(2, dtype=torch.int32))


def test_there_is_no_cpu_path():
    with pytest.raises(_lib.NA1DError, match="no CPU path"):
        streaming.sink_attention(*_on("cpu"), 4)


def _sink(**kw):
    args = dict(dtype=0, heads=8, kv_heads=2, head_dim=64, scale=0.125, N=2, T=100, window=10, sinks=1)
    strides = {n: kw.pop(n) for n in list(kw) if n.endswith("strides")}
    args.update(kw)
    h = streaming._Sink(**args)
    for n, heads in (("q", 8), ("k", 2), ("v", 2)):
        setattr(h, n + "_strides", (ctypes.c_int64 * 3)(*strides.get(n + "_strides", (100 * heads * 64, 64, heads * 64))))
    return h


@pytest.mark.parametrize("change,status", [
    (dict(dtype=2), -2), (dict(head_dim=60), -3), (dict(head_dim=0), -3), (dict(head_dim=136), -8), (dict(window=0), -4), (dict(sinks=-1), -4), (dict(N=-1), -5),
    (dict(T=-1), -5), (dict(kv_heads=3), -5), (dict(kv_heads=0), -5), (dict(scale=0.0), -11), (dict(scale=float("nan")), -11), (dict(scale=float("inf")), -11),
    (dict(T=(1 << 24) + 1), -8), (dict(N=1 << 40), -8), (dict(q_strides=(0, 64, 56)), -5), (dict(k_strides=(0, -8, 128)), -5), (dict(v_strides=(0, 64, 132)), -6),
    (dict(q_strides=(4, 64, 512)), -6), (dict(q_strides=(0, 0, (1 << 20) + 8)), -8), (dict(heads=1 << 20, kv_heads=1 << 20), -8)])
def test_the_native_call_refuses(change, status):
    lib, h = _lib.load(), _sink(**change)
    assert lib.na1d_sink_saved_bytes(ctypes.byref(h)) == status
    assert lib.na1d_sink_backward_workspace_bytes(ctypes.byref(h)) == status
    assert lib.na1d_sink_forward(ctypes.byref(h), 16, None, 0, 16, 16, 16, None, None) == status
    assert lib.na1d_sink_backward(ctypes.byref(h), *[16] * 9, 1 << 40, None, 16, 1 << 40, None) == status


def test_the_native_call_asks_for_its_pointers_and_workspaces():
    lib, h = _lib.load(), ctypes.byref(_sink())
    nsaved, nws = lib.na1d_sink_saved_bytes(h), lib.na1d_sink_backward_workspace_bytes(h)
    assert nsaved == 4 * 1600 + 16 * 7 * 16 * 64 and nws >= 4 * 1600
    assert lib.na1d_sink_forward(None, 16, None, 0, 16, 16, 16, None, None) == -1
    assert lib.na1d_sink_forward(h, 16, None, 0, None, 16, 16, None, None) == -1
    assert lib.na1d_sink_forward(h, 16, None, 0, 24, 16, 16, None, None) == -6
    assert lib.na1d_sink_forward(h, 16, 16, nsaved - 1, 16, 16, 16, None, None) == -10
    assert lib.na1d_sink_backward(h, *[16] * 9, nsaved - 1, None, 16, nws, None) == -10
    assert lib.na1d_sink_backward(h, *[16] * 9, nsaved, None, 16, nws - 1, None) == -10
    assert lib.na1d_sink_backward(h, *[16] * 8, None, nsaved, None, 16, nws, None) == -1
    for nothing in (dict(N=0), dict(T=0)):
        e = ctypes.byref(_sink(**nothing))
        assert lib.na1d_sink_saved_bytes(e) == 0 and lib.na1d_sink_forward(e, None, None, 0, None, None, None, None, None) == 0


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 1), (32, 8), (64, 64)])
def test_a_backwards_sums_stay_small(heads, kv_heads):
    """No more than 1024 workgroups share strips for their sinks, no more than 512 because there are few strips: 128 rows of dk and dv in fp32 each."""
    for N in (1, 3, 64):
        for T in (1, 63, 1000, 16384, 1 << 20):
            for window, sinks in ((1, 0), (1, 1), (2000, 4), (64, 1 << 24), (1 << 24, 0)):
                h = _sink(N=N, T=T, heads=heads, kv_heads=kv_heads, head_dim=128, window=window, sinks=sinks)
                sums = _lib.load().na1d_sink_backward_workspace_bytes(ctypes.byref(h)) - 4 * ((N * heads * T + 3) // 4 * 4)
                assert 0 <= sums <= (1024 + 512) * 2 * 128 * 128 * 4, (N, T, window, sinks)


def test_the_oracle_agrees_with_automatic_differentiation():
    g = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(2, 23, h, 8, generator=g, dtype=torch.float64) for h in (6, 2, 2, 6))
    lengths = torch.tensor([23, 11])
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    o = torch.zeros(2, 23, 6, 8, dtype=torch.float64)
    for n in range(2):
        for h in range(6):
            for t in range(int(lengths[n])):
                us = [u for u in range(t + 1) if t - u < 5 or u < 2]
                p = torch.softmax(torch.stack([q[n, t, h] @ k[n, u, h // 3] for u in us]) * 8 ** -0.5, 0)
                o[n, t, h] = sum(p[i] * v[n, u, h // 3] for i, u in enumerate(us))
    grads = torch.autograd.grad(o, [q, k, v], dout)
    got = O.attention(*[x.detach() for x in (q, k, v)], 5, 2, t_valid=lengths, dout=dout)
    for name, want in zip(("out", "dq", "dk", "dv"), (o,) + grads):
        assert torch.allclose(got[name][0], want, atol=1e-12), name


# ------------------------------------------------------------------------------------------------ caches
def _caches(bits=16, N=2, K=2, S=20, C=32, dtype=torch.bfloat16, device="meta"):
    return streaming.new_cache(N, K, S, C, bits, dtype, device)


def _call(q=None, k=None, v=None, caches=None, lengths=None, window=8, sinks=1, bits=16):
    tokens = _on("meta", T=3, C=32)
    q, k, v = (given if given is not None else x for given, x in zip((q, k, v), tokens))
    caches = _caches(bits) if caches is None else caches
    lengths = torch.zeros(2, dtype=torch.int32, device="meta") if lengths is None else lengths
    return streaming.cache_step(q, k, v, *caches, lengths, window, sinks)


@pytest.mark.parametrize("bits", [16, 4])
def test_caches_and_tokens_that_do_not_fit(bits):
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, dtype=dtype, device="meta")  # noqa: E731
    with pytest.raises(_lib.NA1DError, match="no CPU path"):        # everything but the device is right
        _call(bits=bits)
    for wrong, error in ((dict(q=meta(2, 3, 3, 32)), ValueError), (dict(q=meta(2, 2, 4, 32)), ValueError), (dict(k=meta(2, 3, 4, 32)), ValueError),
                         (dict(v=meta(2, 4, 2, 32)), ValueError), (dict(k=meta(1, 3, 2, 32)), ValueError), (dict(q=meta(2, 3, 4, 64)), ValueError),
                         (dict(q=meta(2, 3, 4, 32, dtype=torch.float16)), TypeError), (dict(k=torch.empty(2, 3, 2, 32, dtype=torch.bfloat16)), _lib.NA1DError),
                         (dict(lengths=meta(2, dtype=torch.int64)), ValueError), (dict(lengths=meta(3, dtype=torch.int32)), ValueError),
                         (dict(lengths=torch.zeros(2, dtype=torch.int32)), _lib.NA1DError), (dict(window=0), _lib.NA1DError), (dict(window=18), _lib.NA1DError),
                         (dict(sinks=20, window=1), _lib.NA1DError), (dict(sinks=11), _lib.NA1DError), (dict(caches=(_caches(bits)[0], _caches(20 - bits)[1])), ValueError),
                         (dict(caches=(_caches(bits)[0], _caches(bits, S=21)[1])), ValueError), (dict(caches=(_caches(bits)[0], _caches(bits, dtype=torch.float16)[1])), ValueError),
                         (dict(caches=_caches(bits, K=0)), _lib.NA1DError)):
        with pytest.raises(error):
            _call(bits=bits, **wrong)
    with pytest.raises(_lib.NA1DError, match="no CPU path"):
        _call(bits=bits, window=17)                                 # 1 sink, 17, 2 more for three tokens at a time
    with pytest.raises(ValueError, match="cache_attend"):
        streaming.cache_step(_on("meta", C=32)[0], None, None, *_caches(bits), None, 4)
    with pytest.raises(ValueError, match="lengths"):
        streaming.cache_attend(_on("meta", T=3, C=32)[0], *_caches(bits), None, 4)


def test_caches_that_cannot_be_written_to():
    k, v = _caches(device="cpu")
    with pytest.raises(_lib.NA1DError, match="contiguous"):
        streaming._check_caches(k.transpose(1, 2), v.transpose(1, 2), 0)
    with pytest.raises(_lib.NA1DError, match="aligned"):
        streaming._check_caches(torch.zeros(k.numel() + 1, dtype=k.dtype)[1:].view(k.shape), v, 0)
    with pytest.raises(_lib.NA1DError, match="gradient"):
        streaming._check_caches(k.requires_grad_(True), v, 0)
    codes, ranges = _caches(4, device="cpu")[0]
    for bad in (streaming.Rows4(codes.to(torch.int8), ranges), streaming.Rows4(codes, ranges[..., :1]), streaming.Rows4(codes[0], ranges)):
        with pytest.raises(ValueError):
            streaming.cache_rows(bad)
    with pytest.raises(_lib.NA1DError, match="head_dim"):
        streaming.cache_rows(streaming.Rows4(codes[..., :10].contiguous(), ranges))
    for bits, C in ((4, 40), (4, 256), (8, 64)):
        with pytest.raises(_lib.NA1DError, match="bits"):
            _caches(bits, C=C)


def _native_cache(**kw):
    args = dict(dtype=0, bits=16, kv_heads=2, head_dim=64, N=2, capacity=100, sinks=4, k=16, v=16, k_ranges=16, v_ranges=16)
    args.update(kw)
    return streaming._Cache(**args)


@pytest.mark.parametrize("change,call,status", [
    (dict(dtype=2), {}, -2), (dict(bits=8), {}, -2), (dict(head_dim=60), {}, -3), (dict(head_dim=136), {}, -8), (dict(bits=4, head_dim=40), {}, -3), (dict(N=-1), {}, -5),
    (dict(kv_heads=0), {}, -5), ({}, dict(heads=3), -5), ({}, dict(fresh=-1), -5), (dict(sinks=100), {}, -4), (dict(sinks=-1), {}, -4), ({}, dict(window=0), -4),
    ({}, dict(window=97), -4), ({}, dict(window=95, fresh=3), -4), (dict(capacity=(1 << 23) + 1), {}, -8), (dict(N=1 << 24), {}, -8), ({}, dict(fresh=1 << 20), -8)])
def test_native_caches_refuse(change, call, status):
    lib, c = _lib.load(), _native_cache(**change)
    a = dict(fresh=1, heads=4, window=96)
    a.update(call)
    s = (ctypes.c_int64 * 3)(256, 64, 256)
    ref = ctypes.byref(c)
    assert lib.na1d_sink_attend_workspace_bytes(ref, a["fresh"], a["heads"], a["window"]) == status
    assert lib.na1d_sink_attend(ref, 16, 16, s, 16, a["fresh"], a["heads"], a["window"], 0.1, 16, 1 << 40, None) == status
    assert lib.na1d_sink_step(ref, 16, 16, 16, 16, s, s, s, 16, a["fresh"], a["heads"], a["window"], 0.1, 16, 1 << 40, None) == status
    if not call:
        assert lib.na1d_sink_append(ref, 16, 16, s, s, None, None, 5, None) == status


def test_native_caches_ask_for_their_pointers():
    lib, s = _lib.load(), (ctypes.c_int64 * 3)(256, 64, 256)
    step = lambda c, *a: lib.na1d_sink_step(ctypes.byref(c), *a)  # noqa: E731
    good = [16, 16, 16, 16, s, s, s, 16, 1, 4, 96, 0.1, 16, 1 << 40, None]
    for i in (0, 1, 2, 3, 4, 5, 6, 7):
        assert step(_native_cache(), *good[:i], None, *good[i + 1:]) == -1, i
    for name in ("k", "v"):
        assert step(_native_cache(**{name: None}), *good) == -1
        assert step(_native_cache(**{name: 8}), *good) == -6
        assert step(_native_cache(bits=4, **{name + "_ranges": None}), *good) == -1
        assert step(_native_cache(bits=4, **{name + "_ranges": 8}), *good) == -6
    for i in (0, 1, 2, 3):
        assert step(_native_cache(), *good[:i], 24, *good[i + 1:]) == -6
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert step(_native_cache(), *good[:11], scale, *good[12:]) == -11
    for bad, status in (((256, 64, 56), -5), ((256, 64, 68), -6), ((-8, 64, 256), -5), ((256, 64, 1 << 21), -8)):
        for i in (4, 5, 6):
            assert step(_native_cache(), *good[:i], (ctypes.c_int64 * 3)(*bad), *good[i + 1:]) == status
    long = _native_cache(capacity=5000)
    need = lib.na1d_sink_attend_workspace_bytes(ctypes.byref(long), 1, 4, 4000)
    assert need > 0
    args = good[:8] + [1, 4, 4000, 0.1]
    assert step(long, *args, 16, need - 1, None) == -10 and step(long, *args, None, need, None) == -1
    assert step(_native_cache(N=0), *[None] * 4, s, s, s, None, 1, 4, 96, 0.1, None, 0, None) == 0
    for a, status in (((16, 16, 16, 5, 60, 0), -3), ((16, 16, 16, 5, 64, 2), -2), ((16, 16, 16, -1, 64, 0), -5), ((None, 16, 16, 5, 64, 0), -1), ((16, 8, 16, 5, 64, 0), -6),
                      ((16, 16, 16, 5, 160, 0), -8), ((None, None, None, 0, 64, 0), 0)):
        assert lib.na1d_sink_rows(*a, None) == status
    assert lib.na1d_sink_append(ctypes.byref(long), 16, 16, s, s, None, None, -1, None) == -5
    assert lib.na1d_sink_append(ctypes.byref(long), 16, 16, s, s, None, None, (1 << 24) + 1, None) == -8
    assert lib.na1d_sink_append(ctypes.byref(long), None, 16, s, s, None, None, 5, None) == -1
    assert lib.na1d_sink_append(ctypes.byref(long), 16, 16, s, None, None, None, 5, None) == -1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_bytes_that_a_forward_saves(dtype):
    for N, T, H, K, C in ((1, 1, 1, 1, 8), (3, 17, 6, 2, 40), (2, 100, 4, 4, 64), (5, 333, 8, 1, 128), (2, 64, 3, 3, 72)):
        q, k, v = _on("meta", N, T, H, K, C, dtype)
        assert streaming.saved_bytes(q) == streaming._bytes("na1d_sink_saved_bytes", streaming._sink(q, k, v, 5, 1, 0.1))


@pytest.mark.parametrize("bits", [16, 4])
def test_caches_that_share_memory(bits):
    """Of the caches, and with what is put into them: refused wherever something is written."""
    k, v = _caches(bits, device="cpu")
    lengths = torch.zeros(2, dtype=torch.int32)
    q, kx, vx = _on("cpu", T=3, C=32)
    flat = torch.zeros(2 * 2 * 20 * 32 + 64, dtype=torch.bfloat16)                                # a cache that starts inside the other
    near = flat[64:].view(2, 2, 20, 32), flat[:-64].view(2, 2, 20, 32)
    pairs = [(k, k), (k, streaming.Rows4(v.codes, k.ranges)) if bits == 4 else near]
    for pair in pairs:
        with pytest.raises(_lib.NA1DError, match="share memory"):
            streaming.cache_append(kx, vx, *pair)
        with pytest.raises(_lib.NA1DError, match="share memory"):
            streaming.cache_step(q, kx, vx, *pair, lengths, 8)
        with pytest.raises(_lib.NA1DError, match="no CPU path"):                                 # nothing is written
            streaming.cache_attend(q, *pair, lengths, 8)
    rows = k.codes.view(torch.bfloat16).view(-1) if bits == 4 else k.view(-1)
    inside = rows[:2 * 3 * 2 * 32].view(2, 3, 2, 32)
    for tokens in ((inside, vx), (kx, inside)):
        with pytest.raises(_lib.NA1DError, match="share memory"):
            streaming.cache_append(*tokens, k, v)
        with pytest.raises(_lib.NA1DError, match="share memory"):
            streaming.cache_step(q, *tokens, k, v, lengths, 8)
    both = torch.zeros(2, 2, 2, 20, 32, dtype=torch.bfloat16)                                    # halves of one tensor do not
    with pytest.raises(_lib.NA1DError, match="no CPU path"):
        streaming.cache_append(kx, vx, *both)
