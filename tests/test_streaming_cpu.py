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
