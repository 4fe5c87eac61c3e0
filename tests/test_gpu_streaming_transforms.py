"""Attention of streams under forward-mode derivatives, tracers, batching transforms, hooks on what is saved and torch.compile."""
import pytest
import torch
from torch.autograd import forward_ad

from na1d_amd import _lib, ops, streaming

pytestmark = pytest.mark.gpu


def _inputs(N=2, T=70, H=4, K=2, C=32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(N, T, h, C, generator=g).to(torch.bfloat16).cuda() for h in (H, K, K, H)]


def _grads(f, q, k, v, dout):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = f(q, k, v)
    return [out.detach(), *torch.autograd.grad(out, [q, k, v], dout)]


def _same(a, b):
    torch.cuda.synchronize()
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_forward_mode_and_transforms_are_refused():
    q, k, v, _ = _inputs()
    for call in (lambda q, k, v: streaming.sink_attention(q, k, v, 9, 1), lambda q, k, v: ops.sink_attention_op(q, k, v, 9, 1)):
        for at in range(3):
            with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
                call(*[forward_ad.make_dual(x, torch.ones_like(x)) if i == at else x for i, x in enumerate((q, k, v))])
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: streaming.sink_attention(x, k, v, 9))(torch.stack((q, q)))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: streaming.sink_attention(x, k, v, 9).float().sum())(q)


@pytest.mark.parametrize("strided", [False, True])
def test_a_trace_computes(strided):
    q, k, v, _ = _inputs()
    if strided:                                                        # (packed by the Python path)
        q, k, v = (torch.stack((x, x), -1)[..., 0] for x in (q, k, v))
    traced = torch.jit.trace(lambda q, k, v: streaming.sink_attention(q, k, v, 9, 1) + 1, (q, k, v), check_trace=False)
    for seed in (1, 2):
        x = _inputs(seed=seed)
        junk = [torch.full_like(q, 9.0) for _ in range(4)]             # what uninitialised memory would hold
        del junk
        _same([traced(*x[:3])], [streaming.sink_attention(*x[:3], 9, 1) + 1])
    op = torch.jit.trace(lambda q, k, v: ops.sink_attention_op(q, k, v, 9, 1), (q, k, v), check_trace=False)
    x = _inputs(seed=3)
    _same([op(*x[:3])], [streaming.sink_attention(*x[:3], 9, 1)])


@pytest.mark.parametrize("bits", [16, 4])
def test_calls_over_caches_are_not_traced_and_have_no_tangents(bits):
    q, k, v, _ = (x[:, :2].contiguous() for x in _inputs())
    caches, lengths = streaming.new_cache(2, 2, 20, 32, bits), torch.zeros(2, dtype=torch.int32, device="cuda")
    calls = (lambda q, k, v: streaming.cache_append(k, v, *caches), lambda q, k, v: streaming.cache_step(q, k, v, *caches, lengths, 5),
             lambda q, k, v: streaming.cache_attend(q, *caches, lengths, 5))
    for call in calls:
        with pytest.raises(_lib.NA1DError, match="trace"):
            torch.jit.trace(lambda q, k, v: (call(q, k, v), q + 1)[1], (q, k, v), check_trace=False)
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(*[torch.stack((x, x)) for x in (q, k, v)])
    with forward_ad.dual_level():
        for call in calls[1:]:
            with pytest.raises(_lib.NA1DError, match="no gradient"):
                call(forward_ad.make_dual(q, torch.ones_like(q)), k, v)
    assert not any(t.any() for c in caches for t in (c if bits == 4 else (c,)))      # nothing was written


def test_hooks_on_what_is_saved():
    q, k, v, dout = _inputs()
    lengths = torch.tensor([70, 33], dtype=torch.int32, device="cuda")
    want, seen = _grads(lambda *x: streaming.sink_attention(*x, 9, 1, t_valid=lengths), q, k, v, dout), []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.shape) or t.cpu(), lambda t: t.cuda()):
        got = _grads(lambda *x: streaming.sink_attention(*x, 9, 1, t_valid=lengths), q, k, v, dout)
    _same(got, want)
    assert len(seen) == 6


def test_steps_beside_a_compiled_graph():
    """A compiled layer leaves calls over caches out of its graph."""
    q, k, v, _ = (x[:, :2].contiguous() for x in _inputs())
    lengths = torch.tensor([5, 0], dtype=torch.int32, device="cuda")
    a, b = streaming.new_cache(2, 2, 20, 32), streaming.new_cache(2, 2, 20, 32)
    layer = lambda step, cache: step(2 * q, k + 1, v, *cache, lengths, 8, 1) + 1  # noqa: E731
    with torch.no_grad():
        got = torch.compile(lambda: layer(torch.compiler.disable(streaming.cache_step), a), backend="aot_eager")()
        _same([got, *a], [layer(streaming.cache_step, b), *b])


def test_a_call_without_gradients_keeps_nothing(monkeypatch):
    """Through the Python path as through the native one."""
    kept, forward = [], streaming.sink_forward
    monkeypatch.setattr(_lib, "nodes", lambda: None)
    monkeypatch.setattr(streaming, "sink_forward", lambda *a: kept.append(a[-1]) or forward(*a))
    q, k, v, dout = _inputs()
    streaming.sink_attention(q, k, v, 9)
    with torch.no_grad():
        streaming.sink_attention(q.requires_grad_(True), k, v, 9)
    with torch.inference_mode():
        x = [torch.stack((y, y), -1)[..., 0] for y in (q, k, v)]
        assert torch.equal(streaming.sink_attention(*x, 9), streaming.sink_attention(*(y.contiguous() for y in x), 9))
    assert kept == [False] * 4
    assert streaming.sink_attention(q, k, v, 9).requires_grad and kept[-1]
