"""Attention of streams under forward-mode derivatives, tracers and batching transforms, without a GPU: what is not supported is refused, nothing is lost.  The native calls are stubbed."""
import pytest
import torch
from torch.autograd import forward_ad

from na1d_amd import _lib, streaming


def _tokens(N=2, T=9, H=4, K=2, C=16):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(N, T, h, C, generator=g).to(torch.bfloat16) for h in (H, K, K)]


@pytest.fixture
def stubbed(monkeypatch):
    """`sink_attention` gives 2 q, outside of what a tracer sees, as the native call would."""
    def forward(q, k, v, t_valid, win_size, sinks, scale, want_saved):
        calls.append(want_saved)
        out = torch.empty(q.shape, dtype=q.dtype)
        state = torch._C._get_tracing_state()
        torch._C._set_tracing_state(None)
        out.copy_(2 * q.detach())
        torch._C._set_tracing_state(state)
        return out, torch.empty(8 if want_saved else 0, dtype=torch.uint8)
    calls = []
    monkeypatch.setattr(streaming, "sink_forward", forward)
    monkeypatch.setattr(streaming, "_check_gpu", lambda q: None)
    monkeypatch.setattr(_lib, "nodes", lambda: None)
    return calls


def test_forward_mode_is_refused(stubbed):
    q, k, v = _tokens()
    for at in range(3):
        with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
            xs = [forward_ad.make_dual(x, torch.ones_like(x)) if i == at else x for i, x in enumerate((q, k, v))]
            streaming.sink_attention(*xs, 4)


def test_a_trace_holds_the_call(stubbed):
    q, k, v = _tokens()
    traced = torch.jit.trace(lambda q, k, v: streaming.sink_attention(q, k, v, 4) + 1, (q, k, v), check_trace=False)
    for seed in (1, 2):
        other = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).to(q.dtype)
        assert torch.equal(traced(other, k, v), 2 * other + 1)


def test_what_is_kept_for_a_backward(stubbed):
    """Nothing where there is none."""
    q, k, v = _tokens()
    streaming.sink_attention(q, k, v, 4)
    with torch.no_grad():
        assert not streaming.sink_attention(q.requires_grad_(True), k, v, 4).requires_grad
    assert stubbed == [False, False]
    assert streaming.sink_attention(q, k, v, 4).requires_grad and stubbed == [False, False, True]


def test_batching_is_refused(stubbed):
    q, k, v = _tokens()
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda x: streaming.sink_attention(x, k, v, 4))(torch.stack((q, q)))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: streaming.sink_attention(x, k, v, 4).float().sum())(q)


def _cache_calls(bits):
    q, k, v = (x[:, :2, :, :].contiguous() for x in _tokens(C=32))
    caches = streaming.new_cache(2, 2, 20, 32, bits, device="cpu")
    lengths = torch.zeros(2, dtype=torch.int32)
    return (q, k, v), caches, [lambda q, k, v: streaming.cache_append(k, v, *caches), lambda q, k, v: streaming.cache_step(q, k, v, *caches, lengths, 5),
                               lambda q, k, v: streaming.cache_attend(q, *caches, lengths, 5)]


@pytest.mark.parametrize("bits", [16, 4])
def test_calls_over_caches_are_not_traced(bits):
    """A trace would hold neither what is written to a cache nor what is read from it."""
    tokens, caches, calls = _cache_calls(bits)
    for call in calls:
        with pytest.raises(_lib.NA1DError, match="trace"):
            torch.jit.trace(lambda q, k, v: (call(q, k, v), q + 1)[1], tokens, check_trace=False)
    if bits == 4:
        with pytest.raises(_lib.NA1DError, match="trace"):
            torch.jit.trace(lambda codes: streaming.cache_rows(streaming.Rows4(codes, caches[0].ranges)), caches[0].codes, check_trace=False)


@pytest.mark.parametrize("bits", [16, 4])
def test_tangents_over_caches_are_refused(bits):
    tokens, caches, calls = _cache_calls(bits)
    with forward_ad.dual_level():
        for call in calls[1:]:
            for at in range(3 if call is calls[1] else 1):
                with pytest.raises(_lib.NA1DError, match="no gradient"):
                    call(*[forward_ad.make_dual(x, torch.ones_like(x)) if i == at else x for i, x in enumerate(tokens)])
        values = caches[0].ranges if bits == 4 else caches[0]
        dual = forward_ad.make_dual(values, torch.ones_like(values))
        with pytest.raises(_lib.NA1DError, match="gradient"):
            streaming.cache_rows(streaming.Rows4(caches[0].codes, dual) if bits == 4 else dual)


@pytest.mark.parametrize("bits", [16, 4])
def test_batches_of_calls_over_caches_are_refused(bits):
    tokens, caches, calls = _cache_calls(bits)
    for call in calls:
        with pytest.raises(RuntimeError):
            torch.func.vmap(lambda q, k, v: call(q, k, v), in_dims=(0, 0, 0))(*[torch.stack((x, x)) for x in tokens])
