"""Attention of streams in the largest launches."""
import pytest
import torch

from na1d_amd import _lib, streaming

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_sequences_of_one_token_that_fill_a_launch(dtype):
    """2^24 - 16 workgroups: a token sees itself, so the output is v; one sequence more is refused."""
    N, H, C = (1 << 20) - 1, 16, 8
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, dout = (torch.randn(N + 1, 1, H, C, generator=g, device="cuda", dtype=dtype) for _ in range(4))
    with pytest.raises(_lib.NA1DError, match="status -8"):
        streaming.sink_attention(q, k, v, 5)
    q, k, v = (x[:-1].requires_grad_(True) for x in (q, k, v))
    out = streaming.sink_attention(q, k, v, 5)
    dq, dk, dv = torch.autograd.grad(out, [q, k, v], dout[:-1])
    assert torch.equal(out, v) and torch.equal(dv, dout[:-1])
    # dS = P (dP - delta) is what fp32 sums of 8 products in two orders differ by, at most 2^-20 of 8 times 6^2 with these numbers, times a scale and 6
    assert float(dq.abs().max()) < 2.0 ** -20 * 8 * 36 * 8 ** -0.5 * 6 and float(dk.abs().max()) < 2.0 ** -20 * 8 * 36 * 8 ** -0.5 * 6


def test_caches_that_fill_a_launch():
    N, K, C = (1 << 20) - 1, 16, 8
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(N, 1, K, C, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    caches, lengths = streaming.new_cache(N, K, 2, C), torch.zeros(N, dtype=torch.int32, device="cuda")
    streaming.cache_append(k, v, *caches)
    assert torch.equal(caches[1][:, :, 0], v[:, 0]) and not bool(caches[1][:, :, 1].any())
    out = streaming.cache_step(q, k, 2 * v, *caches, lengths + 1, 1)      # sees the token itself alone
    assert torch.equal(out, 2 * v) and torch.equal(caches[0][:, :, 1], k[:, 0]) and torch.equal(caches[0][:, :, 0], k[:, 0])
    more = streaming.new_cache(N + 1, K, 2, C)
    x = torch.zeros(N + 1, 1, K, C, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(_lib.NA1DError, match="status -8"):
        streaming.cache_append(x, x, *more)
    with pytest.raises(_lib.NA1DError, match="status -8"):
        streaming.cache_step(x, x, x, *more, torch.zeros(N + 1, dtype=torch.int32, device="cuda"), 1)
