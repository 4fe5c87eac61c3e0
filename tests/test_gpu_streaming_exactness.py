"""What a backward of streams' attention pays for: the bytes that outputs lost in rounding, and products with P and dS as two numbers each, seen in the gradients' errors as norms."""
import pytest
import torch

from na1d_amd import streaming
from oracle import streaming_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["bf16", "fp16"]


def _whole_outputs(out, saved):
    """Outputs with their bytes, by the layout that the kernels share: behind 4 bytes to a head's row, [N, heads] tiles of 16 rows; channels 32 s + 8 g .. + 7 of row n are the
    eight bytes 512 s + 8 (16 g + n) .., with 16 channels 4 g .. + 3 the four bytes 4 (16 g + n) ..; a byte counts 2^8 (bf16) or 2^5 (fp16) steps of fp32."""
    N, T, H, C = out.shape
    wide = next(w for w in (16, 32, 64, 96, 128) if C <= w)
    tiles, shift = (T + 15) // 16, 8 if out.dtype == torch.bfloat16 else 5
    rest = saved[16 * ((N * H * T + 3) // 4):].view(torch.int8).view(N, H, tiles, 16 * wide)
    if wide == 16:
        rest = rest.view(N, H, tiles, 4, 16, 4).permute(0, 1, 2, 4, 3, 5)
    else:
        rest = rest.view(N, H, tiles, wide // 32, 4, 16, 8).permute(0, 1, 2, 5, 3, 4, 6)
    rest = rest.reshape(N, H, tiles * 16, wide)[:, :, :T, :C].transpose(1, 2).int()
    bits = out.float().view(torch.int32) + rest * 2 ** shift
    return bits.view(torch.float32).double(), rest


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,T,H,K,C,W,Z", [(2, 100, 4, 2, 8, 7, 2), (1, 33, 2, 1, 16, 5, 0), (3, 129, 3, 3, 32, 9, 1), (2, 70, 4, 2, 40, 6, 3), (2, 200, 2, 2, 64, 11, 70), (1, 65, 6, 3, 80, 3, 1),
                                           (1, 150, 4, 1, 96, 13, 2), (2, 90, 2, 1, 112, 10, 0), (4, 333, 8, 2, 128, 30, 5), (9, 900, 16, 8, 64, 300, 2)])
def test_the_bytes_that_outputs_lost(N, T, H, K, C, W, Z, dtype):
    """Queries of zeros make an output the mean of what is seen, to 2^-20 before it is rounded (fp32 sums of powers of two times values, a reciprocal)."""
    g = torch.Generator().manual_seed(C)
    v = torch.randn(N, T, K, C, generator=g).to(dtype).cuda()
    q, k = torch.zeros(N, T, H, C, dtype=dtype, device="cuda"), torch.randn(N, T, K, C, generator=g).to(dtype).cuda()
    lengths = torch.tensor([T, T // 2, 1, 0, T, T, 17, T, T][:N], dtype=torch.int32, device="cuda")
    out, saved = streaming.sink_forward(q, k, v, lengths, W, Z, 0.1, True)
    want, _ = O.attention(q, k, v, W, Z, t_valid=lengths, scale=0.1)["out"]
    size, _ = O.attention(q, k, v.abs(), W, Z, t_valid=lengths, scale=0.1)["out"]
    whole, rest = _whole_outputs(out, saved)
    torch.cuda.synchronize()
    # 2^8 or 2^5 fp32 steps, one of which is 2^-23 of a number at most; fp16 below 2^-14: the byte ends at its range, and half a step of fp16 may be lost
    left, least = (2.0 ** -15, 0.0) if dtype == torch.bfloat16 else (2.0 ** -18, 2.0 ** -25 * (want.abs() < 2.0 ** -13))
    off = (whole - want).abs()
    assert bool((off <= left * want.abs() + 2.0 ** -20 * size + least + 2.0 ** -126).all()), float((off / want.abs()).nan_to_num(0).max())
    assert int((rest != 0).sum()) > 0.9 * int((want != 0).sum()) - T * K * C * N // W - 64 * H * C       # (means of one value, and a few others, lose nothing)
    assert not bool(rest[want == 0].any())



@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("mean", [0.0, 3.0])
@pytest.mark.parametrize("N,T,H,K,C,W,Z,ragged", [(2, 300, 2, 1, 16, 300, 0, False), (2, 300, 4, 2, 32, 20, 100, True), (1, 500, 4, 4, 64, 60, 3, False), (4, 400, 6, 2, 64, 400, 1, True),
                                                 (2, 260, 2, 2, 80, 100, 0, False), (3, 500, 10, 2, 96, 100, 3, True), (1, 700, 2, 1, 128, 700, 5, False), (3, 513, 8, 4, 120, 129, 70, True),
                                                 (2, 200, 3, 3, 8, 50, 2, True)])
def test_errors_of_gradients_as_norms(N, T, H, K, C, W, Z, ragged, mean, dtype):
    """Values of mean 0 show a P or dS that is one number; with a mean of 3, which drops out of dP - delta, an output without its byte or with a wrong one (tests/test_streaming_exactness_cpu.py
    has what each of them would make of it, and why right ones stay below 0.1 u more than the results' rounding)."""
    q, k, v, dout = O.centred(N, T, H, K, C, dtype, mean)
    lengths = torch.tensor([T, T - 37, T // 3, 0][:N], dtype=torch.int32) if ragged else None
    want = O.attention(q, k, v, W, Z, t_valid=lengths, dout=dout)
    xs = [x.cuda().requires_grad_(True) for x in (q, k, v)]
    out = streaming.sink_attention(*xs, W, Z, t_valid=None if lengths is None else lengths.cuda())
    got = torch.autograd.grad(out, xs, dout.cuda())
    for name, x in zip(("dq", "dk", "dv"), got):
        more = O.more_than_rounding(x.cpu(), want[name][0])
        assert more < 0.1, "%s: %.3f u more than its rounding" % (name, more)
