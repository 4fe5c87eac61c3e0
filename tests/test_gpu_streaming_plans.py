"""The ways in which large problems of streams' attention are cut: each case asserts that it takes its way."""
import ctypes

import pytest
import torch

from na1d_amd import _lib, streaming
from oracle import streaming_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["bf16", "fp16"]


def _near(name, got, value, bound):
    off = (got.double() - value).abs()
    if not bool((off <= bound).all()):
        worst = (off / bound).nan_to_num(torch.inf).argmax()
        pytest.fail("%s: off by %.3g where %.3g is allowed" % (name, off.flatten()[worst], bound.flatten()[worst]))


def _last_kernel(call):
    """`call()` and the kernel that it launched last on this thread."""
    lib = _lib.load()
    events = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    for e in events:
        e.record()
    assert lib.na1d_profile_events(*[ctypes.c_void_p(e.cuda_event) for e in events]) == 0
    try:
        result = call()
        return result, lib.na1d_profile_last_kernel().decode()
    finally:
        lib.na1d_profile_events(None, None)


def _key_plan(q, k, v, W):
    """Strips of keys with a workgroup of their own, and workgroups that share each of the others, without sinks: a backward's workspace has 128 rows of fp32 for each of these."""
    N, T, H, C = q.shape
    wide = next(w for w in (16, 32, 64, 96, 128) if C <= w)
    floats = (N * H * T + 3) // 4 * 4 + (N * H * (-(-T // 64)) * 4 if q.dtype == torch.float16 else 0)
    shares = (streaming._bytes("na1d_sink_backward_workspace_bytes", streaming._sink(q, k, v, W, 0, 0.1)) // 4 - floats) // (128 * wide)
    strips, card = N * k.shape[2] * (-(-T // 64)), 256 * (2 if C > 64 else 4 if C > 32 else 6)
    over = strips % card
    return (strips - over, shares // over) if shares else (strips, 1)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,T,H,K,C,W,Z,tiles,plan", [
    (4, 1100, 32, 32, 64, 700, 2, 2, (2048, 3)), (8, 513, 32, 8, 16, 300, 0, 2, (0, 2)), (3, 700, 60, 20, 32, 256, 3, 2, (0, 2)), (5, 801, 32, 4, 72, 400, 40, 2, (260, 1)),
    (4, 1030, 32, 8, 96, 1030, 1, 2, (512, 16)), (6, 900, 24, 6, 128, 300, 130, 2, (512, 6)), (4, 1025, 32, 16, 120, 500, 0, 2, (1024, 4)), (5, 1400, 24, 12, 64, 400, 1, 2, (1024, 3)),
    (2, 1500, 24, 12, 128, 300, 2, 1, (512, 3)), (6, 1000, 16, 8, 128, 300, 2, 1, (512, 2)), (3, 1500, 16, 8, 80, 200, 66, 1, (512, 2)), (5, 1400, 44, 22, 64, 250, 5, 1, (2048, 2)),
    (3, 1500, 64, 32, 16, 200, 1, 1, (1536, 2))])
def test_large_launches(N, T, H, K, C, W, Z, tiles, plan, dtype):
    """Forwards with one and two tiles of queries to a wave; strips of keys with workgroups of their own beside strips in parts, with sinks among both."""
    g = torch.Generator().manual_seed(C)
    q, k, v, dout = (torch.randn(N, T, h, C, generator=g).to(dtype).cuda() for h in (H, K, K, H))
    lengths = torch.tensor([T, T - 1, T // 2, 65, 1, 0, T, T][:N], dtype=torch.int32, device="cuda")
    assert _key_plan(q, k, v, W) == plan
    for t_valid in (None, lengths):
        xs = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out, kernel = _last_kernel(lambda: streaming.sink_attention(*xs, W, Z, t_valid=t_valid))
        assert kernel.startswith("sink_fwd_kernel") and kernel.endswith(", %d>" % tiles), kernel
        got = (out.detach(),) + torch.autograd.grad(out, xs, dout)
        torch.cuda.synchronize()
        for n in range(N):                                             # (a sample at a time: all pairs of rows in 64 bits)
            want = O.attention(*(x[n:n + 1] for x in (q, k, v)), W, Z, t_valid=None if t_valid is None else t_valid[n:n + 1], dout=dout[n:n + 1])
            for name, x in zip(("out", "dq", "dk", "dv"), got):
                _near(name, x[n:n + 1], *want[name])
                size = float(want[name][0].norm())
                if size > 0:                                           # 0.42 u of a norm are the rounding, other errors less than that
                    assert float((x[n:n + 1].double() - want[name][0]).norm()) < 0.75 * O.half_step(dtype) * size + (2.0 ** -25 if dtype == torch.float16 else 0.0) * x[n].numel() ** 0.5, name
        again = torch.autograd.grad(streaming.sink_attention(*xs, W, Z, t_valid=t_valid), xs, dout)
        assert all(torch.equal(a, b) for a, b in zip(got[1:], again))


def _splits(caches, q, W):
    """Workgroups that share a head's keys: a step's workspace has their sums."""
    four = isinstance(caches[0], streaming.Rows4)
    shape, dtype = streaming._check_caches(*caches, 0)
    N, K, S, C = shape
    c = streaming._cache(*caches, shape, dtype, 2)
    rows = q.shape[1] * q.shape[2] // K
    tiles = 1 if rows <= 16 else 2 if rows <= 32 else 4
    wide = next(w for w in (16, 32, 64, 96, 128) if C <= w)
    each = N * K * (-(-rows // (16 * tiles))) * 16 * tiles * (wide + 4) * 4
    nbytes = _lib.load().na1d_sink_attend_workspace_bytes(ctypes.byref(c), q.shape[1], q.shape[2], W)
    assert nbytes % each == 0
    return nbytes // each or 1


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,K,G,C,W,n,splits", [(36, 8, 2, 128, 2500, 1, (4, 4)), (70, 9, 1, 64, 3000, 1, (3, 3)), (60, 8, 3, 96, 2000, 2, (1, 3)), (70, 8, 1, 32, 2000, 1, (4, 4)),
                                                (67, 4, 8, 128, 2000, 1, (4, 4)), (37, 16, 12, 64, 1500, 3, (4, 4)), (25, 8, 1, 128, 3000, 1, (4, 2)), (50, 8, 1, 128, 3000, 1, (3, 4))])
def test_caches_of_many_streams(N, K, G, C, W, n, splits, bits, dtype):
    """Heads enough for more than half of the workgroups that the card holds at once (and one case with a few less): a head's keys are split so that the last round of them is nearly full."""
    Z, H = 2, K * G
    g = torch.Generator(device="cuda").manual_seed(C)
    T = W + 200
    k, v = (torch.randn(N, T, K, C, generator=g, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(N, n, H, C, generator=g, device="cuda").to(dtype)
    caches = streaming.new_cache(N, K, Z + W + n - 1, C, bits, dtype)
    ages = [T - n if i % 5 else (i * 131) % (T - n) for i in range(N)]
    ages[3] = -1
    lengths = torch.tensor(ages, dtype=torch.int32, device="cuda")
    streaming.cache_append(k, v, *caches, sinks=Z, t_valid=lengths)
    at = lengths.clamp(min=0).long().view(N, 1) + torch.arange(n, device="cuda")
    new = [x.gather(1, at.view(N, n, 1, 1).expand(N, n, K, C)) for x in (k, v)]
    rows = n * G
    tiles = 1 if rows <= 16 else 2 if rows <= 32 else 4
    assert _splits(caches, q, W) == splits[bits == 4]
    out, kernel = _last_kernel(lambda: streaming.cache_step(q, *new, *caches, lengths, W, Z))
    assert kernel.startswith("cache_attend%s_kernel" % ("4" if bits == 4 else "")) and kernel.endswith("%d, 4>" % tiles), kernel
    torch.cuda.synchronize()
    for i in range(0, N, 3):                                           # (the idle one among them)
        value, bound = O.over_history(q[i:i + 1], k[i:i + 1], v[i:i + 1], W, Z, [ages[i] + n if ages[i] >= 0 else 0], four=bits == 4)
        _near("out", out[i:i + 1], value, bound)
    ended = torch.where(lengths < 0, lengths, lengths + n)
    assert torch.equal(out, streaming.cache_attend(q, *caches, ended, W, Z))

