"""Windowed causal attention with sinks on the GPU against its formulas in 64 bits."""
import pytest
import torch

from na1d_amd import streaming
from oracle import streaming_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["bf16", "fp16"]
SIZES = [  # N, T, heads, kv_heads, C, window, sinks
    (1, 1, 1, 1, 8, 1, 0), (2, 1, 4, 2, 64, 5, 1), (3, 2, 2, 1, 16, 1, 0), (1, 17, 3, 3, 24, 4, 2), (2, 63, 4, 4, 32, 63, 0), (2, 64, 2, 1, 40, 64, 1),
    (1, 65, 6, 2, 48, 16, 3), (3, 100, 4, 4, 64, 27, 1), (2, 129, 8, 2, 72, 128, 64), (1, 300, 4, 1, 128, 65, 5), (2, 257, 5, 5, 80, 1, 4), (1, 400, 2, 2, 96, 7, 130),
    (2, 333, 3, 1, 104, 200, 0), (1, 321, 8, 8, 120, 1000, 0), (1, 200, 4, 2, 112, 30, 500), (1, 500, 16, 1, 64, 50, 70),
]
FULL = [  # launches that fill the card: strips of 128 rows, parts by the sinks
    (8, 513, 16, 4, 64, 100, 4), (4, 700, 16, 8, 128, 129, 1), (16, 260, 8, 8, 32, 64, 66), (3, 1100, 32, 8, 16, 200, 2), (2, 1500, 20, 4, 72, 90, 129),
]


def _inputs(N, T, H, K, C, dtype, seed, sinks=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dout = (torch.randn(N, T, h, C, generator=g) for h in (H, K, K, H))
    q += 0.5
    k[:, :sinks] += 1.0
    return [x.to(dtype).cuda() for x in (q, k, v, dout)]


def _near(name, got, want):
    value, bound = want
    assert got.shape == value.shape, name
    off = (got.double() - value).abs()
    if not bool((off <= bound).all()):
        worst = (off / bound).nan_to_num(torch.inf).argmax()
        pytest.fail("%s: off by %.3g where %.3g is allowed" % (name, off.flatten()[worst], bound.flatten()[worst]))


def _train(q, k, v, dout, *args, **kw):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = streaming.sink_attention(q, k, v, *args, **kw)
    grads = torch.autograd.grad(out, [q, k, v], dout)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(),) + grads))


def _check(got, want):
    torch.cuda.synchronize()
    for name, value in got.items():
        _near(name, value, want[name])


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,T,H,K,C,W,Z", SIZES + FULL)
def test_forward_and_gradients(N, T, H, K, C, W, Z, dtype):
    q, k, v, dout = _inputs(N, T, H, K, C, dtype, 1, Z)
    got = _train(q, k, v, dout, W, Z)
    _check(got, O.attention(q, k, v, W, Z, dout=dout))
    assert torch.equal(got["out"], streaming.sink_attention(q, k, v, W, Z))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,T,H,K,C,W,Z", [(5, 100, 4, 2, 64, 27, 3), (6, 200, 2, 2, 80, 64, 0), (4, 513, 16, 4, 128, 100, 70), (5, 700, 16, 16, 32, 31, 1)])
def test_lengths_and_what_lies_behind_them(N, T, H, K, C, W, Z, dtype):
    q, k, v, dout = _inputs(N, T, H, K, C, dtype, 2, Z)
    lengths = torch.tensor([T, 0, 1, T - 1, T // 2, 65][:N], dtype=torch.int32, device="cuda")
    want = O.attention(q, k, v, W, Z, t_valid=lengths, dout=dout)
    behind = torch.arange(T, device="cuda") >= lengths.unsqueeze(1)
    for x, filler in zip((q, k, v, dout), (float("nan"), float("inf"), float("nan"), -float("inf"))):
        x[behind] = filler
    got = _train(q, k, v, dout, W, Z, t_valid=lengths)
    _check(got, want)
    for x in got.values():
        assert not x[behind].any()
    far = torch.where(lengths == T, 2 ** 30, torch.where(lengths == 0, -7, lengths)).int()       # beyond either end: as at the ends
    again = _train(q, k, v, dout, W, Z, t_valid=far)
    assert all(torch.equal(again[n], got[n]) for n in got)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("layout", ["one projection", "heads first", "every other channel", "off the alignment", "rows apart", "samples backwards"])
def test_layouts(layout, dtype):
    N, T, H, K, C, W, Z = 3, 150, 6, 2, 40, 33, 2
    q, k, v, dout = _inputs(N, T, H, K, C, dtype, 3, Z)
    want = O.attention(q, k, v, W, Z, dout=dout)
    if layout == "one projection":
        q, k, v = torch.cat((q, k, v), 2).split([H, K, K], 2)
    elif layout == "heads first":
        q, k, v, dout = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, dout))
    elif layout == "every other channel":
        q, k, v, dout = (torch.stack((x, -x), -1).flatten(3)[..., ::2] for x in (q, k, v, dout))
    elif layout == "off the alignment":
        q, k, v, dout = (torch.cat((x.flatten()[:1], x.flatten()))[1:].view(x.shape) for x in (q, k, v, dout))
    elif layout == "rows apart":
        q, k, v = (torch.stack((x, x), 2).flatten(1, 2)[:, ::2] for x in (q, k, v))
    else:
        q, k, v = (torch.as_strided(x.flip(0), x.shape, x.stride()).flip(0) for x in (q, k, v))
    _check(_train(q, k, v, dout, W, Z), want)


def test_one_key_for_all_and_broadcast_tensors():
    N, T, H, C = 2, 130, 4, 64
    q, k, v, dout = _inputs(N, T, H, 1, C, torch.bfloat16, 4)
    k1, v1 = k[:1, :1].detach().requires_grad_(True), v[:1, :1].detach().requires_grad_(True)
    out = streaming.sink_attention(q, k1.expand(N, T, 1, C), v1.expand(N, T, 1, C), 20, 1)
    dk, dv = torch.autograd.grad(out, [k1, v1], dout)
    want = O.attention(q, k1.detach().expand(N, T, 1, C), v1.detach().expand(N, T, 1, C), 20, 1, dout=dout)
    _near("out", out.detach(), want["out"])
    u = O.half_step(torch.bfloat16)
    for got, name in ((dk, "dk"), (dv, "dv")):               # torch sums the rows' gradients in fp32 and rounds once more
        value, bound = (x.sum((0, 1), keepdim=True) for x in want[name])
        _near(name, got, (value, bound + u * value.abs() + 2.0 ** -16 * want[name][0].abs().sum((0, 1), keepdim=True)))


def test_large_scores_and_a_scale():
    q, k, v, dout = _inputs(2, 200, 4, 2, 64, torch.bfloat16, 5, 3)
    q, k = q * 8, k * 8
    got = _train(q, k, v, dout, 50, 3, scale=0.37)
    _check(got, O.attention(q, k, v, 50, 3, scale=0.37, dout=dout))


def test_some_gradients_only_and_none():
    q, k, v, dout = _inputs(2, 90, 4, 2, 64, torch.float16, 6, 1)
    whole = _train(q, k, v, dout, 16, 1)
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        xs = [x.detach().requires_grad_(i == at) for i, x in enumerate((q, k, v))]
        assert torch.equal(torch.autograd.grad(streaming.sink_attention(*xs, 16, 1), xs[at], dout)[0], whole[name])
    assert not streaming.sink_attention(q, k, v, 16, 1).requires_grad


def test_the_gradients_are_not_differentiated_again():
    q, k, v, dout = _inputs(1, 40, 2, 2, 32, torch.bfloat16, 7)
    q.requires_grad_(True)
    out = streaming.sink_attention(q, k, v, 8)
    (dq,) = torch.autograd.grad(out, q, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dq.sum().backward()


def test_nothing_to_do():
    for N, T in ((0, 5), (3, 0)):
        q, k, v, dout = _inputs(N, T, 4, 2, 64, torch.bfloat16, 8)
        got = _train(q, k, v, dout, 3, 1)
        assert got["out"].shape == (N, T, 4, 64) and got["dk"].shape == (N, T, 2, 64)
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    q, k, v, dout = _inputs(2, 70, 4, 2, 64, torch.bfloat16, 8)
    assert not any(x.any() for x in _train(q, k, v, dout, 3, 1, t_valid=lengths).values())


def test_results_are_the_same_from_call_to_call_and_on_another_stream():
    q, k, v, dout = _inputs(2, 1000, 8, 2, 64, torch.bfloat16, 9, 4)
    first = _train(q, k, v, dout, 100, 4)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        second = _train(q, k, v, dout, 100, 4)
    stream.synchronize()
    assert all(torch.equal(first[n], second[n]) for n in first)


def test_a_captured_training_step():
    q, k, v, dout = _inputs(3, 300, 8, 2, 64, torch.bfloat16, 10, 2)
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))

    def step():
        out = streaming.sink_attention(q, k, v, 40, 2)
        return (out.detach(),) + torch.autograd.grad(out, [q, k, v], dout)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for _ in range(3):
            step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (11, 12, 13):
        with torch.no_grad():
            for x, new in zip((q, k, v, dout), _inputs(3, 300, 8, 2, 64, torch.bfloat16, seed, 2)):
                x.copy_(new)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_gradients_against_differences():
    """A step along a direction changes the sum of out * dout by the gradient's product with it."""
    q, k, v, dout = _inputs(2, 80, 4, 2, 32, torch.float16, 14, 2)
    got = _train(q, k, v, dout, 20, 2)
    g = torch.Generator().manual_seed(15)
    for i, name in enumerate(("dq", "dk", "dv")):
        x = (q, k, v)[i]
        along = torch.randn(x.shape, generator=g).cuda().double()
        value = lambda e: float((O.attention(*[y.double() + e * along if j == i else y.double() for j, y in enumerate((q, k, v))],  # noqa: E731
                                             20, 2)["out"][0] * dout.double()).sum())
        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        bound = O.attention(q, k, v, 20, 2, dout=dout)[name][1]
        assert abs(slope - float((got[name].double() * along).sum())) <= float((bound * along.abs()).sum()) + 1e-5 * abs(slope)
