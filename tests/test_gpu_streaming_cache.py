"""Attention over caches that hold what a window with sinks can see, in 16 bits and in 4, against the definition over all tokens in 64 bits."""
import pytest
import torch

from na1d_amd import _lib, streaming
from oracle import streaming_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["bf16", "fp16"]


def _tokens(N, T, H, K, C, dtype, seed, sinks=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(N, T, h, C, generator=g) for h in (H, K, K))
    q += 0.3
    k[:, :sinks] += 0.7
    return [x.to(dtype).cuda() for x in (q, k, v)]


def _near(got, want):
    torch.cuda.synchronize()
    value, bound = want
    off = (got.double() - value).abs()
    if not bool((off <= bound).all()):
        worst = (off / bound).nan_to_num(torch.inf).argmax()
        pytest.fail("off by %.3g where %.3g is allowed" % (off.flatten()[worst], bound.flatten()[worst]))


def _garbage(cache):
    """What no token has been put into may hold anything."""
    for t in cache if isinstance(cache, streaming.Rows4) else (cache,):
        t.copy_(torch.full(t.shape, 255, dtype=torch.uint8) if t.dtype == torch.uint8 else torch.full(t.shape, float("nan"), dtype=t.dtype))
    return cache


def _caches(N, K, S, C, bits, dtype):
    return [_garbage(c) for c in streaming.new_cache(N, K, S, C, bits, dtype)]


SHAPES = [  # N, heads, kv_heads, C, window, sinks, rows more than needed, tokens of a step, tokens in all
    (1, 1, 1, 32, 1, 0, 0, 1, 5), (2, 4, 2, 64, 7, 2, 0, 1, 40), (3, 2, 2, 32, 33, 1, 5, 2, 120), (2, 8, 2, 128, 64, 4, 0, 3, 201), (1, 6, 3, 96, 20, 30, 1, 5, 130),
    (2, 16, 1, 64, 100, 0, 0, 2, 260), (1, 24, 1, 32, 40, 3, 7, 3, 150), (1, 10, 2, 128, 50, 1, 0, 20, 240), (2, 64, 1, 64, 30, 2, 0, 2, 60),
]
SHAPES16 = [(2, 3, 3, 8, 5, 1, 0, 1, 30), (1, 4, 2, 24, 17, 2, 3, 2, 60), (2, 6, 2, 72, 65, 3, 0, 1, 150), (1, 2, 1, 104, 31, 0, 2, 4, 100), (2, 5, 5, 16, 9, 9, 0, 1, 40)]


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("bits,shape", [(16, s) for s in SHAPES + SHAPES16] + [(4, s) for s in SHAPES])
def test_a_stream_from_its_first_token(bits, shape, dtype):
    N, H, K, C, W, Z, more, n, T = shape
    q, k, v = _tokens(N, T, H, K, C, dtype, 1, Z)
    caches = _caches(N, K, Z + W + n - 1 + more, C, bits, dtype)
    lengths = torch.zeros(N, dtype=torch.int32, device="cuda")
    for t in range(0, T - n + 1, n):
        out = streaming.cache_step(q[:, t:t + n], k[:, t:t + n], v[:, t:t + n], *caches, lengths, W, Z)
        lengths += n
        if t < 3 * n or t % (7 * n) == 0 or t + 2 * n > T:
            _near(out, O.over_history(q[:, t:t + n], k, v, W, Z, lengths, four=bits == 4))
            assert torch.equal(out, streaming.cache_attend(q[:, t:t + n], *caches, lengths, W, Z))
    whole = O.attention(q, k, v, W, Z)["out"][0] if bits == 16 else None
    if whole is not None:
        last = T - T % n
        assert (out.double() - whole[:, last - n:last]).abs().max() < 0.1


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("H,K,C,W,Z,n", [(32, 8, 128, 1500, 4, 1), (8, 8, 64, 2000, 0, 1), (4, 2, 32, 5000, 100, 2), (12, 4, 96, 700, 3, 3), (2, 1, 128, 9000, 1, 4)])
def test_long_windows_and_streams_of_different_ages(H, K, C, W, Z, n, bits, dtype):
    """Several workgroups share a head's keys; streams that are idle, empty, younger than the window and long past it."""
    ages = [-1, 0, 1, W // 3, W + Z - 1, W + Z + 5, 2 * W + 77, 3 * W + 1]
    N, T = len(ages), max(ages) + n
    q, k, v = _tokens(N, T, H, K, C, dtype, 2, Z)
    caches = _caches(N, K, Z + W + n + 3, C, bits, dtype)
    lengths = torch.tensor(ages, dtype=torch.int32, device="cuda")
    streaming.cache_append(k, v, *caches, sinks=Z, t_valid=lengths)
    before = [t.clone() for c in caches for t in (c if bits == 4 else (c,))]
    at = lengths.clamp(min=0).long().view(N, 1) + torch.arange(n, device="cuda")
    new = [x.gather(1, at.view(N, n, 1, 1).expand(N, n, *x.shape[2:])) for x in (q, k, v)]
    out = streaming.cache_step(*new, *caches, lengths, W, Z)
    _near(out, O.over_history(new[0], k, v, W, Z, [a + n if a >= 0 else 0 for a in ages], four=bits == 4))
    for old, t in zip(before, [t for c in caches for t in (c if bits == 4 else (c,))]):
        assert torch.equal(old[0].view(torch.uint8), t[0].view(torch.uint8))             # the idle one
        assert int((old.view(torch.uint8) != t.view(torch.uint8)).any(-1).sum()) <= (N - 1) * K * n
    ended = torch.where(lengths < 0, lengths, lengths + n)
    assert torch.equal(out, streaming.cache_attend(new[0], *caches, ended, W, Z))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("bits", [16, 4])
def test_prompts_in_pieces(bits, dtype):
    """Pieces of any length leave what one append leaves, whatever of them is kept."""
    N, K, C, Z, S = 4, 3, 64, 5, 42
    _, k, v = _tokens(N, 200, K, K, C, dtype, 3)
    total = torch.tensor([200, 3, 0, 61], dtype=torch.int32, device="cuda")
    whole, pieces = _caches(N, K, S, C, bits, dtype), _caches(N, K, S, C, bits, dtype)
    streaming.cache_append(k, v, *whole, sinks=Z, t_valid=total)
    t = 0
    for size in (1, 2, 4, 33, 1, 60, 99):
        lengths, there = torch.full_like(total, t), (total - t).clamp(0, size)
        lengths[there == 0] = -1                                                          # a stream that has ended is idle
        streaming.cache_append(k[:, t:t + size], v[:, t:t + size], *pieces, lengths=lengths, sinks=Z, t_valid=there)
        t += size
    for a, b in zip(whole, pieces):
        for x, y in zip(a, b) if bits == 4 else ((a, b),):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    rows = [streaming.cache_rows(c) for c in whole]
    for i in range(N):
        L = int(total[i])
        for p in range(L):
            if p < Z or p >= L - (S - Z):
                row = p if p < Z else Z + (p - Z) % (S - Z)
                for r, x in zip(rows, (k, v)):
                    want = O.in_4_bits(x[i, p])[3].to(dtype) if bits == 4 else x[i, p]
                    assert torch.equal(r[i, :, row], want)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("C", [32, 64, 96, 128])
def test_rows_in_4_bits(C, dtype):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 50, 3, C, generator=g)
    x[0, 0] = 0.0
    x[0, 1] = -2.5
    x[0, 2] *= 1e-6
    x[0, 3] += 100.0
    x[0, 4] *= 1e3
    x[0, 5, :, 0] = 60000.0
    x[0, 6] = 0.0
    x[0, 6, :, 1] = -0.0
    x[1] = (x[1] * 4).round() / 4                            # halves between codes
    x = x.to(dtype).cuda()
    cache = streaming.new_cache(2, 3, 60, C, 4, dtype)
    streaming.cache_append(x, -x, *cache)
    for c, sign in zip(cache, (1, -1)):
        code, step, low, value = O.in_4_bits(sign * x)
        held = c.codes[:, :, :50].transpose(1, 2)
        assert torch.equal(torch.stack((held & 15, held >> 4), -1).flatten(-2), code.to(torch.uint8))
        assert torch.equal(c.ranges[:, :, :50].transpose(1, 2), torch.cat((step, low), -1))
        assert torch.equal(streaming.cache_rows(c)[:, :, :50].transpose(1, 2), value.float().to(dtype))
        assert not c.codes[:, :, 50:].any() and not c.ranges[:, :, 50:].any()


def test_caches_beyond_32_bits():
    """Heads' rows of 2^30 bytes each, more than 2^32 in all: the last rows of the last head."""
    N, K, C, W, Z = 5, 1, 128, 70, 2
    S = (1 << 29) // C
    _, k, v = _tokens(N, 200, 4, K, C, torch.bfloat16, 5)
    caches = streaming.new_cache(N, K, S, C)
    lengths = torch.tensor([S - 100, 0, 100, S + (S - Z) - 90, S - 150], dtype=torch.int32, device="cuda")
    streaming.cache_append(k, v, *caches, lengths=lengths, sinks=Z)
    q = _tokens(N, 1, 4, K, C, torch.bfloat16, 6)[0]
    out = streaming.cache_attend(q, *caches, lengths + 200, W, Z)
    # as a shorter stream: what was not appended is zeros, and the window's rows are what the last tokens left
    short = [[torch.cat((torch.zeros(100, K, C, dtype=x.dtype, device="cuda"), y)) for y in x] for x in (k, v)]
    for y, x in zip(short, (k, v)):
        y[1][:Z] = x[1, :Z]
    _near(out, O.over_history(q, *short, W, Z, [300] * N))
    assert torch.equal(caches[0][4, 0, S - 1], k[4, 149, 0]) and torch.equal(caches[0][4, 0, Z], k[4, 150, 0])


@pytest.mark.parametrize("bits", [16, 4])
def test_views_of_one_projection(bits):
    N, n, H, K, C, W, Z = 3, 2, 4, 2, 64, 20, 1
    q, k, v = _tokens(N, 60, H, K, C, torch.float16, 7)
    a, b = _caches(N, K, 40, C, bits, torch.float16), _caches(N, K, 40, C, bits, torch.float16)
    lengths = torch.tensor([50, 9, 0], dtype=torch.int32, device="cuda")
    qkv = torch.cat((q, k, v), 2)
    streaming.cache_append(k, v, *a, sinks=Z)
    streaming.cache_append(*qkv[:, :, H:].split([K, K], 2), *b, sinks=Z)
    first = streaming.cache_step(q[:, :n], k[:, 1:n + 1], v[:, 1:n + 1], *a, lengths, W, Z, scale=0.2)
    parts = torch.cat((q[:, :n], k[:, 1:n + 1], v[:, 1:n + 1]), 2).split([H, K, K], 2)
    assert torch.equal(first, streaming.cache_step(*parts, *b, lengths, W, Z, scale=0.2))
    flipped = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in parts]
    assert torch.equal(first, streaming.cache_step(*flipped, *b, lengths, W, Z, scale=0.2))
    odd = [torch.cat((x.flatten()[:1], x.flatten()))[1:].view(x.shape) for x in parts]
    assert torch.equal(first, streaming.cache_step(*odd, *b, lengths, W, Z, scale=0.2))


@pytest.mark.parametrize("bits", [16, 4])
def test_captured_steps_go_on_from_each_other(bits):
    """Two graphs of one stream's steps, replayed in turn, with the lengths counted up inside them."""
    N, H, K, C, W, Z = 2, 8, 2, 64, 600, 3
    q, k, v = _tokens(N, 900, H, K, C, torch.bfloat16, 8, Z)
    caches, again = _caches(N, K, Z + W, C, bits, torch.bfloat16), _caches(N, K, Z + W, C, bits, torch.bfloat16)
    lengths = torch.full((N,), 880, dtype=torch.int32, device="cuda")
    streaming.cache_append(k[:, :880], v[:, :880], *caches, sinks=Z)
    streaming.cache_append(k[:, :880], v[:, :880], *again, sinks=Z)
    token = [x[:, 880:881].clone() for x in (q, k, v)]

    def step():
        out = streaming.cache_step(*token, *caches, lengths, W, Z)
        lengths.add_(1)
        return out

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        streaming.cache_step(*token, *caches, lengths, W, Z)
    stream.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    lengths.fill_(880)
    for t in range(880, 890):
        for x, y in zip(token, (q, k, v)):
            x.copy_(y[:, t:t + 1])
        graph, out = graphs[t % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = streaming.cache_step(q[:, t:t + 1], k[:, t:t + 1], v[:, t:t + 1], *again, torch.full_like(lengths, t), W, Z)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    _near(want, O.over_history(q[:, 889:890], k, v, W, Z, [890, 890], four=bits == 4))


def test_a_prompt_and_what_follows():
    """A run of them together: the prompt's layer, its append, then steps, against the layer over the whole sequence."""
    N, H, K, C, W, Z, T, P = 2, 8, 2, 64, 50, 2, 160, 120
    q, k, v = _tokens(N, T, H, K, C, torch.bfloat16, 9, Z)
    want = O.attention(q, k, v, W, Z)["out"]
    caches = streaming.new_cache(N, K, Z + W + 3, C)
    with torch.no_grad():
        outs = [streaming.sink_attention(q[:, :P], k[:, :P], v[:, :P], W, Z)]
        streaming.cache_append(k[:, :P], v[:, :P], *caches, sinks=Z)
        lengths = torch.full((N,), P, dtype=torch.int32, device="cuda")
        for t in range(P, T, 4):
            outs.append(streaming.cache_step(q[:, t:t + 4], k[:, t:t + 4], v[:, t:t + 4], *caches, lengths, W, Z))
            lengths += 4
    _near(torch.cat(outs, 1), want)


def test_nothing_to_do():
    q, k, v = _tokens(2, 4, 4, 2, 64, torch.bfloat16, 10)
    caches = _caches(2, 2, 10, 64, 16, torch.bfloat16)
    before = [c.clone() for c in caches]
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    streaming.cache_append(k[:, :0], v[:, :0], *caches)
    streaming.cache_append(k, v, *caches, t_valid=zero)
    streaming.cache_append(k, v, *caches, lengths=zero - 1)
    assert streaming.cache_step(q[:, :0], k[:, :0], v[:, :0], *caches, zero, 5).shape == (2, 0, 4, 64)
    for idle in (zero - 1, zero - 2 ** 31, zero + 2 ** 31 - 1):
        assert not streaming.cache_step(q, k, v, *caches, idle, 5).any()
    assert not streaming.cache_attend(q, *caches, zero, 5).any()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(caches, before))
    none = streaming.new_cache(0, 2, 10, 64)
    assert streaming.cache_step(q[:0], k[:0], v[:0], *none, zero[:0], 5).shape == (0, 4, 4, 64)
    assert streaming.cache_rows(streaming.new_cache(0, 2, 10, 64, 4)[0]).shape == (0, 2, 10, 64)


def test_there_is_no_gradient():
    q, k, v = _tokens(1, 2, 4, 2, 64, torch.bfloat16, 11)
    caches = streaming.new_cache(1, 2, 10, 64)
    lengths = torch.zeros(1, dtype=torch.int32, device="cuda")
    with pytest.raises(_lib.NA1DError, match="no gradient"):
        streaming.cache_step(q.requires_grad_(True), k, v, *caches, lengths, 5)
    with torch.no_grad():
        streaming.cache_step(q, k, v, *caches, lengths, 5)
