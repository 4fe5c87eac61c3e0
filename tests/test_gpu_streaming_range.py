"""Attention of streams where numbers are large or small for their 16-bit type, against its formulas in 64 bits.

`u` is half a step of the type.  fp16 rounds below 2^-14 to multiples of 2^-24, half of one off; the kernels lift what they round: a product with a step of 4 bits so that the
largest step is 2^7 at least, so that it is off by 2^-32 of that step; a probability by 2^9, so that it is off by 2^-34 beside one of 1; P and dS of a backward by 2^10 unless dS is large."""
import pytest
import torch

from na1d_amd import streaming
from oracle import streaming_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["bf16", "fp16"]


def _near(got, value, bound):
    torch.cuda.synchronize()
    off = (got.double() - value).abs()
    if not bool((off <= bound).all()):
        worst = (off / bound).nan_to_num(torch.inf).argmax()
        pytest.fail("off by %.3g where %.3g is allowed, of %.3g" % (off.flatten()[worst], bound.flatten()[worst], value.flatten()[worst]))


# ------------------------------------------------------------------------------------------------ rows in 4 bits
def _over_four(q, k, v, W, Z, dtype, scale):
    """One token's attention over a cache in 4 bits that the others have been put into, what it should be, and how far off it may be:
    as over_history counts it, but for what is too small for fp16: 7.5 of 2^-32 of the largest step for every key, and half a step of the result's."""
    N, T, K, C = k.shape
    cache = streaming.new_cache(N, K, Z + W, C, 4, dtype)
    streaming.cache_append(k, v, *cache, sinks=Z)
    lengths = torch.full((N,), T, dtype=torch.int32, device="cuda")
    got = streaming.cache_attend(q, *cache, lengths, W, Z, scale=scale)
    value, bound = O.over_history(q, k, v, W, Z, [T] * N, scale=scale, four=True)
    largest = O.in_4_bits(v)[1].double().max().item()
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    bound = bound - least * (1 + 16 * N * T) + least + (7.5 * 2.0 ** -32 * largest * T if dtype == torch.float16 else 0.0)
    return got, value, bound


def _rising(N, T, K, C, dtype, octaves):
    """Keys whose scores, for queries of ones and a scale of 1 / C, rise by so many octaves from one unit of 64 keys to the next (a wave has every fourth)."""
    rise = torch.arange(T) // 64 * (octaves * 0.6931)
    return rise.view(1, T, 1, 1).expand(N, T, K, C).to(dtype).cuda().contiguous()


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,H,K,C,T,W", [(2, 4, 2, 32, 500, 400), (32, 32, 32, 32, 1200, 1200), (16, 64, 64, 64, 700, 700), (16, 64, 64, 96, 600, 590), (8, 64, 64, 128, 1000, 900),
                                         (2, 4, 2, 128, 2500, 2400)])
def test_wide_values_in_4_bits(N, H, K, C, T, W, dtype):
    """Scores that rise by less than what moves the softmax's reference, so that probabilities pass 1, and values whose steps are 1000 and more.  With many
    heads a wave has several units of a head's keys, one after the other."""
    g = torch.Generator().manual_seed(C)
    q = torch.ones(N, 1, H, C, dtype=dtype, device="cuda")
    v = (torch.randn(N, T, K, C, generator=g) * 4000).clamp(-65000, 65000)
    v[:, T // 2:, 1] *= 4                                              # ranges up to all that fp16 has
    v = v.clamp(-65000, 65000).to(dtype).cuda()
    for octaves in (1.45, 0.7, 0.0):
        got, value, bound = _over_four(q, _rising(N, T, K, C, dtype, octaves), v, W, 0, dtype, 1.0 / C)
        _near(got, value, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,H,K,C,T", [(2, 8, 2, 32, 500), (32, 64, 32, 32, 900), (2, 8, 2, 64, 1100), (16, 64, 64, 96, 600), (8, 64, 64, 128, 700)])
def test_steps_of_very_different_sizes_in_4_bits(N, H, K, C, T, dtype):
    g = torch.Generator().manual_seed(C)
    q, k = (torch.randn(N, t, h, C, generator=g).to(dtype).cuda() for t, h in ((1, H), (T, K)))
    order = torch.randperm(T, generator=g)
    for sizes in (2.0 ** (torch.arange(T) / T * 24 - 12), 2.0 ** (12 - torch.arange(T) / T * 24), (2.0 ** (torch.arange(T) / T * 24 - 12))[order]):
        v = (torch.randn(N, T, K, C, generator=g) * sizes.view(1, T, 1, 1)).to(dtype).cuda()
        got, value, bound = _over_four(q, k, v, T, 0, dtype, None)
        _near(got, value, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("size", [2.0 ** -10, 1.0])
def test_small_shares_in_4_bits(size, dtype):
    """A sink without a value takes nearly all of every row; what is left are products of small probabilities and, possibly, small steps."""
    N, H, K, C, T = 2, 4, 2, 64, 900
    q = torch.ones(N, 1, H, C, dtype=dtype, device="cuda")
    k, v = torch.zeros(N, T, K, C), torch.randn(1, 1, K, C, generator=torch.Generator().manual_seed(1)).expand(N, T, K, C) * size
    k[:, 0] = 8.3                                                      # e^-8.3 is 2^-12
    v = v.clone()
    v[:, 0] = 0.0
    got, value, bound = _over_four(q, k.to(dtype).cuda(), v.to(dtype).cuda(), T - 1, 1, dtype, 1.0 / C)
    assert float(value.abs().max()) > 0.05 * size
    _near(got, value, bound)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_rows_in_4_bits_to_the_ends_of_their_type(dtype):
    """What a finite row stands for is finite: its last code is not beyond the type's largest number where the step was rounded up."""
    largest, C, T = torch.finfo(dtype).max, 32, 64
    x = torch.zeros(1, T, 1, C)
    falls = (1 - torch.arange(T) / (4 * T)).view(1, T, 1, 1)
    x[..., 1::2] = largest if dtype == torch.bfloat16 else largest * falls
    # (bf16: a range that fp32 holds, 255.95 times 2^120 and less, a fifteenth of which is rounded from 17.06 to 17.125)
    x[..., ::2] = -largest / 255 * (0.7 + falls / 4) if dtype == torch.bfloat16 else -largest * falls
    x = x.to(dtype).cuda()
    cache = streaming.new_cache(1, 1, T, C, 4, dtype)
    streaming.cache_append(x, x, *cache)
    value = O.in_4_bits(x)[3]
    assert bool((value.to(dtype).double().abs() > largest).any())      # of these rows some would be
    for c in cache:
        got = streaming.cache_rows(c).transpose(1, 2)
        assert torch.equal(got, value.clamp(-largest, largest).to(dtype))


# ------------------------------------------------------------------------------------------------ small shares
def _sink_and_equals(N, T, H, K, C, dtype, share, rows):
    """A first token without a value that takes nearly all of every row, and others whose keys are alike, each with a probability of 2^share beside it."""
    q, k = torch.ones(N, T, H, C), torch.zeros(N, T, K, C)
    k[:, 0] = -share * 0.6931
    v = 1 + 0.1 * torch.randn(N, T, K, C, generator=torch.Generator().manual_seed(C))
    v[:, 0] = 0.0
    return [x.to(dtype).cuda() for x in (q[:, rows:], k, v)]


def _least(dtype, T, v):
    """Half a step of a result that is small for fp16, and 2^-34 of the largest value for every key (a probability of 1 being the largest at least)."""
    return 2.0 ** -25 + T * 2.0 ** -34 * float(v.abs().max()) if dtype == torch.float16 else 0.0


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("H,K,C,T,W", [(2, 1, 16, 700, 300), (2, 2, 32, 1500, 1500), (4, 1, 64, 2048, 2000), (3, 3, 96, 900, 900), (2, 1, 128, 1100, 700), (64, 8, 64, 2100, 2100)])
def test_small_shares(H, K, C, T, W, dtype):
    """Each probability is rounded by itself (half a step of it), as is their sum's share of it and the result: whatever their size beside the largest."""
    q, k, v = _sink_and_equals(1, T, H, K, C, dtype, -20.4, 0)
    assert torch.equal(q, torch.ones_like(q))
    u, f = O.half_step(dtype), O.FP32 * (1 + 20.4 * 0.6931)
    got = streaming.sink_attention(q, k, v, W, 1, scale=1.0 / C)
    value = O.attention(q[:, :, :1], k[:, :, :1], v[:, :, :1], W, 1, scale=1.0 / C)["out"][0]
    for h in range(K):                                                 # (heads differ in their values alone)
        if h:
            value = O.attention(q[:, :, :1], k[:, :, :1], v[:, :, h:h + 1], W, 1, scale=1.0 / C)["out"][0]
        for i in range(h * (H // K), (h + 1) * (H // K)):
            _near(got[:, :, i:i + 1], value, (3 * u + f) * value.abs() + _least(dtype, W, v))
    assert float(value.max()) > W * 2.0 ** -20.6 * 0.5


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("N,H,K,C,T,n", [(1, 4, 4, 64, 1028, 1), (2, 4, 2, 16, 1500, 1), (3, 8, 2, 128, 3000, 2), (2, 6, 2, 96, 900, 1), (40, 16, 16, 32, 1000, 1), (1, 64, 1, 32, 2000, 3)])
def test_small_shares_over_a_cache(N, H, K, C, T, n, dtype):
    q, k, v = _sink_and_equals(N, T, H, K, C, dtype, -20.4, T - n)
    cache = streaming.new_cache(N, K, T, C, 16, dtype)
    streaming.cache_append(k, v, *cache, sinks=1)
    got = streaming.cache_attend(q, *cache, torch.full((N,), T, dtype=torch.int32, device="cuda"), T - n, 1, scale=1.0 / C)
    value, _ = O.over_history(q, k, v, T - n, 1, [T] * N, scale=1.0 / C)
    u, f = O.half_step(dtype), O.FP32 * (1 + 20.4 * 0.6931)
    _near(got, value, (2 * u + f) * value.abs() + _least(dtype, T, v))


# ------------------------------------------------------------------------------------------------ gradients
def _gradients(q, k, v, dout, *args, **kw):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(streaming.sink_attention(q, k, v, *args, **kw), [q, k, v], dout)))


def _norms_near(got, want, more, part=slice(None)):
    """As norms: the rounding of the results themselves, as it comes out, and `more` of the whole."""
    torch.cuda.synchronize()
    for name, x in got.items():
        x, value = x[:, part], want[name][0][:, part]
        assert bool(x.isfinite().all()), name
        size, off, own = (float(y.norm()) for y in (value, x.double() - value, value.to(x.dtype).double() - value))
        assert off <= own + more * size, "%s: off by %.3g of it, its rounding %.3g and %.3g more allowed" % (name, off / size, own / size, more)


@pytest.mark.parametrize("power", [-16, -12, -8, 0, 6])
@pytest.mark.parametrize("H,K,C,T,W,Z", [(2, 1, 64, 4096, 4096, 0), (1, 1, 16, 4000, 4000, 3), (2, 2, 32, 3000, 2000, 100), (2, 1, 96, 2500, 2500, 1), (1, 1, 128, 4096, 3000, 4)])
def test_fp16_gradients_for_any_size_of_what_comes_back(H, K, C, T, W, Z, power):
    """Beside the results' rounding a delta has what the output's sum lost to roundings of probabilities: independent ones, half a step each at most, u / sqrt(3) of a term of its size;
    all else (two numbers for P and dS each, fp32) is below a twentieth of u."""
    g = torch.Generator().manual_seed(C)
    q, k, v, dout = (torch.randn(1, T, h, C, generator=g) for h in (H, K, K, H))
    q, k, v, dout = (x.to(torch.float16).cuda() for x in (q, 4 * k, v, 2.0 ** power * dout))
    u = O.half_step(torch.float16)
    _norms_near(_gradients(q, k, v, dout, W, Z), O.attention(q, k, v, W, Z, dout=dout), u * (3 ** -0.5 + 0.05))


@pytest.mark.parametrize("N,H,K,C,T,W,Z", [(1, 2, 1, 64, 500, 400, 0), (2, 4, 4, 16, 300, 300, 2), (1, 2, 2, 32, 700, 100, 5), (2, 4, 2, 96, 260, 260, 1), (4, 16, 8, 128, 513, 129, 66)])
def test_fp16_gradients_beyond_the_range_of_their_parts(N, H, K, C, T, W, Z):
    """dS is beyond 65504 in places where scale * dS * k is not."""
    g = torch.Generator().manual_seed(C)
    q, k, v, dout = (torch.randn(N, T, h, C, generator=g) for h in (H, K, K, H))
    q, k, v, dout = (x.to(torch.float16).cuda() for x in (2 * q, 0.5 * k, 8 * v, 4000 * dout))
    scale = 1 / 64
    want = O.attention(q, k, v, W, Z, scale=scale, dout=dout)
    q_, k_, v_, g_ = (x[:, :64].double().transpose(1, 2).repeat_interleave(H // x.shape[2], 1) for x in (q, k, v, dout))
    p = torch.softmax((q_ @ k_.transpose(-1, -2) * scale).masked_fill(~torch.ones(64, 64, dtype=torch.bool, device="cuda").tril(), -torch.inf), -1)
    dp = g_ @ v_.transpose(-1, -2)
    assert float((p * (dp - (p * dp).sum(-1, keepdim=True))).abs().max()) > 65504
    assert all(float(want[n][0].abs().max()) < 60000 for n in ("dq", "dk", "dv"))
    u = O.half_step(torch.float16)
    _norms_near(_gradients(q, k, v, dout, W, Z, scale=scale), want, u * (3 ** -0.5 + 0.05))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("H,K,C,T,W", [(2, 1, 16, 700, 300), (2, 2, 32, 1500, 1500), (4, 1, 64, 2048, 2000), (2, 1, 128, 1100, 700)])
def test_gradients_of_small_shares(H, K, C, T, W, dtype):
    """The keys beside a first token that takes nearly all of every row: their P and dS are 2^-20 of it."""
    q, k, v = _sink_and_equals(1, T, H, K, C, dtype, -20.4, 0)
    k[:, 1:] = (0.05 * torch.randn(1, T - 1, K, C, generator=torch.Generator().manual_seed(1))).to(dtype)
    dout = (1 + 0.1 * torch.randn(1, T, H, C, generator=torch.Generator().manual_seed(2))).to(dtype).cuda()
    want = O.attention(q, k, v, W, 1, scale=1.0 / C, dout=dout)
    got = _gradients(q, k, v, dout, W, 1, scale=1.0 / C)
    _norms_near({n: got[n] for n in ("dk", "dv")}, want, O.half_step(dtype) * (3 ** -0.5 + 0.05), slice(1, None))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("filler", [float("inf"), float("nan")])
def test_what_comes_back_infinite_stays_where_it_belongs(filler, dtype):
    """As where a loss's scale was too large: such gradients are no numbers, so that whoever looks for that finds it, and rows that have nothing to do with them are as without."""
    N, T, H, K, C, W = 2, 640, 4, 2, 64, 64
    g = torch.Generator().manual_seed(5)
    q, k, v, dout = (torch.randn(N, T, h, C, generator=g).to(dtype).cuda() for h in (H, K, K, H))
    clean = _gradients(q, k, v, dout, W)
    dout[0, 100, 1] = filler
    got = _gradients(q, k, v, dout, W)
    torch.cuda.synchronize()
    bad = torch.zeros(N, T, dtype=torch.bool, device="cuda")
    bad[0, 100] = True
    assert not bool(got["dq"][0, 100, 1].isfinite().any())
    assert torch.equal(got["dq"][~bad], clean["dq"][~bad]) and torch.equal(got["dq"][0, 100, [0, 2, 3]], clean["dq"][0, 100, [0, 2, 3]])
    for name in ("dk", "dv"):
        assert not bool(got[name][0, 37:101, 0].isfinite().any())
        assert torch.equal(got[name][1], clean[name][1]) and torch.equal(got[name][0, :, 1], clean[name][0, :, 1])
        assert torch.equal(got[name][0, 128:, 0], clean[name][0, 128:, 0])            # (strips of 64 keys that the row's chunk of queries does not see)


# ------------------------------------------------------------------------------------------------ large scores
@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("size", [300.0, 1500.0, 6000.0])
def test_scores_of_many_millions(size, dtype):
    """Where fp32 has few or no digits behind a score's point a row's output is the value of its largest score, if that is larger than the next by more than sums of 64 products are off by."""
    N, T, H, K, C, W, Z = 2, 300, 4, 2, 64, 250, 2
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(N, T, h, C, generator=g) for h in (H, K, K))
    q, k, v = (x.to(dtype).cuda() for x in (size * q, size * k, v))
    at = torch.arange(T, device="cuda")
    s = (q.double().transpose(1, 2) @ k.double().transpose(1, 2).repeat_interleave(H // K, 1).transpose(-1, -2) * C ** -0.5).masked_fill(~O.visible(at, at, W, Z), -torch.inf)
    top = s.topk(2, -1)
    off = 2.0 ** -20 * (q.double().abs().transpose(1, 2) @ k.double().abs().transpose(1, 2).repeat_interleave(H // K, 1).transpose(-1, -2) * C ** -0.5).amax(-1)
    clear = top.values[..., 0] - top.values[..., 1] > off + 12          # e^-12 is below half a step
    assert float(clear.double().mean()) > 0.8
    want = v.transpose(1, 2).repeat_interleave(H // K, 1).gather(2, top.indices[..., :1].expand(N, H, T, C))
    out = streaming.sink_attention(q, k, v, W, Z).transpose(1, 2)
    cache = streaming.new_cache(N, K, T, C, 16, dtype)
    streaming.cache_append(k, v, *cache, sinks=Z)
    step = streaming.cache_attend(q[:, -1:], *cache, torch.full((N,), T, dtype=torch.int32, device="cuda"), W, Z).transpose(1, 2)
    torch.cuda.synchronize()
    u = O.half_step(dtype)
    assert bool(out.isfinite().all()) and bool(step.isfinite().all())
    assert float((out.double() - want)[clear].abs().max()) < 2 * u * float(v.abs().max())
    assert float((step.double() - want[:, :, -1:])[clear[:, :, -1:]].abs().max()) < 2 * u * float(v.abs().max())


def test_a_captured_fp16_step_for_gradients_of_any_size():
    """What one replay's dS was taken down by is not the next one's."""
    N, T, H, K, C, W = 2, 300, 4, 2, 64, 100
    g = torch.Generator().manual_seed(7)
    q, k, v, base = (torch.randn(N, T, h, C, generator=g).to(torch.float16).cuda() for h in (H, K, K, H))
    q, k, v = (x.requires_grad_(True) for x in (q, k, v))
    dout = base.clone()

    def step():
        return torch.autograd.grad(streaming.sink_attention(q, k, v, W, 2), [q, k, v], dout)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for power in (11, -10, 0, 11, -12):
        dout.copy_(base * 2.0 ** power)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and all(bool(x.isfinite().all()) for x in want)
