"""Windowed causal attention with sinks in 64 bits by its formulas, with all pairs of a query and a key in memory; caches by a loop over
positions; and how far results in the kernels' number formats may be off.  Test infrastructure only."""
import torch

# fp32 work on a score of at most `s` in size, relative to a probability: sums of up to 128 products, a scale, a power of two
# to 2^-21, and row sums of up to 2^14 terms in a tree of chunks
FP32 = 2.0 ** -16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(t, u, window, sinks):
    """Whether the tokens at positions t see those at u."""
    t, u = t.unsqueeze(-1), u.unsqueeze(-2)
    return (u >= 0) & (u <= t) & ((t - u < window) | (u < sinks))


def softmax_rows(scores, seen):
    """Probabilities of what is seen; zeros for a row that sees nothing."""
    scores = scores.masked_fill(~seen, -torch.inf)
    high = scores.amax(-1, keepdim=True)
    e = torch.where(seen, (scores - high).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0)


def _heads(x, H):
    """[N, T, heads, C] in 64 bits as [N, H, T, C], every head as often as its group has heads."""
    x = x.double().transpose(1, 2)
    return x.repeat_interleave(H // x.shape[1], 1)


def attention(q, k, v, window, sinks=0, t_valid=None, scale=None, dout=None):
    """{"out", and with dout "dq", "dk", "dv"}: (value, how far a kernel's may be off), each like its tensor.

    The bounds count half steps u of the 16-bit type: a probability is rounded where it is multiplied (u) and divided by a sum of rounded ones
    (u); dS is rounded (u); an output is (u); delta = rowsum(dO O) has what O lost: u of it with fp16, and the byte that goes with
    bf16 leaves 2^-16; the fp32 work, FP32 times the size of a score."""
    N, T, H, C = q.shape
    K, dtype, u = k.shape[2], q.dtype, half_step(q.dtype)
    scale = C ** -0.5 if scale is None else scale
    real = torch.ones(N, T, dtype=torch.bool, device=q.device) if t_valid is None else torch.arange(T, device=q.device) < t_valid.unsqueeze(1)
    clean = lambda x: torch.where(real[:, :, None, None], x, torch.zeros_like(x))  # noqa: E731
    q_, k_, v_ = (_heads(clean(x), H) for x in (q, k, v))
    at = torch.arange(T, device=q.device)
    seen = visible(at, at, window, sinks) & real[:, None, :, None] & real[:, None, None, :]
    s = q_ @ k_.transpose(-1, -2) * scale
    p = softmax_rows(s, seen)
    f = FP32 * (1 + (q_.abs() @ k_.abs().transpose(-1, -2) * scale).amax().item())
    out, size = p @ v_, p @ v_.abs()
    got = {"out": (out, u * out.abs() + (2 * u + f) * size)}
    if dout is not None:
        g = _heads(clean(dout), H)
        dp, delta = g @ v_.transpose(-1, -2), (g * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        ddelta = ((2 * u + f) * (g.abs() * size) + ((u if dtype == torch.float16 else 2.0 ** -16) + f) * (g * out).abs()).sum(-1, keepdim=True)
        dds = p * (ddelta + f * (g.abs() @ v_.abs().transpose(-1, -2))) + (2 * u + f) * ds.abs()
        groups = lambda x: x.view(N, K, H // K, T, C).sum(2)  # noqa: E731
        dq, dk, dv = scale * ds @ k_, groups(scale * ds.transpose(-1, -2) @ q_), groups(p.transpose(-1, -2) @ g)
        got["dq"] = (dq, u * dq.abs() + scale * dds @ k_.abs())
        got["dk"] = (dk, u * dk.abs() + groups(scale * dds.transpose(-1, -2) @ q_.abs()))
        got["dv"] = (dv, u * dv.abs() + (2 * u + f) * groups(p.transpose(-1, -2) @ g.abs()))
    # What is too small for its format.  A power of two below fp32's (and bf16's) least normal value, 2^-126, is 0, and so is a dS or a result: each is off
    # by that at most.  fp16 rounds p, dS and results to multiples of 2^-24, half of one off.  A term's share counts times what it is multiplied by
    # (dP - delta and then k or q, or dout, or v), for every term of a sum.
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    most = lambda x: float(x.double().nan_to_num(0, 0, 0).abs().max()) if x.numel() else 0.0  # noqa: E731
    spread = 1 if dout is None else 1 + most(dp - delta)
    times = {"out": 1 + T * most(v_), "dq": 1 + 2 * scale * T * spread * most(k_), "dk": 1 + 2 * scale * T * H * spread * most(q_)}
    if dout is not None:
        times["dv"] = 1 + T * H * most(g)
    return {n: (a.transpose(1, 2), (b + least * times[n]).transpose(1, 2)) for n, (a, b) in got.items()}


def in_4_bits(x):
    """Rows as a cache in 4 bits holds them: codes, step and least value (as fp32 steps of the stated arithmetic), and the values in 64 bits."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((high.float() - low.float()) / 15).to(x.dtype)
    code = torch.where(step > 0, torch.round((x.float() - low.float()) / step.float()).clamp(0, 15), 0.0)
    return code, step, low, low.double() + code.double() * step.double()


def over_history(q, k, v, window, sinks, ends, scale=None, four=False):
    """The last tokens `q [N, n, H, C]` of sequences whose tokens have been `k[i], v[i] [>= ends[i], K, C]`: (value, how far a kernel's may be off).

    p is rounded where it meets v, in 16 bits (u sum p |v|); rows in 4 bits have p times the step rounded, which meets a code less 7.5
    (u sum p 7.5 step), and their scores and sums are made of parts up to 31 steps and |least| in size (fp32, counted in f)."""
    N, n, H, C = q.shape
    u, scale = half_step(q.dtype), C ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for i in range(N):
        end = max(0, int(ends[i]))
        t = torch.arange(end - n, end, device=q.device)
        at = torch.arange(end, device=q.device)
        seen = visible(t, at, window, sinks)
        if end == 0:
            continue
        values = lambda x: in_4_bits(x[:end])[3] if four else x[:end].double()  # noqa: E731
        wide = lambda x: (lambda c, s, low, _: 31 * s.double() + low.double().abs())(*in_4_bits(x[:end])).expand(x[:end].shape) if four else x[:end].double().abs()  # noqa: E731
        heads = lambda x: x.transpose(0, 1).repeat_interleave(H // x.shape[1], 0)  # noqa: E731
        qi = q[i].double().transpose(0, 1)
        p = softmax_rows(qi @ heads(values(k[i])).transpose(-1, -2) * scale, seen)
        o = p @ heads(values(v[i]))
        f = FP32 * (1 + (qi.abs() @ heads(wide(k[i])).transpose(-1, -2) * scale).amax().item())
        rounded = heads((7.5 * in_4_bits(v[i][:end])[1].double()).expand(v[i][:end].shape)) if four else heads(values(v[i]).abs())
        out[i] = o.transpose(0, 1)
        bound[i] = (u * o.abs() + u * (p @ rounded) + f * (p @ heads(wide(v[i])))).transpose(0, 1)
    least = 2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -126
    return out, bound + least * (1 + 16 * sum(x.shape[0] for x in v))


def centred(N, T, H, K, C, dtype, mean=0.0):
    """Standard normal q, k, v, dout, v with a mean."""
    g = torch.Generator().manual_seed(T + C)
    q, k, v, dout = (torch.randn(N, T, h, C, generator=g) for h in (H, K, K, H))
    return [x.to(dtype) for x in (q, k, v + mean, dout)]


def more_than_rounding(got, value):
    """By how much the error of `got`, as a norm, is more than that of the value's rounding, in half steps."""
    off, own, size = ((x.double() - value).norm() for x in (got, value.to(got.dtype), torch.zeros_like(value)))
    return float((off - own) / size) / half_step(got.dtype)


def rounded_gradients(q, k, v, window, sinks, dout, ds_once=False, p_once=False, bytes_lost=False, bytes_wrong=False):
    """A head's gradients with the roundings that a backward's kernels have, [1, T, 1, C]: probabilities where they meet v and in their sum, which the backward divides by, and results; and,
    if asked for, with those that they avoid."""
    dtype, C, u = q.dtype, q.shape[3], half_step(q.dtype)
    round_ = lambda x: x.float().to(dtype).double()  # noqa: E731
    q_, k_, v_, g = (x.double()[0, :, 0] for x in (q, k, v, dout))
    at = torch.arange(q.shape[1])
    seen, s = visible(at, at, window, sinks), q_ @ k_.t() * C ** -0.5
    e = torch.where(seen, (s - s.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True) + 0.3).exp(), 0.0)       # (a reference that is not quite the largest)
    total = round_(e).sum(-1, keepdim=True)
    p, out = e / total, round_(e) @ v_ / total
    if bytes_lost:
        out = round_(out)
    if bytes_wrong:
        out = round_(out) + (2 * torch.rand(out.shape, generator=torch.Generator().manual_seed(0), dtype=torch.float64) - 1) * u * out.abs()
    ds = p * (g @ v_.t() - (g * out).sum(-1, keepdim=True))
    ds, p = round_(ds) if ds_once else ds, round_(p) if p_once else p
    got = {"dq": ds @ k_ * C ** -0.5, "dk": ds.t() @ q_ * C ** -0.5, "dv": p.t() @ g}
    return {n: x.float().to(dtype)[None, :, None] for n, x in got.items()}
