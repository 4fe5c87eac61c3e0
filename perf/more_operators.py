"""Attention of unbounded streams, as cases for timing: a causal window of any length with a few first tokens that stay visible
(sinks), in training, over prompts and a few tokens at a time over a cache, and the same over a cache held in 4 bits.

  attend    streaming.sink_attention: whole sequences, forward, or forward and backward ("train")
  step      streaming.cache_step: `new` tokens to a sequence are stored in a 16-bit cache and attend to it
  attend4   streaming.cache_attend: the last `new` tokens attend to a cache held in 4 bits that has them already
  fill4     streaming.cache_append into a cache held in 4 bits, and its content by streaming.cache_rows

`heads` are the queries' heads, `kv_heads` those of keys and values.  "ragged" says that sequences have lengths of their own, some
of them none (attend), or have seen anything from nothing to three times what the cache holds, one of them being idle (the others).

A cache has `capacity` rows to a head: position p is in row p where p < sinks, else in row sinks + (p - sinks) % (capacity - sinks).
In 4 bits a row is codes, two to a byte (the even channel low), with the row's lowest value and a fifteenth of its range, both in
the type of the rows.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_SCORES = 3.0e9                  # scores that the plain form of a drawn case of whole sequences has in memory
MOST_PAIRS = 3.2e10                  # visible pairs of query and key times head_dim / 64 of such a case, a training step's three times
MOST_CACHE = 6.0e8                   # values of a cache's keys


def _case(name, kind, dtype, batch, T, heads, kv_heads, head_dim, window, sinks, train=False, ragged=False, new=1, capacity=0):
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "T": T, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "window": window, "sinks": sinks, "train": train, "ragged": ragged, "new": new, "capacity": capacity}


def listed():
    return [
        # one utterance of 3 s through a streaming layer: nothing but latency
        _case("prompt_utterance", "attend", "bf16", 1, 300, 4, 4, 64, 100, 1),
        # prompts of different lengths, everything odd, a sequence that is empty
        _case("prompts_ragged", "attend", "fp16", 6, 1237, 12, 3, 72, 333, 5, ragged=True),
        # a long prompt of a wide model, four query heads to a key head
        _case("prompt_long", "attend", "bf16", 1, 16384, 32, 8, 128, 2048, 4),
        # a training step's layer on crops of 10 s, a key head to every query head
        _case("train_batch", "attend", "bf16", 16, 1000, 16, 16, 64, 128, 1, train=True),
        # a training step with lengths, odd sizes and grouped heads
        _case("train_ragged", "attend", "fp16", 5, 777, 10, 2, 96, 100, 3, train=True, ragged=True),
        # long context in training, grouped heads
        _case("train_long", "attend", "bf16", 2, 8192, 16, 4, 128, 1024, 16, train=True),
        # the next frame of one stream
        _case("step_one", "step", "bf16", 1, 0, 4, 4, 64, 1024, 4, capacity=1028),
        # a few frames at a time for streams that began at different times, an idle one among them, odd sizes
        _case("step_ragged", "step", "fp16", 7, 0, 12, 4, 80, 777, 2, ragged=True, new=3, capacity=781),
        # the next token of many streams: what bounds it is memory
        _case("step_batch", "step", "bf16", 64, 0, 32, 8, 128, 4096, 4, capacity=4100),
        # a few streams, odd sizes, two tokens at a time
        _case("attend4_ragged", "attend4", "fp16", 5, 0, 8, 2, 64, 2000, 7, ragged=True, new=2, capacity=2008),
        # many streams with a long window
        _case("attend4_batch", "attend4", "bf16", 64, 0, 32, 8, 128, 8192, 4, capacity=8196),
        # prompts of different lengths go into the cache, some of them longer than it is
        _case("fill4_ragged", "fill4", "bf16", 8, 5000, 8, 8, 128, 4000, 4, ragged=True, capacity=4010),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "step", "step", "attend4", "attend4", "fill4"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 8]) if kind != "fill4" else 1
    four = kind in ("attend4", "fill4")
    head_dim = rng.choice([32, 64, 96, 128, 128]) if four else rng.choice([64, 128, 8 * rng.randint(2, 16)])
    sinks = rng.choice([0, 1, 4, rng.randint(2, 64)])
    ragged, dtype = rng.random() < 0.4, rng.choice(["bf16", "fp16"])
    heads = group * kv_heads
    case = _case("", kind, dtype, 1, 0, heads, kv_heads, head_dim, 0, sinks, ragged=ragged)
    if kind == "attend":
        case["train"] = rng.random() < 0.6
        case["T"] = T = _log(rng, 1, 16384)
        case["window"] = window = _log(rng, 16, 2048) if T > 2048 else _log(rng, 1, 2048)
        block = min(window, T)
        pairs = T * block * heads * head_dim / 64 * (3 if case["train"] else 1)
        case["batch"] = _log(rng, 1, max(1, min(64, int(MOST_PAIRS / pairs), int(MOST_SCORES / (2 * T * block * heads)))))
    else:
        most = 16384 if four else 8192
        case["window"] = window = _log(rng, 16, most)
        case["new"] = new = 1 if rng.random() < 0.6 else rng.randint(2, 8)
        case["capacity"] = capacity = sinks + window + new - 1 + rng.choice([0, 0, rng.randint(1, 64)])
        case["batch"] = _log(rng, 1, max(1, min(128, int(MOST_CACHE * (1.0 if kind != "fill4" else 0.1) / (capacity * kv_heads * head_dim)))))
        if kind == "fill4":
            case["T"] = _log(rng, 1, 2 * capacity)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ preparation
def _lengths(case):
    """What the sequences have: tokens (attend), tokens to store (fill4), or tokens that the cache has seen; -1: idle."""
    B = case["batch"]
    if case["kind"] in ("attend", "fill4"):
        if not case["ragged"]:
            return [case["T"]] * B
        return [0 if b == 0 and B > 3 else max(1, case["T"] * (B - b) // B) for b in range(B)]
    if not case["ragged"]:
        return [case["capacity"] + 17 * b for b in range(B)]
    return [-1 if b == 0 and B > 3 else 0 if b == 1 and B > 3 else 1 + 3 * case["capacity"] * b // B for b in range(B)]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, kind = DTYPES[case["dtype"]], case["kind"]
    B, T, H, K, D, S = case["batch"], case["T"], case["heads"], case["kv_heads"], case["head_dim"], case["capacity"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    # Queries lean towards one direction of their head, and the first tokens' keys have twice as much of it: that is how
    # first tokens come to hold a large part of every row.
    lean = 0.5 * normal(K, D)
    order = torch.randperm(B, generator=gen, device=dev)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)[order].contiguous()
    s = {"case": case, "lengths": lengths}
    if kind == "attend":
        # views of one projection's output, as a layer has them
        qkv = normal(B, T, H + 2 * K, D)
        qkv[:, :, :H] += lean.repeat_interleave(H // K, 0)
        qkv[:, :case["sinks"], H:H + K] += 2 * lean
        qkv = qkv.to(dtype)
        for name, part in zip("qkv", qkv.split([H, K, K], 2)):
            s[name] = part.detach().requires_grad_(case["train"])
        if case["train"]:
            s["dout"] = normal(B, T, H, D).to(dtype)
        return s
    n = case["new"]
    if kind == "fill4":
        s["k"], s["v"] = normal(B, T, K, D).to(dtype), normal(B, T, K, D).to(dtype)
        s["start"] = torch.zeros_like(lengths)
    else:
        s["q"] = (normal(B, n, H, D) + lean.repeat_interleave(H // K, 0)).to(dtype)
        if kind == "step":
            s["k"], s["v"] = normal(B, n, K, D).to(dtype), normal(B, n, K, D).to(dtype)
    k, v = normal(B, K, S, D), normal(B, K, S, D)
    k[:, :, :case["sinks"]] += 2 * lean.unsqueeze(1)
    k, v = k.to(dtype), v.to(dtype)
    if kind == "step":
        s["k_cache"], s["v_cache"] = k, v
    else:
        s["rows"] = (k, v) if kind == "attend4" else ()
        s["k_cache"], s["v_cache"] = _packed(k), _packed(v)
    return s


def _quantized(x):
    """Codes, the step from one to the next, and the lowest value of rows."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step = ((high.float() - low.float()) / 15).to(x.dtype)
    code = torch.round((x.float() - low.float()) / step.float()).clamp(0, 15)
    return torch.where(step > 0, code, torch.zeros_like(code)), step, low


def _packed(x):
    code, step, low = _quantized(x)
    code = code.to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat((step, low), -1)


def _values(codes, ranges):
    code = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return ranges[..., 1:].float() + code * ranges[..., :1].float()


def _streaming():
    path = os.path.abspath("pcf-nat_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from na1d_amd import streaming
    return streaming


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case, f = s["case"], _streaming()
    if case["kind"] == "attend":
        t_valid = s["lengths"] if case["ragged"] else None
        if not case["train"]:
            return {"out": f.sink_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"], t_valid=t_valid)}
        with torch.enable_grad():
            out = f.sink_attention(s["q"], s["k"], s["v"], case["window"], case["sinks"], t_valid=t_valid)
        dq, dk, dv = torch.autograd.grad(out, [s["q"], s["k"], s["v"]], s["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if case["kind"] == "step":
        out = f.cache_step(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["lengths"], case["window"], case["sinks"])
        return {"out": out, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    k_cache, v_cache = f.Rows4(*s["k_cache"]), f.Rows4(*s["v_cache"])
    if case["kind"] == "attend4":
        return {"out": f.cache_attend(s["q"], k_cache, v_cache, s["lengths"], case["window"], case["sinks"])}
    f.cache_append(s["k"], s["v"], k_cache, v_cache, s["start"], case["sinks"], t_valid=s["lengths"])
    return {"k": f.cache_rows(k_cache), "v": f.cache_rows(v_cache)}


def _run_plain(s):
    """The definitions in 32 bits."""
    with torch.no_grad():
        return {"attend": _attend_plain, "step": _step_plain, "attend4": _attend4_plain, "fill4": _fill4_plain}[s["case"]["kind"]](s)


def _attend_plain(s):
    """Queries in blocks as long as the window, each against the block's keys, the block's before and the sinks."""
    case = s["case"]
    B, T, H, K, D, W = (case[n] for n in ("batch", "T", "heads", "kv_heads", "head_dim", "window"))
    dev, dtype, G, scale = s["q"].device, s["q"].dtype, H // K, D ** -0.5
    w = min(W, T)
    nb = -(-T // w)
    Z = min(case["sinks"], T)
    real = torch.arange(T, device=dev) < s["lengths"].unsqueeze(1)                        # [B, T]

    def blocks(x):                                                                        # [B, T, H, D] -> [B, K, blocks, G * w, D]
        x = torch.where(real[:, :, None, None], x, torch.zeros_like(x)).float()
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nb * w - T))
        return x.view(B, nb, w, K, G, D).permute(0, 3, 1, 4, 2, 5).reshape(B, K, nb, G * w, D)

    def unblocks(x):
        return x.view(B, K, nb, G, w, D).permute(0, 2, 4, 1, 3, 5).reshape(B, nb * w, H, D)[:, :T]

    def keys(x):                                                                          # [B, T, K, D] -> [B, K, w + blocks * w, D]
        x = torch.where(real[:, :, None, None], x, torch.zeros_like(x)).float()
        return torch.nn.functional.pad(x.transpose(1, 2), (0, 0, w, nb * w - T))

    def pairs(x):                                                                         # a block's keys: [B, K, blocks, 2 * w, D]
        x = x.view(B, K, nb + 1, w, D)
        return torch.cat((x[:, :, :-1], x[:, :, 1:]), 3)

    q, k, v = blocks(s["q"]), keys(s["k"]), keys(s["v"])
    ks, vs = k[:, :, None, w:w + Z], v[:, :, None, w:w + Z]
    kb, vb = pairs(k), pairs(v)
    t = torch.arange(nb * w, device=dev).view(nb, 1, w, 1)
    u = (torch.arange(nb, device=dev) * w - w).view(nb, 1, 1, 1) + torch.arange(2 * w, device=dev)
    near = ((u >= 0) & (u <= t) & (t - u < W)).expand(nb, G, w, 2 * w).reshape(nb, G * w, 2 * w)
    z = torch.arange(Z, device=dev)
    far = (t - z >= W).expand(nb, G, w, Z).reshape(nb, G * w, Z)
    scores = torch.cat((torch.matmul(q, ks.transpose(-1, -2)), torch.matmul(q, kb.transpose(-1, -2))), -1) * scale
    scores = scores.masked_fill_(~torch.cat((far, near), -1), -torch.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :Z], vs) + torch.matmul(p[..., Z:], vb)
    out = torch.where(real[:, :, None, None], unblocks(o), 0.0).to(dtype)
    if not case["train"]:
        return {"out": out}
    g = blocks(s["dout"])
    ds = torch.cat((torch.matmul(g, vs.transpose(-1, -2)), torch.matmul(g, vb.transpose(-1, -2))), -1)
    ds -= (g * o).sum(-1, keepdim=True)
    ds *= p
    ds *= scale
    dq = torch.matmul(ds[..., :Z], ks) + torch.matmul(ds[..., Z:], kb)

    def of_keys(p, x):
        both = torch.matmul(p[..., Z:].transpose(-1, -2), x).view(B, K, nb, 2, w, D)
        d = both[:, :, :, 1].reshape(B, K, nb * w, D)
        d[:, :, :-w] += both[:, :, 1:, 0].reshape(B, K, (nb - 1) * w, D)
        d[:, :, :Z] += torch.matmul(p[..., :Z].transpose(-1, -2), x).sum(2)
        return d[:, :, :T].transpose(1, 2).to(dtype)

    return {"out": out, "dq": unblocks(dq).to(dtype), "dk": of_keys(ds, q), "dv": of_keys(p, g)}


def _cache_plain(s, k, v, end):
    """The last `new` of `end` tokens attend to a cache whose rows are k and v, in 32 bits."""
    case = s["case"]
    B, n, H, K, D, W, S, Z = (case[x] for x in ("batch", "new", "heads", "kv_heads", "head_dim", "window", "capacity", "sinks"))
    dev, G = k.device, H // K
    row = torch.arange(S, device=dev)
    end = end.long().view(B, 1)
    last = end - 1 - (end - 1 - row) % (S - Z)                                             # the newest position that row has
    position = torch.where(row < Z, row, last)
    position = torch.where((row >= Z) & (last < Z), -1, position).view(B, 1, 1, 1, S)
    t = (end - n + torch.arange(n, device=dev)).view(B, 1, 1, n, 1)
    seen = (position >= 0) & (position <= t) & ((t - position < W) | (position < Z))
    q = s["q"].float().view(B, n, K, G, D).permute(0, 2, 3, 1, 4).reshape(B, K, G * n, D)
    scores = torch.matmul(q, k.transpose(-1, -2)).view(B, K, G, n, S) * D ** -0.5
    scores = scores.masked_fill_(~seen, -torch.inf)
    high = scores.amax(-1, keepdim=True)
    p = torch.where(seen, (scores - high).exp(), 0.0)
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0).view(B, K, G * n, S)
    return torch.matmul(p, v).view(B, K, G, n, D).permute(0, 3, 1, 2, 4).reshape(B, n, H, D).to(s["q"].dtype)


def _step_plain(s):
    case = s["case"]
    B, n, S, Z = (case[x] for x in ("batch", "new", "capacity", "sinks"))
    busy = s["lengths"] >= 0
    position = s["lengths"].clamp(min=0).long().view(B, 1) + torch.arange(n, device=s["q"].device)
    row = torch.where(position < Z, position, Z + (position - Z) % (S - Z))
    b = torch.arange(B, device=row.device).view(B, 1)
    for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        cache[b, :, row] = torch.where(busy.view(B, 1, 1, 1), new, cache[b, :, row])
    end = torch.where(busy, s["lengths"] + n, -1)
    return {"out": _cache_plain(s, s["k_cache"].float(), s["v_cache"].float(), end), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend4_plain(s):
    return {"out": _cache_plain(s, _values(*s["k_cache"]), _values(*s["v_cache"]), s["lengths"])}


def _fill4_plain(s):
    case = s["case"]
    B, K, D, S, Z = (case[x] for x in ("batch", "kv_heads", "head_dim", "capacity", "sinks"))
    row = torch.arange(S, device=s["k"].device)
    end = s["lengths"].long().view(B, 1)
    position = torch.where(row < Z, row, end - 1 - (end - 1 - row) % (S - Z))
    stored = ((position >= 0) & (position < end) & ((row < Z) | (position >= Z))).view(B, 1, S, 1)
    index = position.clamp(0, case["T"] - 1).view(B, S, 1, 1).expand(B, S, K, D)

    def filled(new, cache):
        code, step, low = _quantized(new.gather(1, index).transpose(1, 2))
        return torch.where(stored, low.float() + code * step.float(), _values(*cache)).to(new.dtype)

    return {"k": filled(s["k"], s["k_cache"]), "v": filled(s["v"], s["v_cache"])}


# ------------------------------------------------------------------------------------------------ definition in 64 bits
def _exact_row_values(x):
    """What rows stand for once they are held in 4 bits."""
    a = x.double()
    low = a.min(-1, keepdim=True).values
    step = ((a.max(-1, keepdim=True).values - low) / 15).to(x.dtype).double()
    return torch.where(step > 0, low + step * torch.round((a - low) / torch.where(step > 0, step, 1.0)).clamp(0, 15), low)


def exact(case, seed):
    """A head of a sequence at a time, with all pairs of a query and a key; gradients by automatic differentiation."""
    s = prepare(case, seed)
    B, H, K, W, Z, n = (case[x] for x in ("batch", "heads", "kv_heads", "window", "sinks", "new"))
    G = H // K
    lengths = s["lengths"].tolist()

    def attention(q, k, v, t, u):
        seen = (u <= t[:, None]) & ((u > t[:, None] - W) | (u < Z))
        a = (q @ k.t()) / math.sqrt(q.shape[-1])
        return torch.softmax(a.masked_fill(~seen, -torch.inf), 1) @ v

    if case["kind"] == "attend":
        got = {x: torch.zeros(s[y].shape, dtype=torch.float64, device=s[y].device) for x, y in
               (("out", "q"),) + ((("dq", "q"), ("dk", "k"), ("dv", "v")) if case["train"] else ())}
        for b in range(B):
            L = lengths[b] if case["ragged"] else case["T"]
            at = torch.arange(L, device=s["q"].device)
            for h in range(H if L else 0):
                q, k, v = (x[b, :L, i].detach().double().requires_grad_(case["train"]) for x, i in ((s["q"], h), (s["k"], h // G), (s["v"], h // G)))
                with torch.set_grad_enabled(case["train"]):
                    o = attention(q, k, v, at, at)
                got["out"][b, :L, h] = o.detach()
                if case["train"]:
                    dq, dk, dv = torch.autograd.grad(o, [q, k, v], s["dout"][b, :L, h].double())
                    got["dq"][b, :L, h] = dq
                    got["dk"][b, :L, h // G] += dk
                    got["dv"][b, :L, h // G] += dv
        return got

    S = case["capacity"]

    def row_of(p):
        return p if p < Z else Z + (p - Z) % (S - Z)

    if case["kind"] == "fill4":
        got = {}
        for name in "kv":
            codes, ranges = s[name + "_cache"]
            wide = torch.empty(codes.shape[:-1] + (2 * codes.shape[-1],), dtype=torch.float64, device=codes.device)
            wide[..., ::2], wide[..., 1::2] = (codes % 16).double(), (codes // 16).double()
            got[name] = wide.mul_(ranges[..., :1].double()).add_(ranges[..., 1:].double())
            for b in range(B):
                held = [p for p in range(lengths[b]) if p < Z or p >= lengths[b] - (S - Z)]
                if held:
                    got[name][b][:, [row_of(p) for p in held]] = _exact_row_values(s[name][b, held].transpose(0, 1))
        return got

    if case["kind"] == "step":
        k_all, v_all = s["k_cache"].double(), s["v_cache"].double()
        for b in range(B):
            if lengths[b] >= 0:
                rows = [row_of(lengths[b] + i) for i in range(n)]
                k_all[b][:, rows], v_all[b][:, rows] = s["k"][b].transpose(0, 1).double(), s["v"][b].transpose(0, 1).double()
        ends = [x + n if x >= 0 else 0 for x in lengths]
    else:
        k_all, v_all = (_exact_row_values(x) for x in s["rows"])
        ends = lengths
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(B):
        first = max(0, ends[b] - n)
        held = [p for p in range(max(0, ends[b])) if p < Z or p >= ends[b] - (S - Z)]
        if not held:
            continue
        rows = torch.tensor([row_of(p) for p in held], device=out.device)
        u, t = torch.tensor(held, device=out.device), torch.arange(first, ends[b], device=out.device)
        for h in range(H):
            q = s["q"][b, n - (ends[b] - first):, h].double()
            out[b, n - (ends[b] - first):, h] = attention(q, k_all[b, h // G, rows], v_all[b, h // G, rows], t, u)
    return {"out": out, "k_cache": k_all, "v_cache": v_all} if case["kind"] == "step" else {"out": out}


def work(case):
    """The pairs of a query and a key that see each other: 2 products forward, 5 more backward (probabilities are not kept)."""
    B, T, H, K, D, W, Z, S, n = (case[x] for x in ("batch", "T", "heads", "kv_heads", "head_dim", "window", "sinks", "capacity", "new"))
    lengths = _lengths(case)

    def seen(t):                                                                          # keys of queries at positions t
        return float((np.minimum(t + 1, W) + np.maximum(0, np.minimum(Z, t + 1 - W))).sum())

    if case["kind"] == "attend":
        pairs, tokens = sum(seen(np.arange(x)) for x in lengths), sum(lengths)
        times = 3 if case["train"] else 1                                                 # q, k, v, dout, dq, dk, dv, and out
        rows = 2.0 * D * (tokens * ((H + 2 * K) + (2 * H + 2 * K if case["train"] else 0)) + B * T * H)
        return {"bytes": rows, "flops": 4.0 * D * H * pairs * (3.5 if times == 3 else 1.0)}
    if case["kind"] == "fill4":
        held = sum(min(x, S) for x in lengths)
        return {"bytes": 2.0 * K * (held * (2 * D + D / 2 + 4) + B * S * (D / 2 + 4 + 2 * D)), "flops": 8.0 * K * D * (held + B * S)}
    ends = [x + n if x >= 0 else 0 for x in lengths] if case["kind"] == "step" else [max(0, x) for x in lengths]
    pairs = sum(seen(np.arange(max(0, e - n), e)) for e in ends)
    held = sum(min(e, W + n - 1 + min(Z, max(0, e - W - n + 1))) for e in ends)
    row = 2.0 * D if case["kind"] == "step" else D / 2 + 4.0
    return {"bytes": 2.0 * K * held * row + 4.0 * B * n * H * D + (4.0 * K * D * B * n if case["kind"] == "step" else 0.0), "flops": 4.0 * D * H * pairs}
