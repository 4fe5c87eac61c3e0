"""Losses over a large number of classes without the logits in memory, as cases for timing: what a training step of a
speaker-embedding model has behind its embeddings, and the same heads at the sizes of a vocabulary.

  ce        linear_cross_entropy: softmax cross entropy of a linear head
  margin    margin_cross_entropy: additive angular margin on cosines, `subcenters` weight rows to a class
  distil    linear_distillation: divergence from a teacher that left its `top` largest logits of each row

"train" says that a pass runs the backward too and returns the gradients of the rows and of the weight; the upstream gradient
is 1 with bf16 and, with fp16, a loss scale that keeps a row's share at about 16.  "ragged" says that some rows have no target
(ce, margin), or that rows have teachers of different lengths, some of them none (distil).
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST_PRODUCTS = 8192 * 1024 * 65536          # rows * weight rows * channels of a drawn case
MOST_LOGITS = 8192 * 65536                   # rows * weight rows
IGNORE = -100
SINE_FLOOR = 1e-6                            # of the squared sine in the margin's derivative


def _case(name, kind, dtype, rows, dim, classes, train, ragged=False, subcenters=1, top=0, temperature=1.0, reduction="mean"):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "dim": dim, "classes": classes, "train": train,
            "ragged": ragged, "subcenters": subcenters, "top": top, "temperature": temperature, "reduction": reduction}


def listed():
    return [
        # the log likelihood of one embedding among the speakers of the training set: nothing but latency
        _case("ce_one_row", "ce", "bf16", 1, 192, 17982, False, reduction="none"),
        # a training step of a plain softmax head: 128 crops, the training set's speakers at three speeds
        _case("ce_train_batch", "ce", "fp16", 128, 192, 17982, True),
        # everything odd at once, rows without a target among them
        _case("ce_train_ragged", "ce", "fp16", 1237, 328, 30011, True, ragged=True),
        # scoring of long token streams: the loss of every row
        _case("ce_score_tokens", "ce", "bf16", 16384, 512, 32768, False, reduction="none"),
        # a training step over a vocabulary: the largest
        _case("ce_train_vocabulary", "ce", "bf16", 8192, 1024, 65536, True),
        # the models' own head at their training batch: three sub-centres to a speaker
        _case("margin_train_batch", "margin", "fp16", 128, 192, 17982, True, subcenters=3),
        # validation of a small set, odd sizes, two sub-centres
        _case("margin_score_ragged", "margin", "bf16", 37, 200, 1211, False, ragged=True, subcenters=2, reduction="none"),
        # a hundred thousand speakers, large batches of wide embeddings
        _case("margin_train_speakers", "margin", "bf16", 1024, 512, 100000, True),
        # a student of a speaker model: the 16 best classes of its teacher
        _case("distil_train_batch", "distil", "fp16", 128, 192, 5994, True, top=16, temperature=4.0),
        # teachers of different lengths, rows without one, odd sizes
        _case("distil_train_ragged", "distil", "bf16", 999, 136, 9973, True, ragged=True, top=7, temperature=2.0),
        # distillation over a vocabulary
        _case("distil_train_vocabulary", "distil", "bf16", 4096, 768, 48000, True, top=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["ce", "margin", "distil"])
    dim = 8 * _log(rng, 8, 128)
    classes = _log(rng, 500, 131072)
    subcenters = rng.choice([1, 1, 2, 3, 4]) if kind == "margin" else 1
    if classes * subcenters > 200000:
        subcenters = 1
    most = min(16384, MOST_LOGITS // (classes * subcenters), MOST_PRODUCTS // (classes * subcenters * dim))
    rows = _log(rng, 1, most)
    train = rng.random() < 0.7
    case = _case("", kind, rng.choice(["bf16", "fp16"]), rows, dim, classes, train, ragged=rng.random() < 0.4, subcenters=subcenters,
                 top=_log(rng, 1, 128) if kind == "distil" else 0,
                 temperature=rng.choice([1.0, 2.0, 4.0]) if kind == "distil" else 1.0,
                 reduction=rng.choice(["mean", "sum"]) if train else rng.choice(["none", "none", "mean"]))
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------ preparation
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    N, D, V, K = case["rows"], case["dim"], case["classes"], case["subcenters"]
    # Rows lean towards their class, as a head's do after some training: the target's logit is some 4 above the others, whose
    # deviation is 1 (cosines: about 0.4).
    weight = (torch.randn(V * K, D, generator=gen, device=dev) * D ** -0.5).to(dtype)
    target = torch.randint(0, V, (N,), generator=gen, device=dev)
    lean = (4.0 if kind != "margin" else 0.4 * D ** 0.5) * weight[target * K].float()
    x = (torch.randn(N, D, generator=gen, device=dev) + lean).to(dtype)
    s = {"case": case, "x": x, "weight": weight.view(V, K, D) if kind == "margin" and K > 1 else weight}
    if kind == "distil":
        top = case["top"]
        # The teacher's best class is the row's own, the others are the next ones of a random order of the classes.
        first = torch.randint(0, V, (N, 1), generator=gen, device=dev)
        step = torch.randint(1, max(2, V // top), (N, 1), generator=gen, device=dev)
        ids = (first + step * torch.arange(top, device=dev)) % V
        ids[:, 0] = target
        logits = 2.0 * torch.randn(N, top, generator=gen, device=dev)
        logits[:, 0] += 6.0
        if case["ragged"]:
            length = torch.randint(0, top + 1, (N, 1), generator=gen, device=dev)
            ids = torch.where(torch.arange(top, device=dev) < length, ids, -1)
        s["ids"], s["logits"] = ids, logits.to(dtype)
        counted = (ids >= 0).any(1)
    else:
        if case["ragged"]:
            target = torch.where(torch.rand(N, generator=gen, device=dev) < 0.1, IGNORE, target)
        s["target"] = target
        counted = target >= 0
    if case["train"]:
        up = 1.0
        if dtype == torch.float16:
            share = max(1, int(counted.sum())) if case["reduction"] == "mean" else 1
            up = 2.0 ** min(16, round(math.log2(16 * share)))
        s["dloss"] = torch.tensor(up, device=dev)
    if own:
        s["losses"] = _losses()
        if case["train"]:
            s["x"].requires_grad_(True)
            s["weight"].requires_grad_(True)
    return s


def _losses():
    path = os.path.abspath("pcf-nat_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from na1d_amd import losses
    return losses


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    case, f = s["case"], s["losses"]
    with torch.set_grad_enabled(case["train"]):
        if case["kind"] == "ce":
            loss = f.linear_cross_entropy(s["x"], s["weight"], s["target"], ignore_index=IGNORE, reduction=case["reduction"])
        elif case["kind"] == "margin":
            loss = f.margin_cross_entropy(s["x"], s["weight"], s["target"], margin=0.2, scale=32.0, ignore_index=IGNORE,
                                          reduction=case["reduction"])
        else:
            loss = f.linear_distillation(s["x"], s["weight"], s["logits"], s["ids"], temperature=case["temperature"],
                                         reduction=case["reduction"])
    if not case["train"]:
        return {"loss": loss}
    dx, dweight = torch.autograd.grad(loss, [s["x"], s["weight"]], s["dloss"])
    return {"loss": loss.detach(), "dx": dx, "dweight": dweight}


def _reduced(case, rows, counted):
    """The loss, and what a row's loss has to do with it."""
    if case["reduction"] == "none":
        return rows, None
    share = counted.to(rows.dtype)
    if case["reduction"] == "mean":
        share = share / counted.sum().clamp(min=1)
    return (rows * share).sum(), share


def _run_plain(s):
    """The definitions in 32 bits, with the logits in memory."""
    with torch.no_grad():
        return _margin_plain(s) if s["case"]["kind"] == "margin" else _linear_plain(s)


def _linear_plain(s):
    case = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    N, V = x.shape[0], w.shape[0]
    T = case["temperature"]
    z = x @ w.t()
    if case["kind"] == "ce":
        counted = s["target"] >= 0
        ids, q = s["target"].clamp(min=0).unsqueeze(1), counted.float().unsqueeze(1)
        own_entropy = 0.0
    else:
        z = z / T
        there = s["ids"] >= 0
        counted = there.any(1)
        ids = s["ids"].clamp(min=0)
        t = torch.where(there, s["logits"].float() / T, torch.tensor(-torch.inf, device=x.device))
        top = t.amax(1, keepdim=True)
        e = torch.where(there, torch.exp(t - top), torch.zeros_like(t))
        total = e.sum(1, keepdim=True)
        q = torch.where(there, e / total, torch.zeros_like(e))
        own_entropy = torch.where(there, q * (t - top - torch.log(total)), torch.zeros_like(t)).sum(1)
    high = z.amax(1, keepdim=True)
    p = torch.exp(z - high)
    total = p.sum(1, keepdim=True)
    lse = high + torch.log(total)
    rows = own_entropy - (q * (z.gather(1, ids) - lse)).sum(1)
    rows = torch.where(counted, T * T * rows, torch.zeros_like(rows))
    loss, share = _reduced(case, rows, counted)
    if not case["train"]:
        return {"loss": loss}
    g = (s["dloss"] * share * T).unsqueeze(1)
    p /= total
    p.scatter_add_(1, ids, -q)
    p *= g
    return {"loss": loss, "dx": (p @ w).to(s["x"].dtype), "dweight": (p.t() @ x).to(s["weight"].dtype)}


def _margin_plain(s, margin=0.2, scale=32.0):
    case = s["case"]
    x, w = s["x"].float(), s["weight"].float()
    V, K = case["classes"], case["subcenters"]
    w = w.view(V * K, -1)
    x_norm, w_norm = (x * x).sum(1, keepdim=True).sqrt(), (w * w).sum(1, keepdim=True).sqrt()
    xn, wn = x / x_norm, w / w_norm
    counted = s["target"] >= 0
    t = s["target"].clamp(min=0).unsqueeze(1)
    cosine, which = (xn @ wn.t()).view(-1, V, K).max(2)
    at = cosine.gather(1, t)
    sine2 = 1.0 - at * at
    far = at <= math.cos(math.pi - margin)
    shifted = torch.where(far, at - math.sin(math.pi - margin) * margin,
                          at * math.cos(margin) - torch.sqrt(sine2.clamp(min=0.0)) * math.sin(margin))
    z = (cosine * scale).scatter(1, t, shifted * scale)
    high = z.amax(1, keepdim=True)
    p = torch.exp(z - high)
    total = p.sum(1, keepdim=True)
    rows = (high + torch.log(total) - shifted * scale).squeeze(1)
    rows = torch.where(counted, rows, torch.zeros_like(rows))
    loss, share = _reduced(case, rows, counted)
    if not case["train"]:
        return {"loss": loss}
    slope = torch.where(far, torch.ones_like(at), math.cos(margin) + math.sin(margin) * at / torch.sqrt(sine2.clamp(min=SINE_FLOOR)))
    p /= total
    p.scatter_(1, t, (p.gather(1, t) - 1.0) * slope)
    p *= (s["dloss"] * share * scale).unsqueeze(1)
    d = torch.zeros(p.shape + (K,), device=x.device).scatter_(2, which.unsqueeze(2), p.unsqueeze(2)).view(-1, V * K)
    ax, aw = d @ wn, d.t() @ xn
    dx = (ax - xn * (ax * xn).sum(1, keepdim=True)) / x_norm
    dw = (aw - wn * (aw * wn).sum(1, keepdim=True)) / w_norm
    return {"loss": loss, "dx": dx.to(s["x"].dtype), "dweight": dw.view(s["weight"].shape).to(s["weight"].dtype)}


# ------------------------------------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    """By automatic differentiation of the definition, written with log-probabilities."""
    s = prepare(case, seed)
    dev = s["x"].device
    x, w = (s[name].detach().double().requires_grad_(case["train"]) for name in ("x", "weight"))
    V, K = case["classes"], case["subcenters"]
    n = torch.arange(case["rows"], device=dev)
    if case["kind"] == "margin":
        unit_x, unit_w = x / x.norm(dim=-1, keepdim=True), w / w.norm(dim=-1, keepdim=True)
        cosine = unit_x @ unit_w.reshape(V * K, -1).t()
        if K > 1:
            cosine = cosine.view(-1, V, K).amax(2)
        ok = s["target"] != IGNORE
        t = torch.where(ok, s["target"], 0)
        theta = torch.arccos(cosine[n, t])
        near = theta < math.pi - 0.2
        moved = torch.where(near, torch.cos(torch.where(near, theta, 0.0) + 0.2), cosine[n, t] - 0.2 * math.sin(math.pi - 0.2))
        delta = torch.zeros(case["rows"], V, device=dev, dtype=torch.float64)
        delta[n, t] = 1.0
        z = 32.0 * (cosine + delta * (moved - cosine[n, t]).unsqueeze(1))
        rows = torch.where(ok, torch.logsumexp(z, 1) - z[n, t], 0.0)
    else:
        z = x @ w.t() / case["temperature"]
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        if case["kind"] == "ce":
            ok = s["target"] != IGNORE
            rows = torch.where(ok, -logp[n, torch.where(ok, s["target"], 0)], 0.0)
        else:
            there = s["ids"] >= 0
            ok = there.any(1)
            teacher = torch.where(there, s["logits"].double() / case["temperature"], -1e300)
            logq = torch.log_softmax(teacher, 1)
            divergence = torch.where(there, logq.exp() * (logq - logp.gather(1, s["ids"].clamp(min=0))), 0.0).sum(1)
            rows = torch.where(ok, divergence * case["temperature"] ** 2, 0.0)
    if case["reduction"] == "none":
        return {"loss": rows}
    loss = rows.sum() / (max(1, int(ok.sum())) if case["reduction"] == "mean" else 1)
    if not case["train"]:
        return {"loss": loss}
    dx, dweight = torch.autograd.grad(loss, [x, w], s["dloss"].double())
    return {"loss": loss.detach(), "dx": dx, "dweight": dweight}


def work(case):
    N, D, VK = case["rows"], case["dim"], case["classes"] * case["subcenters"]
    flops, nbytes = 2.0 * N * VK * D, 2.0 * (N + VK) * D
    nbytes += N * (8.0 if case["kind"] != "distil" else 10.0 * case["top"]) + 4.0 * (N if case["reduction"] == "none" else 1)
    if case["train"]:
        flops, nbytes = 3 * flops, nbytes + 2.0 * (N + VK) * D + 4.0
    return {"bytes": nbytes, "flops": flops}
