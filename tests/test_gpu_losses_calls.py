"""Losses over many classes as they are called: layouts, masks, streams, graphs, compiled, in the models, and together."""
import math
import threading

import pytest
import torch
import torch.nn.functional as F
import torch.utils.checkpoint

from na1d_amd import _lib, losses, models
from oracle import losses_oracle as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(N=33, D=72, V=300, dtype=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype).cuda()
    target = torch.randint(0, V, (N,), generator=g).cuda()
    x = (torch.randn(N, D, generator=g).cuda() + 3 * w[target].float()).to(dtype)
    ids = torch.randint(-1, V, (N, 6), generator=g).cuda()
    logits = torch.randn(N, 6, generator=g).cuda()
    return x, w, target, ids, logits


def _calls(target, ids, logits, reduction="mean"):
    """Each loss as a function of x and weight."""
    return {"ce": lambda x, w: losses.linear_cross_entropy(x, w, target, reduction=reduction),
            "margin": lambda x, w: losses.margin_cross_entropy(x, w.unflatten(0, (-1, 3)), target // 3, reduction=reduction),
            "distil": lambda x, w: losses.linear_distillation(x, w, logits, ids, 2.0, reduction)}


KINDS = ["ce", "margin", "distil"]


def _both(call, x, w, up=None):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = call(x, w)
    return [loss.detach(), *torch.autograd.grad(loss, [x, w], up)]


def _same(a, b):
    return all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("kind", KINDS)
def test_any_layout_gives_the_same(kind):
    x, w, target, ids, logits = _inputs()
    call = _calls(target, ids, logits)[kind]
    want = _both(call, x, w)

    def laid(t, how):
        if how == "wide rows":
            out = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device="cuda")[:, 8:8 + t.shape[1]]
        elif how == "odd rows":
            out = torch.full((t.shape[0], t.shape[1] + 3), float("nan"), dtype=t.dtype, device="cuda")[:, :t.shape[1]]
        elif how == "every other":
            out = torch.full((2 * t.shape[0], t.shape[1]), float("nan"), dtype=t.dtype, device="cuda")[::2]
        elif how == "columns":
            out = torch.empty(t.shape[1], t.shape[0], dtype=t.dtype, device="cuda").t()
        else:
            out = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return out.copy_(t)

    for how in ("wide rows", "odd rows", "every other", "columns", "misaligned"):
        leaf_x, leaf_w = laid(x, how).requires_grad_(True), laid(w, how).requires_grad_(True)
        loss = call(leaf_x, leaf_w)
        assert _same([loss.detach(), *torch.autograd.grad(loss, [leaf_x, leaf_w])], want), how
    # leading dimensions, and an upstream gradient that is one number expanded
    t = x.view(3, 11, 72)
    more = {"ce": lambda a, b: losses.linear_cross_entropy(a, b, target.view(3, 11), reduction="none"),
            "margin": lambda a, b: losses.margin_cross_entropy(a, b.unflatten(0, (-1, 3)), target.view(3, 11) // 3, reduction="none"),
            "distil": lambda a, b: losses.linear_distillation(a, b, logits.view(3, 11, 6), ids.view(3, 11, 6), 2.0, "none")}[kind]
    flat = _both(_calls(target, ids, logits, "none")[kind], x, w, torch.ones(33, device="cuda"))
    loss, dx, dw = _both(more, t, w, torch.ones(1, device="cuda").expand(3, 11))
    assert loss.shape == (3, 11) and dx.shape == t.shape and _same([loss.view(-1), dx.view(33, 72), dw], flat)


@pytest.mark.parametrize("kind", KINDS)
def test_only_the_gradients_that_are_asked_for(kind):
    x, w, target, ids, logits = _inputs(N=130, V=600)
    call = _calls(target, ids, logits)[kind]
    _, dx, dw = _both(call, x, w)
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(call(a, w), a)[0], dx)
    assert torch.equal(torch.autograd.grad(call(x, b), b)[0], dw)
    assert not call(x, w).requires_grad
    with torch.no_grad():
        assert not call(a, b).requires_grad


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_rows_without_a_target(reduction):
    x, w, target, ids, logits = _inputs()
    target[:], ids[:] = -100, -1
    up = torch.ones(33, device="cuda") if reduction == "none" else None
    for call in (lambda x, w: losses.linear_cross_entropy(x, w, target, reduction=reduction),
                 lambda x, w: losses.margin_cross_entropy(x, w, target, reduction=reduction),
                 lambda x, w: losses.linear_distillation(x, w, logits, ids, reduction=reduction),
                 lambda x, w: losses.linear_distillation(x, w, logits - math.inf, ids.abs(), reduction=reduction)):
        assert all(not t.any() for t in _both(call, x, w, up))
    # no rows at all
    empty = x[:0]
    none, no_ids = target[:0], ids[:0]
    for call in (lambda x, w: losses.linear_cross_entropy(x, w, none, reduction=reduction), lambda x, w: losses.margin_cross_entropy(x, w, none, reduction=reduction),
                 lambda x, w: losses.linear_distillation(x, w, logits[:0], no_ids, reduction=reduction)):
        loss, dx, dw = _both(call, empty, w, up[:0] if reduction == "none" else None)
        assert dx.shape == (0, 72) and not dw.any() and not loss.any() and loss.shape == ((0,) if reduction == "none" else ())
    _, hits = losses.linear_cross_entropy(empty, w, none, reduction=reduction, return_hits=True)
    assert hits.shape == (0,)


def test_targets_and_ids_that_are_no_classes():
    """Such a row's loss is no number, it has no gradient, and the others' are as if it were ignored."""
    x, w, target, ids, logits = _inputs()
    ids[2] = torch.arange(6)
    ignored = target.clone()
    ignored[2] = -100
    up = torch.rand(33, device="cuda")
    for bad in (300, -1, -99, 1 << 40, -(1 << 40), 2 ** 31 - 1):
        wrong = target.clone()
        wrong[2] = bad
        for f in (losses.linear_cross_entropy, losses.margin_cross_entropy):
            got, want = (_both(lambda x, w: f(x, w, t, reduction="none"), x, w, up) for t in (wrong, ignored))
            assert math.isnan(got[0][2]) and not got[1][2].any()
            got[0][2] = 0
            assert _same(got, want)
            assert math.isnan(f(x, w, wrong))
    absent, wrong = ids.clone(), ids.clone()
    absent[2], wrong[2, 4] = -1, 300
    for bad in (300, 1 << 40, 2 ** 31 - 1):
        wrong[2, 4] = bad
        got, want = (_both(lambda x, w: losses.linear_distillation(x, w, logits, i, reduction="none"), x, w, up) for i in (wrong, absent))
        assert math.isnan(got[0][2]) and not got[1][2].any()
        got[0][2] = 0
        assert _same(got, want)
    wrong[2, 4] = -(1 << 40)                                         # below 0: not there
    assert torch.isfinite(losses.linear_distillation(x, w, logits, wrong))
    other = losses.linear_cross_entropy(x, w, torch.where(target == 5, 7, target).masked_fill(torch.arange(33, device="cuda") == 2, 5), ignore_index=5, reduction="none")
    assert other[2] == 0 and (other != 0).sum() == 32


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite_stay_in_their_rows(kind):
    x, w, target, ids, logits = _inputs()
    call = _calls(target, ids, logits, "none")[kind]
    want = call(x, w)
    for bad in (float("nan"), float("inf"), -float("inf")):
        broken = x.clone()
        broken[4, 7] = bad
        got = call(broken, w)
        keep = torch.arange(33, device="cuda") != 4
        assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[4])
    weight = w.clone()
    weight[9, 3] = float("nan")
    assert call(x, weight).isnan().all()
    if kind == "distil":
        for bad in (float("nan"), float("inf")):
            t = logits.clone()
            t[4, 0] = bad
            i = ids.abs()
            got, plain = (losses.linear_distillation(x, w, l, i, 2.0, "none") for l in (t, logits))
            assert not torch.isfinite(got[4]) and torch.equal(got[keep], plain[keep])


def test_rows_of_zeros_have_no_angle():
    x, w, target, _, _ = _inputs(dtype=BF16)
    x[5], w[target[7]], w[11] = 0, 0, 0
    target[target == 11] = 12
    loss, dx, dw = _both(lambda x, w: losses.margin_cross_entropy(x, w, target, reduction="none"), x, w, torch.ones(33, device="cuda"))
    rows, ok, e, _ = O.margin(x, w.unsqueeze(1), target)
    assert torch.isfinite(loss).all() and ((loss - rows).abs() <= O.logit_bound(O.unit(x.double()), O.unit(w.double()), 32.0)).all()
    assert not dx[5].any() and not dw[11].any() and not dw[target[7]].any() and torch.isfinite(dx).all() and torch.isfinite(dw).all()


def test_certain_rows_and_large_logits():
    """A loss far below one keeps its digits, and logits of thousands neither overflow nor lose the others."""
    x, w, target, _, _ = _inputs(D=64)
    for scale in (10.0, 300.0, 3000.0):
        rows, ok, e = O.softmax_targets(x, w, target, scale)
        loss, dx, dw = _both(lambda x, w: losses.linear_cross_entropy(x, w, target, scale=scale, reduction="none"), x, w, torch.ones(33, device="cuda"))
        delta = O.logit_bound(x, w, scale)
        # An error of delta in the exponents moves a loss by that factor, and by no more than delta.
        assert ((loss - rows).abs() <= torch.minimum(torch.expm1(2 * delta) * rows, 2 * delta) + 2.0 ** -20 * rows + 1e-38).all()
        gx, gw, magnitudes = O.linear_gradients(x, w, e, torch.ones_like(rows))
        bx, bw = O.gradient_bounds(gx, gw, magnitudes, delta, x.dtype, 1e-30)
        assert ((dx.double() - gx).abs() <= bx).all() and ((dw.double() - gw).abs() <= bw).all()


@pytest.mark.parametrize("kind", KINDS)
def test_gradients_by_differences(kind):
    """The change of every row's loss along a direction that 16 bits hold exactly (steps of 2^-5 on values of steps 2^-5)."""
    x, w, target, ids, logits = _inputs(N=16, D=64, V=90, dtype=FP16)
    x, w = (x * 32).round() / 32, (w * 64).round() / 64
    call = _calls(target, ids, logits, "none")[kind]
    g = torch.Generator().manual_seed(3)
    to_x = (torch.randint(-1, 2, x.shape, generator=g) / 32).half().cuda()
    to_w = (torch.randint(-1, 2, w.shape, generator=g) / 128).half().cuda()
    for dx, dw in ((to_x, 0 * to_w), (0 * to_x, to_w)):
        step = lambda h: call(x + h * dx, w + h * dw).double().sum()
        # central differences of steps 1 and 2, extrapolated: an error of the fourth order
        slope = (4 * (step(1) - step(-1)) / 2 - (step(2) - step(-2)) / 4) / 3
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        ga, gb = torch.autograd.grad(call(a, b).sum(), [a, b])
        along = (ga.double() * dx.double()).sum() + (gb.double() * dw.double()).sum()
        size = (ga.double() * dx.double()).abs().sum() + (gb.double() * dw.double()).abs().sum()
        assert abs(slope - along) <= 0.01 * size, (slope, along, size)


@pytest.mark.parametrize("kind", KINDS)
def test_results_are_the_same_from_call_to_call(kind):
    x, w, target, ids, logits = _inputs(N=700, D=136, V=6000, dtype=FP16)
    call = _calls(target, ids, logits)[kind]
    want = _both(call, x, w)
    for _ in range(3):
        assert _same(_both(call, x, w), want)


@pytest.mark.parametrize("kind", KINDS)
def test_streams_of_their_own(kind):
    x, w, target, ids, logits = _inputs(N=260, D=136, V=6000)
    call = _calls(target, ids, logits)[kind]
    want = _both(call, x, w)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:                                                  # side by side
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append(_both(call, x, w))
    torch.cuda.synchronize()
    assert all(_same(g, want) for g in got)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("kind", KINDS)
def test_captured_passes_replay(kind, reduction):
    x, w, target, ids, logits = _inputs(N=130, D=136, V=3000, dtype=FP16)
    call = _calls(target, ids, logits, reduction)[kind]
    up = torch.full((130,) if reduction == "none" else (), 4.0, device="cuda")
    a, b = x.clone(), w.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _both(call, a, b, up)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                                 # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_both(call, a, b, up))
        graphs.append(graph)
    for i in range(4):
        a.copy_(x * (1 + i / 8))
        b.copy_(w * (1 - i / 16))
        want = _both(call, a, b, up)
        torch.cuda.synchronize()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert _same(out, want), i


def test_offsets_past_32_bits():
    """Weights of 4.9 GB and rows of 4.5 GB: the last ones' losses and gradients."""
    V, D = 600_000, 4096
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(V, D, dtype=BF16, device="cuda")
    for i in range(0, V, 50_000):
        w[i:i + 50_000] = torch.randn(50_000, D, generator=g, device="cuda") / 64
    target = torch.tensor([V - 1, 0, V - 70_000], device="cuda")
    x = (torch.randn(3, D, generator=g, device="cuda") + 6 * w[target].float()).to(BF16)
    loss, dx, dw = _both(lambda x, w: losses.linear_cross_entropy(x, w, target, reduction="none"), x, w, torch.ones(3, device="cuda"))
    z = torch.cat([x.double() @ w[i:i + 50_000].double().t() for i in range(0, V, 50_000)], 1)
    lse = torch.logsumexp(z, 1)
    rows = lse - z[torch.arange(3), target]
    assert ((loss - rows).abs() <= 1e-4 * rows + 1e-4).all()            # 4096 roundings of sums of magnitude 50
    p = torch.exp(z - lse.unsqueeze(1))
    p[torch.arange(3), target] -= 1
    for c in (V - 1, V - 70_000, V - 2, 123_456, 0):
        want = p[:, c] @ x.double()
        assert ((dw[c].double() - want).abs() <= 2.0 ** -7 * (p[:, c].abs() @ x.double().abs()) + 1e-30).all()
    del w, dw
    N = (1 << 20) - 3
    x = torch.randn(N, 2136, generator=g, device="cuda", dtype=BF16)
    w = (torch.randn(16, 2136, generator=g, device="cuda") / 16).to(BF16)
    target = torch.randint(0, 16, (N,), generator=g, device="cuda")
    loss, dx, dw = _both(lambda x, w: losses.linear_cross_entropy(x, w, target, reduction="none"), x, w, torch.ones(N, device="cuda"))
    tail = slice(N - 1000, N)
    rows, _, e = O.softmax_targets(x[tail], w, target[tail])
    assert ((loss[tail] - rows).abs() <= O.logit_bound(x[tail], w, 1.0)).all()
    want, want_dw, magnitudes = O.linear_gradients(x[tail], w, e, torch.ones(1000, device="cuda"))
    assert ((dx[tail].double() - want).abs() <= O.gradient_bounds(want, want_dw, magnitudes, O.logit_bound(x[tail], w, 1.0), BF16)[0]).all()


def test_calls_of_several_threads_at_once():
    sizes = ((128, 192, 3000, BF16), (700, 256, 5001, FP16), (33, 64, 900, BF16), (1, 128, 21000, FP16))
    cases = [_inputs(N, D, V, dtype, seed=i) for i, (N, D, V, dtype) in enumerate(sizes)]
    pairs = [(_calls(target, ids, logits)["margin"], x, w) for x, w, target, ids, logits in cases]
    want = [_both(*p) for p in pairs]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [((i + k) % 4, _both(*pairs[(i + k) % 4])) for i in range(20)]
        stream.synchronize()
        wrong.extend(j for j, g in got if not _same(g, want[j]))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("kind", KINDS)
def test_a_graph_of_one_loss_and_other_nodes(kind):
    """Kept for a second backward, recomputed under checkpointing, with a weight that makes x too, and one that is written to in between."""
    x, w, target, ids, logits = _inputs()
    call = _calls(target, ids, logits)[kind]
    want = _both(call, x, w)[1:]
    a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = call(a, b)
    assert _same(torch.autograd.grad(loss, [a, b], retain_graph=True), want) and _same(torch.autograd.grad(loss, [a, b]), want)
    loss = torch.utils.checkpoint.checkpoint(call, a, b, use_reentrant=False)
    assert _same(torch.autograd.grad(loss, [a, b]), want)
    tied, = torch.autograd.grad(call(b[:33], b), b)
    apart = _both(call, w[:33], w)[1:]
    assert torch.equal(tied, torch.cat([apart[1][:33] + apart[0], apart[1][33:]]))
    loss = call(a, b)
    with torch.no_grad():
        b.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_the_largest_launches():
    """2^36 logits, and as many cosines of four weight rows: some rows against the same rows by themselves.  Losses are off by the
    logits' fp32 sums (8 products) alone; gradients, in norm, by half a step of dz and one of their own on either side."""
    g = torch.Generator(device="cuda").manual_seed(0)
    for N, V, K in ((1 << 14, 1 << 22, 4), (1 << 20, 1 << 16, 1)):
        x = torch.randn(N, 8, generator=g, device="cuda", dtype=BF16)
        w = torch.randn(V, K, 8, generator=g, device="cuda", dtype=BF16)
        target = torch.randint(0, V, (N,), generator=g, device="cuda")
        call = losses.margin_cross_entropy if K > 1 else losses.linear_cross_entropy
        some = torch.tensor([0, 1, 77, N // 2, *range(N - 40, N)], device="cuda")
        if K > 1:
            loss, few = call(x, w, target, reduction="none"), call(x[some], w, target[some], reduction="none")
        else:
            loss, dx, _ = _both(lambda a, b: call(a, b, target, reduction="none"), x, w[:, 0], torch.ones(N, device="cuda"))
            few, dx_few, _ = _both(lambda a, b: call(a, b, target[some], reduction="none"), x[some], w[:, 0], torch.ones(len(some), device="cuda"))
            assert ((dx[some].double() - dx_few.double()).norm(dim=1) <= 4 * 2.0 ** -8 * dx_few.double().norm(dim=1)).all()
            up = torch.zeros(N, device="cuda")
            up[some] = 1.0                                                   # the weight's gradient of these rows alone
            _, _, dw = _both(lambda a, b: call(a, b, target, reduction="none"), x, w[:, 0], up)
            _, _, dw_few = _both(lambda a, b: call(a, b, target[some], reduction="none"), x[some], w[:, 0], torch.ones(len(some), device="cuda"))
            assert (dw.double() - dw_few.double()).norm() <= 4 * 2.0 ** -8 * dw_few.double().norm()
        assert ((loss[some] - few).abs() <= 2.0 ** -17 * (few.abs() + 32 * 8)).all()


def test_hits():
    x, w, target, _, _ = _inputs(N=500)
    target[::3] = torch.randint(0, 300, (167,), generator=torch.Generator().manual_seed(1)).cuda()
    target[4] = -100
    best = (x.double() @ w.double().t()).argmax(1)
    loss, hits = losses.linear_cross_entropy(x, w, target, return_hits=True)
    assert torch.equal(hits, best == target) and torch.equal(loss, losses.linear_cross_entropy(x, w, target)) and 0 < hits.sum() < 500
    best = (O.unit(x.double()) @ O.unit(w.double()).t()).view(500, 100, 3).amax(2).argmax(1)
    _, hits = losses.margin_cross_entropy(x, w.view(100, 3, 72), target.clamp(min=0) // 3, return_hits=True)
    assert torch.equal(hits, best == target.clamp(min=0) // 3)
    w[7] = w[9]                                                        # a shared first place
    _, hits = losses.linear_cross_entropy(50 * w[[7, 9]], w, torch.tensor([7, 7], device="cuda"), return_hits=True)
    assert hits.all()


def test_equal_subcenters_take_the_first():
    x, w, target, _, _ = _inputs(N=40, V=90)
    three = w[::3].unsqueeze(1).repeat(1, 3, 1).contiguous()
    _, dx, dw = _both(lambda x, w: losses.margin_cross_entropy(x, w, target // 3), x, three)
    _, one_dx, one_dw = _both(lambda x, w: losses.margin_cross_entropy(x, w, target // 3), x, three[:, :1].contiguous())
    assert not dw[:, 1:].any() and dw[:, 0].any()
    assert torch.allclose(dx.float(), one_dx.float(), atol=2.0 ** -8 * one_dx.abs().max().item())


def test_compiled_ops_equal_the_functions():
    from na1d_amd import ops
    x, w, target, ids, logits = _inputs(N=130, V=600)
    for kind, f in {"ce": lambda x, w: ops.linear_cross_entropy_op(x, w, target, 1.5), "margin": lambda x, w: ops.margin_cross_entropy_op(x, w, target),
                    "distil": lambda x, w: ops.linear_distillation_op(x, w, logits, ids, 2.0)}.items():
        plain = {"ce": lambda x, w: losses.linear_cross_entropy(x, w, target, 1.5), "margin": lambda x, w: losses.margin_cross_entropy(x, w, target),
                 "distil": lambda x, w: losses.linear_distillation(x, w, logits, ids, 2.0)}[kind]
        want = _both(plain, x, w)
        assert _same(_both(f, x, w), want), kind
        compiled = torch.compile(lambda x, w: 2 * f(x * 1, w), backend="aot_eager", fullgraph=True)
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        loss = compiled(a, b)
        grads = torch.autograd.grad(loss, [a, b], torch.tensor(0.5, device="cuda"))
        assert torch.equal(loss, 2 * want[0]) and _same(grads, want[1:]), kind


def test_a_compiled_op_takes_batches_of_any_size():
    from na1d_amd import ops
    compiled = torch.compile(lambda x, w, t: ops.linear_cross_entropy_op(x, w, t), backend="aot_eager", fullgraph=True, dynamic=True)
    for N in (33, 40, 7):
        x, w, target, _, _ = _inputs(N=N)
        got = _both(lambda a, b: compiled(a, b, target), x, w)
        assert _same(got, _both(lambda a, b: losses.linear_cross_entropy(a, b, target), x, w)), N


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("kind", KINDS)
def test_upstream_gradients_that_are_not_finite_or_zero(kind, dtype):
    """A loss scale that has run over reaches the gradients, a zero leaves none; a row's own stays in its row of dx."""
    x, w, target, ids, logits = _inputs(dtype=dtype)
    for bad in (float("inf"), float("nan")):
        for reduction in ("mean", "none"):
            call = _calls(target, ids, logits, reduction)[kind]
            up = torch.tensor(bad, device="cuda") if reduction == "mean" else torch.ones(33, device="cuda").index_fill(0, torch.tensor([4], device="cuda"), bad)
            _, dx, dw = _both(call, x, w, up)
            assert not torch.isfinite(dx[4]).all() and not torch.isfinite(dw).all()
            if reduction == "none":
                assert torch.isfinite(dx[:4]).all() and torch.isfinite(dx[5:]).all()
    _, dx, dw = _both(_calls(target, ids, logits)[kind], x, w, torch.tensor(0.0, device="cuda"))
    assert not dx.any() and not dw.any()


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_the_models_head(dtype):
    """The fused head beside the torch one: the same parameters, losses and gradients to what products in 16 bits give."""
    torch.manual_seed(0)
    plain = models.ArcMarginSubCenters(192, 1000, subcenters=3).cuda()
    fused = models.ArcMarginSubCenters(192, 1000, subcenters=3, head="fused", dtype=dtype).cuda()
    fused.load_state_dict(plain.state_dict())
    with torch.no_grad():                                              # as 16 bits hold them
        for head in (plain, fused):
            head.W.copy_(head.W.to(dtype))
    labels = torch.randint(0, 1000, (64,), device="cuda")
    x = (torch.randn(64, 192, device="cuda") / 8 + 30 * plain.W[labels, 1].detach()).to(dtype).float().requires_grad_(True)
    up = torch.tensor(1024.0, device="cuda")
    (loss, acc), (want, want_acc) = fused(x, labels), plain(x, labels)
    assert loss.dtype == torch.float32 and acc == want_acc and abs(loss - want) < 1e-4 * want
    got = torch.autograd.grad(loss, [x, fused.W], up)
    for a, b in zip(got, torch.autograd.grad(want, [x, plain.W], up)):
        assert a.dtype == torch.float32 and a.shape == b.shape and O_rel(a, b) < (1e-2 if dtype == BF16 else 2e-3)


def O_rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_a_training_step_with_a_teacher():
    """As they are used together: a model's embeddings, its margin head, a plain head and a teacher's top classes, one backward."""
    torch.manual_seed(0)
    model = models.MFA_NATransformer(depths=(2, 1), num_heads=16, win_size=[[27, 0], 27], na="fused_qkv", frames=200, dtype=FP16).cuda().train()
    head = models.ArcMarginSubCenters(192, 700, subcenters=2, head="fused", dtype=FP16).cuda()
    student = torch.nn.Parameter(torch.randn(700, 192, device="cuda") / 14)
    teacher = torch.randn(16, 700, device="cuda").topk(8)
    labels = torch.randint(0, 700, (16,), device="cuda")
    x = torch.randn(16, 80, 200, device="cuda")
    params = [*model.parameters(), head.W, student]

    def step(plain):
        torch.manual_seed(1)
        with torch.autocast("cuda", dtype=FP16):
            emb = model(x)
        emb16, w16 = emb.to(FP16), student.to(FP16)
        margin, _ = head(emb.float(), labels)
        if plain:
            z = emb16.float() @ w16.float().t()
            ce = F.cross_entropy(z, labels)
            q = torch.softmax(teacher.values / 2, 1)
            kd = 4 * (q * (q.log() - F.log_softmax(z / 2, 1).gather(1, teacher.indices))).sum(1).mean()
        else:
            ce = losses.linear_cross_entropy(emb16, w16, labels)
            kd = losses.linear_distillation(emb16, w16, teacher.values, teacher.indices, 2.0)
        return margin + ce + kd, torch.autograd.grad(1024 * (margin + ce + kd), params)

    loss, grads = step(False)
    want, want_grads = step(True)
    assert abs(loss - want) < 1e-4 * want and all(torch.isfinite(g).all() for g in grads)
    assert O_rel(grads[-1], want_grads[-1]) < 2e-3 and torch.equal(grads[-2], want_grads[-2])
