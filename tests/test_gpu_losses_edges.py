"""Losses over many classes at the edges of what they take: rows that do not count beside upstream gradients that are not finite,
losses that are written to, rows far apart, workgroups' rows behind the last, the largest weights and batches, and ops called by themselves."""
import math

import pytest
import torch

from na1d_amd import losses, ops
from oracle import losses_oracle as O

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16
KINDS = ["ce", "margin", "distil"]


def _inputs(N=33, D=72, V=300, dtype=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype).cuda()
    target = torch.randint(0, V, (N,), generator=g).cuda()
    x = (torch.randn(N, D, generator=g).cuda() + 3 * w[target].float()).to(dtype)
    ids = torch.stack([torch.randperm(V, generator=g)[:6] for _ in range(N)]).cuda()
    logits = torch.randn(N, 6, generator=g).cuda()
    return x, w, target, ids, logits


def _calls(target, ids, logits, reduction="mean"):
    return {"ce": lambda x, w: losses.linear_cross_entropy(x, w, target, reduction=reduction),
            "margin": lambda x, w: losses.margin_cross_entropy(x, w.unflatten(0, (-1, 3)), target // 3, reduction=reduction),
            "distil": lambda x, w: losses.linear_distillation(x, w, logits, ids, 2.0, reduction)}


def _both(call, x, w, up=None):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = call(x, w)
    return [loss.detach(), *torch.autograd.grad(loss, [x, w], up)]


def _same(a, b):
    return all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_do_not_count_have_no_use_for_an_upstream_gradient(kind, dtype):
    """Whatever comes to such a row, its gradient is zero and the others' are the same to the bit.  (A bad target's loss is no number,
    so what is built on it mostly hands none back.)"""
    x, w, target, ids, logits = _inputs(N=130, dtype=dtype)
    rows = torch.tensor([4, 60, 129], device="cuda")
    ways = {"ignored": -100, "no class": 300} if kind != "distil" else {"absent": -1, "no class": 300, "all -inf": None}
    for name, bad in ways.items():
        t, i, l = target.clone(), ids.clone(), logits.clone()
        if kind == "margin":
            t[rows] = -100 if name == "ignored" else 900
        elif kind == "ce":
            t[rows] = bad
        elif name == "all -inf":
            l[rows] = -math.inf
        elif name == "absent":
            i[rows] = -1
        else:
            i[rows, 2] = bad
        if kind == "margin":
            call = lambda x, w: losses.margin_cross_entropy(x, w.unflatten(0, (-1, 3)), torch.where(t < 0, t, t // 3), reduction="none")
        else:
            call = _calls(t, i, l, "none")[kind]
        up = torch.rand(130, generator=torch.Generator().manual_seed(2)).cuda()
        want = _both(call, x, w, up)[1:]
        assert not want[0][rows].any() and all(torch.isfinite(g).all() and g.any() for g in want)
        for value in (math.nan, math.inf, -math.inf, 3e38, 0.0):
            got = _both(call, x, w, up.index_fill(0, rows, value))[1:]
            assert _same(got, want), (name, value)


@pytest.mark.parametrize("kind", KINDS)
def test_losses_are_written_to(kind):
    """A loss is a tensor of its own, whichever node it comes from: divided, added to and cut off in place."""
    x, w, target, ids, logits = _inputs()
    for reduction in ("mean", "none"):
        call = _calls(target, ids, logits, reduction)[kind]
        want = _both(lambda a, b: call(a, b).sum() / 4, x, w)
        for lay in (lambda t: t.detach().clone(), lambda t: t.detach().t().contiguous().t()):          # by the native node, and the other
            a, b = lay(x).requires_grad_(True), lay(w).requires_grad_(True)
            loss = call(a, b)
            assert not loss._is_view()
            loss /= 4
            total = loss.sum()
            total += 1
            assert _same(torch.autograd.grad(total, [a, b]), want[1:])
            loss = call(a, b)
            assert not loss.detach_().requires_grad


@pytest.mark.parametrize("kind", KINDS)
def test_rows_very_far_apart(kind):
    """The last state of long sequences is a view whose rows are more than 2^20 elements apart, and so may a weight's be."""
    x, w, target, ids, logits = _inputs(N=5, V=30)
    want = _both(_calls(target, ids, logits)[kind], x, w)
    far = (1 << 20) + 8
    hidden, table = torch.empty(5, far, dtype=BF16, device="cuda"), torch.empty(30, far, dtype=BF16, device="cuda")
    last, rows = hidden[:, -72:], table[:, 8:80]
    last.copy_(x), rows.copy_(w)
    a, b = last.requires_grad_(True), rows.requires_grad_(True)
    assert a.stride(0) == far and b.stride(0) == far
    loss = _calls(target, ids, logits)[kind](a, b)
    assert _same([loss.detach(), *torch.autograd.grad(loss, [a, b])], want)
    if kind == "margin":                                                   # a class's three rows together reach further than that
        near = torch.empty(30, 1 << 19, dtype=BF16, device="cuda")[:, :72].copy_(w).unflatten(0, (10, 3)).requires_grad_(True)
        loss = losses.margin_cross_entropy(x, near, target // 3)
        assert near.stride() == (3 << 19, 1 << 19, 1) and torch.equal(loss.detach(), want[0])
        assert torch.equal(torch.autograd.grad(loss, near)[0].view(30, 72), want[2])


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("V,K", [(1, 1), (2, 1), (2, 2), (2, 3), (2, 5)])
def test_a_last_row_that_is_far_from_every_class(V, K, dtype):
    """All its cosines are near -1 and the scale is large, so that the logarithm of its sum is far below zero: what stands behind it in
    its tile has no share in any gradient."""
    g = torch.Generator().manual_seed(V * 10 + K)
    for N in (1, 37, 130):
        base = torch.randn(64, generator=g)
        w = (base + 0.02 * torch.randn(V, K, 64, generator=g)).to(dtype).cuda()
        x = (-base + 0.02 * torch.randn(N, 64, generator=g)).to(dtype).cuda()
        target = torch.randint(0, V, (N,), generator=g).cuda()
        for scale in (128.0, 500.0):
            rows, ok, e, cosines = O.margin(x, w, target, scale=scale)
            up = torch.full((N,), 16.0, device="cuda")
            loss, dx, dw = _both(lambda a, b: losses.margin_cross_entropy(a, b, target, scale=scale, reduction="none"), x, w, up)
            delta = O.logit_bound(O.unit(x.double()), O.unit(w.double().view(V * K, 64)), scale)
            assert ((loss - rows).abs() <= 2 * delta + 2.0 ** -20 * rows).all()
            gx, gw, magnitudes = O.margin_gradients(x, w, e, up)
            far = O.undecided(x, w, e, cosines, up)
            # fp16: half a step of the smallest dz, 2^-39 of the largest, in up to 130 terms
            bx, bw = O.gradient_bounds(gx, gw, magnitudes, 2 * delta, dtype, 2.0 ** -31 * 4 * scale)
            assert ((dx.double() - gx).abs() <= bx + far[0]).all() and ((dw.double().view(V * K, 64) - gw).abs() <= bw + far[1]).all()


def test_the_largest_weight_that_many_rows_share():
    """2^24 weight rows, four to a class, and a batch of which the weight's gradient is summed in parts: some rows' share of both
    gradients against the same rows by themselves.  In norm they differ by half a step of dz and one of their own on either side."""
    g = torch.Generator(device="cuda").manual_seed(0)
    N, V, K = 1 << 14, 1 << 22, 4
    x = torch.randn(N, 8, generator=g, device="cuda", dtype=BF16)
    w = torch.randn(V, K, 8, generator=g, device="cuda", dtype=BF16)
    target = torch.randint(0, V, (N,), generator=g, device="cuda")
    some = torch.tensor([0, 1, 77, N // 2, *range(N - 40, N)], device="cuda")
    up = torch.zeros(N, device="cuda").index_fill(0, some, 1.0)
    call = lambda t: lambda a, b: losses.margin_cross_entropy(a, b, t, reduction="none")
    loss, dx, dw = _both(call(target), x, w, up)
    few, dx_few, dw_few = _both(call(target[some]), x[some], w, torch.ones(len(some), device="cuda"))
    # A row's two nearest of a class may be closer than fp32 tells: tiles of either batch add in another order.
    assert ((loss[some] - few).abs() <= 2.0 ** -17 * (few.abs() + 32 * 8)).all()
    assert ((dx[some].double() - dx_few.double()).norm(dim=1) <= 4 * 2.0 ** -8 * dx_few.double().norm(dim=1)).all()
    assert (dw.double() - dw_few.double()).norm() <= 4 * 2.0 ** -8 * dw_few.double().norm()


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_rows_that_the_backward_takes_in_batches(dtype, monkeypatch):
    """More than 2^19 rows have ranges of few classes, and more than 2^21 times weight rows of a class are worked on some at a time:
    the whole against 64 bits.

    In fp16 a class has up to some 1500 rows whose upstream gradients are 16 each: with 1 - P up to 1 and |x| beyond 3, elements of its
    gradient pass 65504, fp16's largest, and have to be infinite (or, within the bound of that, may be)."""
    import test_gpu_losses as T
    near = T._near

    def near_or_beyond(name, got, want, bound):
        beyond = got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound > torch.finfo(got.dtype).max)
        near(name, torch.where(beyond, want.to(torch.float64), got.double()), want, bound)

    monkeypatch.setattr(T, "_near", near_or_beyond)
    T.test_cross_entropy((530_001, 8, 300), dtype)
    T._distillation((530_001, 8, 300), 3, dtype)
    for size, subs in (((600_000, 8, 300), 1), ((270_001, 16, 300), 2), ((3000, 16, 300), 200), ((11_001, 16, 300), 200)):
        T._margin(size, subs, dtype)


@pytest.mark.parametrize("kind", KINDS)
def test_weights_whose_gradient_is_summed_in_parts_range_by_range(kind):
    """So many rows that a range has few classes, and its weight rows' gradients are sums of many parts: against 64 bits in the norm, by
    what rounding once leaves (half a step of dz in every term, and of the sum at the end)."""
    x, w, target, ids, logits = _inputs(N=70_000, D=64, V=9_000)
    call = _calls(target, ids, logits)[kind]
    _, dx, dw = _both(call, x, w)
    if kind == "margin":
        rows, ok, e, _ = O.margin(x, w.view(3000, 3, 64), target // 3)
        want = O.margin_gradients(x, w, e, O.shares(ok, "mean", 1.0))[:2]
    else:
        rows, ok, e = O.softmax_targets(x, w, target) if kind == "ce" else O.teacher(x, w, logits, ids, 2.0)
        want = O.linear_gradients(x, w, e, O.shares(ok, "mean", 1.0))[:2]
    for got, exact in zip((dx, dw), want):
        assert (got.double() - exact).norm() <= 2 * 2.0 ** -8 * exact.norm()


@pytest.mark.parametrize("way", ["native node", "Python node", "op"])
@pytest.mark.parametrize("kind", KINDS)
def test_a_penalty_on_a_gradient_is_refused(kind, way):
    """The gradients are the same with create_graph, and a loss that holds them is not differentiated without them."""
    x, w, target, ids, logits = _inputs()
    call = _calls(target, ids, logits)[kind]
    if way == "op":
        call = {"ce": lambda x, w: ops.linear_cross_entropy_op(x, w, target), "margin": lambda x, w: ops.margin_cross_entropy_op(x, w.unflatten(0, (-1, 3)), target // 3),
                "distil": lambda x, w: ops.linear_distillation_op(x, w, logits, ids, 2.0)}[kind]
    lay = (lambda t: t.t().contiguous().t()) if way == "Python node" else (lambda t: t.clone())
    want = _both(call, x, w)[1:]
    for both in (True, False):
        a, b = lay(x).requires_grad_(True), lay(w).requires_grad_(both)
        leaves = [a, b] if both else [a]
        loss = call(a, b)
        grads = torch.autograd.grad(loss, leaves, create_graph=True)
        assert _same(grads, want[:len(grads)])
        with pytest.raises(RuntimeError, match="differentiated again"):
            (loss + grads[0].float().square().sum()).backward()


@pytest.mark.parametrize("kind", KINDS)
def test_the_ops_by_themselves(kind):
    """As torch.ops has them: schema and fake kernels, the functions' results, and operands that do not fit refused before any kernel."""
    x, w, target, ids, logits = _inputs()
    number = KINDS.index(kind)
    operands = (x, w.unflatten(0, (-1, 3)) if kind == "margin" else w, ids if kind == "distil" else target // 3 if kind == "margin" else target,
                logits if kind == "distil" else None)
    rest = (number, {"ce": 1.0, "margin": 32.0, "distil": 2.0}[kind], 0.2 if kind == "margin" else 0.0, -100)
    f, b = torch.ops.na_cuda.class_loss_forward, torch.ops.na_cuda.class_loss_backward
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(f.default, (*operands, *rest, 1), test_utils=tests)
    want = _both(_calls(target, ids, logits)[kind], x, w)
    loss, saved = f(*operands, *rest, 1)
    one = torch.ones((), device="cuda")
    torch.library.opcheck(b.default, (one, *operands, saved, *rest, 1, True, True), test_utils=tests)
    dx, dw = b(one, *operands, saved, *rest, 1, True, True)
    assert _same([loss, dx, dw.view_as(w)], want)
    short = (x, operands[1], operands[2][:30], None if operands[3] is None else operands[3][:30])
    for call in (lambda: f(*short, *rest, 1), lambda: b(one, *short, saved, *rest, 1, True, True), lambda: b(one.expand(33), *operands, saved, *rest, 1, True, True),
                 lambda: b(one, *operands, saved[:64], *rest, 1, True, True), lambda: f(x, operands[1].cpu(), *operands[2:], *rest, 1)):
        with pytest.raises((RuntimeError, ValueError)):
            call()


def test_rows_whose_length_fp32_does_not_hold():
    """bfloat16 reaches 3e38, whose square fp32 does not: such a row's cosines are no numbers, where 0 would be a wrong one.  Short rows
    have theirs down to 1e-12, below which a row counts as zeros."""
    x, w, target, _, _ = _inputs()
    x, w = torch.nn.functional.normalize(x.float()).to(BF16), torch.nn.functional.normalize(w.float()).to(BF16)
    call = lambda a, b: losses.margin_cross_entropy(a, b, target, reduction="none")
    want, up = call(x, w), torch.ones(33, device="cuda")
    other = torch.arange(33, device="cuda") != 4
    for size, fine in ((2.0 ** 62, True), (2.0 ** 66, False), (2.0 ** -38, True)):
        a = torch.where(other.unsqueeze(1), x, x * size)
        loss, dx, _ = _both(call, a, w, up)
        assert torch.equal(loss[other], want[other])
        if fine:
            assert abs(loss[4] - want[4]) <= 1e-5 * want[4] and dx[4].any() and torch.isfinite(dx[4]).all()
        else:
            assert loss[4].isnan() and dx[4].isnan().all()
    short = torch.where(other.unsqueeze(1), x, x * 2.0 ** -41)
    loss, dx, _ = _both(call, short, w, up)
    zeros = torch.where(other.unsqueeze(1), x, torch.zeros_like(x))
    assert torch.equal(loss, call(zeros, w)) and not dx[4].any()
    long = torch.where(other.unsqueeze(1), x, x * 2.0 ** 66)                # an ignored one has no say, as any other
    ignored = target.masked_fill(~other, -100)
    ignore = lambda a, b: losses.margin_cross_entropy(a, b, ignored, reduction="none", return_hits=True)[0]
    assert _same(_both(ignore, long, w, up), _both(ignore, x, w, up))
    assert not losses.margin_cross_entropy(long, w, target, return_hits=True)[1][4]
    heavy = w.clone()
    heavy[9] *= 2.0 ** 66
    assert call(x, heavy).isnan().all()


def test_under_compiled_autograd():
    from torch._dynamo import compiled_autograd
    x, w, target, ids, logits = _inputs()
    for kind in KINDS:
        call = _calls(target, ids, logits)[kind]
        want = _both(call, x, w)
        a, b = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        with compiled_autograd._enable(lambda graph: torch.compile(graph, backend="eager")):
            call(a, b).backward()
        assert torch.equal(a.grad, want[1]) and torch.equal(b.grad, want[2]), kind
