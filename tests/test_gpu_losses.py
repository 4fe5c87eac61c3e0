"""Losses over many classes on the GPU against their formulas in 64 bits."""
import math

import pytest
import torch

from na1d_amd import losses
from oracle import losses_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAMES = ["bf16", "fp16"]
SIZES = [  # rows, channels, classes: one of each; below, at and above the tiles' 32, 64 and 128; several tiles each way
    (1, 8, 1), (1, 192, 3001), (5, 16, 2), (32, 72, 65), (33, 64, 63), (31, 136, 300), (128, 192, 1000), (130, 200, 129), (129, 128, 64),
    (257, 328, 1211), (1030, 40, 300), (4100, 64, 130), (300, 1032, 501),
]
LARGE = [  # launches that fill the card: tiles of 128 x 128 and of 256 x 256, products of either, several ranges of classes
    (1000, 264, 9001), (2100, 72, 5003), (700, 1032, 13000), (2050, 512, 16390), (16390, 16, 8300), (1500, 192, 9001), (1024, 512, 8000),
    (1500, 192, 3000), (1500, 960, 9000), (2050, 1024, 12000), (3000, 1024, 16000),
]


FEW_ROWS = [(1, 128, 50001), (20, 128, 50000), (32, 264, 30001), (31, 1032, 9000)]       # and a weight whose gradient fills the card


def _inputs(N, D, V, dtype, seed, strength=3.0):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype)
    target = torch.randint(0, V, (N,), generator=g)
    x = (torch.randn(N, D, generator=g) + strength * w[target].float()).to(dtype)
    return x.cuda(), w.cuda(), target.cuda()


def _upstream(reduction, ok, dtype, seed=5):
    n = len(ok)
    if reduction == "none":
        return torch.randn(n, generator=torch.Generator().manual_seed(seed)).cuda()
    return torch.tensor(16.0 * (max(1, int(ok.sum())) if reduction == "mean" else 1) if dtype == torch.float16 else 1.5, device="cuda")


def _near(name, got, want, bound):
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= bound).all()), "%s: off by %.3g where %.3g is allowed" % (
        name, off.max(), bound.flatten()[(off - bound).flatten().argmax()])


def _check(loss, grads, rows, ok, reduction, want_dx, want_dw, magnitudes, delta, up, dtype, extra_loss=1.0):
    torch.cuda.synchronize()
    want = O.reduced(rows, ok, reduction)
    _near("loss", loss, want, extra_loss * O.reduced(torch.where(ok, delta, 0.0), ok, reduction) + 2.0 ** -22 * want.abs())
    least = 2.0 ** -30 * float(O.shares(ok, reduction, up).abs().max())          # fp16: what is lost of scaled dz, 2^-38 a term
    bound_x, bound_w = O.gradient_bounds(want_dx, want_dw, magnitudes, delta, dtype, least)
    _near("dx", grads[0], want_dx, bound_x)
    _near("dweight", grads[1].reshape(want_dw.shape), want_dw, bound_w)


def _train(call, x, w, up):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = call(x, w)
    return loss.detach(), torch.autograd.grad(loss, [x, w], up)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("size", SIZES + LARGE + FEW_ROWS, ids=lambda s: "x".join(map(str, s)))
def test_cross_entropy(size, dtype):
    N, D, V = size
    print("cross entropy", size, dtype, flush=True)
    x, w, target = _inputs(N, D, V, dtype, 1)
    if N > 4:
        target[2::5] = -100
    for reduction, scale, ids in (("mean", 1.0, target), ("none", 2.5, target.int()), ("sum", 1.0, target)):
        rows, ok, e = O.softmax_targets(x, w, target, scale)
        up = _upstream(reduction, ok, dtype)
        loss, grads = _train(lambda a, b: losses.linear_cross_entropy(a, b, ids, scale=scale, reduction=reduction), x, w, up)
        _check(loss, grads, rows, ok, reduction, *O.linear_gradients(x, w, e, O.shares(ok, reduction, up)), O.logit_bound(x, w, scale), up, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("subs", [1, 2, 3, 5])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_margin(size, subs, dtype):
    _margin(size, subs, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("size,subs", [(s, 1) for s in LARGE] + [((2100, 72, 3003), 2), ((16390, 16, 4200), 3), ((260, 1024, 3000), 3), ((260, 512, 3000), 3)], ids=lambda s: str(s))
def test_margin_of_large_launches(size, subs, dtype):
    _margin(size, subs, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("subs", [2, 3, 4, 6, 20])
@pytest.mark.parametrize("size", [(40, 72, 70), (33, 64, 33), (200, 136, 97), (700, 200, 1003), (130, 1024, 1)], ids=lambda s: "x".join(map(str, s)))
def test_margin_of_many_weight_rows(size, subs, dtype):
    """Classes whose number ends in or short of a tile of as many classes as there is room for, and steps of 64 of them that the last tile leaves."""
    _margin(size, subs, dtype)


def _margin(size, subs, dtype):
    N, D, V = size
    print("margin", size, subs, dtype, flush=True)
    x, w, target = _inputs(N, D, V * subs, dtype, 2, strength=0.4 * D ** 0.5)
    w = w.view(V, subs, D)
    target = target // subs
    if N > 4:
        target[1::7] = -100
        x[3] = -w[int(target[3]), 0].float().to(dtype)            # an angle next to pi: past the margin's end
    reduction = "none" if subs == 2 else "mean"
    rows, ok, e, cosines = O.margin(x, w, target)
    up = _upstream(reduction, ok, dtype)
    given = w if subs > 1 else w.view(V, D)
    loss, grads = _train(lambda a, b: losses.margin_cross_entropy(a, b, target, reduction=reduction), x, given, up)
    ux, uw = O.unit(x.double()), O.unit(w.double().view(V * subs, D))
    # With a margin a target's logit moves 1 + sin(m) / sine times as far as its cosine, the slope sin(m) / sine^3 times.
    c = torch.where(ok.unsqueeze(1), cosines.view(N, V, subs).amax(2).gather(1, target.clamp(min=0).unsqueeze(1)), 0.0).squeeze(1)
    sine = torch.sqrt((1 - c * c).clamp(min=1e-6))
    delta = O.logit_bound(ux, uw, 32.0) * torch.where(c > math.cos(math.pi - 0.2), 1 + 0.2 / sine ** 3, 1.0)
    # 14 million cosines have classes whose two nearest rows differ by 3e-9, less than fp32 tells apart: such a share goes to either.
    dx, dw, magnitudes = O.margin_gradients(x, w, e, O.shares(ok, reduction, up))
    either_x, either_w = O.undecided(x, w, e, cosines, O.shares(ok, reduction, up))
    _check(loss, grads, rows, ok, reduction, dx, dw, lambda f: (magnitudes(f)[0] + either_x, magnitudes(f)[1] + either_w), delta, up, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("seed", range(8))
def test_a_single_rows_target_loses_little_in_rounding(seed, dtype):
    """Gradients of logits are scaled so that the target's, one number here, lies in the last eighth of a factor of two, where half a
    step is at most 2^(1/8) / 2 = 0.546 of u relative to it; the other classes' are off by u at most, each in a weight row of its own."""
    x, w, target = _inputs(1, 64, 500, dtype, 40 + seed, strength=3.0)
    w[(target + 1) % 500] *= 0.3 + 0.04 * seed                                           # a short row, by which alone no scale may go
    rows, ok, e, _ = O.margin(x, w.view(500, 1, 64), target)
    up = _upstream("mean", ok, dtype)
    _, (_, dw) = _train(lambda a, b: losses.margin_cross_entropy(a, b, target), x, w, up)
    _, want, _ = O.margin_gradients(x, w, e, O.shares(ok, "mean", up))
    u, mine = torch.finfo(dtype).eps / 2, torch.arange(500, device="cuda") == target
    once = (want.to(dtype).double() - want).norm()
    bound = u * torch.sqrt((0.546 * want[mine].norm()) ** 2 + want[~mine].norm() ** 2) + 1.1 * once + 2.0 ** -13 * want.norm() * u
    assert (dw.double() - want).norm() <= bound + 2.0 ** -17 * want.norm()               # and what fp32 logits are off


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("top", [1, 3, 64, 100, 256])
@pytest.mark.parametrize("size", [(1, 8, 1), (1, 64, 500), (33, 72, 63), (128, 192, 1000), (1030, 40, 300), (4100, 64, 130)],
                         ids=lambda s: "x".join(map(str, s)))
def test_distillation(size, top, dtype):
    _distillation(size, top, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("size", LARGE, ids=lambda s: "x".join(map(str, s)))
def test_distillation_of_large_launches(size, dtype):
    _distillation(size, 5, dtype)


def _distillation(size, top, dtype):
    N, D, V = size
    print("distillation", size, top, dtype, flush=True)
    x, w, target = _inputs(N, D, V, dtype, 3)
    g = torch.Generator().manual_seed(top)
    ids = torch.randint(-1, V, (N, top), generator=g)               # classes twice and more where there are few, and absent ones
    ids[:, 0] = target.cpu()
    logits = 2 * torch.randn(N, top, generator=g)
    logits[:, -1:] = -math.inf if top > 1 else logits[:, -1:]
    if N > 4:
        ids[4] = -1
        ids[N // 2, top // 2:] = -7
    ids, logits = ids.cuda(), logits.cuda()
    for reduction, temperature, logits_as, ids_as in (("mean", 2.0, logits.to(dtype), ids), ("none", 1.0, logits, ids.int()),
                                                      ("sum", 4.0, logits.to(torch.float16), ids)):
        rows, ok, e = O.teacher(x, w, logits_as, ids, temperature)
        up = _upstream(reduction, ok, dtype)
        loss, grads = _train(lambda a, b: losses.linear_distillation(a, b, logits_as, ids_as, temperature, reduction), x, w, up)
        g = O.shares(ok, reduction, up)
        dx, dw, magnitudes = O.linear_gradients(x, w, e, g)
        # What stands at an entry is the difference of two shares, each with an error of its own.
        p = torch.softmax(x.double() @ w.double().t() / temperature, 1) * temperature * ok.unsqueeze(1)
        both = O.linear_gradients(x, w, p, g)[2]
        delta = O.logit_bound(x, w, 1 / temperature) + 2.0 ** -18
        more = lambda f: tuple(a + b for a, b in zip(magnitudes(f), both(2 * delta + 2.0 ** -18)))
        _check(loss, grads, rows, ok, reduction, dx, dw, more, 2 * delta, up, dtype, extra_loss=temperature ** 2)


def test_gradients_that_are_differentiated_again_are_refused():
    x, w, target = _inputs(33, 64, 63, torch.float16, 4)
    x.requires_grad_(True)
    for call in (lambda: losses.linear_cross_entropy(x, w, target), lambda: losses.linear_cross_entropy(x[:, :], w.t().contiguous().t(), target)):
        plain = torch.autograd.grad(call(), x)[0]
        (dx,) = torch.autograd.grad(call(), x, create_graph=True)
        assert torch.equal(dx, plain)
        with pytest.raises(RuntimeError):
            dx.sum().backward()
