"""Attention of streams as it is called: compiled, by several threads, kept and recomputed, under autocast, by a layer, beside the other paths."""
import threading

import pytest
import torch

from na1d_amd import _lib, ops, streaming
from oracle import streaming_oracle as O

pytestmark = pytest.mark.gpu


def _inputs(N, T, H, K, C, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(N, T, h, C, generator=g).to(dtype).cuda() for h in (H, K, K, H)]


def _grads(f, q, k, v, dout):
    q, k, v = (x.detach().requires_grad_(True) for x in (q, k, v))
    out = f(q, k, v)
    return (out.detach(),) + torch.autograd.grad(out, [q, k, v], dout)


def _same(a, b):
    torch.cuda.synchronize()
    assert len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_the_registered_op(dtype):
    q, k, v, dout = _inputs(2, 130, 4, 2, 40, dtype, 1)
    lengths = torch.tensor([130, 61], dtype=torch.int32, device="cuda")
    for t_valid in (None, lengths):
        want = _grads(lambda q, k, v: 2 * streaming.sink_attention(q, k, v, 20, 3, t_valid=t_valid), q, k, v, dout)
        _same(_grads(lambda q, k, v: 2 * ops.sink_attention_op(q, k, v, 20, 3, t_valid=t_valid), q, k, v, dout), want)
        compiled = torch.compile(lambda q, k, v: 2 * ops.sink_attention_op(q * 1, k, v, 20, 3, t_valid=t_valid), backend="aot_eager", fullgraph=True)
        _same(_grads(compiled, q, k, v, dout), want)
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(torch.ops.na_cuda.sink_attention_forward.default, (q, k, v, lengths, 20, 3, 0.2), test_utils=checks)
    out, saved = torch.ops.na_cuda.sink_attention_forward(q, k, v, None, 20, 3, 0.2)
    torch.library.opcheck(torch.ops.na_cuda.sink_attention_backward.default, (dout, q, k, v, None, out, saved, 20, 3, 0.2), test_utils=checks)


def test_the_op_compiled_for_any_length():
    compiled = torch.compile(lambda q, k, v: ops.sink_attention_op(q, k, v, 20, 3), backend="aot_eager", fullgraph=True, dynamic=True)
    for N, T in ((2, 50), (3, 77), (2, 131)):
        q, k, v, dout = _inputs(N, T, 4, 2, 64, torch.bfloat16, N + T)
        _same(_grads(compiled, q, k, v, dout), _grads(lambda q, k, v: streaming.sink_attention(q, k, v, 20, 3), q, k, v, dout))


def test_the_ops_gradients_are_not_differentiated_again():
    q, k, v, dout = _inputs(1, 40, 2, 2, 32, torch.bfloat16, 2)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(ops.sink_attention_op(q, k, v, 8), q, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dq.sum().backward()


def test_the_op_refuses_what_does_not_fit():
    q, k, v, dout = _inputs(1, 40, 2, 2, 32, torch.bfloat16, 3)
    out, saved = torch.ops.na_cuda.sink_attention_forward(q, k, v, None, 8, 0, 0.2)
    f, b = torch.ops.na_cuda.sink_attention_forward, torch.ops.na_cuda.sink_attention_backward
    for call in (lambda: f(q, k[:, :5], v, None, 8, 0, 0.2), lambda: f(q, k, v, None, 0, 0, 0.2), lambda: f(q, k, v, None, 8, -1, 0.2),
                 lambda: b(dout[:, :5], q, k, v, None, out, saved, 8, 0, 0.2), lambda: b(dout, q, k, v, None, out, saved[:-1], 8, 0, 0.2),
                 lambda: b(dout, q, k, v, None, out, saved.float(), 8, 0, 0.2), lambda: f(q, k, v, None, 8, 0, -1.0)):
        with pytest.raises((RuntimeError, ValueError)):
            call()


def test_the_python_node_does_what_the_native_one_does(monkeypatch):
    q, k, v, dout = _inputs(2, 200, 6, 2, 64, torch.bfloat16, 4)
    caches = [streaming.new_cache(2, 2, 80, 64, bits) for bits in (16, 4, 16, 4)]
    lengths = torch.tensor([150, 7], dtype=torch.int32, device="cuda")

    def calls(pair):
        got = list(_grads(lambda q, k, v: streaming.sink_attention(q, k, v, 33, 2), q, k, v, dout))
        for c in pair:
            streaming.cache_append(k, v, *c, sinks=2, t_valid=lengths)
            got.append(streaming.cache_step(q[:, :3], k[:, :3], v[:, :3], *c, lengths, 70, 2, scale=0.1))
            got.append(streaming.cache_attend(q[:, :2], *c, lengths + 3, 70, 2))
            got += [streaming.cache_rows(x) for x in c]
        return got

    first = calls(caches[:2])
    monkeypatch.setattr(_lib, "nodes", lambda: None)
    _same(first, calls(caches[2:]))


def test_several_threads_at_once():
    shapes = [(2, 300, 4, 2, 64), (1, 500, 8, 8, 32), (3, 130, 2, 1, 128), (2, 257, 6, 3, 80)]
    data = [_inputs(*s, torch.bfloat16, i) for i, s in enumerate(shapes)]
    call = lambda q, k, v: streaming.sink_attention(q, k, v, 50, 4)  # noqa: E731
    want = [_grads(call, *d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None] * len(data), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = _grads(call, *data[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(data))]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors
    for a, b in zip(got, want):
        _same(a, b)


def test_kept_graphs_recomputation_and_saved_inputs_that_change():
    q, k, v, dout = _inputs(2, 100, 4, 2, 64, torch.bfloat16, 5)
    want = _grads(lambda q, k, v: streaming.sink_attention(q, k, v, 30, 1), q, k, v, dout)
    again = _grads(lambda q, k, v: torch.utils.checkpoint.checkpoint(streaming.sink_attention, q, k, v, 30, 1, use_reentrant=False), q, k, v, dout)
    _same(want, again)
    qg = q.detach().requires_grad_(True)
    out = streaming.sink_attention(qg, k, v, 30, 1)
    first = torch.autograd.grad(out, qg, dout, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(out, qg, dout, retain_graph=True)[0])
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, qg, dout)


def test_a_cache_that_a_graph_needs_has_been_written_to():
    """What a cache's rows are used for beside attention sees that they change."""
    _, k, v, _ = _inputs(1, 4, 2, 2, 32, torch.bfloat16, 6)
    cache = streaming.new_cache(1, 2, 8, 32)
    weight = torch.ones(32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    for write in (lambda: streaming.cache_append(k, v, *cache),
                  lambda: streaming.cache_step(k, k, v, *cache, torch.zeros(1, dtype=torch.int32, device="cuda"), 4)):
        out = (cache[0] * weight).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()
    with torch.inference_mode():
        mine = streaming.new_cache(1, 2, 8, 32)
        streaming.cache_append(k, v, *mine)
        assert torch.equal(mine[0][:, :, :4].transpose(1, 2), k)


def test_inside_a_layer_under_autocast():
    """A pre-norm layer whose projection's output is read in place: gradients of its weights against the same layer in 64 bits."""
    torch.manual_seed(7)
    N, T, H, K, C, dim = 2, 150, 4, 2, 32, 64
    qkv, proj = torch.nn.Linear(dim, (H + 2 * K) * C).cuda(), torch.nn.Linear(H * C, dim).cuda()
    x = torch.randn(N, T, dim, device="cuda")

    def layer(x, attention, qkv, proj):
        q, k, v = qkv(x).view(N, T, H + 2 * K, C).split([H, K, K], 2)
        return x + proj(attention(q, k, v).reshape(N, T, H * C))

    params = [*qkv.parameters(), *proj.parameters()]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = layer(x, lambda q, k, v: streaming.sink_attention(q, k, v, 40, 2), qkv, proj)
    got = torch.autograd.grad(out.float().square().mean(), params)
    wide = [torch.nn.Linear(m.in_features, m.out_features).cuda().double() for m in (qkv, proj)]
    for a, b in zip(wide, (qkv, proj)):
        a.load_state_dict(b.state_dict())
    ref = layer(x.double(), lambda q, k, v: _attention64(q, k, v, 40, 2), *wide)
    want = torch.autograd.grad(ref.square().mean(), [p for m in wide for p in m.parameters()])
    # every tensor on the way is rounded to bf16 about ten times, each 2^-8 of it at most: the sum of independent ones stays under 2^-8 * 10
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) < 10 * 2.0 ** -8


def _attention64(q, k, v, window, sinks):
    H = q.shape[2]
    q, k, v = (x.transpose(1, 2).repeat_interleave(H // x.shape[2], 1) for x in (q, k, v))
    at = torch.arange(q.shape[2], device=q.device)
    s = (q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5).masked_fill(~O.visible(at, at, window, sinks), -torch.inf)
    return (torch.softmax(s, -1) @ v).transpose(1, 2)


def test_windows_that_see_everything_agree_with_the_dense_operator_on_the_last_row():
    """A query that sees all keys is a query of dense attention."""
    from na1d_amd.dense import global_attention
    q, k, v, _ = _inputs(3, 140, 4, 4, 64, torch.float16, 8)
    heads_first = lambda x: x.transpose(1, 2).reshape(12, 140, 64).contiguous()  # noqa: E731
    dense = global_attention(*map(heads_first, (q, k, v)), 4).view(3, 4, 140, 64)[:, :, -1]
    mine = streaming.sink_attention(q, k, v, 140)[:, -1]
    assert (mine.float() - dense.float()).abs().max() <= 2.0 ** -9 * float(v.abs().max())


def test_errors_of_the_native_call_carry_its_reason():
    q, k, v, _ = _inputs(1, 10, 2, 2, 32, torch.bfloat16, 9)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(_lib.NA1DError, match="scale"):
            streaming.sink_attention(q, k, v, 4, scale=scale)
        with pytest.raises(_lib.NA1DError, match="scale"):
            streaming.cache_step(q[:, :1], k[:, :1], v[:, :1], *streaming.new_cache(1, 2, 8, 32), torch.zeros(1, dtype=torch.int32, device="cuda"), 4, scale=scale)


@pytest.mark.parametrize("bits", [16, 4])
def test_caches_that_share_memory_are_refused(bits):
    """By the native path too, which passes them on to the checks."""
    q, kx, vx, _ = _inputs(2, 3, 4, 2, 32, torch.bfloat16, 50)
    k, v = streaming.new_cache(2, 2, 20, 32, bits)
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    rows = k.codes.view(torch.bfloat16).view(-1) if bits == 4 else k.view(-1)
    inside = rows[-2 * 3 * 2 * 32:].view(2, 3, 2, 32)
    for pair, tokens in (((k, k), (kx, vx)), ((k, v), (inside, vx)), ((v, k), (kx, inside))):
        with pytest.raises(_lib.NA1DError, match="share memory"):
            streaming.cache_append(*tokens, *pair)
        with pytest.raises(_lib.NA1DError, match="share memory"):
            streaming.cache_step(q, *tokens, *pair, lengths, 8)
    both = streaming.cache_attend(q, k, k, lengths + 3, 8)                # read only
    _same([both], [streaming.cache_attend(q, k, streaming.Rows4(*(t.clone() for t in k)) if bits == 4 else k.clone(), lengths + 3, 8)])


def test_a_sequence_beyond_32_bits():
    """Offsets of a head's rows pass 2^31 bytes: its last rows are those of a short sequence that ends with the same tokens.

    Both round what differs by sums in another order (2^-20 of the value at most: some hundred fp32 terms) to bf16, half a step each: a step in all, 2^-8 * 2, of
    which a norm keeps the same bound."""
    T, part, W = 560128, 1024, 70                     # T a multiple of a strip
    g = torch.Generator(device="cuda").manual_seed(51)
    q, k, v, dout = (torch.randn(1, T, 16, 128, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(4))
    assert q.numel() * 2 > 2 ** 31
    whole = _grads(lambda *x: streaming.sink_attention(*x, W), q, k, v, dout)
    short = _grads(lambda *x: streaming.sink_attention(*x, W), *(t[:, -part:].clone() for t in (q, k, v, dout)))
    for name, a, b in zip(("out", "dq", "dk", "dv"), whole, short):
        a, b = a[:, 2 * W - part:].double(), b[:, 2 * W:].double()
        assert float((a - b).norm()) <= (2 ** -7 + 2 ** -20) * float(b.norm()), name
    for t in whole:
        assert bool(torch.isfinite(t[:, ::4097]).all()) and float(t[:, -part:].abs().max()) > 0


@pytest.mark.parametrize("bits", [16, 4])
def test_streams_of_two_to_the_thirty_tokens(bits):
    """A stream's age matters by its place in the ring alone, up to 2^30 tokens; one that is older is idle."""
    N, K, C, W, Z, n = 3, 2, 64, 40, 3, 2
    ring = W + n - 1
    q, k, v, _ = _inputs(N, 200, 4, K, C, torch.float16, 52)
    old = 200 - n
    laps = ((1 << 30) - n - old) // ring              # as many as leave the stream at 2^30 or just below once the step is done

    def step(add):
        caches = streaming.new_cache(N, K, Z + ring, C, bits, torch.float16)
        streaming.cache_append(k[:, :old], v[:, :old], *caches, sinks=Z)
        lengths = torch.full((N,), old + add, dtype=torch.int32, device="cuda")
        outs = [streaming.cache_step(q[:, old:], k[:, old:], v[:, old:], *caches, lengths, W, Z), streaming.cache_attend(q[:, old:], *caches, lengths + n, W, Z)]
        return outs + [t for c in caches for t in (c if bits == 4 else (c,))]
    young = step(0)
    _same(young, step(ring * laps))
    assert old + ring * laps + n <= 1 << 30 < old + ring * (laps + 1) + n
    over = step(ring * (laps + 2))
    assert not bool(over[0].any()) and not bool(over[1].any()) and bool(young[0].any())
