"""That the errors of gradients, as norms, tell a backward with P and dS as one number each, or without the bytes that outputs lost in rounding, from one with them."""
import pytest
import torch

from oracle import streaming_oracle as O

SHAPES = [(300, 16, 300, 0), (500, 64, 60, 3), (400, 128, 400, 5), (300, 32, 20, 100), (200, 8, 50, 2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("T,C,W,Z", SHAPES)
def test_what_shows_in_the_norms(T, C, W, Z, dtype):
    """The results' rounding is 0.42 u of a norm (uniform within half a step), and independent errors add as squares: another rounding of every term makes 0.59 u of it, 0.17 more.  A row's sum of
    rounded probabilities, by which all of its P and dS are divided, and the output in its delta are 0.42 u of a term over the root of the number of keys that matter each: 0.3 u and less with
    these rows, and 0.1 u more.  An output rounded without its byte, its mean 3 times what the values vary by, is 1.2 u by itself."""
    for mean in (0.0, 3.0):
        q, k, v, dout = O.centred(1, T, 1, 1, C, dtype, mean)
        want = O.attention(q, k, v, W, Z, dout=dout)
        more = lambda **kw: {n: O.more_than_rounding(x, want[n][0]) for n, x in O.rounded_gradients(q, k, v, W, Z, dout, **kw).items()}  # noqa: E731
        assert all(x < 0.1 for x in more().values())
        single = more(ds_once=True)
        assert single["dq"] > 0.13 and single["dk"] > 0.13
        assert more(p_once=True)["dv"] > 0.13
        if mean:
            lost = more(bytes_lost=True)
            assert lost["dq"] > 0.5 and lost["dk"] > 0.5
            wrong = more(bytes_wrong=True)
            assert wrong["dq"] > 0.5 and wrong["dk"] > 0.5
