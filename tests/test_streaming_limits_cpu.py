"""Sizes at the limits of the native calls of streams' attention: what a launch does not hold is refused before it."""
import ctypes

import pytest

from na1d_amd import _lib, streaming

UNSUPPORTED, SCALE = -8, -11


def _sink(N, T, heads, kv_heads, head_dim=8, dtype=0, window=64, sinks=0, scale=0.125):
    h = streaming._Sink(dtype, heads, kv_heads, head_dim, scale, N, T, window, sinks)
    for n, k in (("q", heads), ("k", kv_heads), ("v", kv_heads)):
        setattr(h, n + "_strides", (ctypes.c_int64 * 3)(T * k * head_dim, head_dim, k * head_dim))
    return h


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("N,T,heads,kv_heads", [(1 << 24, 1, 1, 1), (1 << 20, 1, 16, 1), (1 << 10, 64, 1 << 14, 1 << 14), (1 << 10, 1 << 14, 64, 1), (1, 1 << 24, 64, 1), (1 << 18, 65, 32, 32)])
def test_sequences_of_more_workgroups_than_a_launch_has(N, T, heads, kv_heads, dtype):
    """2^24 of 256 threads are 2^32."""
    assert N * heads * -(-T // 64) >= 1 << 24
    lib, h = _lib.load(), ctypes.byref(_sink(N, T, heads, kv_heads, dtype=dtype))
    assert lib.na1d_sink_forward(h, 16, None, 0, 16, 16, 16, None, None) == UNSUPPORTED
    assert lib.na1d_sink_backward(h, *[16] * 9, 1 << 50, None, 16, 1 << 50, None) == UNSUPPORTED


@pytest.mark.parametrize("bits,head_dim", [(16, 8), (4, 32)])
@pytest.mark.parametrize("N,kv_heads,heads,fresh", [(1 << 24, 1, 1, 1), (1 << 12, 1 << 12, 1 << 12, 1), (1 << 20, 8, 8 * 65, 2), (1 << 20, 1, 1, 1 << 10)])
def test_caches_of_more_workgroups_than_a_launch_has(bits, head_dim, N, kv_heads, heads, fresh):
    lib, c = _lib.load(), streaming._Cache(0, bits, kv_heads, head_dim, N, fresh + 3, 1, 16, 16, 16, 16)
    s, ref = (ctypes.c_int64 * 3)(1 << 20, head_dim, 1 << 20), ctypes.byref(c)
    assert lib.na1d_sink_attend(ref, 16, 16, s, 16, fresh, heads, 2, 0.1, 16, 1 << 50, None) == UNSUPPORTED
    assert lib.na1d_sink_step(ref, 16, 16, 16, 16, s, s, s, 16, fresh, heads, 2, 0.1, 16, 1 << 50, None) == UNSUPPORTED
    if N * kv_heads == 1 << 24:
        assert lib.na1d_sink_append(ref, 16, 16, s, s, None, None, 5, None) == UNSUPPORTED


@pytest.mark.parametrize("scale", [2.4e38, 3.0e38])
def test_scales_whose_product_with_log2_e_is_infinite(scale):
    """An infinite factor times a score of 0 is no number."""
    lib, h = _lib.load(), ctypes.byref(_sink(1, 10, 2, 1, scale=scale))
    assert lib.na1d_sink_saved_bytes(h) == SCALE and lib.na1d_sink_backward_workspace_bytes(h) == SCALE
    assert lib.na1d_sink_forward(h, 16, None, 0, 16, 16, 16, None, None) == SCALE
    c, s = ctypes.byref(streaming._Cache(0, 16, 2, 8, 1, 9, 1, 16, 16, None, None)), (ctypes.c_int64 * 3)(16, 8, 16)
    assert lib.na1d_sink_attend(c, 16, 16, s, 16, 1, 2, 8, scale, 16, 1 << 50, None) == SCALE
    assert lib.na1d_sink_step(c, 16, 16, 16, 16, s, s, s, 16, 1, 2, 8, scale, 16, 1 << 50, None) == SCALE


def test_the_largest_scale():
    assert _lib.load().na1d_sink_saved_bytes(ctypes.byref(_sink(1, 10, 2, 1, scale=2.3e38))) > 0
