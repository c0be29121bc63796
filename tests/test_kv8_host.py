"""The paged 8-bit KV cache on the host side, beside test_kv8.py: where rotary
frequencies leave the usual contexts, what is refused before a GPU is asked, and
calls that have nothing to do."""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

from .test_kv8 import P, desc, rope_desc


@pytest.mark.parametrize("dims,base,factor,ctx", [(128, 10000.0, 16.0, 65536.0), (128, 10000.0, 4.0, 131072.0),
                                                  (64, 10000.0, 8.0, 1048576.0), (128, 1000000.0, 4.0, 32768.0)])
def test_frequencies_yarn_past_the_last_pair(dims, base, factor, ctx):
    """Long original contexts: the slowest pair still makes more than beta_slow
    turns, so the ramp ends past it and no pair is interpolated whole. F32
    results of a formula in 64 bits: half a unit, 2^-24."""
    got, _ = F.rope_frequencies(dims, base, "yarn", factor, ctx)
    j = np.arange(dims // 2)
    f = base ** (-2.0 * j / dims)
    at = lambda turns: dims * np.log(ctx / (2 * np.pi * turns)) / (2 * np.log(base))  # noqa: E731
    lo, hi = np.floor(at(32.0)), np.ceil(at(1.0))
    assert 0 <= lo < hi <= dims - 1 and (hi > dims // 2 - 1) == (ctx > 32768)
    ramp = np.clip((j - lo) / (hi - lo), 0, 1)
    want = f * (1 - ramp) + f / factor * ramp
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * want * (1 + 1e-6))


def test_unknown_format_is_a_value_error():
    with pytest.raises(ValueError, match="e4m3"):
        F.KV8Cache.empty(4, 2, 16, 64, "int4", device="cpu")


def test_no_rows_need_no_rows():
    """Rows of an empty tensor have no address: with a count of 0 none is asked for, and the rest is still checked."""
    cache, turn = C.byref(desc()), C.byref(rope_desc())

    def append(k_stride=128, heads=4, q_stride=256):
        return F.lib.fyb_kv8_append(cache, None, 0, 0, None, k_stride, None, 128, turn, None, None, q_stride, None, 256,
                                    heads, None, None)
    assert append() == 0 and append(heads=0) == 0
    assert append(k_stride=127) == append(q_stride=255) == -1
    assert F.lib.fyb_kv8_read(cache, None, 0, None, None, None, None) == 0

    def rope(heads=2, kv_heads=1, q_stride=128):
        return F.lib.fyb_rope(turn, None, 0, 64, 0, None, q_stride, None, 128, heads, None, 64, None, 64, kv_heads, None,
                              None)
    assert rope() == 0 and rope(heads=0) == 0 and rope(kv_heads=0) == 0
    assert rope(q_stride=127) == rope(heads=0, kv_heads=0) == -1

    def attention(lengths=P, starts=P):
        return F.lib.fyb_kv8_attention(cache, lengths, starts, 1, 1, 0, P, 1, 0, None, 256, None, 256, 4, 0.1, P, 1 << 40,
                                       None, None)
    assert attention() == 0
    assert attention(lengths=None) == attention(starts=None) == -1


def test_a_batch_that_was_never_made_closes():
    batch = F.Batch.__new__(F.Batch)
    assert batch.ptr is None
    batch.close()
