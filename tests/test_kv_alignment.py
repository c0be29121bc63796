"""Rows that begin off a whole element are refused by every entry point of the
paged caches before anything reaches a device, so no GPU is needed: a kernel's
access to them would be misaligned."""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

BUF = np.zeros(4096, np.float32)
AT = (BUF.ctypes.data + 255) // 256 * 256
P = C.c_void_p(AT)  # never read: every call below is refused
WIDTH = {0: 4, 1: 2, 30: 2}  # F32, F16, BF16


def caches():
    four = F.KV4CacheDesc(k=AT, v=AT, k_scale=AT, v_scale=AT, blocks=4, kv_heads=2, block_size=16, head_dim=64)
    eight = F.KV8CacheDesc(k=AT, v=AT, k_scale=AT, v_scale=AT, blocks=4, kv_heads=2, block_size=16, head_dim=64, format=0)
    return [(F.lib.fyb_kv4_append, F.lib.fyb_kv4_attention, four), (F.lib.fyb_kv8_append, F.lib.fyb_kv8_attention, eight)]


@pytest.mark.parametrize("type_", sorted(WIDTH))
@pytest.mark.parametrize("which", [0, 1])
def test_cache_rows(type_, which):
    append, attention, cache = caches()[which]
    rope = F.RopeDesc(cos_table=AT, sin_table=AT, table_rows=8, dims=64, layout=0)
    for off in range(1, WIDTH[type_]):
        bad = C.c_void_p(AT + off)
        for k, v in ((bad, P), (P, bad)):
            assert append(C.byref(cache), P, 1, type_, k, 128, v, 128, None, None, None, 0, None, 0, 0, None, None) == -1
        for q, o in ((bad, P), (P, bad)):
            assert append(C.byref(cache), P, 1, type_, P, 128, P, 128, C.byref(rope), P, q, 256, o, 256, 4, None, None) == -1
            assert attention(C.byref(cache), P, None, 1, 1, 1, P, 1, type_, q, 256, o, 256, 4, 0.1, P, 1 << 40, None, None) == -1


@pytest.mark.parametrize("type_", sorted(WIDTH))
def test_rope_rows(type_):
    rope = F.RopeDesc(cos_table=AT, sin_table=AT, table_rows=8, dims=64, layout=0)
    for off in range(1, WIDTH[type_]):
        for i in range(4):
            q, qo, k, ko = (C.c_void_p(AT + off) if j == i else P for j in range(4))
            assert F.lib.fyb_rope(C.byref(rope), P, 1, 64, type_, q, 256, qo, 256, 4, k, 128, ko, 128, 2, None, None) == -1
