"""GPU tests of the paged 8-bit KV cache beside test_gpu_kv8.py: appends whose
tables, rows or slots are not as regular as a model's, to the byte."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv8 import ROW_TYPES, RefCache, i32, same_cache, tables  # noqa: E402


def shifted(t, by):
    """A copy of t that begins `by` floats into its allocation."""
    big = torch.empty(t.numel() + by, device="cuda")
    big[by:] = t.reshape(-1)
    return big[by:].view(t.shape)


@pytest.mark.parametrize("layout,dims", [("interleaved", 6), ("interleaved", 66), ("interleaved", 126),
                                         ("interleaved", 64), ("half", 8), ("half", 120)])
@pytest.mark.parametrize("kind,hd", [("f32", 128), ("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("rows", [5, 900])
def test_append_turns_k_alone(layout, dims, kind, hd, rows):
    """K rotated and no q: odd numbers of pairs, whose table rows begin on any
    4 bytes, and tables that begin there; single rows and windows of rows."""
    dims = min(dims, hd - 2) if dims % 4 else min(dims, hd)
    kv, size, ctx = 4, 16, 1000
    k, v = (torch.randn(rows, kv, hd).to(ROW_TYPES[kind]) for _ in "kv")
    pos, slots = list(range(1, 1 + rows)), list(range(size, size + rows))
    blocks = -(-rows // size) + 2
    for by in (0, 1, 2):
        cos, sin = (shifted(t, by) for t in tables(ctx, dims))
        cache, ref = F.KV8Cache.empty(blocks, kv, size, hd), RefCache(blocks, kv, size, hd, "int8")
        turned = torch.empty(rows, kv, hd, device="cuda")
        F.rope(k.cuda().float(), None, i32(pos), cos, sin, layout, turned, None)
        cache.append(k.cuda(), v.cuda(), i32(slots), i32(pos), cos, sin, layout)
        ref.append("k", turned.cpu(), slots)
        ref.append("v", v, slots)
        same_cache(cache, ref)
