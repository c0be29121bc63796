"""GPU test of how far fp16 rows of attention over the 4-bit cache are off as a
whole."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv4 import i32, reference  # noqa: E402


@pytest.mark.parametrize("heads,kv,new", [(16, 2, 1), (8, 2, 2), (8, 2, 8), (8, 2, 16), (8, 2, 60), (6, 2, 100)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [600, 9000])
def test_error_of_fp16_rows(heads, kv, new, hd, n):
    """The norm of the error of fp16 rows with K and V as a model has them: row tiles of 8, 32, 64 and 256.

    V, a weight and the output are each rounded to fp16 once, K too: with weights and values of random sign such a rounding
    is uniform, 2^-11 / sqrt(3) of the value at the worst (a value just above a power of two), and independent from
    position to position, so each of the first three moves an output by that much of itself in the norm. K's moves a score
    by that of the root of the sum of (q k scale)^2, a product's size being about 1 / sqrt(hd) of the score's spread, which
    is 1 here: a weight by as much. Together at the most 4 x 2^-11 / sqrt(3) = 1.13e-3, if no two of them cancelled."""
    g = torch.Generator(device="cuda").manual_seed(n + hd + new)
    size = 64
    blocks = -(-n // size)
    cache = F.KV4Cache.empty(blocks, kv, size, hd)
    k, v = (torch.randn((n, kv, hd), generator=g, device="cuda") for _ in "kv")
    cache.append(k, v, i32(range(n)))
    q = torch.randn((new, heads, hd), generator=g, device="cuda").half()
    out, table = torch.empty_like(q), np.arange(blocks, dtype=np.int32)[None]
    cache.attention(q, i32([n]), i32(table), out, cache.attention_workspace(1, new, heads), row_start=i32([0, new]), most_rows=new)
    want, _, _ = reference(cache, table, [n], [0, new], q, hd ** -0.5, "f16")
    off = float((out.cpu().double() - want).norm() / want.norm())
    print("fp16 rows: %d heads of %d, %d rows, %d tokens: %.2e (rounded output alone %.2e)" %
          (heads // kv, hd, new, n, off, float((want.half().double() - want).norm() / want.norm())))
    assert off <= 4 * 2.0 ** -11 / 3 ** 0.5
