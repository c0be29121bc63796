"""GPU tests of attention over the 4-bit cache with query rows of 16 bits: how
far fp16 rows are off as a whole, and scores that are very large."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv4 import i32, make, reference  # noqa: E402


@pytest.mark.parametrize("new", [1, 2, 8, 9, 30, 65, 130])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("power", [24, 28, 33, 40])
def test_scores_beyond_the_resolution(new, hd, power):
    """Largest scores of some 2^power, where F32 numbers lie up to 2^(power - 23) apart: the weights stay finite, and an
    output lies within its group's values."""
    heads, kv, n = 8, 2, 700
    cache, table = make([n], heads, kv, hd, 32, power, junk=False)
    g = torch.Generator(device="cuda").manual_seed(power + new)
    q = torch.randn(new, heads, hd, generator=g, device="cuda").to(torch.bfloat16)
    out, err = torch.full_like(q, 7.0), i32([0])
    for sign in (1.0, -1.0):
        cache.attention(q, i32([n]), i32(table), out, cache.attention_workspace(1, new, heads), row_start=i32([0, new]),
                        most_rows=new, scale=sign * 2.0 ** (power - 6), error=err)
        assert err.item() == 0 and out.isfinite().all()
        use = cache.tensors[3][torch.tensor(table[0], device="cuda").long()].float()  # scale, low
        top = (15 * use[..., 0] + use[..., 1].abs()).amax((0, 2)).repeat_interleave(64, -1)  # [kv][hd]
        assert (out.float().unflatten(1, (kv, heads // kv)).abs() <= 1.01 * top[None, :, None]).all()


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
