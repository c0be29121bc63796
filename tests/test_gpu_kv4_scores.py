"""GPU tests of attention over the 4-bit cache with query rows of 16 bits whose
scores are very large."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv4 import i32, make  # noqa: E402


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


@pytest.mark.parametrize("new", [9, 30, 130])
def test_large_scores_stay_in_their_row(new):
    """A row of scores beyond the resolution among ordinary ones changes no bit of theirs."""
    cache, table = make([300], 8, 2, 128, 32, new, junk=False)
    g = torch.Generator(device="cuda").manual_seed(new)
    q = torch.randn(new, 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    a, b, ws = torch.empty_like(q), torch.empty_like(q), cache.attention_workspace(1, new, 8)
    args = dict(row_start=i32([0, new]), most_rows=new)
    cache.attention(q, i32([300]), i32(table), a, ws, **args)
    for power in (22, 30, 60):
        q2 = q.clone()
        q2[new // 2, 3] *= 2.0 ** power
        cache.attention(q2, i32([300]), i32(table), b, ws, **args)
        assert b.isfinite().all()
        b[new // 2, 3] = a[new // 2, 3]
        assert torch.equal(a, b)
