"""GPU tests of the 4-bit cache with many KV heads (rows that several CTAs append
and read), many requests (several to a thread of the placement) and score
factors at the edges."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv4 import HALF_UNIT, ROW_TYPES, check_append, i32, make, reference, rope_tables, run_attention, slot_values  # noqa: E402


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("kv,hd", [(17, 128), (40, 128), (33, 64), (64, 64)])
def test_many_kv_heads(kind, kv, hd):
    g = torch.Generator().manual_seed(kv)
    rows, size, heads = 150, 16, 2 * kv
    y = torch.randn(rows, heads + 2 * kv, hd, generator=g).to(ROW_TYPES[kind]).cuda()
    q, k, v = y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    cache = F.KV4Cache.empty(rows // size + 3, kv, size, hd)
    slots = torch.randperm((rows // size + 3) * size, generator=g)[:rows].numpy()
    cos, sin = rope_tables(64, hd)
    pos = np.arange(rows) % 64
    for n in (3, rows):  # q in the same launch, and in one of its own
        check_append(k[:n], v[:n], slots[:n], cache, size)
        got = check_append(k[:n], v[:n], slots[:n], cache, size, pos[:n], (cos, sin), "half", q=q[:n])
        want = torch.empty_like(got)
        F.rope(q[:n], None, i32(pos[:n]), cos, sin, "half", want, None)
        assert torch.equal(got, want)
    ko, vo = (torch.empty(rows, kv, hd, device="cuda") for _ in "kv")
    cache.read(i32(slots), ko, vo)
    for name, out in (("k", ko), ("v", vo)):
        want = slot_values(cache, name, slots)
        assert (np.abs(out.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -24).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,hd", [(64, 64, 64), (80, 40, 128)])
def test_attention_of_many_kv_heads(kind, heads, kv, hd):
    for new in ([1, 1], [20, 3]):
        run_attention([300, 70], new, heads, kv, hd, 32, kind, seed=kv)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("most", [1, 3, 13, 40])
def test_a_thousand_requests(kind, most):
    """Of all lengths to 500, none among them, some without rows, over the same blocks."""
    n, heads, kv, hd = 1100, 4, 2, 64
    cache, table = make([500], heads, kv, hd, 32, most, junk=False)
    rng = np.random.default_rng(most)
    lengths = rng.integers(0, 501, n)
    lengths[::97] = 0
    new = np.ones(n, int) if most == 1 else np.minimum(rng.integers(0, most + 1, n), 2 ** 31)
    starts = [0] + list(np.cumsum(new))
    q = torch.randn(starts[-1], heads, hd, device="cuda").to(ROW_TYPES[kind])
    out, err = torch.full_like(q, 7.0), i32([0])
    tables = np.repeat(table, n, 0)
    cache.attention(q, i32(lengths), i32(tables), out, cache.attention_workspace(n, most, heads),
                    row_start=None if most == 1 else i32(starts), most_rows=most, error=err)
    want, tol, _ = reference(cache, tables, lengths.tolist(), starts, q, hd ** -0.5, kind)
    assert err.item() == 0
    assert ((out.cpu().double() - want).abs() <= tol + want.abs() * HALF_UNIT[kind] + 2.0 ** -25).all()


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-30, -1e-38, 1e-6])
def test_scales_next_to_nothing(kind, scale):
    """All weights are alike, whichever kernel runs."""
    for new in ([1, 1], [9, 2], [70, 33]):
        run_attention([200, 131], new, 8, 2, 128, 16, kind, seed=5, scale=scale)


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
def test_scale_that_is_no_number(kind):
    for new in (1, 9, 70):
        cache, table = make([200], 8, 2, 128, 16, 1)
        q = torch.randn(new, 8, 128, device="cuda").to(ROW_TYPES[kind])
        out = torch.zeros_like(q)
        cache.attention(q, i32([200]), i32(table), out, cache.attention_workspace(1, new, 8), row_start=i32([0, new]),
                        most_rows=new, scale=float("nan"))
        assert out.isnan().all()
