"""GPU tests of the numbers that the 4-bit cache holds, byte for byte, where a
group's low and high, rounded to F16, no longer enclose its values: x lies below
low or above low + 15 scale, and the number is 0 or 15 all the same."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from . import test_gpu_kv4  # noqa: E402
from .test_gpu_kv4 import ROW_TYPES, check_append, i32, rope_tables, slot_values  # noqa: E402


@pytest.fixture(autouse=True)
def minus_zero_is_less(monkeypatch):
    """The definition's least value: of zeros of both signs -0, where numpy's minimum is whichever it meets. (The sign of low
    is a bit that is held; the values are the same.)"""
    plain = test_gpu_kv4.hold

    def hold(x):
        n, scale, low = plain(x)
        groups = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], -1, 64)
        minus = ((groups == 0) & np.signbit(groups)).any(-1) & (np.where(np.isfinite(groups), groups, np.inf).min(-1) == 0)
        return n, scale, np.where(minus, np.float16(-0.0), low)

    monkeypatch.setattr(test_gpu_kv4, "hold", hold)

BASES = [1.0, -1.0, 10.0, 100.0, -100.0, 6e4, -6e4]
UNITS = [0.5, 1.0, 2.0, 3.0, 5.0, 8.0, 12.0, 20.0]  # ranges, in steps of F16 at the base
SMALL = [1e-8, 1e-7, 4e-7, 1e-6, 3e-6, 1e-5, 1e-4]


def narrow_rows(hd, seed):
    """[rows][2][hd] F32: groups of a small range about a base or about zero, in both heads."""
    g = torch.Generator().manual_seed(seed)
    rows = []
    for base in BASES:
        step = float(np.spacing(np.float16(abs(base))))
        for units in UNITS:
            rows.append(base + units * step * (torch.rand(2, hd, generator=g) - 0.5))
        rows.append(base + step * torch.linspace(-3.0, 4.0, hd).repeat(2, 1))
        rows.append(base + base * 0.0005 * torch.randn(2, hd, generator=g))
    for s in SMALL:
        rows += [s * torch.randn(2, hd, generator=g), s * torch.linspace(-1.5, 1.5, hd).repeat(2, 1), s * torch.rand(2, hd, generator=g)]
    return torch.stack(rows).float()


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("aligned", [True, False])
def test_narrow_groups(kind, hd, aligned):
    x = narrow_rows(hd, hd).to(ROW_TYPES[kind]).cuda()
    if not aligned:
        x = torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(x.shape)
    rows, size = len(x), 16
    cache = F.KV4Cache.empty(2 * rows // size + 2, 2, size, hd)
    check_append(x, -x, np.arange(rows), cache, size)
    # what is held is at most half a step, or what low and high lost by rounding, away
    ko, vo = (torch.empty(rows, 2, hd, device="cuda") for _ in "kv")
    cache.read(i32(np.arange(rows)), ko, vo)
    assert torch.equal(ko.cpu().double(), torch.from_numpy(slot_values(cache, "k", np.arange(rows))).float().double())
    y = x.float().cpu().double()
    far = (ko.cpu().double() - y).abs().unflatten(-1, (hd // 64, 64)).amax(-1)
    top, wide = (t.unflatten(-1, (hd // 64, 64)) for t in (y.abs(), y))
    step = (wide.amax(-1) - wide.amin(-1)) / 15
    lost = top.amax(-1) * 2.0 ** -11 + 2.0 ** -25  # of low and of high; scale is off by as much of itself, 15 times
    assert (far <= step / 2 + 2 * lost + step * 15 * 2.0 ** -11 + 15 * 2.0 ** -25).all()


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_narrow_groups_rotated(kind, layout):
    """Positions 0, whose rotation changes nothing, and others."""
    hd, size = 128, 32
    x = narrow_rows(hd, 3).to(ROW_TYPES[kind]).cuda()
    rows = len(x)
    cos, sin = rope_tables(50, hd)
    cache = F.KV4Cache.empty(rows // size + 2, 2, size, hd)
    for pos in (np.zeros(rows, int), np.arange(rows) % 50):
        check_append(x, x, np.arange(rows), cache, size, pos, (cos, sin), layout)
        check_append(x, x, np.arange(rows), cache, size, pos, (cos, sin), layout, q=x[:, :1].contiguous())
