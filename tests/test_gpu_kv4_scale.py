"""GPU test of the 4-bit cache's scale: (high - low) / 15 as a real number, rounded
to F16 once. With low and high many bits apart the difference does not fit F32,
or the quotient in F32 falls on a border between two halves that the real one
does not lie on."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv4 import check_append, hold  # noqa: E402

#: (low, high), both halves: real quotients next to a border between two halves, on either side of it
PAIRS = [(511 * 2.0 ** -24, 1.00390625), (511 * 2.0 ** -24, float.fromhex("0x1.22cp0")), (-511 * 2.0 ** -23, float.fromhex("0x1.264p1")),
         (float.fromhex("0x1.ff4p-9"), float.fromhex("0x1.6ap7")), (float.fromhex("0x1.ff4p-14"), float.fromhex("0x1.cb8p2")),
         (float.fromhex("0x1.804p-10"), float.fromhex("0x1.17cp4")), (float.fromhex("0x1.ffcp-10"), float.fromhex("0x1.178p6")),
         (-511 * 2.0 ** -23, float.fromhex("0x1.78cp1")), (float.fromhex("0x1.ffcp-12"), float.fromhex("0x1.40cp4"))]


@pytest.mark.parametrize("hd", [64, 128])
def test_scale_is_rounded_once(hd):
    rows = []
    g = torch.Generator().manual_seed(1)
    for low, high in PAIRS:
        for a, b in ((low, high), (-high, -low)):
            row = a + (b - a) * torch.rand(1, hd, generator=g, dtype=torch.float64)
            row[0, ::64], row[0, 37::64] = a, b
            rows.append(row.clamp(a, b).float())
    x = torch.stack(rows)
    _, scale, _ = hold(x.numpy())
    narrow = [np.float16(np.float32(np.float32(np.float32(b) - np.float32(a)) / np.float32(15))) for a, b in PAIRS]
    assert sum(n != s for n, s in zip(narrow, scale[::2, 0, 0])) > len(PAIRS) // 2  # pairs that F32 does not settle
    cache = F.KV4Cache.empty(4, 1, 16, hd)
    check_append(x.cuda(), x.flip(-1).contiguous().cuda(), np.arange(len(x)), cache, 16)


def test_scales_of_all_kinds():
    """Random low and high of every pair of magnitudes."""
    rng = np.random.default_rng(2)
    halves = np.arange(0x7b81, dtype=np.uint16).view(np.float16).astype(np.float64)
    halves = np.concatenate([halves[halves <= 61440], -halves[halves <= 61440]])
    ends = np.sort(rng.choice(halves, (4000, 4, 2)), -1)
    x = ends[..., :1] + (ends[..., 1:] - ends[..., :1]) * rng.random((4000, 4, 64))
    x[..., 5], x[..., 50] = ends[..., 0], ends[..., 1]
    x = torch.from_numpy(np.clip(x, ends[..., :1], ends[..., 1:])).float().reshape(4000, 2, 128).cuda()
    check_append(x, -x, np.arange(4000), F.KV4Cache.empty(32, 2, 128, 128), 128)
