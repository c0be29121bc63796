"""GPU tests of attention over the paged 4-bit cache with many query rows of 16
bits per KV head (row tiles of 32, 64 and 256): long requests in many parts, bad
tables, streams and graphs, large pools, rows that are not aligned. The
definition in 64 bits and its tolerances are test_gpu_kv4's.
"""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402
from .test_gpu_kv4 import ROW_TYPES, HALF_UNIT, i32, make, reference, run_attention  # noqa: E402

TILES = [8, 16, 60]  # rows of a request that fill row tiles of 32, 64 and 256 with four heads a group


@pytest.mark.parametrize("rows", [8, 9, 16, 17, 32, 33, 40, 64, 65, 96])
@pytest.mark.parametrize("hd,kind", [(64, "f16"), (128, "bf16")])
def test_many_parts(rows, hd, kind):
    """One long request: its segments are shared by many CTAs. Row tiles full and with one row more."""
    run_attention([7001], [rows], 8, 2, hd, 64, kind, seed=rows)
    run_attention([300, 4500], [3, rows], 4, 1, hd, 16, kind, seed=rows + 1)


@pytest.mark.parametrize("group", [3, 5, 7, 33, 64])
def test_groups(group):
    """Row tiles that a group's heads do not fill."""
    for rows in (1, 2, 5, 40):
        run_attention([77 + rows, 1300], [rows, rows], group, 1, 128, 32, "f16", seed=group + rows)


@pytest.mark.parametrize("most", TILES)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_bad_tables_and_lengths(most, kind):
    lengths = [100, 90, 400]
    cache, table = make(lengths, 8, 2, 128, 16, 4)
    starts = i32([0, most, 2 * most, 3 * most])
    q = torch.randn(3 * most, 8, 128, device="cuda").to(ROW_TYPES[kind])
    good, bad = torch.empty_like(q), torch.empty_like(q)
    ws, err = cache.attention_workspace(3, most, 8), i32([0])
    call = lambda t, le, out: cache.attention(q, i32(le), i32(t), out, ws, row_start=starts, most_rows=most, error=err)  # noqa: E731
    call(table, lengths, good)
    assert err.item() == 0
    rest = torch.tensor([*range(most), *range(2 * most, 3 * most)], device="cuda")
    for value in (-1, 10 ** 6, 2 ** 31 - 1):
        t = table.copy()
        t[1, 2] = value
        err.zero_()
        call(t, lengths, bad)
        assert err.item() == 4 and torch.equal(bad[rest], good[rest]) and bad.isfinite().all()
    err.zero_()
    call(table, [100, table.shape[1] * 16 + 1, 400], bad)
    assert err.item() == 4 and torch.equal(bad[rest], good[rest]) and (bad[most:2 * most] == 0).all()
    # a length below zero holds nothing
    err.zero_()
    call(table, [100, -5, 400], bad)
    assert torch.equal(bad[rest], good[rest]) and (bad[most:2 * most] == 0).all()


@pytest.mark.parametrize("rows", TILES)
def test_graphs_share_a_workspace(rows):
    """Two captured calls, one of them of single tokens, replayed in turn on one workspace and one stream, at lengths that
    change between replays: parts, counters and joins of one leave nothing for the other."""
    lengths = [[3000, 200], [150, 2900], [1, 70]]
    cache, table = make([3000, 3000], 8, 2, 128, 32, 4, junk=False)
    t, le = i32(table), i32(lengths[0])
    q = torch.randn(2 * rows, 8, 128, device="cuda").to(torch.bfloat16)
    q1 = q[:2].contiguous()
    args = dict(row_start=i32([0, rows, 2 * rows]), most_rows=rows)
    want = []
    for n in lengths:
        a, b = torch.empty_like(q), torch.empty_like(q1)
        cache.attention(q, i32(n), t, a, cache.attention_workspace(2, rows, 8), **args)
        cache.attention(q1, i32(n), t, b, cache.attention_workspace(2, 1, 8))
        want.append((a, b))
    ws, out, out1 = cache.attention_workspace(2, rows, 8), torch.empty_like(q), torch.empty_like(q1)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        cache.attention(q, le, t, out, ws, **args)
    with torch.cuda.graph(graphs[1]):
        cache.attention(q1, le, t, out1, ws)
    for i in (0, 1, 2, 1, 0):
        le.copy_(i32(lengths[i]))
        out.fill_(3.0)
        out1.fill_(3.0)
        graphs[0].replay()
        graphs[1].replay()
        graphs[0].replay()
        assert torch.equal(out, want[i][0]) and torch.equal(out1, want[i][1]), i


@pytest.mark.parametrize("rows", TILES)
def test_streams(rows):
    """On another stream behind work of its own, and two calls at once with a workspace each."""
    cache, table = make([3000, 1700], 8, 2, 128, 32, 4, junk=False)
    q = torch.randn(2 * rows, 8, 128, device="cuda").to(torch.float16)
    args = dict(row_start=i32([0, rows, 2 * rows]), most_rows=rows)
    le, t, want = i32([3000, 1700]), i32(table), torch.empty_like(q)
    cache.attention(q, le, t, want, cache.attention_workspace(2, rows, 8), **args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, spaces = [torch.empty_like(q) for _ in streams], [cache.attention_workspace(2, rows, 8) for _ in streams]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big  # the stream is busy; q changes behind it
        q2 = torch.zeros_like(q).copy_(q)
        cache.attention(q2, le, t, outs[0], spaces[0], **args)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    for _ in range(20):
        for s, o, w in zip(streams, outs, spaces):
            cache.attention(q, le, t, o, w, stream=s.cuda_stream, **args)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("rows", TILES)
def test_rows_that_are_not_aligned(rows):
    """q and out that begin on any element, with gaps between their rows that are left as they were."""
    lengths, hd = [90 + rows, 2500], 128
    cache, table = make(lengths, 8, 2, hd, 16, rows)
    args = dict(row_start=i32([0, rows, 2 * rows]), most_rows=rows)
    ws = cache.attention_workspace(2, rows, 8)
    for kind in ("f16", "bf16"):
        q = torch.randn(2 * rows, 8, hd, device="cuda").to(ROW_TYPES[kind])
        want, tol, _ = reference(cache, table, lengths, [0, rows, 2 * rows], q, hd ** -0.5, kind)
        for off, gap in ((1, 3), (8, 8), (4, 12)):
            def wide(fill):
                return torch.full((off + 2 * rows * (8 * hd + gap),), fill, dtype=ROW_TYPES[kind], device="cuda")
            def rows_of(x):
                return x[off:].unflatten(0, (2 * rows, 8 * hd + gap))[:, :8 * hd].unflatten(1, (8, hd))
            qs, outs = wide(float("nan")), wide(7.0)
            rows_of(qs).copy_(q)
            cache.attention(rows_of(qs), i32(lengths), i32(table), rows_of(outs), ws, **args)
            got = rows_of(outs).cpu().double()
            assert ((got - want).abs() <= tol + want.abs() * HALF_UNIT[kind] + 2.0 ** -25).all()
            rows_of(outs).fill_(7.0)
            assert (outs == 7).all()


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB: the same blocks at its two ends give the same output."""
    kv, size, hd = 2, 256, 128
    blocks = (1 << 32) // (kv * size * hd // 2) + 40
    cache = F.KV4Cache.empty(blocks, kv, size, hd)
    low, high = [1, 2, 3], [blocks - 1, blocks - 20, blocks - 3]
    for t in cache.tensors[:2]:
        t[low] = torch.randint(0, 256, (3, kv, size, hd // 2), device="cuda").to(torch.uint8)
        t[high] = t[low]
    for t in cache.tensors[2:]:
        t[low] = torch.randn(3, kv, size, 2, 2, device="cuda").to(torch.float16) * 0.1
        t[high] = t[low]
    for new in TILES:
        q = torch.randn(new, 8, hd, device="cuda").to(torch.bfloat16)
        q2, out = torch.cat([q, q]), torch.empty(2 * new, 8, hd, dtype=torch.bfloat16, device="cuda")
        cache.attention(q2, i32([2 * size + 81] * 2), i32([low, high]), out, cache.attention_workspace(2, new, 8),
                        row_start=i32([0, new, 2 * new]), most_rows=new)
        assert torch.equal(out[:new], out[new:]) and (out != 0).any()


def test_many_requests():
    """Requests that attend the same blocks, some with no rows."""
    cache, table = make([900], 8, 2, 128, 32, 3, junk=False)
    n = 70
    new = [(5 * r) % 23 for r in range(n)]
    starts = [0] + list(np.cumsum(new))
    q = torch.randn(starts[-1], 8, 128, device="cuda").to(torch.bfloat16)
    lengths = [900 - 11 * r for r in range(n)]
    out = torch.empty_like(q)
    cache.attention(q, i32(lengths), i32(np.repeat(table, n, 0)), out, cache.attention_workspace(n, max(new), 8),
                    row_start=i32(starts), most_rows=max(new))
    want, tol, _ = reference(cache, np.repeat(table, n, 0), lengths, starts, q, 128 ** -0.5, "bf16")
    assert ((out.cpu().double() - want).abs() <= tol + want.abs() * HALF_UNIT["bf16"] + 2.0 ** -25).all()
