"""GPU tests of the paged 8-bit KV cache beside test_gpu_kv8.py: lengths at
their end, operands that are left out, appends whose tables, rows or slots are
not as regular as a model's (to the byte), scores and value scales far apart."""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv8 import ROW_TYPES, RefCache, i32, run_attention, same_cache, tables  # noqa: E402


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


def left_out(ref, name, rows, slots, drop):
    """ref.append of rows of which `drop` have a slot but are not stored: they belong to their block's rows (the first
    of which says where its older tokens end), and neither count for its scale nor change its bytes."""
    size = ref.size
    lost = {b for b in (int(s) // size for s in slots if s >= 0)
            if all(drop[i] for i, s in enumerate(slots) if s >= 0 and s // size == b)}
    slots = [-1 if s >= 0 and s // size in lost else s for s in slots]
    rows, kept = rows.float().clone(), {}
    for i, s in enumerate(slots):
        if drop[i] and s >= 0:
            rows[i] = 0
            kept[s] = ref.x[name][s // size, :, s % size].clone()
    ref.append(name, rows, slots)
    for s, x in kept.items():
        ref.x[name][s // size, :, s % size] = x


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("kind,hd,size", [("f32", 128, 16), ("bf16", 64, 32), ("f16", 128, 256)])
@pytest.mark.parametrize("rows", [7, 40, 1500])
def test_rows_left_out_of_a_block(fmt, kind, hd, size, rows):
    """Rows with a position outside the table, without a slot or with one past the pool, among rows of their block:
    the others are stored as if alone, from a single row a CTA to windows of a block. The blocks had another owner
    before, with larger scales, and the first has older tokens of its own."""
    kv, heads, ctx, first = 3, 2, 2000, 5
    rng = np.random.default_rng(rows + size)
    blocks = -(-(first + rows) // size) + 3
    order = rng.permutation(blocks).tolist()
    slot = lambda p: order[p // size] * size + p % size  # noqa: E731
    cos, sin = tables(ctx, hd)
    cache, ref = F.KV8Cache.empty(blocks, kv, size, hd, fmt), RefCache(blocks, kv, size, hd, fmt)

    def append(k, v, slots, pos):
        q = torch.randn(len(slots), heads, hd).to(ROW_TYPES[kind]).cuda()
        qo, turned = torch.empty_like(q), torch.empty(len(slots), kv, hd, device="cuda")
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        cache.append(k.cuda(), v.cuda(), i32(slots), i32(pos), cos, sin, "half", q, qo, error=err)
        F.rope(k.cuda().float(), None, i32(pos), cos, sin, "half", turned, None)
        mine = [s if s < blocks * size else -1 for s in slots]
        left_out(ref, "k", turned.cpu(), mine, [not 0 <= p < ctx for p in pos])
        ref.append("v", v, mine)
        same_cache(cache, ref)
        return err.item()

    whole = [b * size + t for b in range(blocks) for t in range(size)]
    k, v = (torch.randn(len(whole), kv, hd).to(ROW_TYPES[kind]) * 50 for _ in "kv")
    append(k, v, whole, [0] * len(whole))
    k, v = (torch.randn(first, kv, hd).to(ROW_TYPES[kind]) for _ in "kv")
    assert append(k, v, [slot(p) for p in range(first)], list(range(first))) == 0
    for what in ("middle", "edges", "many", "slots"):
        k, v = (torch.randn(rows, kv, hd).to(ROW_TYPES[kind]) for _ in "kv")
        at = np.arange(first, first + rows)
        pos, slots = at.copy(), [slot(int(p)) for p in at]
        if what == "middle":
            pos[at % size == size // 2] = ctx
        if what == "edges":
            pos[(at % size == 0) | (at % size == size - 1) | (at == first)] = -1
        if what == "many":
            pos[rng.random(rows) < 0.7] = ctx + 7
        if what == "slots":  # rows of a block stay within its size of one another
            gone = rng.random(rows) < 0.3
            slots = [(-1 if p % 2 else 2 ** 31 - 1) if g else s for g, p, s in zip(gone, at, slots)]
        err = append(k, v, slots, [int(p) for p in pos])
        assert err == (4 if any(not 0 <= p < ctx for p in pos) or any(s > blocks * size for s in slots) else 0)


@pytest.mark.parametrize("kind,hd,dims", [("bf16", 128, 128), ("f32", 64, 32)])
@pytest.mark.parametrize("rows", [3, 9001])
def test_rope_of_k_alone(kind, hd, dims, rows):
    """No q, from a few rows to enough that they go through shared memory: k as it is beside a q."""
    kv, ctx = 8, 700
    cos, sin = tables(ctx, dims)
    pos = torch.randint(0, ctx, (rows,), dtype=torch.int32).cuda()
    k = torch.randn(rows, kv, hd, device="cuda").to(ROW_TYPES[kind])
    beside, alone, none = torch.empty_like(k), torch.full_like(k, 7.0), k[:, :0]
    F.rope(k, k, pos, cos, sin, "half", torch.empty_like(k), beside)
    desc = F.RopeDesc(cos.data_ptr(), sin.data_ptr(), ctx, dims, 1)
    stream = torch.cuda.current_stream().cuda_stream
    type_ = {"f32": 0, "bf16": 30}[kind]
    assert F.lib.fyb_rope(C.byref(desc), pos.data_ptr(), rows, hd, type_, None, 0, None, 0, 0, k.data_ptr(), kv * hd,
                          alone.data_ptr(), kv * hd, kv, None, stream) == 0
    assert torch.equal(alone, beside)
    alone.fill_(7.0)
    F.rope(none, k, pos, cos, sin, "half", none, alone)
    assert torch.equal(alone, beside)


def test_cache_of_another_gpu_is_refused():
    """A cache whose tensors are not on the current device, beside tensors that are: as for any tensor, nothing is
    launched. (One GPU is enough: the cache only says that it is elsewhere.)"""
    cache = F.KV8Cache.empty(4, 2, 16, 64)
    k, v = torch.randn(2, 3, 2, 64, device="cuda")
    q, lengths, table, slots = torch.randn(1, 4, 64, device="cuda"), i32([3]), i32([[0]]), i32([0, 1, 2])
    ws = cache.attention_workspace(1, 1, 4)
    ko, vo = torch.full((2, 3, 2, 64), 7.0, device="cuda")
    out = torch.full_like(q, 7.0)
    calls = [lambda: cache.append(k, v, slots), lambda: cache.read(slots, ko, vo),
             lambda: cache.attention(q, lengths, table, out, ws)]
    here = torch.cuda.current_device()
    assert cache._held.device == here
    cache._held.device = here + 1
    for call in calls:
        with pytest.raises(ValueError, match="cache"):
            call()
    assert all((t.view(torch.uint8) == 0).all() for t in cache.tensors)
    assert (ko == 7.0).all() and (vo == 7.0).all() and (out == 7.0).all()
    cache._held.device = here
    for call in calls:
        call()
    assert (ko != 7.0).all() and (out != 7.0).all()


def test_no_rows():
    """Steps without a row, as torch makes them (empty tensors have no address): nothing is done and nothing refused."""
    cache, empty = F.KV8Cache.empty(4, 2, 16, 64), i32([])
    before = [t.clone() for t in cache.tensors]
    k, q = torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 4, 64, device="cuda")
    cos, sin = tables(8, 64)
    F.rope(q, k, empty, cos, sin, "half", q, k)
    F.rope(q, None, empty, cos, sin, "interleaved", torch.empty_like(q), None)
    cache.append(k, k, empty)
    cache.append(k, k, empty, empty, cos, sin, "half", q, q)
    cache.read(empty, k, k)
    cache.attention(q, i32([3, 7]), i32([[0], [1]]), q, cache.attention_workspace(2, 4, 4), row_start=i32([0, 0, 0]),
                    most_rows=4)
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache.tensors, before))


def test_more_tokens_than_31_bits():
    """A table wide enough for more than 2^31 tokens: a request that would pass 2^31 - 1 is invalid by itself, and the
    requests after it get their blocks."""
    block, width = 1 << 19, 4097
    lengths, new = i32([5, 2 ** 31 - 1, 2 ** 31 - 2, 0]), i32([1, 1, 1, 3])
    table = torch.arange(4 * width, dtype=torch.int32, device="cuda").reshape(4, width) % 4000
    free, count = i32(range(100, 110)), i32([10])
    out, left, start, status = (torch.full((m,), 77, dtype=torch.int32, device="cuda") for m in (4, 1, 5, 4))
    slots, pos, who = (torch.full((8,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
    F.kv_blocks(lengths, new, table, free, count, block, out, left, start, slots, pos, who, status)
    assert status.tolist() == [0, 2, 0, 0] and left.item() == 9
    assert out.tolist() == [6, 2 ** 31 - 1, 2 ** 31 - 1, 3] and start.tolist() == [0, 1, 1, 2, 5]
    assert table[3, 0].item() == 109 and slots[2:5].tolist() == [109 * block + i for i in range(3)]
    assert pos.tolist() == [5, 2 ** 31 - 2, 0, 1, 2, 0, 0, 0] and who.tolist() == [0, 2, 3, 3, 3, -1, -1, -1]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("group,new,hd", [(4, 1, 128), (8, 1, 64), (4, 5, 128), (1, 40, 64)])
@pytest.mark.parametrize("rising", [False, True])
def test_scores_beyond_their_resolution(fmt, group, new, hd, rising):
    """Scores of 2^26 to 2^30, where neighbouring F32 numbers are 8 to 64 apart: which weight a token gets is down to
    rounding, but every row is still a mean of its values (all of them 1 to 2 here)."""
    n, kv, size, length, top = 24, 2, 32, 300, {"int8": 127.0, "e4m3": 448.0}[fmt]
    g = torch.Generator(device="cuda").manual_seed(group + new)
    blocks = n * -(-length // size)
    k = torch.zeros(blocks, kv, size, hd, device="cuda")
    k[..., 0] = 96
    k[..., 1] = torch.randint(0, 8, k.shape[:3], generator=g, device="cuda").float()
    if rising:  # the largest scores of a request in its later tiles
        k[..., 1] = 2 * (torch.arange(blocks, device="cuda") % -(-length // size) // 4)[:, None, None] + k[..., 1] // 4
    v = torch.randint(64, 97, k.shape, generator=g, device="cuda").float()
    kind = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    one = torch.ones(blocks, kv, device="cuda")
    cache = F.KV8Cache(k.to(kind), v.to(kind), one, one / 64)
    table = torch.arange(blocks, dtype=torch.int32, device="cuda").reshape(n, -1)
    q = torch.zeros(n * new, kv * group, hd, device="cuda")
    q[..., 0] = 2.0 ** (26 + 4 * torch.rand(q.shape[:2], generator=g, device="cuda")) / 96
    q[..., 1] = 2.0 ** torch.randint(1, 5, q.shape[:2], generator=g, device="cuda")
    out, ws = torch.empty_like(q), cache.attention_workspace(n, new, kv * group)
    for sign in (1, -1):
        cache.attention(sign * q, i32([length] * n), table, out, ws, row_start=i32(range(0, n * new + 1, new)),
                        most_rows=new, scale=0.6931472)
        assert out.isfinite().all(), int((~out.isfinite()).any(2).sum())
        # a mean to 22 bits a weight, as far as sums of 300 weights in F32 go
        assert (out >= 1 - 300 * 2.0 ** -22).all() and (out <= 1.5 + 300 * 2.0 ** -22).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv,hd,size", [(2, 2, 128, 16), (2, 2, 64, 32), (8, 2, 128, 16), (6, 2, 64, 16)])
@pytest.mark.parametrize("lengths,new", [([60], [60]), ([200, 131, 40], [60, 64, 33]), ([700, 9], [300, 9]), ([90], [8])])
def test_values_that_grow(fmt, heads, kv, hd, size, lengths, new):
    """Value scales that grow from block to block by a factor of a hundred: a token's result is as near as its own
    values allow, whatever the tokens after it bring (the bound is test_gpu_kv8's, by the values a row attends)."""
    def grow(cache, table):
        vs = cache.tensors[3]
        for row in table:
            for i, b in enumerate(row):
                if b >= 0:
                    vs[int(b)] *= 100.0 ** (i % 7)
    run_attention(lengths, new, heads, kv, hd, size, fmt, "f32", seed=sum(new), change=grow)
