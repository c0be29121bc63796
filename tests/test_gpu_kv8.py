"""GPU tests of the paged 8-bit KV cache: block tables, rotary positions,
append and read back, attention, and all of them together, each against a
plain restatement of its definition (whole numbers and stored bytes exactly,
floating sums in 64 bits).

Attention tolerances: a score is a sum of hd products, so its F32 error is at
most (hd + 8) 2^-24 sum|q k| scale =: e (the fp16 halves of q and p keep 22
bits, inside the same bound); a softmax weight then moves by a factor within
exp(+-2e), and the sums over n positions add n 2^-23 at the worst. So |out -
ref| <= max|v| (2 e + (n + 16) 2^-23), plus half a unit of the output type.
"""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

ROW_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
STORED = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}


def i32(v):
    return torch.tensor(np.asarray(v, np.int64).astype(np.int32), device="cuda")


# ---------------------------------------------------------------- block tables
def blocks_ref(lengths, new, table, free, count, block, max_rows):
    table, n, width = table.copy(), len(lengths), table.shape[1]
    start, status, out, rows = [0], [], list(lengths), []
    total, used, full = 0, 0, False
    ends = []
    for r in range(n):
        ok = lengths[r] >= 0 and new[r] >= 0 and lengths[r] + new[r] <= width * block
        total += new[r] if ok else 0
        ends.append(total)
        start.append(min(total, max_rows))
        ok = ok and total <= max_rows
        need = -(-(lengths[r] + new[r]) // block) - -(-lengths[r] // block) if ok else 0
        if not ok:
            status.append(2)
        elif need and (full or used + need > count):
            full = True
            status.append(1)
        else:
            status.append(0)
            first = -(-lengths[r] // block)
            for j in range(need):
                table[r, first + j] = free[count - 1 - used - j]
            used += need
            out[r] += new[r]
        for i in range(new[r] if new[r] > 0 and (ok or status[-1] == 2 and lengths[r] >= 0) else 0):
            if start[r] + i < start[r + 1]:
                p = lengths[r] + i
                rows.append((table[r, p // block] * block + p % block if status[-1] == 0 else -1, p, r))
    rows += [(-1, 0, -1)] * (max_rows - len(rows))
    return table, out, count - used, start, rows, status


def run_blocks(lengths, new, block, width, spare, max_rows, seed=0):
    rng = np.random.default_rng(seed)
    n = len(lengths)
    held = [min(width, max(0, -(-x // block))) for x in lengths]
    ids = rng.permutation(sum(held) + spare + 2).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    free = np.concatenate([ids[at:at + spare], [-7]]).astype(np.int32)  # an entry above the top is not used
    want = blocks_ref(lengths, new, table, free, spare, block, max_rows)
    d = {"lengths": i32(lengths), "new_tokens": i32(new), "table": i32(table), "free_list": i32(free),
         "free_count": i32([spare])}
    for name, m in (("lengths_out", n), ("free_count_out", 1), ("row_start", n + 1), ("slots", max_rows),
                    ("positions", max_rows), ("row_request", max_rows), ("status", n)):
        d[name] = torch.full((m,), 77, dtype=torch.int32, device="cuda")
    for _ in range(2):  # a step can be repeated: inputs stay
        F.kv_blocks(block_size=block, **d)
        g = {k: v.cpu().numpy() for k, v in d.items()}
        assert (g["table"] == want[0]).all()
        assert list(g["lengths_out"]) == want[1] and g["free_count_out"][0] == want[2]
        assert list(g["row_start"]) == want[3] and list(g["status"]) == want[5]
        assert [tuple(x) for x in np.stack([g["slots"], g["positions"], g["row_request"]], 1)] == want[4]
        assert list(g["lengths"]) == list(lengths) and g["free_count"][0] == spare


@pytest.mark.parametrize("block", [1, 16, 64])
@pytest.mark.parametrize("n", [1, 16, 511, 513, 2000])
def test_blocks(n, block):
    rng = np.random.default_rng(n + block)
    lengths = [int(x) for x in rng.integers(0, 200, n)]
    new = [int(x) for x in rng.choice([0, 1, 1, 1, 37, 130], n)]
    width = -(-340 // block)
    need = sum(-(-(a + b) // block) - -(-a // block) for a, b in zip(lengths, new))
    for spare in (need, need + 5, need // 2, 0):
        run_blocks(lengths, new, block, width, spare, sum(new) + 3, seed=spare)


def test_blocks_edges():
    run_blocks([0], [0], 16, 1, 3, 1)
    run_blocks([15, 16, 17, 0], [1, 1, 1, 1], 16, 3, 4, 4)
    run_blocks([5, -1, 7, 40, 9], [2, 3, -4, 30, 1], 16, 4, 8, 12)       # negative counts, over the table
    run_blocks([5, 6, 7, 8], [4, 4, 4, 4], 16, 4, 8, 10)                  # the third crosses max_rows
    run_blocks([0] * 40, [16] * 40, 16, 1, 13, 640)                       # the pool runs out inside
    run_blocks([16, 3, 16, 3], [1, 1, 1, 1], 16, 2, 1, 4)                 # after it, only those that need none
    run_blocks([2 ** 31 - 1, 3], [2 ** 31 - 1, 1], 16, 2, 4, 4)           # sums beyond 31 bits
    run_blocks([3] * 16384, [1] * 16384, 16, 1, 0, 16384)


def test_release_gives_blocks_back():
    n, width, block = 700, 9, 16
    rng = np.random.default_rng(5)
    lengths = rng.integers(0, width * block + 1, n)
    held = -(-lengths // block)
    ids = rng.permutation(int(held.sum()) + 11).astype(np.int32)
    table, at = np.full((n, width), -1, np.int32), 0
    for r in range(n):
        table[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    free = np.full(len(ids), -5, np.int32)
    free[:11] = ids[at:]
    # finished, shortened, shortened to more than they hold, and a negative count
    keep = np.where(rng.random(n) < 0.3, 0, rng.integers(-3, width * block + 20, n))
    left = np.minimum(np.maximum(keep, 0), lengths)
    stay = -(-left // block)
    want = np.concatenate([free[:11]] + [table[r, stay[r]:held[r]] for r in range(n)])
    t, le, fr, fc = i32(table), i32(lengths), i32(free), i32([11])
    F.kv_release(le, i32(keep), t, fr, fc, block)
    assert fc.item() == len(want) and (fr.cpu().numpy()[:len(want)] == want).all()
    assert (le.cpu().numpy() == left).all()
    assert (t.cpu().numpy() == np.where(np.arange(width)[None] < stay[:, None], table, -1)).all()
    F.kv_release(le, i32(keep), t, fr, fc, block)  # nothing left to give
    assert fc.item() == len(want) and (le.cpu().numpy() == left).all()
    # a free list with room for the first blocks only keeps the rest with their requests
    t, le, fr, fc = i32([[1, 2], [3, 4], [5, -1]]), i32([32, 20, 3]), i32([9, 0, 0, 0]), i32([1])
    F.kv_release(le, i32([0, 0, 0]), t, fr, fc, 16)
    assert fc.item() == 3 and fr.tolist() == [9, 1, 2, 0] and le.tolist() == [0, 20, 3]
    assert t.tolist() == [[-1, -1], [3, 4], [5, -1]]


# ---------------------------------------------------------------- rotary positions
def turn(x, cos, sin, layout):
    """x [rows][heads][hd] in 64 bits."""
    y, pairs = x.double().clone(), cos.shape[1]
    i = torch.arange(0, 2 * pairs, 2) if layout == "interleaved" else torch.arange(pairs)
    j = i + (1 if layout == "interleaved" else pairs)
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = x[..., i].double(), x[..., j].double()
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def tables(rows, dims, seed=0):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * torch.tensor(10000.0 ** (-np.arange(dims // 2) / (dims // 2)))
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def rope_bound(x, want, kind):
    # three roundings of values at most |a| + |b|, then one to the row's type
    return x.double().abs().amax() * 2 * 4 * 2.0 ** -24 + want.abs() * HALF_UNIT[kind] + 2.0 ** -25


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("hd,dims", [(128, 128), (128, 64), (64, 16), (80, 20), (6, 2), (96, 96), (256, 128)])
def test_rope(kind, layout, hd, dims):
    rng = torch.Generator().manual_seed(hd + dims)
    rows, heads, kv, ctx = 37, 5, 2, 300
    cos, sin = tables(ctx, dims)
    pos = torch.randint(0, ctx, (rows,), generator=rng, dtype=torch.int32)
    pos[0], pos[1] = 0, ctx - 1
    y = torch.randn((rows, heads + kv, hd), generator=rng).to(ROW_TYPES[kind]).cuda()
    q, k = y[:, :heads], y[:, heads:]  # strided rows
    c, s = cos[pos.long()], sin[pos.long()]
    for inplace in (False, True):
        qi, ki = (q, k) if not inplace else (q.clone(), k.clone())
        qo, ko = (torch.full(t.shape, 7.0, dtype=t.dtype, device="cuda") for t in (q, k))
        if inplace:
            qo, ko = qi, ki
        F.rope(qi, ki, pos.cuda(), cos, sin, layout, qo, ko)
        for x, got in ((q, qo), (k, ko)):
            want = turn(x.cpu(), c.cpu(), s.cpu(), layout)
            assert ((got.cpu().double() - want).abs() <= rope_bound(x.cpu(), want, kind)).all()
            assert (got[..., dims:] == x[..., dims:]).all()


@pytest.mark.parametrize("kind,layout,hd,dims", [("f32", "half", 128, 128), ("bf16", "interleaved", 128, 64),
                                                 ("f16", "half", 64, 32), ("f32", "interleaved", 64, 64)])
@pytest.mark.parametrize("heads,kv", [(32, 8), (7, 0)])
def test_rope_many_rows(kind, layout, hd, dims, heads, kv):
    """Enough rows that they go through shared memory: strided, in place, with
    positions outside the table, and beside a row count that is no multiple of anything."""
    rows, ctx = 9001, 500
    cos, sin = tables(ctx, dims)
    pos = torch.randint(0, ctx, (rows,), dtype=torch.int32)
    pos[[5, rows - 1]] = torch.tensor([-1, ctx], dtype=torch.int32)
    fine = ((pos >= 0) & (pos < ctx))
    y = torch.randn((rows, heads + kv + 1, hd), device="cuda").to(ROW_TYPES[kind])
    q, k = y[:, :heads], y[:, heads:heads + kv] if kv else None
    c, s = (t[pos.clamp(0, ctx - 1).long().cuda()].cpu() for t in (cos, sin))
    for inplace in (False, True):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        base = y.clone()
        qi, ki = base[:, :heads], base[:, heads:heads + kv] if kv else None
        qo, ko = (qi, ki) if inplace else (torch.full_like(q, 7.0), torch.full_like(k, 7.0) if kv else None)
        F.rope(qi, ki, pos.cuda(), cos, sin, layout, qo, ko, error=err)
        assert err.item() == 4
        for x, got in ((q, qo), (k, ko)) if kv else ((q, qo),):
            want = turn(x.cpu(), c, s, layout)
            assert ((got.cpu().double() - want).abs() <= rope_bound(x.cpu(), want, kind))[fine].all()
            assert (got[..., dims:] == x[..., dims:])[fine.cuda()].all()
            left = x if inplace else torch.full_like(x, 7.0)
            assert torch.equal(got[~fine.cuda()], left[~fine.cuda()])
        assert torch.equal(base[:, heads + kv:], y[:, heads + kv:])


def test_rope_unaligned_and_out_of_table():
    """Odd strides and offsets take the scalar path; positions outside the
    table leave their rows as they were and raise the error word."""
    big = torch.randn(4, 3 * 64 + 3, device="cuda")
    q = big[:, 1:129].as_strided((4, 2, 64), (195, 64, 1), 1)
    cos, sin = tables(10, 64)
    pos, err = i32([3, -1, 10, 9]), torch.zeros(1, dtype=torch.int32, device="cuda")
    for layout in ("interleaved", "half"):
        out = torch.full((4, 2, 64), 7.0, device="cuda")
        F.rope(q, None, pos, cos, sin, layout, out, None, error=err)
        want = turn(q.cpu(), cos[pos.clamp(0, 9).long()].cpu(), sin[pos.clamp(0, 9).long()].cpu(), layout)
        assert ((out.cpu().double() - want).abs() <= rope_bound(q.cpu(), want, "f32"))[[0, 3]].all()
        assert (out[1:3] == 7.0).all() and err.item() == 4


def test_rope_turns_back():
    """A rotation by the negative angles undoes it (what a gradient needs)."""
    cos, sin = tables(50, 64)
    x, pos = torch.randn(9, 3, 64, device="cuda"), i32(range(9))
    y, z = torch.empty_like(x), torch.empty_like(x)
    F.rope(x, None, pos, cos, sin, "half", y, None)
    F.rope(y, None, pos, cos, -sin, "half", z, None)
    assert ((z - x).abs() <= 16 * 2.0 ** -24 * x.abs().max()).all()


@pytest.mark.parametrize("kind,kw", [("plain", {}), ("yarn", dict(factor=4.0, original_context=64.0))])
def test_rope_tables(kind, kw):
    freq, mag = F.rope_frequencies(64, 10000.0, kind, **kw)
    c, s = F.rope_tables(torch.tensor(freq).cuda(), mag, 1000, first=130000)
    angle = (np.arange(130000, 131000).astype(np.float32)[:, None] * freq[None]).astype(np.float64)  # F32 angles
    for got, want in ((c, np.cos(angle)), (s, np.sin(angle))):
        assert np.abs(got.cpu().numpy() - want * mag).max() <= 4 * 2.0 ** -24 * mag


# ---------------------------------------------------------------- append and read
def store(y, fmt):
    """round(y) of a format, as the numbers stored (F32 in, F32 out)."""
    y = y.clamp(-TOP[fmt], TOP[fmt])
    return y.round() if fmt == "int8" else y.to(torch.float8_e4m3fn).float()


class RefCache:
    """The cache in plain F32: numbers [blocks][heads][size][hd] and scales."""

    def __init__(self, blocks, heads, size, hd, fmt):
        self.fmt, self.size = fmt, size
        self.x = {n: torch.zeros(blocks, heads, size, hd) for n in "kv"}
        self.s = {n: torch.zeros(blocks, heads) for n in "kv"}

    def append(self, name, rows, slots):
        x, s, inv = self.x[name], self.s[name], torch.tensor(1.0) / TOP[self.fmt]
        for b in dict.fromkeys(int(t) // self.size for t in slots if t >= 0):
            at = [i for i, t in enumerate(slots) if t >= 0 and t // self.size == b]
            new = rows[at].float().transpose(0, 1)
            first = min(int(slots[i]) % self.size for i in at)
            fine = torch.where(new.isfinite(), new.abs(), 0.0)
            was = s[b] if first else torch.zeros_like(s[b])
            now = torch.maximum(was, fine.amax((1, 2)) * inv)
            grown = (now > was)[:, None, None]
            x[b, :, :first] = torch.where(grown, store(x[b, :, :first] * (was / now)[:, None, None], self.fmt), x[b, :, :first])
            y = torch.where(now[:, None, None] > 0, new / now[:, None, None], 0.0)
            y = torch.where(new.isfinite(), y, torch.where(new.isnan(), 0.0, new.sign() * TOP[self.fmt]))
            for i, a in enumerate(at):
                x[b, :, int(slots[a]) % self.size] = store(y[:, i], self.fmt)
            s[b] = now

    def values(self, name, slots):
        b, t = torch.tensor(slots) // self.size, torch.tensor(slots) % self.size
        return self.x[name][b, :, t] * self.s[name][b][:, :, None]


def same_cache(cache, ref):
    k, v, ks, vs = cache.tensors
    for name, q, s in (("k", k, ks), ("v", v, vs)):
        assert torch.equal(s.cpu(), ref.s[name])
        got = q.cpu().float() if q.dtype == torch.int8 else q.view(torch.float8_e4m3fn).cpu().float()
        assert torch.equal(got, ref.x[name] + 0.0), name


@pytest.mark.parametrize("fmt", sorted(STORED))
@pytest.mark.parametrize("kind,hd,size", [("f32", 128, 16), ("bf16", 128, 64), ("f16", 64, 32), ("f32", 64, 256)])
def test_append_steps(fmt, kind, hd, size):
    """Prompts, single tokens and drafts of three requests, step after step, to the byte."""
    g = torch.Generator().manual_seed(size)
    heads, blocks = 3, 12
    cache, ref = F.KV8Cache.empty(blocks, heads, size, hd, fmt), RefCache(blocks, heads, size, hd, fmt)
    order = torch.randperm(blocks, generator=g).tolist()
    own, length = [order[0:4], order[4:8], order[8:12]], [0, 0, 0]
    held = []
    for step, new in enumerate([[size + 3, 0, 1], [1, 5, 1], [1, size * 2, 0], [7, 1, 2], [1, 1, 1]]):
        slots = []
        for r, m in enumerate(new):
            slots += [own[r][p // size] * size + p % size for p in range(length[r], length[r] + m)]
            length[r] += m
        k, v = (torch.randn(len(slots), heads, hd, generator=g) * (1 + step) for _ in "kv")
        k[:, 0] = 0 if step < 2 else k[:, 0]  # a head that is zero at first: scale 0
        k, v = k.to(ROW_TYPES[kind]), v.to(ROW_TYPES[kind])
        cache.append(k.cuda(), v.cuda(), i32(slots))
        ref.append("k", k, slots)
        ref.append("v", v, slots)
        same_cache(cache, ref)
        held += slots
    ko, vo = (torch.empty(len(held), heads, hd, device="cuda") for _ in "kv")
    cache.read(i32(held), ko, vo)
    assert torch.equal(ko.cpu(), ref.values("k", held)) and torch.equal(vo.cpu(), ref.values("v", held))


@pytest.mark.parametrize("fmt", sorted(STORED))
@pytest.mark.parametrize("kind,hd,size,layout", [("bf16", 128, 64, "interleaved"), ("f32", 64, 256, "half"),
                                                 ("f16", 128, 16, None)])
def test_append_prompts(fmt, kind, hd, size, layout):
    """Prompts of several requests, long enough that CTAs take runs of rows: to the byte, q as by fyb_rope."""
    g = torch.Generator().manual_seed(size)
    kv, heads, ctx = 4, 6, 1500
    news, starts, used, slots, pos = [700, 1, 1311, 260], [0, 5, 77, 256], 0, [], []
    order = torch.randperm(400, generator=g).tolist()
    for n, p0 in zip(news, starts):
        own = order[used:used + -(-(p0 + n) // size)]
        used += len(own)
        slots += [own[p // size] * size + p % size for p in range(p0, p0 + n)]
        pos += range(p0, p0 + n)
    cache, ref = F.KV8Cache.empty(400, kv, size, hd, fmt), RefCache(400, kv, size, hd, fmt)
    k, v = (torch.randn(len(slots), kv, hd, generator=g).to(ROW_TYPES[kind]) for _ in "kv")
    q = torch.randn(len(slots), heads, hd, generator=g).to(ROW_TYPES[kind]).cuda()
    kw, rotated = {}, k
    if layout:
        cos, sin = tables(ctx, hd)
        qa, qb, kb = torch.empty_like(q), torch.empty_like(q), torch.empty(len(slots), kv, hd, device="cuda")
        F.rope(q, None, i32(pos), cos, sin, layout, qb, None)
        F.rope(k.cuda().float(), None, i32(pos), cos, sin, layout, kb, None)
        rotated, kw = kb.cpu(), dict(positions=i32(pos), cos=cos, sin=sin, layout=layout, q=q, q_out=qa)
    cache.append(k.cuda(), v.cuda(), i32(slots), **kw)
    ref.append("k", rotated, slots)
    ref.append("v", v, slots)
    same_cache(cache, ref)
    assert not layout or torch.equal(qa, qb)


def test_append_refuses_rows_and_values():
    """Negative slots are skipped, slots and positions out of range are left
    out with the error word raised; infinities saturate, NaN is 0."""
    fmt, hd = "int8", 64
    cache, ref = F.KV8Cache.empty(3, 2, 16, hd, fmt), RefCache(3, 2, 16, hd, fmt)
    k, v = torch.randn(5, 2, hd), torch.randn(5, 2, hd)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(k.cuda(), v.cuda(), i32([-1, 16, 17, -1, 0]), error=err)
    for n, x in (("k", k), ("v", v)):
        ref.append(n, x, [-1, 16, 17, -1, 0])
    same_cache(cache, ref)
    assert err.item() == 0
    cache.append(k[:2].cuda(), v[:2].cuda(), i32([48, 2 ** 31 - 1]), error=err)
    same_cache(cache, ref)
    assert err.item() == 4
    k[0, 0, 3], k[0, 1, 5], v[0, 0, 0], v[0, 1] = float("inf"), float("nan"), -float("inf"), float("nan")
    err.zero_()
    cache.append(k[:1].cuda(), v[:1].cuda(), i32([32]), error=err)
    for n, x in (("k", k), ("v", v)):
        ref.append(n, x[:1], [32])
    same_cache(cache, ref)
    assert err.item() == 2
    cos, sin = tables(4, hd)
    err.zero_()
    cache.append(k[1:3].cuda(), v[1:3].cuda(), i32([33, 40]), i32([4, -1]), cos, sin, error=err)
    assert err.item() == 4  # K is left out where its position is; V has no position
    ko, vo = (torch.full((2, 2, hd), 7.0, device="cuda") for _ in "kv")
    err.zero_()
    cache.read(i32([-1, 48]), ko, vo, error=err)
    assert (ko == 0).all() and (vo == 0).all() and err.item() == 4


@pytest.mark.parametrize("layout,dims", [("interleaved", 128), ("half", 128), ("half", 64), ("interleaved", 6)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_append_rotates(layout, dims, kind):
    """K rotated in the append is K rotated by fyb_rope and appended, q likewise, to the bit; on rows that are
    slices of a fused buffer, aligned or not."""
    hd, heads, kv, rows = 128, 6, 2, 33
    cos, sin = tables(64, dims)
    pos, slots = i32(range(5, 5 + rows)), i32(range(16, 16 + rows))
    for pad in (0, 1):
        y = torch.randn(rows, (heads + 2 * kv) * hd + pad, device="cuda").to(ROW_TYPES[kind])
        part = lambda a, n: y.as_strided((rows, n, hd), (y.shape[1], hd, 1), a * hd + pad)  # noqa: E731
        y2 = torch.empty(rows, heads + 2 * kv, hd, device="cuda", dtype=y.dtype)
        q, k, v = part(0, heads), part(heads, kv), part(heads + kv, kv) if not pad else part(heads + kv, kv).clone()
        one, two = (F.KV8Cache.empty(4, kv, 16, hd) for _ in range(2))
        qa, qb, kb = torch.empty_like(y2[:, :heads]), torch.empty_like(y2[:, :heads]), torch.empty_like(y2[:, :kv])
        one.append(k, v, slots, pos, cos, sin, layout, q, qa)
        F.rope(q, k, pos, cos, sin, layout, qb, kb)
        assert torch.equal(qa, qb)
        if kind == "f32":  # the rotated K is not rounded to the rows' type on its way to the cache
            two.append(kb, v, slots)
            for a, b in zip(one.tensors, two.tensors):
                assert torch.equal(a, b)
        ko, vo = (torch.empty(rows, kv, hd, device="cuda") for _ in "kv")
        one.read(slots, ko, vo)
        want = turn(k.cpu(), cos[pos.long()].cpu(), sin[pos.long()].cpu(), layout)
        assert ((ko.cpu().double() - want).abs() <= want.abs().amax() * (0.51 / 127)).all()


# ---------------------------------------------------------------- attention
def make(lengths, heads, kv, hd, size, fmt, seed, width=None, extra=2):
    """A cache with requests' blocks in random order, garbage everywhere that is not a token of theirs."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-n // size) for n in lengths]
    blocks = sum(counts) + extra
    x = {n: torch.randn((blocks, kv, size, hd), generator=g, device="cuda") for n in "kv"}
    bad = {}
    for n in "kv":
        s = x[n].abs().amax((2, 3)) / TOP[fmt]
        y = x[n] / s[:, :, None, None]
        bad[n] = [(y.round() if fmt == "int8" else y).to(STORED[fmt]), s]
    order = torch.randperm(blocks, generator=g, device="cuda").tolist()
    table = np.full((len(lengths), width or max(1, max(counts))), -1, np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
        if lengths[r] % size:  # what lies past the length: NaN of the format, or its lowest value
            junk = 0x7f if fmt == "e4m3" else -128
            for n in "kv":
                bad[n][0].view(torch.int8)[order[at - 1], :, lengths[r] % size:] = junk
    for b in order[at:]:
        bad["k"][1][b], bad["v"][1][b] = float("nan"), float("inf")
    return F.KV8Cache(bad["k"][0], bad["v"][0], bad["k"][1].contiguous(), bad["v"][1].contiguous()), table


def reference(cache, table, lengths, starts, q, scale):
    """(out, bound) in 64 bits; rows [rows][heads][hd] on the CPU."""
    k, v, ks, vs = (t.cpu() for t in cache.tensors)
    kv, size, hd = k.shape[1:]
    q = q.cpu().double()
    rows, heads, _ = q.shape
    out, tol = torch.zeros(rows, heads, hd, dtype=torch.float64), torch.zeros(rows, heads, 1, dtype=torch.float64)
    num = lambda t: t.double() if t.dtype == torch.int8 else t.float().double()  # noqa: E731
    for r, n in enumerate(lengths):
        use = table[r, :-(-n // size)].tolist()
        if not use:
            continue
        kk, vv = (torch.cat([num(t[b]) * s[b].double()[:, None, None] for b in use], 1)[:, :n] for t, s in ((k, ks), (v, vs)))
        m = starts[r + 1] - starts[r]
        for j in range(m):
            end = n - m + j + 1
            if end <= 0:
                continue
            row = q[starts[r] + j].reshape(kv, heads // kv, hd)
            sc = torch.einsum("ghd,gtd->ght", row, kk[:, :end]) * scale
            mag = torch.einsum("ghd,gtd->ght", row.abs(), kk[:, :end].abs()).amax(2) * abs(scale)
            p = torch.softmax(sc, 2)
            out[starts[r] + j] = torch.einsum("ght,gtd->ghd", p, vv[:, :end]).reshape(heads, hd)
            top = vv[:, :end].abs().amax((1, 2))[:, None]
            e = (hd + 8) * 2.0 ** -24 * mag
            tol[starts[r] + j] = (top * (2 * e + (end + 16) * 2.0 ** -23)).reshape(heads, 1)
    return out, tol


def run_attention(lengths, new, heads, kv, hd, size, fmt, kind, seed=0, scale=None, q=None, ws=None, change=None, stride=0):
    cache, table = make(lengths, heads, kv, hd, size, fmt, seed, width=-(-max(max(lengths), 1) // size) + seed % 3)
    if change:
        change(cache, table)
    starts = [0] + list(np.cumsum(new))
    rows = starts[-1]
    scale = hd ** -0.5 if scale is None else scale
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    if q is None:
        q = torch.randn((rows, heads, hd), generator=g, device="cuda")
    q = q.to(ROW_TYPES[kind])
    if stride:
        q = torch.cat([q.reshape(rows, -1), q.new_full((rows, stride), 7.0)], 1)[:, :heads * hd].unflatten(1, (heads, hd))
    out = torch.full((rows, heads, hd), 7.0, dtype=q.dtype, device="cuda")
    ws = cache.attention_workspace(len(lengths), max(new), heads) if ws is None else ws
    args = dict(row_start=None if all(m == 1 for m in new) else i32(starts), most_rows=max(new), scale=scale)
    cache.attention(q, i32(lengths), i32(table), out, ws, **args)
    again = torch.full_like(out, 3.0)
    cache.attention(q, i32(lengths), i32(table), again, ws, **args)  # the workspace is left as it has to be
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))
    want, tol = reference(cache, table, lengths, starts, q, scale)
    got = out.cpu().double()
    assert got.isfinite().all()
    far = (got - want).abs() - tol - want.abs() * HALF_UNIT[kind] - 2.0 ** -25
    assert (far <= 0).all(), float(far.max())
    # and in the mean far nearer than the worst case: single roundings, not a lost half of q or p
    if want.norm() > 0 and kind == "f32":
        assert (got - want).norm() <= 2e-5 * want.norm()
    return out


EDGES = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000]


@pytest.mark.parametrize("fmt", sorted(STORED))
@pytest.mark.parametrize("size", [16, 32, 64, 128, 256])
def test_decode_lengths(fmt, size):
    run_attention(EDGES, [1] * len(EDGES), 8, 2, 128, size, fmt, "f32", seed=size)
    run_attention(EDGES, [1] * len(EDGES), 8, 2, 64, size, fmt, "f32", seed=size + 1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 31, 64])
def test_decode_groups(group, hd):
    for fmt in STORED:
        run_attention([77, 300, 1], [1, 1, 1], group * 2, 2, hd, 32, fmt, "f32", seed=group)


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("fmt", sorted(STORED))
def test_decode_types(kind, fmt):
    run_attention([500, 3, 64, 129], [1] * 4, 16, 4, 128, 16, fmt, kind, seed=3)
    run_attention([500, 3, 64, 129], [1] * 4, 16, 4, 64, 64, fmt, kind, seed=4, stride=8)
    run_attention([500, 3, 64, 129], [1] * 4, 16, 4, 64, 64, fmt, kind, seed=4, stride=1)


@pytest.mark.parametrize("fmt", sorted(STORED))
@pytest.mark.parametrize("new", [[2, 2, 2], [8, 5, 1], [16, 16, 3], [17, 40, 2], [130, 65, 64]])
@pytest.mark.parametrize("heads,kv,hd,size", [(8, 2, 128, 64), (16, 2, 64, 16), (3, 3, 128, 32), (12, 2, 128, 128)])
def test_rows(new, heads, kv, hd, size, fmt):
    """Drafts and chunks: causal inside, at the start of a context and behind a long one."""
    run_attention([m + d for m, d in zip(new, (0, 77, 400))], new, heads, kv, hd, size, fmt, "f32", seed=sum(new))
    run_attention([m + d for m, d in zip(new, (63, 0, 1))], new, heads, kv, hd, size, fmt, "bf16", seed=sum(new))


def test_empty_rows_and_requests():
    """Requests with no tokens or no rows, and rows that attend nothing, among others."""
    for new in ([1, 1, 1, 1], [3, 0, 2, 5], [20, 0, 33, 2]):
        for fmt in STORED:
            out = run_attention([0, 0, 70, 4], new, 8, 2, 128, 16, fmt, "f32", seed=9)
            assert (out[:new[0]] == 0).all()
    # more rows than tokens: the first rows attend nothing
    out = run_attention([2, 90], [6, 30], 8, 2, 64, 32, "int8", "f32", seed=2)
    assert (out[:4] == 0).all() and (out[4:6] != 0).any()


def test_wide_scales_and_scores():
    """Block scales many orders apart (0 among them), scores in the hundreds, queries of very different size."""
    def spread(cache, table):
        k, v, ks, vs = cache.tensors
        for i, b in enumerate(table[0]):
            if b >= 0:
                vs[b] *= 10.0 ** (i % 7 - 3)
                ks[b] *= [1.0, 30.0, 1e-3][i % 3]
                if i == 4:
                    vs[b], ks[b] = 0.0, 0.0
    for new in ([1], [9], [40]):
        for fmt in STORED:
            run_attention([333], new, 8, 2, 128, 16, fmt, "f32", seed=1, change=spread)
    q = torch.randn(2, 8, 128, device="cuda") * torch.tensor([1e-6, 1e-3, 0.1, 1, 10, 1e3, 1e-20, 0.0], device="cuda")[None, :, None]
    run_attention([100, 200], [1, 1], 8, 2, 128, 32, "int8", "f32", q=q, scale=0.01)
    run_attention([100, 200], [1, 1], 8, 2, 128, 32, "int8", "f32", q=q.clamp(-1, 1), scale=-3.0)


def test_long_tail_of_small_weights():
    """One token takes nearly all weight, 20000 others share the rest: their sum has to survive."""
    n, hd = 20000, 64
    cache, table = make([n], 1, 1, hd, 64, "int8", 11)
    k, v, ks, vs = cache.tensors
    k.zero_()
    k[table[0, 100], 0, 7] = 127
    ks.fill_(1.0 / 127)
    v.fill_(127)
    v[table[0, 100], 0, 7] = 0
    vs.fill_(1.0 / 127)
    q = torch.full((1, 1, hd), 1.0, device="cuda")
    out = torch.empty_like(q)
    scale = 16.0 / hd  # the strong score is 16, all others 0
    cache.attention(q, i32([n]), i32(table), out, cache.attention_workspace(1, 1, 1), scale=scale)
    want = (n - 1) / (n - 1 + np.exp(16.0))
    assert np.abs(out.cpu().numpy() / want - 1).max() <= n * 2.0 ** -23


def test_bad_tables_and_lengths():
    """Blocks outside the pool and lengths beyond the table are left out and raise the error word; other requests
    are as ever."""
    lengths, new = [100, 90, 64], [1, 1, 1]
    cache, table = make(lengths, 8, 2, 128, 16, "int8", 4)
    q = torch.randn(3, 8, 128, device="cuda")
    good, bad = torch.empty_like(q), torch.empty_like(q)
    ws, err = cache.attention_workspace(3, 1, 8), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.attention(q, i32(lengths), i32(table), good, ws, error=err)
    assert err.item() == 0
    for value in (-1, 10 ** 6, 2 ** 31 - 1):
        t = table.copy()
        t[1, 2] = value
        err.zero_()
        cache.attention(q, i32(lengths), i32(t), bad, ws, error=err)
        assert err.item() == 4 and torch.equal(bad[[0, 2]], good[[0, 2]]) and bad.isfinite().all()
    err.zero_()
    cache.attention(q, i32([100, table.shape[1] * 16 + 1, 64]), i32(table), bad, ws, error=err)
    assert err.item() == 4 and torch.equal(bad[[0, 2]], good[[0, 2]])
    # more rows than the caller said: those past most_rows are left out
    err.zero_()
    bad.fill_(7.0)
    cache.attention(q, i32([100]), i32(table[:1]), bad, ws, row_start=i32([0, 3]), most_rows=2, error=err)
    assert err.item() == 4 and (bad[2] == 7.0).all() and (bad[:2] != 7.0).any()


def test_nan_query_stays_in_its_row():
    for new in ([1, 1], [9, 30]):
        lengths = [100, 80]
        cache, table = make(lengths, 8, 2, 128, 16, "int8", 4)
        starts = [0] + list(np.cumsum(new))
        q = torch.randn(starts[-1], 8, 128, device="cuda")
        args = dict(row_start=i32(starts), most_rows=max(new))
        a, b, ws = torch.empty_like(q), torch.empty_like(q), cache.attention_workspace(2, max(new), 8)
        cache.attention(q, i32(lengths), i32(table), a, ws, **args)
        q[1, 3, 5] = float("nan")
        cache.attention(q, i32(lengths), i32(table), b, ws, **args)
        assert b[1, 3].isnan().all()
        b[1, 3] = a[1, 3]
        assert torch.equal(a, b)


def test_other_stream_and_graph():
    """The calls run on torch's current stream and can be captured: the graph then serves other lengths."""
    lengths = [100, 33]
    cache, table = make([200, 200], 8, 2, 128, 16, "int8", 4)
    q, le, t = torch.randn(2, 8, 128, device="cuda"), i32(lengths), i32(table)
    want, out, ws = torch.empty_like(q), torch.empty_like(q), cache.attention_workspace(2, 1, 8)
    cache.attention(q, le, t, want, ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big  # the stream is busy; q changes behind it
        q2 = torch.zeros_like(q).copy_(q)
        cache.attention(q2, le, t, out, ws)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attention(q, le, t, out, ws)
    for n in ([200, 1], [100, 33]):
        le.copy_(i32(n))
        graph.replay()
    assert torch.equal(out, want)


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB: the same blocks at its two ends give the same output."""
    kv, size, hd = 2, 256, 128
    blocks = (1 << 32) // (kv * size * hd) + 40
    cache = F.KV8Cache.empty(blocks, kv, size, hd)
    low, high = [1, 2, 3], [blocks - 1, blocks - 20, blocks - 3]
    for t in cache.tensors[:2]:
        t[low] = torch.randint(-127, 128, (3, kv, size, hd), device="cuda").to(torch.int8)
        t[high] = t[low]
    for t in cache.tensors[2:]:
        t[low] = torch.rand(3, kv, device="cuda") * 0.01
        t[high] = t[low]
    k, v = torch.randn(2, kv, hd, device="cuda"), torch.randn(2, kv, hd, device="cuda")
    cache.append(torch.cat([k[:1]] * 2), torch.cat([v[:1]] * 2), i32([low[2] * size + 80, high[2] * size + 80]))
    for new in (1, 12):
        q = torch.randn(new, 8, hd, device="cuda")
        q2, out = torch.cat([q, q]), torch.empty(2 * new, 8, hd, device="cuda")
        cache.attention(q2, i32([2 * size + 81] * 2), i32([low, high]), out, cache.attention_workspace(2, new, 8),
                        row_start=i32([0, new, 2 * new]), most_rows=new)
        assert torch.equal(out[:new], out[new:]) and (out != 0).any()
    ko, vo = (torch.empty(2, kv, hd, device="cuda") for _ in "kv")
    cache.read(i32([low[1] * size + 255, high[1] * size + 255]), ko, vo)
    assert torch.equal(ko[0], ko[1]) and (ko != 0).any()


def test_steps_together():
    """Blocks, append with rotation, attention: a prompt and then single tokens of three requests, against
    attention in 64 bits over the values the cache reads back."""
    heads, kv, hd, size, n = 8, 2, 128, 16, 3
    cache = F.KV8Cache.empty(40, kv, size, hd)
    cos, sin = tables(256, hd)
    lengths, table = i32([0] * n), torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    free, count = i32(range(40)), i32([40])
    ws = cache.attention_workspace(n, 37, heads)
    for step, new in enumerate([[37, 5, 16], [1, 1, 1], [1, 0, 1], [8, 3, 1], [1, 1, 1]]):
        rows = sum(new)
        e = lambda m: torch.empty(m, dtype=torch.int32, device="cuda")  # noqa: E731
        out_len, out_count, start, slots, pos, who, status = e(n), e(1), e(n + 1), e(rows), e(rows), e(rows), e(n)
        F.kv_blocks(lengths, i32(new), table, free, count, size, out_len, out_count, start, slots, pos, who, status)
        lengths, count = out_len, out_count
        assert status.tolist() == [0] * n and start.tolist() == [0] + list(np.cumsum(new))
        y = torch.randn(rows, heads + 2 * kv, hd, device="cuda")
        q, out = torch.empty(rows, heads, hd, device="cuda"), torch.empty(rows, heads, hd, device="cuda")
        cache.append(y[:, heads:heads + kv], y[:, heads + kv:], slots, pos, cos, sin, "interleaved", y[:, :heads], q)
        cache.attention(q, lengths, table, out, ws, row_start=start, most_rows=max(new))
        want, tol = reference(cache, table.cpu().numpy(), lengths.tolist(), start.tolist(), q, hd ** -0.5)
        assert ((out.cpu().double() - want).abs() <= tol + want.abs() * 2.0 ** -24 + 2.0 ** -25).all(), step
    F.kv_release(lengths, i32([0, 999, -1]), table, free, count, size)
    assert lengths.tolist()[0] == 0 and count.item() == 40 - -(-lengths.tolist()[1] // size)


# ---------------------------------------------------------------- a plan's batched decode over the cache
CFG = dict(layers=2, embedding=512, heads=8, kv_heads=2, feed_forward=1024, vocabulary=1024, context=64,
           matrix_type=F.Q4_K, seed=21, norm_mode=2)


class RefModel:
    """The engine's dense LLaMA step (llm_cpu.c:424-578) in 64 bits, its cache in the 8 bits of RefCache."""

    def __init__(self, model, fmt, size):
        import oracle as O
        self.w, self.m = {}, model
        for i in range(3 + 9 * model.layers):
            t = model.tensor(i)
            shape = [int(t.dimensions[d]) for d in range(t.dimension_count)][::-1]
            x = O.dequantize(model.tensor_bytes(i), t.type, int(np.prod(shape)))
            self.w[t.name.decode()] = x.reshape(shape).astype(np.float64)
        self.fmt, self.size = fmt, size
        self.freq = F.rope_frequencies(model.head_dim, 500000.0)[0]

    def session(self, capacity):
        return [RefCache(-(-capacity // self.size), self.m.kv_heads, self.size, self.m.head_dim, self.fmt)
                for _ in range(self.m.layers)]

    def norm(self, x, name):
        return x / np.sqrt(np.mean(x * x) + 1e-5) * self.w[name]

    def turn(self, x, pos):
        angle = (np.float32(pos) * self.freq).astype(np.float64)
        c, s = np.cos(angle), np.sin(angle)
        y = np.empty_like(x)
        y[:, 0::2], y[:, 1::2] = x[:, 0::2] * c - x[:, 1::2] * s, x[:, 0::2] * s + x[:, 1::2] * c
        return y

    def step(self, session, token, pos):
        m, w = self.m, self.w
        x = w["token_embd.weight"][token].copy()
        for l in range(m.layers):
            n = "blk.%d." % l
            h = self.norm(x, n + "attn_norm.weight")
            q, k, v = (w[n + "attn_%s.weight" % c] @ h for c in "qkv")
            q = self.turn(q.reshape(m.heads, m.head_dim), pos)
            k = self.turn(k.reshape(m.kv_heads, m.head_dim), pos)
            cache = session[l]
            for name, row in (("k", k), ("v", v.reshape(m.kv_heads, m.head_dim))):
                cache.append(name, torch.tensor(row, dtype=torch.float32)[None], [pos])
            kk, vv = (cache.values(c, list(range(pos + 1))).double().numpy() for c in "kv")
            out = np.empty_like(q)
            for g in range(m.heads):
                s = kk[:, g // (m.heads // m.kv_heads)] @ q[g] / np.sqrt(m.head_dim)
                p = np.exp(s - s.max())
                out[g] = p @ vv[:, g // (m.heads // m.kv_heads)] / p.sum()
            x = x + w[n + "attn_output.weight"] @ out.reshape(-1)
            h = self.norm(x, n + "ffn_norm.weight")
            gate, up = w[n + "ffn_gate.weight"] @ h, w[n + "ffn_up.weight"] @ h
            x = x + w[n + "ffn_down.weight"] @ (gate / (1 + np.exp(-gate)) * up)
        return w["output.weight"] @ self.norm(x, "output_norm.weight")


@pytest.mark.parametrize("kv", sorted(STORED))
@pytest.mark.parametrize("nseq", [1, 5, 12])
def test_batch_over_the_cache(provider, nseq, kv):
    """Batched decode with the paged 8-bit cache against the same step in 64
    bits over the same 8-bit cache: logits within 1e-3 of the logit scale, the
    bound of every plan test. Sequences go on at ragged positions, some going
    back over rows they have written."""
    m = F.SynthModel(**CFG)
    plan = provider.plan(m, CFG["context"])
    batch = F.Batch(plan, nseq, kv=kv, blocks=4 * nseq, block_size=16)
    ref = RefModel(m, kv, 16)
    refs = [ref.session(CFG["context"]) for _ in range(nseq)]
    rng = np.random.default_rng(nseq)
    pos = np.zeros(nseq, np.uint32)
    worst = 0.0
    for s in range(24):
        toks = rng.integers(0, m.vocabulary, nseq).astype(np.uint32)
        lg, am = batch.step(toks, pos)
        assert (am == lg.argmax(1)).all()
        for b in range(nseq):
            e = ref.step(refs[b], int(toks[b]), int(pos[b]))
            worst = max(worst, float(np.max(np.abs(lg[b] - e)) / (1 + np.max(np.abs(e)))))
        held = int(sum(-(-(int(p) + 1) // 16) for p in pos))
        assert batch.free_blocks() == 4 * nseq - held
        pos = np.where(rng.random(nseq) < 0.1, pos * 2 // 3, pos + 1).astype(np.uint32)
    assert worst <= 1e-3
    batch.close()
    plan.close()
    m.close()


def test_batch_greedy_and_refusals(provider):
    """Greedy steps on the device are the same steps one by one; a gap, a
    position past the plan's capacity and a step that needs more blocks than the
    pool has are refused, and the batch goes on after them."""
    m = F.SynthModel(**CFG)
    plan = provider.plan(m, CFG["context"])
    nseq = 3
    batch, other = (F.Batch(plan, nseq, kv="int8", blocks=4 * nseq, block_size=16) for _ in range(2))
    rng = np.random.default_rng(3)
    for s in range(20):  # the same history in both: a block keeps the scale of rows that were taken back
        toks = rng.integers(0, m.vocabulary, nseq).astype(np.uint32)
        for x in (batch, other):
            x.step(toks, np.full(nseq, s, np.uint32))
    start, first = np.full(nseq, 17, np.uint32), rng.integers(0, m.vocabulary, nseq).astype(np.uint32)
    got = other.decode_greedy(first, start, 8)
    assert other.free_blocks() == 2 * nseq
    cur = first
    for i in range(8):
        _, cur = batch.step(cur, start + np.uint32(i))
        assert (cur == got[i]).all(), i
    with pytest.raises(RuntimeError):
        batch.step(cur, np.full(nseq, 26, np.uint32))
    with pytest.raises(RuntimeError):
        batch.decode_greedy(cur, np.full(nseq, 25, np.uint32), 40)
    batch.step(cur, np.full(nseq, 25, np.uint32))
    tight = F.Batch(plan, nseq, kv="e4m3", blocks=nseq, block_size=16)
    assert tight.decode_greedy(cur, np.zeros(nseq, np.uint32), 16).shape == (16, nseq)
    with pytest.raises(RuntimeError):
        tight.step(cur, np.full(nseq, 16, np.uint32))
    assert tight.free_blocks() == 0
    tight.step(cur, np.full(nseq, 15, np.uint32))
    assert tight.time_greedy(cur, np.full(nseq, 3, np.uint32), 4) > 0
    assert not F.lib.fyb_batch_create_kv8(C.c_void_p(plan.ptr), 4, 16, 24, 0)
    assert not F.lib.fyb_batch_create_kv8(C.c_void_p(plan.ptr), 17, 16, 16, 0)
    assert not F.lib.fyb_batch_create_kv8(C.c_void_p(plan.ptr), 4, 0, 16, 0)
    for x in (tight, other, batch):
        x.close()
    plan.close()
    m.close()
