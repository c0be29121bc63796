"""GPU tests of the paged 4-bit KV cache: append and read back, attention, and
both together, each against a plain restatement of its definition (stored bits
exactly, floating sums in 64 bits).

Attention tolerances. A score is a sum over a group's values of q n, times scale,
plus low times the sum of q: hd products and sums of magnitudes at most |q| (15
scale + |low|), so its F32 error is at most (hd + 16) 2^-24 sum |q| (15 scale +
|low|) =: e; a softmax weight then moves by a factor within exp(+-2e), and the
sums over n positions add n 2^-23 at the worst: |out - ref| <= vtop (2 e + (n +
16) 2^-23), vtop the largest 15 scale + |low| of V, plus half a unit of the
output type. With rows of 16 bits K, V and the weights may be rounded to fp16
once, half a step (2^-11) each: e grows by 2^-11 of the same sum (and 2^-25 |q|
where K is below fp16's normal numbers), the output by vtop 2^-11 for V and twice
that for the weights and their sum, and 2^-25.
"""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

ROW_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
MOST = 61440.0


def i32(v):
    return torch.tensor(np.asarray(v, np.int64).astype(np.int32), device="cuda")


def rope_tables(rows, dims):
    angle = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(dims // 2) / (dims // 2))
    return (torch.tensor(f(angle), dtype=torch.float32, device="cuda") for f in (np.cos, np.sin))


# ---------------------------------------------------------------- the format
def hold(x):
    """Rows [..., hd] (F32) as they are held: numbers, scale and low, in 64 bits on the CPU."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], -1, 64)
    fine = np.isfinite(g)
    none = ~fine.any(-1)
    low = np.where(none, 0.0, np.clip(np.where(fine, g, np.inf).min(-1), -MOST, MOST)).astype(np.float16)
    high = np.where(none, 0.0, np.clip(np.where(fine, g, -np.inf).max(-1), -MOST, MOST)).astype(np.float16)
    scale = ((high.astype(np.float64) - low.astype(np.float64)) / 15).astype(np.float16)
    lo, unit = (t.astype(np.float64)[..., None] for t in (low, scale))
    y = np.where(np.isnan(g), 0.0, g)
    n = np.zeros(y.shape)
    for k in range(15):  # borders between k and k + 1; a tie goes to the even one
        border = lo + (k + 0.5) * unit
        n += (y > border) | ((y == border) & (k % 2 == 1))
    return np.where(unit > 0, n, 0.0).astype(np.uint32), scale, low


def packed(n):
    """Numbers [..., groups, 64] as bytes [..., hd / 2]: words of eight, the groups' words in turn."""
    w = n.reshape(*n.shape[:-1], 8, 8)
    w = (w << (4 * np.arange(8, dtype=np.uint32))).sum(-1).astype(np.uint32)
    return np.ascontiguousarray(np.swapaxes(w, -1, -2)).reshape(*w.shape[:-2], -1).view(np.uint8)


def numbers(cache, name):
    """(numbers [blocks][kv][size][groups][64], scale, low) of a cache's K or V, in 64 bits on the CPU."""
    b, s = cache.tensors["kv".index(name)].cpu().numpy(), cache.tensors[2 + "kv".index(name)].cpu().numpy()
    w = b.view(np.uint32)
    groups = s.shape[-2]
    n = (w[..., None] >> (4 * np.arange(8, dtype=np.uint32))) & 15
    n = np.swapaxes(n.reshape(*w.shape[:-1], 8, groups, 8), -3, -2).reshape(*w.shape[:-1], groups, 64)
    return n.astype(np.float64), s[..., 0].astype(np.float64), s[..., 1].astype(np.float64)


def values(cache, name):
    n, s, low = numbers(cache, name)
    x = low[..., None] + s[..., None] * n
    return x.reshape(*x.shape[:-2], -1)


def slot_values(cache, name, slots):
    x = values(cache, name)
    slots = np.asarray(slots)
    size = x.shape[2]
    return x[slots // size, :, slots % size]


# ---------------------------------------------------------------- append and read
def turn32(x, pos, cos, sin, layout):
    """x [rows][heads][hd] F32 rotated, each product and sum rounded."""
    x, c, s = x.float().cpu().numpy().copy(), cos.cpu().numpy()[pos][:, None], sin.cpu().numpy()[pos][:, None]
    pairs = c.shape[-1]
    i = np.arange(0, 2 * pairs, 2) if layout == "interleaved" else np.arange(pairs)
    j = i + (1 if layout == "interleaved" else pairs)
    a, b = x[..., i], x[..., j]
    x[..., i], x[..., j] = a * c - b * s, a * s + b * c
    return x


def check_append(k, v, slots, cache, size, pos=None, rope=None, layout="interleaved", q=None, skip_k=(), error=0):
    """Append rows and compare every byte of the cache with what it has to hold."""
    want = []
    for name, x in (("k", k), ("v", v)):
        b, s = (t.cpu().numpy().copy() for t in (cache.tensors["kv".index(name)], cache.tensors[2 + "kv".index(name)]))
        y = turn32(x, np.clip(pos, 0, len(rope[0]) - 1), *rope, layout) if name == "k" and rope else x.float().cpu().numpy()
        n, scale, low = hold(y)
        n = packed(n)
        for r, slot in enumerate(slots):
            if 0 <= slot < len(b) * size and not (name == "k" and r in skip_k):
                b[slot // size, :, slot % size] = n[r]
                s[slot // size, :, slot % size, :, 0], s[slot // size, :, slot % size, :, 1] = scale[r], low[r]
        want += [b, s]
    err = i32([0])
    args = {}
    if rope:
        args = dict(positions=i32(pos), cos=rope[0], sin=rope[1], layout=layout)
        if q is not None:
            args |= dict(q=q, q_out=torch.empty_like(q))
    cache.append(k, v, i32(slots), error=err, **args)
    assert err.item() == error
    got = cache.tensors
    for t, w in zip((got[0], got[2], got[1], got[3]), want):
        assert (t.cpu().numpy().view(np.uint8) == np.ascontiguousarray(w).view(np.uint8)).all()
    return args.get("q_out")


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size,rows,kv", [(16, 1, 1), (32, 16, 3), (256, 300, 2)])
def test_append(kind, hd, size, rows, kv):
    g = torch.Generator().manual_seed(rows + hd)
    blocks = rows // size + 3
    cache = F.KV4Cache.empty(blocks, kv, size, hd)
    cache.tensors[0].fill_(0xA5)
    cache.tensors[3].fill_(float("nan"))
    y = (torch.randn(rows, 2 * kv + 2, hd, generator=g) * 3).to(ROW_TYPES[kind]).cuda()
    slots = torch.randperm(blocks * size, generator=g)[:rows].numpy()  # any order
    if rows > 4:
        slots[3], slots[rows // 2] = -1, -7
    check_append(y[:, 1:1 + kv], y[:, 1 + kv:1 + 2 * kv], slots, cache, size)                       # strided rows
    check_append(y[:, 1:1 + kv].contiguous(), y[:, :kv].contiguous(), slots[::-1], cache, size)     # written again
    odd = torch.cat([y.reshape(-1), y.reshape(-1)[:1]])[1:].view(y.shape)                            # rows off 16 bytes
    check_append(odd[:, :kv], odd[:, kv:2 * kv], slots, cache, size)
    use = np.concatenate([slots, [-1]])
    ko, vo = (torch.full((rows + 1, kv, hd), 7.0, device="cuda") for _ in "kv")
    cache.read(i32(use), ko, vo)
    for name, out in (("k", ko), ("v", vo)):
        want = np.where((use >= 0)[:, None, None], slot_values(cache, name, np.maximum(use, 0)), 0.0)
        assert (np.abs(out.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -24).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("layout,hd,dims", [("interleaved", 128, 128), ("half", 128, 128), ("interleaved", 64, 6),
                                            ("half", 64, 10), ("half", 128, 72), ("interleaved", 128, 66), ("half", 64, 32),
                                            ("interleaved", 128, 64)])
@pytest.mark.parametrize("rows", [5, 200])
def test_append_rotated(kind, layout, hd, dims, rows):
    kv, heads, size, ctx = 2, 6, 16, 400
    g = torch.Generator().manual_seed(rows + dims)
    cos, sin = rope_tables(ctx, dims)
    y = torch.randn(rows, heads + 2 * kv, hd, generator=g).to(ROW_TYPES[kind]).cuda()
    q, k, v = y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    pos = torch.randint(0, ctx, (rows,), generator=g).numpy()
    pos[0] = ctx - 1
    cache = F.KV4Cache.empty(rows // size + 2, kv, size, hd)
    slots = np.arange(rows) + 3
    got = check_append(k, v, slots, cache, size, pos, (cos, sin), layout, q=q)
    want = torch.empty_like(got)
    F.rope(q, None, i32(pos), cos, sin, layout, want, None)
    assert torch.equal(got, want)
    check_append(v, k, slots, cache, size, pos, (cos, sin), layout)  # K alone
    turned = q.clone()
    cache.append(k, v, i32(slots), i32(pos), cos, sin, layout, q=turned, q_out=turned)  # in place
    assert torch.equal(turned, want)
    shift = torch.cat([cos.reshape(-1)[:1], cos.reshape(-1)])[1:].view(cos.shape)  # tables off 16 bytes
    check_append(k, v, slots, cache, size, pos, (shift, sin), layout, q=q)


def test_append_values_at_the_edges():
    """Constant and zero groups, one value, ties between numbers, ranges below F16's, values beyond it, infinities
    and NaN (error 2)."""
    hd, kv, size = 128, 1, 16
    rows = []
    base = torch.linspace(-1.5, 1.5, hd)
    add = lambda f: rows.append(f.clone().float())  # noqa: E731
    add(torch.zeros(hd))
    add(torch.full((hd,), 3.25))
    add(torch.full((hd,), -1e-9))
    add(base * 1e-7)
    add(base * 1e-10)
    add(base * 40000.0)                       # to +-60000
    add(base * 1e6)                           # beyond: as +-61440
    add(base * 1e37)
    add((torch.arange(hd) % 61) * 0.25)       # 0 .. 15 in quarters: scale 1, ties at every half
    add(-(torch.arange(hd) % 61) * 0.5 + 7)   # 15 steps of 2, odd offsets
    add((torch.arange(hd) % 31) * 2.0 ** -15 + 1)
    one = torch.zeros(hd); one[70] = -5.0
    add(one)
    add(torch.full((hd,), 2.0 ** -140))
    for i in range(40):  # ties as a 16-bit row has them
        add((torch.randn(hd, generator=torch.Generator().manual_seed(i)) * 4).to(torch.bfloat16))
    x = torch.stack(rows)[:, None].cuda()
    cache = F.KV4Cache.empty(8, kv, size, hd)
    check_append(x, -x, np.arange(len(x)), cache, size)
    assert np.isfinite(values(cache, "k")).all()
    x = x[:8].clone()
    x[0, 0, 5] = float("inf")
    x[1, 0, 5], x[1, 0, 6] = float("-inf"), float("nan")
    x[2, 0, :64] = float("nan")
    x[3, 0] = float("inf")
    x[4, 0, 64:] = float("-inf")
    check_append(x, x, np.arange(8) + 40, cache, size, error=2)
    assert np.isfinite(values(cache, "k")).all() and (slot_values(cache, "k", [42])[0, 0, :64] == 0).all()


def test_append_leaves_rows_out():
    """Slots past the pool and positions past the table: error 4, the row left out (of K alone for its position), the
    rest as ever."""
    kv, hd, size, ctx = 2, 64, 16, 32
    cos, sin = rope_tables(ctx, hd)
    cache = F.KV4Cache.empty(3, kv, size, hd)
    y = torch.randn(12, 2 * kv + 4, hd, device="cuda")
    k, v, q = y[:, :kv], y[:, kv:2 * kv], y[:, 2 * kv:]
    pos = np.arange(12)
    pos[2], pos[5] = ctx, -1
    slots = np.arange(12) + 20
    slots[7], slots[8] = 48, 2 ** 31 - 1
    check_append(k, v, slots, cache, size, pos, (cos, sin), "interleaved", skip_k=(2, 5), error=4)
    out, err = torch.full((12, 4, hd), 7.0, device="cuda"), i32([0])
    cache.append(k, v, i32(slots), i32(pos), cos, sin, "interleaved", q=q, q_out=out, error=err)
    assert err.item() == 4 and (out[[2, 5]] == 7).all() and (out[[0, 7, 11]] != 7).any()
    ko, vo = (torch.full((3, kv, hd), 7.0, device="cuda") for _ in "kv")
    err.zero_()
    cache.read(i32([20, 48, -5]), ko, vo, error=err)
    assert err.item() == 4 and (ko[1:] == 0).all() and (vo[1:] == 0).all() and (ko[0] != 0).any()


def test_calls_refuse():
    cache = F.KV4Cache.empty(2, 2, 16, 64)
    x, s = torch.zeros(3, 2, 64, device="cuda"), i32([0, 1, 2])
    for k, v, slots in ((x, x, s[:2]), (x, x[:2], s), (x[..., :32], x[..., :32], s), (x, x.half(), s), (x.double(), x.double(), s),
                        (x, x, s.long()), (x.cpu(), x, s), (x[:, :1], x, s), (x.transpose(1, 2), x, s)):
        with pytest.raises(ValueError):
            cache.append(k, v, slots)
    with pytest.raises(ValueError):
        cache.append(x, x, s, q=x, q_out=x)
    with pytest.raises(ValueError):
        cache.read(s, x[:2], x)
    ws = cache.attention_workspace(3, 1, 4)
    q, t = torch.zeros(3, 4, 64, device="cuda"), i32([[0], [0], [1]])
    for a in ((q, s, t[:2], q, ws), (q[:2], s, t, q, ws), (q, s, t, q.half(), ws), (q, s, t, q, ws[:256]), (q[:, :3], s, t, q[:, :3], ws),
              (q, s, t, q, ws[1:])):
        with pytest.raises(ValueError):
            cache.attention(*a)
    with pytest.raises(ValueError):
        cache.attention_workspace(3, 1, 3)
    empty = x[:0]
    cache.append(empty, empty, s[:0])
    cache.read(s[:0], empty, empty)


# ---------------------------------------------------------------- attention
def make(lengths, heads, kv, hd, size, seed, width=None, extra=2, junk=True):
    """A cache with requests' blocks in random order, garbage everywhere that is not a token of theirs."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-n // size) for n in lengths]
    blocks = sum(counts) + extra
    cache = F.KV4Cache.empty(blocks, kv, size, hd)
    for t in cache.tensors[:2]:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda"))
    for t in cache.tensors[2:]:
        t[..., 0] = 0.05 + 0.3 * torch.rand(t.shape[:-1], generator=g, device="cuda")
        t[..., 1] = t[..., 0] * (-7.5 + torch.randn(t.shape[:-1], generator=g, device="cuda"))
    order = torch.randperm(blocks, generator=g, device="cuda").tolist()
    table = np.full((len(lengths), width or max(1, max(counts))), -1, np.int32)
    at = 0
    for r, c in enumerate(counts):
        table[r, :c] = order[at:at + c]
        at += c
        if lengths[r] % size and junk:  # what lies past the length
            for i, t in enumerate(cache.tensors[2:]):
                t[order[at - 1], :, lengths[r] % size:] = [float("nan"), float("inf"), float("-inf"), 65504.0][(r + i) % 4]
    for b in order[at:]:
        cache.tensors[2][b], cache.tensors[3][b] = float("nan"), float("inf")
    return cache, table


def reference(cache, table, lengths, starts, q, scale, kind):
    """(out, bound) in 64 bits; rows [rows][heads][hd] on the CPU."""
    parts = {}
    for n in "kv":
        num, s, low = (torch.from_numpy(t) for t in numbers(cache, n))
        mag = 15 * s + low.abs()
        parts[n] = (low[..., None] + s[..., None] * num).flatten(-2), mag[..., None].expand(num.shape).flatten(-2)
    _, kv, size, hd = parts["k"][0].shape
    q = q.cpu().double()
    rows, heads, _ = q.shape
    out, tol = torch.zeros(rows, heads, hd, dtype=torch.float64), torch.zeros(rows, heads, 1, dtype=torch.float64)
    wide, peak = kind == "f32", 0.0
    for r, n in enumerate(lengths):
        use = table[r, :-(-n // size)].tolist()
        if not use:
            continue
        kk, km, vv, vm = (torch.cat([t[b] for b in use], 1)[:, :n] for x in "kv" for t in parts[x])
        m = starts[r + 1] - starts[r]
        for j in range(m):
            end = n - m + j + 1
            if end <= 0:
                continue
            row = q[starts[r] + j].reshape(kv, heads // kv, hd)
            sc = torch.einsum("ghd,gtd->ght", row, kk[:, :end]) * scale
            peak = max(peak, float(sc.abs().amax()))
            mag = torch.einsum("ghd,gtd->ght", row.abs(), km[:, :end]).amax(2) * abs(scale)
            p = torch.softmax(sc, 2)
            out[starts[r] + j] = torch.einsum("ght,gtd->ghd", p, vv[:, :end]).reshape(heads, hd)
            top = vm[:, :end].amax((1, 2))[:, None]
            e = ((hd + 16) * 2.0 ** -24 + (0 if wide else 2.0 ** -11)) * mag
            if not wide:
                e = e + row.abs().sum(2) * abs(scale) * 2.0 ** -25
            bound = top * (2 * e + (end + 16) * 2.0 ** -23 + (0 if wide else 3 * 2.0 ** -11)) + (0 if wide else 2.0 ** -25)
            tol[starts[r] + j] = bound.reshape(heads, 1)
    return out, tol, peak


def run_attention(lengths, new, heads, kv, hd, size, kind, seed=0, scale=None, q=None, change=None, stride=0):
    cache, table = make(lengths, heads, kv, hd, size, seed, width=-(-max(max(lengths), 1) // size) + seed % 3)
    if change:
        change(cache, table)
    starts = [0] + list(np.cumsum(new))
    rows = starts[-1]
    scale = hd ** -0.5 if scale is None else scale
    if q is None:
        q = torch.randn((rows, heads, hd), generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda")
    q = q.to(ROW_TYPES[kind])
    if stride:
        q = torch.cat([q.reshape(rows, -1), q.new_full((rows, stride), 7.0)], 1)[:, :heads * hd].unflatten(1, (heads, hd))
    out = torch.full((rows, heads, hd), 7.0, dtype=q.dtype, device="cuda")
    ws, err = cache.attention_workspace(len(lengths), max(new), heads), i32([0])
    args = dict(row_start=None if all(m == 1 for m in new) else i32(starts), most_rows=max(new), scale=scale, error=err)
    cache.attention(q, i32(lengths), i32(table), out, ws, **args)
    again = torch.full_like(out, 3.0)
    cache.attention(q, i32(lengths), i32(table), again, ws, **args)  # the workspace is left as it has to be
    assert err.item() == 0
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))
    want, tol, peak = reference(cache, table, lengths, starts, q, scale, kind)
    got = out.cpu().double()
    assert got.isfinite().all()
    far = (got - want).abs() - tol - want.abs() * HALF_UNIT[kind] - 2.0 ** -25
    assert (far <= 0).all(), float(far.max())
    # and in the mean far nearer than the worst case. A score s in 32 bits is off by up to 2^-24 |s|, its weight by as much
    # of itself; weights and their sum together move an output by up to twice that of the values' size: 2^-23 |s|
    if want.norm() > 0:
        assert (got - want).norm() <= ((2e-5 if kind == "f32" else 1e-2) + 2.0 ** -23 * peak) * want.norm()
    return out


EDGES = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000]


@pytest.mark.parametrize("size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_decode_lengths(size, kind):
    run_attention(EDGES, [1] * len(EDGES), 8, 2, 128, size, kind, seed=size)
    run_attention(EDGES, [1] * len(EDGES), 8, 2, 64, size, kind, seed=size + 1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 31, 64])
def test_decode_groups(group, hd, kind):
    run_attention([77, 300, 1], [1, 1, 1], group * 2, 2, hd, 32, kind, seed=group)


@pytest.mark.parametrize("kind", sorted(ROW_TYPES))
def test_decode_types(kind):
    run_attention([500, 3, 64, 129], [1] * 4, 16, 4, 128, 16, kind, seed=3)
    run_attention([500, 3, 64, 129], [1] * 4, 16, 4, 64, 64, kind, seed=4, stride=8)
    run_attention([500, 3, 64, 129], [1] * 4, 16, 4, 64, 64, kind, seed=4, stride=1)
    run_attention([5000, 1, 2047], [1] * 3, 8, 1, 128, 64, kind, seed=5)


@pytest.mark.parametrize("new", [[2, 2, 2], [8, 5, 1], [16, 16, 3], [17, 40, 2], [130, 65, 64]])
@pytest.mark.parametrize("heads,kv,hd,size", [(8, 2, 128, 64), (16, 2, 64, 16), (3, 3, 128, 32), (12, 2, 128, 128)])
def test_rows(new, heads, kv, hd, size):
    """Drafts and chunks: causal inside, at the start of a context and behind a long one."""
    run_attention([m + d for m, d in zip(new, (0, 77, 400))], new, heads, kv, hd, size, "f32", seed=sum(new))
    run_attention([m + d for m, d in zip(new, (63, 0, 1))], new, heads, kv, hd, size, "bf16", seed=sum(new))
    run_attention([m + d for m, d in zip(new, (5, 1500, 127))], new, heads, kv, hd, size, "f16", seed=sum(new) + 1)


def test_empty_rows_and_requests():
    """Requests with no tokens or no rows, and rows that attend nothing, among others."""
    for kind in ("f32", "bf16"):
        for new in ([1, 1, 1, 1], [3, 0, 2, 5], [20, 0, 33, 2]):
            out = run_attention([0, 0, 70, 4], new, 8, 2, 128, 16, kind, seed=9)
            assert (out[:new[0]] == 0).all()
        # more rows than tokens: the first rows attend nothing
        out = run_attention([2, 90], [6, 30], 8, 2, 64, 32, kind, seed=2)
        assert (out[:4] == 0).all() and (out[4:6] != 0).any()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_wide_scales_and_scores(kind):
    """Scales many orders apart (0 among them), scores in the hundreds, queries of very different size."""
    def spread(cache, table):
        k, v, ks, vs = cache.tensors
        for i, b in enumerate(table[0]):
            if b >= 0:
                vs[b] *= 10.0 ** (i % 7 - 3)
                ks[b] *= [1.0, 30.0, 1e-3][i % 3]
                if i == 4:
                    vs[b], ks[b] = 0.0, 0.0
                if i == 5:
                    vs[b, :, 3], ks[b, :, ::2] = 0.0, 0.0
    for new in ([1], [9], [40]):
        run_attention([333], new, 8, 2, 128, 16, kind, seed=1, change=spread)
    sizes = [1e-6, 1e-3, 0.1, 1, 10, 1e3, 1e-20, 0.0] if kind == "f32" else [1e-4, 1e-3, 0.1, 1, 10, 1e3, 6e-8, 0.0]
    for rows in (1, 9):
        q = torch.randn(2 * rows, 8, 128, device="cuda") * torch.tensor(sizes, device="cuda")[None, :, None]
        run_attention([100, 200], [rows] * 2, 8, 2, 128, 32, kind, q=q, scale=0.01)
        run_attention([100, 200], [rows] * 2, 8, 2, 128, 32, kind, q=q.clamp(-1, 1), scale=-3.0)


@pytest.mark.parametrize("rows", [1, 12])
def test_values_that_grow(rows):
    """The largest values behind the largest weights, and far smaller ones before them and after."""
    def grow(cache, table):
        vs = cache.tensors[3]
        for i, b in enumerate(table[0]):
            if b >= 0:
                vs[b] *= 2.0 ** (i - 12)
    run_attention([400], [rows], 4, 1, 128, 16, "f32", seed=1, change=grow)
    run_attention([400], [rows], 4, 1, 64, 16, "f32", seed=3, change=lambda c, t: grow(c, t[:, ::-1]))


@pytest.mark.parametrize("rows", [1, 12])
def test_scores_beyond_the_resolution(rows):
    """Scores of 2^27 and more, where one more or less is lost: weights stay finite."""
    q = torch.randn(rows, 8, 128, device="cuda") * 1e7
    cache, table = make([300], 8, 2, 128, 16, 3)
    out = torch.empty_like(q)
    cache.attention(q, i32([300]), i32(table), out, cache.attention_workspace(1, rows, 8), row_start=i32([0, rows]),
                    most_rows=rows, scale=50.0)
    assert out.isfinite().all()


def test_long_tail_of_small_weights():
    """One token takes nearly all weight, 20000 others share the rest: their sum has to survive."""
    n, hd = 20000, 64
    for rows in (1, 16):
        cache, table = make([n], 1, 1, hd, 64, 11, junk=False)
        k, v, ks, vs = cache.tensors
        k.zero_()
        k[table[0, 100], 0, 7] = 0xff
        v.fill_(0xff)
        v[table[0, 100], 0, 7] = 0
        ks[..., 0], vs[..., 0], ks[..., 1], vs[..., 1] = 1 / 15, 1 / 15, 0, 0
        unit = np.float64(np.float16(1 / 15)) * 15
        q = torch.full((rows, 1, hd), 1.0, device="cuda")
        out = torch.empty_like(q)
        scale = 16.0 / hd  # the strong score is 16, all others 0
        cache.attention(q, i32([n]), i32(table), out, cache.attention_workspace(1, rows, 1), row_start=i32([0, rows]),
                        most_rows=rows, scale=scale)
        want = np.array([unit * (m - 1) / (m - 1 + np.exp(16.0 * unit)) for m in range(n - rows + 1, n + 1)])
        # the strong score is off by (hd + 16) 2^-24 x 16, its weight by as much
        assert np.abs(out.cpu().numpy()[:, 0] / want[:, None] - 1).max() <= n * 2.0 ** -23 + 2 * 16 * (hd + 16) * 2.0 ** -24


@pytest.mark.parametrize("n", [257, 4000, 30000])
@pytest.mark.parametrize("heads", [2, 8, 16, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_outputs_far_smaller_than_the_values(n, heads, hd):
    """Values of either sign and nearly equal weights: an output is some 1 / sqrt(n) of a value.

    Tolerance: the tensor cores line 16 products w (m 2^-22), m < 16 or 16 m, up at the exponent 2^-14 of a subnormal
    operand and round 24 bits below it towards zero: by up to 2^-38 w, 2^-16 w of a step of the cache, half of that in the
    mean, once for 16 positions, so 2^-21 of the sum of w. An output has the norm of sqrt(n) w values of 15 / sqrt(12)
    steps, n w of the sum of w: 2^-21 sqrt(n) / 4.3 of it. Weights, scores and the rest: 2^-20."""
    g = torch.Generator(device="cuda").manual_seed(n + heads)
    blocks = -(-n // 64)
    cache = F.KV4Cache.empty(blocks, 2, 64, hd)
    k, v = (torch.randn((n, 2, hd), generator=g, device="cuda") for _ in "kv")
    cache.append(k, v, i32(range(n)))
    q = torch.randn((1, heads, hd), generator=g, device="cuda")
    out, table = torch.empty_like(q), np.arange(blocks, dtype=np.int32)[None]
    cache.attention(q, i32([n]), i32(table), out, cache.attention_workspace(1, 1, heads), scale=0.02)
    want, _, _ = reference(cache, table, [n], [0, 1], q, 0.02, "f32")
    assert (out.cpu().double() - want).norm() <= (2.0 ** -21 * n ** 0.5 / 4.3 + 2.0 ** -20) * want.norm()


@pytest.mark.parametrize("most", [1, 20])
def test_bad_tables_and_lengths(most):
    """Blocks outside the pool and lengths beyond the table are left out and raise the error word; other requests
    are as ever."""
    lengths = [100, 90, 64]
    cache, table = make(lengths, 8, 2, 128, 16, 4)
    starts = i32([0, most, 2 * most, 3 * most])
    q = torch.randn(3 * most, 8, 128, device="cuda")
    good, bad = torch.empty_like(q), torch.empty_like(q)
    ws, err = cache.attention_workspace(3, most, 8), i32([0])
    call = lambda t, le, out, **kw: cache.attention(q, i32(le), i32(t), out, ws, error=err,  # noqa: E731
                                                    **(dict(row_start=starts, most_rows=most) | kw))
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
    call(table, [100, table.shape[1] * 16 + 1, 64], bad)
    assert err.item() == 4 and torch.equal(bad[rest], good[rest]) and (bad[most:2 * most] == 0).all()
    # more rows than the caller said: those past most_rows are left out
    err.zero_()
    bad.fill_(7.0)
    ws1 = cache.attention_workspace(1, most + 1, 8)
    cache.attention(q[:most + 3] if most > 1 else q, i32([100]), i32(table[:1]), bad[:most + 3] if most > 1 else bad, ws1,
                    row_start=i32([0, most + 2]), most_rows=most + 1, error=err)
    assert err.item() == 4 and (bad[most + 1:] == 7.0).all() and (bad[:most + 1] != 7.0).any()


def test_rows_behind_the_last_request_stay():
    for kind in ("f32", "bf16"):
        for new in ([1, 2], [30, 9]):
            cache, table = make([100, 80], 8, 2, 128, 16, 4)
            rows = sum(new) + 5
            q = torch.randn(rows, 8, 128, device="cuda").to(ROW_TYPES[kind])
            out = torch.full_like(q, 7.0)
            cache.attention(q, i32([100, 80]), i32(table), out, cache.attention_workspace(2, max(new), 8),
                            row_start=i32([0, new[0], sum(new)]), most_rows=max(new))
            assert (out[sum(new):] == 7).all() and (out[:sum(new)] != 7).any()


def test_nan_query_stays_in_its_row():
    for kind in ("f32", "f16"):
        for new in ([1, 1], [9, 30]):
            cache, table = make([100, 80], 8, 2, 128, 16, 4)
            starts = [0] + list(np.cumsum(new))
            q = torch.randn(starts[-1], 8, 128, device="cuda").to(ROW_TYPES[kind])
            args = dict(row_start=i32(starts), most_rows=max(new))
            a, b, ws = torch.empty_like(q), torch.empty_like(q), cache.attention_workspace(2, max(new), 8)
            cache.attention(q, i32([100, 80]), i32(table), a, ws, **args)
            for value in ("nan", "inf"):
                q2 = q.clone()
                q2[1, 3, 5] = float(value)
                cache.attention(q2, i32([100, 80]), i32(table), b, ws, **args)
                assert b[1, 3].isnan().all()
                b[1, 3] = a[1, 3]
                assert torch.equal(a, b)


def test_other_stream_and_graph():
    """The calls run on torch's current stream and can be captured: the graph then serves other lengths."""
    for rows in (1, 12):
        cache, table = make([200, 200], 8, 2, 128, 16, 4, junk=False)
        q, le, t = torch.randn(2 * rows, 8, 128, device="cuda"), i32([100, 33]), i32(table)
        want, out, ws = torch.empty_like(q), torch.empty_like(q), cache.attention_workspace(2, rows, 8)
        args = dict(row_start=i32([0, rows, 2 * rows]), most_rows=rows)
        cache.attention(q, le, t, want, ws, **args)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            big = torch.randn(4096, 4096, device="cuda")
            for _ in range(4):
                big = big @ big  # the stream is busy; q changes behind it
            q2 = torch.zeros_like(q).copy_(q)
            cache.attention(q2, le, t, out, ws, **args)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(out, want)
        k, v, slots = torch.randn(2, 2, 128, device="cuda"), torch.randn(2, 2, 128, device="cuda"), i32([-1, -1])
        ko, vo = torch.empty_like(k), torch.empty_like(v)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.append(k, v, slots)
            cache.read(slots, ko, vo)
            cache.attention(q, le, t, out, ws, **args)
        for n in ([200, 1], [100, 33]):
            le.copy_(i32(n))
            graph.replay()
        assert torch.equal(out, want) and (ko == 0).all()
        slots.copy_(i32([table[0, 12] * 16 + 9, table[1, 12] * 16 + 9]))  # past every length
        graph.replay()
        assert (np.abs(ko.cpu().numpy() - slot_values(cache, "k", slots.cpu().numpy())) <= 1e-6).all() and (ko != 0).any()


def test_two_streams_at_once():
    """Two calls in flight on two streams, each with a workspace of its own."""
    cache, table = make([3000, 1700], 8, 2, 128, 32, 4, junk=False)
    for rows in (1, 12):
        q = torch.randn(2 * rows, 8, 128, device="cuda")
        args = dict(row_start=i32([0, rows, 2 * rows]), most_rows=rows)
        le, t = i32([3000, 1700]), i32(table)
        want = torch.empty_like(q)
        cache.attention(q, le, t, want, cache.attention_workspace(2, rows, 8), **args)
        outs, streams = [torch.empty_like(q) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
        spaces = [cache.attention_workspace(2, rows, 8) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(20):
            for s, o, w in zip(streams, outs, spaces):
                cache.attention(q, le, t, o, w, stream=s.cuda_stream, **args)
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


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
    k, v = torch.randn(2, kv, hd, device="cuda"), torch.randn(2, kv, hd, device="cuda")
    cache.append(torch.cat([k[:1]] * 2), torch.cat([v[:1]] * 2), i32([low[2] * size + 80, high[2] * size + 80]))
    for new in (1, 12):
        q = torch.randn(new, 8, hd, device="cuda")
        q2, out = torch.cat([q, q]), torch.empty(2 * new, 8, hd, device="cuda")
        cache.attention(q2, i32([2 * size + 81] * 2), i32([low, high]), out, cache.attention_workspace(2, new, 8),
                        row_start=i32([0, new, 2 * new]), most_rows=new)
        assert torch.equal(out[:new], out[new:]) and (out != 0).any()
    ko, vo = (torch.empty(2, kv, hd, device="cuda") for _ in "kv")
    cache.read(i32([low[2] * size + 80, high[2] * size + 80]), ko, vo)
    assert torch.equal(ko[0], ko[1]) and (ko != 0).any()


def test_steps_together():
    """Blocks, append with rotation, attention: a prompt and then single tokens of three requests, against
    attention in 64 bits over what the cache holds."""
    heads, kv, hd, size, n = 8, 2, 128, 16, 3
    cache = F.KV4Cache.empty(40, kv, size, hd)
    cos, sin = rope_tables(256, hd)
    lengths, table = i32([0] * n), torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    free, count = i32(range(40)), i32([40])
    ws = {most: cache.attention_workspace(n, most, heads) for most in (1, 8, 37)}
    for step, new in enumerate([[37, 5, 16], [1, 1, 1], [1, 0, 1], [8, 3, 1], [1, 1, 1]]):
        rows = sum(new)
        e = lambda m: torch.empty(m, dtype=torch.int32, device="cuda")  # noqa: E731
        out_len, out_count, start, slots, pos, who, status = e(n), e(1), e(n + 1), e(rows), e(rows), e(rows), e(n)
        F.kv_blocks(lengths, i32(new), table, free, count, size, out_len, out_count, start, slots, pos, who, status)
        lengths, count = out_len, out_count
        assert status.tolist() == [0] * n
        y = torch.randn(rows, heads + 2 * kv, hd, device="cuda")
        q, out = torch.empty(rows, heads, hd, device="cuda"), torch.empty(rows, heads, hd, device="cuda")
        cache.append(y[:, heads:heads + kv], y[:, heads + kv:], slots, pos, cos, sin, "interleaved", y[:, :heads], q)
        cache.attention(q, lengths, table, out, ws[max(new)], row_start=start, most_rows=max(new))
        want, tol, _ = reference(cache, table.cpu().numpy(), lengths.tolist(), start.tolist(), q, hd ** -0.5, "f32")
        assert ((out.cpu().double() - want).abs() <= tol + want.abs() * 2.0 ** -24 + 2.0 ** -25).all(), step
    F.kv_release(lengths, i32([0, 999, -1]), table, free, count, size)
    assert lengths.tolist()[0] == 0 and count.item() == 40 - -(-lengths.tolist()[1] // size)
