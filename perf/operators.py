"""The operators of serving from a paged 8-bit KV cache, with the sizes they are timed at.

  blocks     block tables and slot maps built on the GPU from request lengths
  rope       rotary positions of q and k: interleaved or half pairs, all of a head or a part of it
  append     new K/V rows into the cache in 8 bits with one scale for each block of tokens and KV head (q and K
             rotated on the way where the case says so), then the touched blocks read back as the values they hold
  attention  causal attention of each request's newest tokens over its blocks

With `own` false, run() computes an operator in its plain form, elementary torch operations in 32 bits; with `own`
true it makes the calls a user of fyodor_b200 makes. Geometries (32/8, 64/8, 16/2 and 8/8 heads of 64 or 128,
contexts to 32768, batches of 16 and 32, drafts of 8) are those of the package's tests and benchmark."""
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
WIDTH = {"f32": 4, "f16": 2, "bf16": 2}
QMAX = {"int8": 127.0, "e4m3": 448.0}
STORED = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
#: (query heads, KV heads, head dimension)
GEOMETRY = {"32/8x128": (32, 8, 128), "64/8x128": (64, 8, 128), "16/2x64": (16, 2, 64), "8/8x128": (8, 8, 128),
            "32/8x64": (32, 8, 64)}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a batched decode step of 16 sequences: one new token each, latency is all there is
        {"name": "blocks step of 16", "op": "blocks", "requests": 16, "block": 16, "most": 768, "prompts": 0,
         "prompt": 0, "short": False, "pick": 1},
        # a serving step that admits prompts beside many decoding requests, with too few free blocks for the last ones
        {"name": "blocks 1021 requests, 40 prompts", "op": "blocks", "requests": 1021, "block": 32, "most": 32768,
         "prompts": 40, "prompt": 2500, "short": True, "pick": 2},
        # q and k of one decode step of 16 sequences
        {"name": "rope step of 16", "op": "rope", "rows": 16, "geometry": "32/8x128", "type": "f32", "dims": 128,
         "layout": "interleaved", "context": 8192, "fused": True, "pick": 3},
        # a long prompt of a model that rotates half of each head, in half pairs
        {"name": "rope prompt of 8191, half of the head", "op": "rope", "rows": 8191, "geometry": "64/8x128",
         "type": "bf16", "dims": 64, "layout": "half", "context": 131072, "fused": False, "pick": 4},
        # the cache rows of one decode step of 16 sequences, rotated on the way
        {"name": "append step of 16, rotated", "op": "append", "requests": 16, "most": 768, "new": 1,
         "geometry": "32/8x128", "type": "f32", "format": "int8", "block": 16, "rope": True, "fused": True, "pick": 5},
        # drafts of up to 8 tokens of 32 sequences, heads of 64
        {"name": "append drafts of 8", "op": "append", "requests": 32, "most": 4000, "new": 8, "geometry": "16/2x64",
         "type": "f16", "format": "e4m3", "block": 32, "rope": False, "fused": False, "pick": 6},
        # prompts of four requests
        {"name": "append 4 prompts of to 2100, rotated", "op": "append", "requests": 4, "most": 0, "new": 2100,
         "geometry": "32/8x128", "type": "bf16", "format": "int8", "block": 64, "rope": True, "fused": True, "pick": 7},
        # one sequence a little into its context
        {"name": "attention one of 257", "op": "attention", "requests": 1, "least": 257, "most": 257, "new": 1,
         "geometry": "32/8x128", "type": "f32", "format": "int8", "block": 16, "fused": False, "pick": 8},
        # the ragged decode batch of the benchmark
        {"name": "attention ragged 32 to 32768", "op": "attention", "requests": 32, "least": 128, "most": 32768,
         "new": 1, "geometry": "32/8x128", "type": "f32", "format": "int8", "block": 64, "fused": False, "pick": 9},
        # the same batch checking drafts of up to 8 tokens
        {"name": "attention drafts of 8, ragged 32", "op": "attention", "requests": 32, "least": 128, "most": 32768,
         "new": 8, "geometry": "32/8x128", "type": "bf16", "format": "e4m3", "block": 64, "fused": True, "pick": 10},
        # sixteen sequences of a 64/8-head model near 8192 positions
        {"name": "attention 16 at 8100, 64 heads", "op": "attention", "requests": 16, "least": 7800, "most": 8192,
         "new": 1, "geometry": "64/8x128", "type": "f16", "format": "int8", "block": 32, "fused": True, "pick": 11},
        # a prompt chunk of 500 tokens behind a long context
        {"name": "attention chunk of 500 at 16000", "op": "attention", "requests": 1, "least": 16001, "most": 16001,
         "new": 500, "geometry": "32/8x128", "type": "f32", "format": "int8", "block": 128, "fused": False,
         "pick": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["blocks", "rope", "append", "append", "attention", "attention", "attention"])
    pick, block = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128])
    geometry, type_ = rng.choice(sorted(GEOMETRY)), rng.choice(sorted(TYPES))
    if op == "blocks":
        n = _log_int(rng, 1, 1021)
        return {"op": op, "requests": n, "block": block, "most": _log_int(rng, 16, 32768),
                "prompts": rng.randint(0, min(n, 40)), "prompt": _log_int(rng, 1, 2500), "short": rng.random() < 0.3,
                "pick": pick}
    if op == "rope":
        hd = GEOMETRY[geometry][2]
        return {"op": op, "rows": _log_int(rng, 1, 8191), "geometry": geometry, "type": type_,
                "dims": rng.choice([hd, hd, hd // 2, hd // 4]), "layout": rng.choice(["interleaved", "half"]),
                "context": 8192, "fused": rng.random() < 0.5, "pick": pick}
    if op == "append":
        n = _log_int(rng, 1, 64)
        return {"op": op, "requests": n, "most": rng.choice([0, _log_int(rng, 1, 4000)]),
                "new": _log_int(rng, 1, max(1, min(2100, 8400 // n))), "geometry": geometry, "type": type_,
                "format": rng.choice(sorted(QMAX)), "block": block, "rope": rng.random() < 0.5,
                "fused": rng.random() < 0.5, "pick": pick}
    heads, kv, hd = GEOMETRY[geometry]
    new = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 500)])
    n = _log_int(rng, 1, 64 if new <= 16 else 4)
    most = _log_int(rng, 1, min(32768, (1 << 20) // n, (1 << 28) // (n * new * heads)))
    return {"op": op, "requests": n, "least": _log_int(rng, 1, most), "most": most, "new": min(new, most),
            "geometry": geometry, "type": type_, "format": rng.choice(sorted(QMAX)), "block": block,
            "fused": rng.random() < 0.5, "pick": pick}


def _shape(case):
    """Lengths and new rows of a case's requests: plain numbers that follow from the case alone."""
    r, n = random.Random(case["pick"]), case.get("requests", 0)
    if case["op"] == "blocks":
        cached = [r.randint(1, case["most"]) for _ in range(n)]
        new = [1] * n
        for i in r.sample(range(n), case["prompts"]):
            cached[i], new[i] = 0, r.randint(1, case["prompt"])
        if n > 8:
            new[r.randrange(n)] = 0  # a request that waits in this step
        return cached, new
    if case["op"] == "append":
        new = [r.randint(1, case["new"]) for _ in range(n)]
        new[0] = case["new"]
        return [r.randint(0, case["most"]) for _ in range(n)], new
    lengths = [r.randint(case["least"], case["most"]) for _ in range(n)]
    new = [1] * n if case["new"] == 1 else [min(t, r.randint(1, case["new"])) for t in lengths]
    new[0] = min(case["new"], lengths[0])
    return [t - m for t, m in zip(lengths, new)], new


def _ceil(a, b):
    return -(-a // b)


def work(case):
    """What one pass cannot do without: each input read once, each output written once."""
    op = case["op"]
    if op == "blocks":
        cached, new = _shape(case)
        rows = sum(new)
        fresh = sum(_ceil(c + m, case["block"]) - _ceil(c, case["block"]) for c, m in zip(cached, new))
        return {"bytes": 4 * (len(cached) * 5 + 3 * rows + 2 * fresh), "flops": 0}
    heads, kv, hd = GEOMETRY[case["geometry"]]
    w = WIDTH[case["type"]]
    if op == "rope":
        values = case["rows"] * (heads + kv) * hd
        return {"bytes": 2 * w * values + case["rows"] * (4 + 4 * case["dims"]),
                "flops": 3 * case["rows"] * (heads + kv) * case["dims"]}
    cached, new = _shape(case)
    rows = sum(new)
    if op == "append":
        block = case["block"]
        touched = sum(_ceil(c + m, block) - c // block for c, m in zip(cached, new))
        held = sum(c + m - c // block * block for c, m in zip(cached, new))  # tokens of the touched blocks
        scales = 8 * kv * touched
        traffic = 2 * w * rows * kv * hd + 2 * rows * kv * hd + scales + 4 * rows  # rows in, bytes and scales out
        traffic += 2 * held * kv * hd * (1 + 4) + scales + 4 * held  # read back: bytes and scales in, values out
        flops = 6 * rows * kv * hd
        if case["rope"]:
            traffic += 2 * w * rows * heads * hd + rows * (4 + 4 * hd)
            flops += 3 * rows * (heads + kv) * hd
        return {"bytes": traffic, "flops": flops}
    total = sum(c + m for c, m in zip(cached, new))
    attended = sum(m * c + m * (m + 1) // 2 for c, m in zip(cached, new))
    blocks = sum(_ceil(c + m, case["block"]) for c, m in zip(cached, new))
    return {"bytes": 2 * total * kv * hd + blocks * (8 * kv + 4) + 2 * w * rows * heads * hd + 8 * len(cached),
            "flops": 4 * attended * heads * hd}


# ---------------------------------------------------------------- inputs
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(new):
    return _ints(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))


def _rows(g, rows, case):
    """q, k and v rows: slices of one fused row buffer, or buffers of their own."""
    heads, kv, hd = GEOMETRY[case["geometry"]]
    y = torch.randn((rows, heads + 2 * kv, hd), generator=g, device=DEV)
    y[:, heads:heads + kv, :: hd // 4] *= 4.0  # a few strong channels, as keys have
    y = y.to(TYPES[case["type"]])
    parts = y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    return parts if case["fused"] else tuple(p.contiguous() for p in parts)


def _rope_tables(dims, context, rows):
    """cos and sin of position x frequency, the frequencies halved for the slow half as a long-context model does."""
    f = 500000.0 ** (-np.arange(dims // 2) / (dims // 2))
    f[dims // 4:] /= 2.0
    angle = torch.arange(context, device=DEV, dtype=torch.float64)[:, None] * torch.tensor(f, device=DEV)
    return angle.cos().float(), angle.sin().float()


def _pool(g, blocks, case):
    """A cache of `blocks` blocks filled with quantised rows, made in pieces."""
    kv, hd = GEOMETRY[case["geometry"]][1:]
    top, out = QMAX[case["format"]], []
    for strong in (4.0, 1.0):
        stored = torch.empty((blocks, kv, case["block"], hd), dtype=STORED[case["format"]], device=DEV)
        scale = torch.empty((blocks, kv), device=DEV)
        step = max(1, (1 << 27) // stored[0].numel())
        for b in range(0, blocks, step):
            x = torch.randn(stored[b:b + step].shape, generator=g, device=DEV)
            x[..., :: hd // 4] *= strong
            s = x.abs().amax((2, 3)) / top
            y = x / s[:, :, None, None]
            stored[b:b + step] = (y.round() if case["format"] == "int8" else y).to(stored.dtype)
            scale[b:b + step] = s
        out += [stored, scale]
    return out[0], out[2], out[1], out[3]


def _tables(g, counts, blocks):
    """Block tables of requests whose blocks lie in any order in the pool (-1 where a request has none), and the rest."""
    order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    counts = torch.tensor(counts, device=DEV)
    width = max(1, int(counts.max()))
    at = torch.arange(width, device=DEV)[None] + (counts.cumsum(0) - counts)[:, None]
    has = torch.arange(width, device=DEV)[None] < counts[:, None]
    table = torch.where(has, order[at.clamp(max=blocks - 1)], torch.full_like(order[:1], -1))
    return table, order[int(counts.sum()):].contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "rope":
        rows = case["rows"]
        s["q"], s["k"], _ = _rows(g, rows, case)
        s["positions"] = torch.randint(0, case["context"], (rows,), generator=g, device=DEV, dtype=torch.int32)
        s["cos"], s["sin"] = _rope_tables(case["dims"], case["context"], rows)
        s["q_out"], s["k_out"] = (torch.empty(s[x].shape, dtype=s[x].dtype, device=DEV) for x in "qk")
        return s
    cached, new = _shape(case)
    block, rows, n = case["block"], sum(new), len(new)
    lengths, fresh = _ints(cached), _ints(new)
    if case["op"] == "blocks":
        before = [_ceil(c, block) for c in cached]
        want = sum(_ceil(c + m, block) for c, m in zip(cached, new)) - sum(before)
        spare = max(0, want * 9 // 10 if case["short"] else want + 7)
        table, free = _tables(g, before, sum(before) + max(1, spare))
        width = max(_ceil(c + m, block) for c, m in zip(cached, new))
        s["table"] = torch.full((n, max(width, table.shape[1])), -1, dtype=torch.int32, device=DEV)
        s["table"][:, :table.shape[1]] = table
        s |= {"lengths": lengths, "new": fresh, "free": free, "free_count": _ints([spare])}
        most = rows + 5  # a fixed number of rows, as a captured step has
        for x, m in (("lengths_out", n), ("row_start", n + 1), ("status", n), ("free_count_out", 1), ("slots", most),
                     ("positions", most), ("row_request", most)):
            s[x] = torch.empty(m, dtype=torch.int32, device=DEV)
        return s
    counts = [_ceil(c + m, block) for c, m in zip(cached, new)]
    blocks = sum(counts) + 3
    s["table"], _ = _tables(g, counts, blocks)
    s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = _pool(g, blocks, case)
    s["q"], s["k"], s["v"] = _rows(g, rows, case)
    s["row_start"], s["lengths"] = _starts(new), lengths + fresh
    if case["op"] == "attention":
        heads, kv, hd = GEOMETRY[case["geometry"]]
        s["out"] = torch.empty((rows, heads, hd), dtype=TYPES[case["type"]], device=DEV)
        s["most_rows"], s["scale"] = max(new), hd ** -0.5
        if case["new"] == 1:
            s["row_start"] = None
        return s
    at = lambda lo, hi: _ints([t for a, b in zip(lo, hi) for t in range(a, b)])  # noqa: E731
    slot = lambda who, pos: s["table"][who.long(), (pos // block).long()] * block + pos % block  # noqa: E731
    who = lambda lo, hi: _ints([i for i, (a, b) in enumerate(zip(lo, hi)) for _ in range(a, b)])  # noqa: E731
    end, floor = [c + m for c, m in zip(cached, new)], [c // block * block for c in cached]
    s["positions"] = at(cached, end)
    s["slots"] = slot(who(cached, end), s["positions"])
    s["held"] = slot(who(floor, end), at(floor, end))  # every token of the touched blocks
    hd = GEOMETRY[case["geometry"]][2]
    if case["rope"]:
        s["cos"], s["sin"] = _rope_tables(hd, max(end), rows)
        s["q_out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV)
    s["k_held"], s["v_held"] = (torch.empty((len(s["held"]), s["k"].shape[1], hd), device=DEV) for _ in "kv")
    return s


# ---------------------------------------------------------------- plain forms
def _plain_blocks(s):
    block, n, width = s["case"]["block"], len(s["lengths"]), s["table"].shape[1]
    most = len(s["slots"])
    length, new, free, count = (s[x].long() for x in ("lengths", "new", "free", "free_count"))
    valid = (length >= 0) & (new >= 0) & (length + new <= width * block)
    end = torch.where(valid, new, 0).cumsum(0)
    start = torch.cat([end.new_zeros(1), end]).clamp(max=most)
    valid &= end <= most
    old = (length + block - 1) // block
    need = torch.where(valid, (length + new + block - 1) // block - old, 0)
    upto = need.cumsum(0)
    served = valid & ((need == 0) | (upto <= count))
    status = torch.where(valid, torch.where(served, 0, 1), 2)
    taken = torch.where(served, need, 0).sum().reshape(1)
    b = torch.arange(width, device=DEV)[None]
    fresh = served[:, None] & (b >= old[:, None]) & (b < (old + need)[:, None])
    pop = (count - 1 - (upto - need)[:, None] - (b - old[:, None])).clamp(0, len(free) - 1)
    table = torch.where(fresh, free[pop], s["table"].long())
    row = torch.arange(most, device=DEV)
    who = torch.searchsorted(start[1:].contiguous(), row, right=True)
    real, who = who < n, who.clamp(max=n - 1)
    position = torch.where(real, length[who] + row - start[who], 0)
    slot = table[who, (position // block).clamp(0, width - 1)] * block + position % block
    slot = torch.where(real & served[who], slot, -1)
    r = {"table": table, "lengths": torch.where(served, length + new, length), "row_start": start, "slots": slot,
         "positions": position, "row_request": torch.where(real, who, -1), "status": status,
         "free_count": count - taken}
    return {k: v.to(torch.int32) for k, v in r.items()}


def _rotate(x, cos, sin, layout):
    """x [rows, heads, hd] in 32 bits, its first 2 * cos.shape[1] dimensions rotated."""
    pairs = cos.shape[1]
    c, z, part = cos[:, None], sin[:, None], x[..., :2 * pairs]
    if layout == "half":
        a, b = part[..., :pairs], part[..., pairs:]
        turned = torch.cat([a * c - b * z, a * z + b * c], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * c - b * z, a * z + b * c], -1).flatten(-2)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _plain_rope(s):
    at, layout = s["positions"].long(), s["case"]["layout"]
    cos, sin = s["cos"][at], s["sin"][at]
    return {x: _rotate(s[x].float(), cos, sin, layout).to(s[x].dtype) for x in "qk"}


def _plain_store(s, rows, cache, scale):
    """`rows` (32 bits) into their slots of `cache`. A block's scale is the largest magnitude it was ever given over
    the largest stored value; where it grows, what the block holds is stored anew."""
    block, top, exact = s["case"]["block"], QMAX[s["case"]["format"]], s["case"]["format"] == "int8"
    slots = s["slots"].long()
    touched, at = torch.unique(slots // block, return_inverse=True)
    peak = rows.new_zeros((len(touched), rows.shape[1]))
    peak.scatter_reduce_(0, at[:, None].expand(-1, rows.shape[1]), rows.abs().amax(2), "amax")
    first = torch.full_like(touched, block).scatter_reduce_(0, at, slots % block, "amin")
    was = torch.where(first[:, None] > 0, scale[touched], 0.0)
    now = torch.maximum(was, peak / top)
    keep = torch.where(now > 0, was / now, 0.0)
    held = cache[touched].float() * keep[:, :, None, None]
    held = held.round() if exact else held
    older = (torch.arange(block, device=DEV)[None] < first[:, None])[:, None, :, None]
    cache[touched] = torch.where(older, held, cache[touched].float()).to(cache.dtype)
    unit = now[at][:, :, None]
    y = torch.where(unit > 0, rows / unit, 0.0)
    y = y.round() if exact else y
    cache[slots // block, :, slots % block] = y.clamp(-top, top).to(cache.dtype)
    scale[touched] = now


def _plain_values(s, cache, scale, slots):
    block = s["case"]["block"]
    b, t = slots.long() // block, slots.long() % block
    return cache[b, :, t].float() * scale[b][:, :, None]


def _plain_append(s):
    r, k, case = {}, s["k"].float(), s["case"]
    if case["rope"]:
        cos, sin = (s[x][s["positions"].long()] for x in ("cos", "sin"))
        k = _rotate(k, cos, sin, "interleaved")
        r["q"] = _rotate(s["q"].float(), cos, sin, "interleaved").to(s["q"].dtype)
    _plain_store(s, k, s["k_cache"], s["k_scale"])
    _plain_store(s, s["v"].float(), s["v_cache"], s["v_scale"])
    for x in "kv":
        r[x] = _plain_values(s, s[x + "_cache"], s[x + "_scale"], s["held"])
        r[x + "_scale"] = s[x + "_scale"]
    return r


def _plain_attention(s):
    block, n = s["case"]["block"], len(s["lengths"])
    heads, kv, hd = GEOMETRY[s["case"]["geometry"]]
    length, table = s["lengths"].long(), s["table"].long().clamp(min=0)
    start = torch.arange(n + 1, device=DEV) if s["row_start"] is None else s["row_start"].long()
    new = start[1:] - start[:-1]
    most, width = s["most_rows"], table.shape[1] * block
    position = torch.arange(width, device=DEV)
    inside = position[None] < length[:, None]

    def whole(cache, scale):
        x = cache[table].float() * scale[table][..., None, None]
        x = x.permute(0, 2, 1, 3, 4).reshape(n, kv, width, hd)
        return torch.where(inside[:, None, :, None], x, 0.0)

    j = torch.arange(most, device=DEV)
    real = j[None] < new[:, None]
    row = (start[:-1, None] + j[None]).clamp(max=len(s["q"]) - 1)
    q = s["q"].float()[row].reshape(n, most, kv, heads // kv, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, hd)
    score = (q @ whole(s["k_cache"], s["k_scale"]).transpose(2, 3)) * s["scale"]
    last = (length - new)[:, None] + j[None]  # the newest position that row j attends
    seen = (position[None, None] <= last[:, :, None]) & real[:, :, None]
    score = score.reshape(n, kv, most, heads // kv, width).masked_fill_(~seen[:, None, :, None], -torch.inf)
    peak = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(peak > -torch.inf, peak, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(n, kv, -1, width) @ whole(s["v_cache"], s["v_scale"])).reshape(n, kv, most, heads // kv, hd)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(n, most, heads, hd)
    who = torch.searchsorted(start[1:].contiguous(), torch.arange(len(s["q"]), device=DEV), right=True)
    return o[who, torch.arange(len(s["q"]), device=DEV) - start[who]].to(s["q"].dtype)


# ---------------------------------------------------------------- the framework's operators
def _cache(s):
    """The cache handle that a serving program keeps."""
    if "cache" not in s:
        import fyodor_b200 as F
        s["cache"] = F.KV8Cache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s["cache"]


def _own_blocks(s):
    import fyodor_b200 as F
    F.kv_blocks(s["lengths"], s["new"], s["table"], s["free"], s["free_count"], s["case"]["block"], s["lengths_out"],
                s["free_count_out"], s["row_start"], s["slots"], s["positions"], s["row_request"], s["status"])
    return {"table": s["table"], "lengths": s["lengths_out"], "row_start": s["row_start"], "slots": s["slots"],
            "positions": s["positions"], "row_request": s["row_request"], "status": s["status"],
            "free_count": s["free_count_out"]}


def _own_rope(s):
    import fyodor_b200 as F
    F.rope(s["q"], s["k"], s["positions"], s["cos"], s["sin"], s["case"]["layout"], s["q_out"], s["k_out"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_append(s):
    cache, r = _cache(s), {}
    if s["case"]["rope"]:
        cache.append(s["k"], s["v"], s["slots"], positions=s["positions"], cos=s["cos"], sin=s["sin"],
                     layout="interleaved", q=s["q"], q_out=s["q_out"])
        r["q"] = s["q_out"]
    else:
        cache.append(s["k"], s["v"], s["slots"])
    cache.read(s["held"], s["k_held"], s["v_held"])
    return r | {"k": s["k_held"], "v": s["v_held"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _own_attention(s):
    cache = _cache(s)
    if "workspace" not in s:
        s["workspace"] = cache.attention_workspace(len(s["lengths"]), s["most_rows"], s["q"].shape[1])
    cache.attention(s["q"], s["lengths"], s["table"], s["out"], s["workspace"], row_start=s["row_start"],
                    most_rows=s["most_rows"], scale=s["scale"])
    return s["out"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"blocks": _own_blocks, "rope": _own_rope, "append": _own_append, "attention": _own_attention}[op](state)
    return {"blocks": _plain_blocks, "rope": _plain_rope, "append": _plain_append,
            "attention": _plain_attention}[op](state)


# ---------------------------------------------------------------- in 64 bits
def _exact_turn(x, angle_cos, angle_sin, layout):
    y, pairs = x.double().clone(), angle_cos.shape[1]
    first = range(0, 2 * pairs, 2) if layout == "interleaved" else range(pairs)
    second = range(1, 2 * pairs, 2) if layout == "interleaved" else range(pairs, 2 * pairs)
    i, j = torch.tensor(list(first), device=DEV), torch.tensor(list(second), device=DEV)
    z = torch.complex(x[..., i].double(), x[..., j].double())
    z = z * torch.complex(angle_cos.double(), angle_sin.double())[:, None]
    y[..., i], y[..., j] = z.real, z.imag
    return y


def _exact_append(s):
    case, out = s["case"], {}
    block, top = case["block"], QMAX[case["format"]]
    k = s["k"]
    if case["rope"]:
        at = s["positions"].long()
        k = _exact_turn(k, s["cos"][at], s["sin"][at], "interleaved")
        out["q"] = _exact_turn(s["q"], s["cos"][at], s["sin"][at], "interleaved")
    slots = s["slots"].tolist()
    runs = [[0]]  # rows of one block lie together
    for i in range(1, len(slots)):
        if slots[i] // block == slots[i - 1] // block:
            runs[-1].append(i)
        else:
            runs.append([i])

    def near(y):
        return y.round() if case["format"] == "int8" else y.float().to(STORED["e4m3"]).double()

    for name, x in (("k", k), ("v", s["v"])):
        held, scale = s[name + "_cache"], s[name + "_scale"].double().clone()
        value = held.double() * scale[:, :, None, None] if held.numel() < 1 << 28 else None
        if value is None:
            return None
        for r in runs:
            b, t = slots[r[0]] // block, slots[r[0]] % block
            new = x[r[0]:r[-1] + 1].double().transpose(0, 1)  # [heads, tokens, hd]
            was = scale[b] if t else torch.zeros_like(scale[b])
            now = torch.maximum(was, new.abs().amax((1, 2)) / top)
            unit = torch.where(now > 0, now, 1.0)[:, None, None]
            if t:
                value[b, :, :t] = near(value[b, :, :t] / unit) * unit
            value[b, :, t:t + len(r)] = near((new / unit).clamp(-top, top)) * unit
            scale[b] = now
        at = s["held"].long()
        out[name], out[name + "_scale"] = value[at // block, :, at % block], scale
    return out


def _exact_attention(s):
    block = s["case"]["block"]
    heads, kv, hd = GEOMETRY[s["case"]["geometry"]]
    n = len(s["lengths"])
    start = list(range(n + 1)) if s["row_start"] is None else s["row_start"].tolist()
    out = torch.zeros((len(s["q"]), heads, hd), dtype=torch.float64, device=DEV)
    for r, length in enumerate(s["lengths"].tolist()):
        use = s["table"][r, :_ceil(length, block)].long()
        k, v = (s[x + "_cache"][use].transpose(0, 1).double() * s[x + "_scale"][use].double().t()[:, :, None, None]
                for x in "kv")
        k, v = (x.reshape(kv, -1, hd)[:, :length] for x in (k, v))
        rows = start[r + 1] - start[r]
        last = length - rows + torch.arange(rows, device=DEV)
        hidden = torch.arange(length, device=DEV)[None] > last[:, None]
        for h in range(heads):
            score = (s["q"][start[r]:start[r + 1], h].double() @ k[h // (heads // kv)].t()) * s["scale"]
            p = torch.softmax(score.masked_fill(hidden, -torch.inf), -1)
            out[start[r]:start[r + 1], h] = torch.nan_to_num(p, nan=0.0) @ v[h // (heads // kv)]
    return out


def exact(case, seed):
    """run()'s outputs from the operators' definitions in 64 bits; None where an output is whole numbers."""
    if case["op"] == "blocks":
        return None
    s = prepare(case, seed)
    if case["op"] == "rope":
        at = s["positions"].long()
        return {x: _exact_turn(s[x], s["cos"][at], s["sin"][at], case["layout"]) for x in "qk"}
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
