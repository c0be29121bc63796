"""The operators of serving from a paged 4-bit KV cache and of scoring what is answered, with the sizes they are timed at.

  append     new K/V rows into the cache in 4 bits, each group of 64 values of a head with a 16-bit scale and low (q and
             K rotated on the way where the case says so), then the same rows read back as the values they are held as
  attention  causal attention of each request's newest tokens over its 4-bit blocks
  logprobs   of rows of logits: log probability and rank of a given token, entropy, the most probable alternatives

With `own` false, run() computes an operator in its plain form, elementary torch operations in 32 bits (the stored
numbers in 64: a quotient near the border of two of them); with `own` true it makes the calls a user of fyodor_b200
makes. Geometries (32/8, 64/8, 16/2 and 8/8 heads of 64 or 128, contexts to 32768, batches of 16 and 32, drafts of 8, a
vocabulary of 128256) are those of the package's tests and benchmark.

K is rotated in 32 bits, each product and sum rounded. A group is held as value = low + scale * n, n = 0..15: low and
high are the group's least and greatest finite value (at most 61440 in magnitude) rounded to 16 bits, scale is
(high - low) / 15 rounded to 16 bits, n is (x - low) / scale rounded to nearest, ties to even. A token's row of one
head is packed eight values to a 32-bit word, the first in the lowest bits; with heads of 128 the words of the two
groups take turns."""
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
WIDTH = {"f32": 4, "f16": 2, "bf16": 2}
GROUP = 64        # values that share a scale and a low
MOST = 61440.0    # largest magnitude held
#: (query heads, KV heads, head dimension)
GEOMETRY = {"32/8x128": (32, 8, 128), "64/8x128": (64, 8, 128), "16/2x64": (16, 2, 64), "8/8x128": (8, 8, 128),
            "32/8x64": (32, 8, 64)}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the cache rows of one decode step of 16 sequences, rotated on the way: latency is all there is
        {"name": "append step of 16, rotated", "op": "append", "requests": 16, "most": 768, "new": 1,
         "geometry": "32/8x128", "type": "f32", "block": 16, "rope": True, "fused": True, "pick": 1},
        # drafts of up to 8 tokens of 32 sequences, heads of 64
        {"name": "append drafts of 8", "op": "append", "requests": 32, "most": 4000, "new": 8, "geometry": "16/2x64",
         "type": "f16", "block": 32, "rope": False, "fused": False, "pick": 2},
        # prompts of four requests
        {"name": "append 4 prompts of to 2100, rotated", "op": "append", "requests": 4, "most": 0, "new": 2100,
         "geometry": "32/8x128", "type": "bf16", "block": 64, "rope": True, "fused": True, "pick": 3},
        # one sequence a little into its context
        {"name": "attention one of 257", "op": "attention", "requests": 1, "least": 257, "most": 257, "new": 1,
         "geometry": "32/8x128", "type": "f32", "block": 16, "fused": False, "pick": 4},
        # the ragged decode batch of the benchmark
        {"name": "attention ragged 32 to 32768", "op": "attention", "requests": 32, "least": 128, "most": 32768,
         "new": 1, "geometry": "32/8x128", "type": "f32", "block": 64, "fused": False, "pick": 5},
        # the same batch checking drafts of up to 8 tokens
        {"name": "attention drafts of 8, ragged 32", "op": "attention", "requests": 32, "least": 128, "most": 32768,
         "new": 8, "geometry": "32/8x128", "type": "bf16", "block": 64, "fused": True, "pick": 6},
        # sixteen sequences of a 64/8-head model near 8192 positions
        {"name": "attention 16 at 8100, 64 heads", "op": "attention", "requests": 16, "least": 7800, "most": 8192,
         "new": 1, "geometry": "64/8x128", "type": "f16", "block": 32, "fused": True, "pick": 7},
        # a prompt chunk of 500 tokens behind a long context
        {"name": "attention chunk of 500 at 16000", "op": "attention", "requests": 1, "least": 16001, "most": 16001,
         "new": 500, "geometry": "32/8x128", "type": "bf16", "block": 128, "fused": False, "pick": 8},
        # the tokens that one decode step of 16 sequences chose, five alternatives each
        {"name": "logprobs step of 16", "op": "logprobs", "rows": 16, "vocabulary": 128256, "type": "f32", "top": 5,
         "pad": 0, "suppressed": True, "pick": 9},
        # a draft of 5 tokens, a small vocabulary of odd size in rows of odd stride
        {"name": "logprobs draft of 5, odd vocabulary", "op": "logprobs", "rows": 5, "vocabulary": 32003,
         "type": "f16", "top": 1, "pad": 6, "suppressed": False, "pick": 10},
        # the loss of a text of 1000 tokens
        {"name": "logprobs text of 1000", "op": "logprobs", "rows": 1000, "vocabulary": 128256, "type": "bf16",
         "top": 0, "pad": 0, "suppressed": False, "pick": 11},
        # a prompt of 400 tokens scored with 20 alternatives
        {"name": "logprobs prompt of 400, top 20", "op": "logprobs", "rows": 400, "vocabulary": 128256, "type": "f32",
         "top": 20, "pad": 64, "suppressed": True, "pick": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["append", "append", "attention", "attention", "attention", "logprobs", "logprobs"])
    pick, block = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128])
    geometry, type_ = rng.choice(sorted(GEOMETRY)), rng.choice(sorted(TYPES))
    if op == "logprobs":
        vocabulary = rng.choice([128256, _log_int(rng, 300, 128256)])
        return {"op": op, "rows": _log_int(rng, 1, 1000 if WIDTH[type_] == 2 else 400), "vocabulary": vocabulary,
                "type": type_, "top": rng.choice([0, 1, rng.randint(2, 20)]), "pad": rng.choice([0, 0, 5, 64]),
                "suppressed": rng.random() < 0.5, "pick": pick}
    if op == "append":
        n = _log_int(rng, 1, 64)
        return {"op": op, "requests": n, "most": rng.choice([0, _log_int(rng, 1, 4000)]),
                "new": _log_int(rng, 1, max(1, min(2100, 8400 // n))), "geometry": geometry, "type": type_,
                "block": block, "rope": rng.random() < 0.5, "fused": rng.random() < 0.5, "pick": pick}
    heads, kv, hd = GEOMETRY[geometry]
    new = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 500)])
    n = _log_int(rng, 1, 64 if new <= 16 else 4)
    most = _log_int(rng, 1, min(32768, (1 << 20) // n, (1 << 28) // (n * new * heads)))
    return {"op": op, "requests": n, "least": _log_int(rng, 1, most), "most": most, "new": min(new, most),
            "geometry": geometry, "type": type_, "block": block, "fused": rng.random() < 0.5, "pick": pick}


def _shape(case):
    """Lengths and new rows of a case's requests: plain numbers that follow from the case alone."""
    r, n = random.Random(case["pick"]), case["requests"]
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
    w = WIDTH[case["type"]]
    if case["op"] == "logprobs":
        rows, values = case["rows"], case["rows"] * case["vocabulary"]
        return {"bytes": w * values + rows * (16 + 8 * case["top"]), "flops": 5 * values}
    heads, kv, hd = GEOMETRY[case["geometry"]]
    token = kv * (hd // 2 + hd // GROUP * 4)  # bytes of K or of V of a token
    cached, new = _shape(case)
    rows = sum(new)
    if case["op"] == "append":
        traffic = 2 * w * rows * kv * hd + 2 * rows * token + 4 * rows  # rows in, held out
        traffic += 2 * rows * token + 2 * 4 * rows * kv * hd + 4 * rows  # read back: held in, values out
        flops = 8 * rows * kv * hd
        if case["rope"]:
            traffic += 2 * w * rows * heads * hd + rows * (4 + 4 * hd)
            flops += 3 * rows * (heads + kv) * hd
        return {"bytes": traffic, "flops": flops}
    total = sum(c + m for c, m in zip(cached, new))
    attended = sum(m * c + m * (m + 1) // 2 for c, m in zip(cached, new))
    blocks = sum(_ceil(c + m, case["block"]) for c, m in zip(cached, new))
    return {"bytes": 2 * total * token + 4 * blocks + 2 * w * rows * heads * hd + 8 * len(cached),
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


def _rope_tables(dims, context):
    """cos and sin of position x frequency, the frequencies halved for the slow half as a long-context model does."""
    f = 500000.0 ** (-np.arange(dims // 2) / (dims // 2))
    f[dims // 4:] /= 2.0
    angle = torch.arange(context, device=DEV, dtype=torch.float64)[:, None] * torch.tensor(f, device=DEV)
    return angle.cos().float(), angle.sin().float()


def _pool(g, blocks, case):
    """A cache of `blocks` blocks filled with quantised rows, made in pieces."""
    kv, hd = GEOMETRY[case["geometry"]][1:]
    out = []
    for strong in (4.0, 1.0):
        held = torch.empty((blocks, kv, case["block"], hd // 2), dtype=torch.uint8, device=DEV)
        scale = torch.empty((blocks, kv, case["block"], hd // GROUP, 2), dtype=torch.float16, device=DEV)
        step = max(1, (1 << 26) // (2 * held[0].numel()))
        for b in range(0, blocks, step):
            x = torch.randn((*held[b:b + step].shape[:3], hd), generator=g, device=DEV)
            x[..., :: hd // 4] *= strong
            held[b:b + step], scale[b:b + step] = _hold(x)
        out += [held, scale]
    return out[0], out[2], out[1], out[3]


def _tables(g, counts, blocks):
    """Block tables of requests whose blocks lie in any order in the pool (-1 where a request has none)."""
    order = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    counts = torch.tensor(counts, device=DEV)
    width = max(1, int(counts.max()))
    at = torch.arange(width, device=DEV)[None] + (counts.cumsum(0) - counts)[:, None]
    has = torch.arange(width, device=DEV)[None] < counts[:, None]
    return torch.where(has, order[at.clamp(max=blocks - 1)], torch.full_like(order[:1], -1))


def _logits(g, case):
    """Rows of logits as a model gives them, most of a row's weight on some fifty tokens, and the tokens asked for."""
    rows, n = case["rows"], case["vocabulary"]
    wide = torch.empty((rows, n + case["pad"]), dtype=TYPES[case["type"]], device=DEV)
    step = max(1, (1 << 26) // n)
    likely = torch.randint(0, n, (rows, 50), generator=g, device=DEV)
    for r in range(0, rows, step):
        x = 2.0 * torch.randn((len(likely[r:r + step]), n), generator=g, device=DEV)
        x.scatter_add_(1, likely[r:r + step], 7.0 + 3.0 * torch.randn(likely[r:r + step].shape, generator=g, device=DEV))
        wide[r:r + step, :n] = x.to(wide.dtype)
    wide[:, n:] = torch.nan  # behind a row's end lies anything
    if case["suppressed"]:
        wide[:, 7:n:1009] = -torch.inf  # tokens that may not be answered
    some = torch.rand(rows, generator=g, device=DEV) < 0.6
    tokens = torch.where(some, likely[:, 0], torch.randint(0, n, (rows,), generator=g, device=DEV))
    return wide[:, :n], tokens.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "logprobs":
        s["logits"], s["tokens"] = _logits(g, case)
        rows, top = case["rows"], case["top"]
        s["logprob"], s["entropy"] = (torch.empty(rows, device=DEV) for _ in range(2))
        s["rank"] = torch.empty(rows, dtype=torch.int32, device=DEV)
        s["top_tokens"] = torch.empty((rows, top), dtype=torch.int32, device=DEV)
        s["top_logprobs"] = torch.empty((rows, top), device=DEV)
        return s
    cached, new = _shape(case)
    block, rows = case["block"], sum(new)
    lengths, fresh = _ints(cached), _ints(new)
    counts = [_ceil(c + m, block) for c, m in zip(cached, new)]
    blocks = sum(counts) + 3
    s["table"] = _tables(g, counts, blocks)
    s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = _pool(g, blocks, case)
    s["q"], s["k"], s["v"] = _rows(g, rows, case)
    s["row_start"], s["lengths"] = _starts(new), lengths + fresh
    heads, kv, hd = GEOMETRY[case["geometry"]]
    if case["op"] == "attention":
        s["out"] = torch.empty((rows, heads, hd), dtype=TYPES[case["type"]], device=DEV)
        s["most_rows"], s["scale"] = max(new), hd ** -0.5
        if case["new"] == 1:
            s["row_start"] = None
        return s
    end = [c + m for c, m in zip(cached, new)]
    s["positions"] = _ints([t for a, b in zip(cached, end) for t in range(a, b)])
    who = _ints([i for i, (a, b) in enumerate(zip(cached, end)) for _ in range(a, b)]).long()
    s["slots"] = s["table"][who, (s["positions"] // block).long()] * block + s["positions"] % block
    if case["rope"]:
        s["cos"], s["sin"] = _rope_tables(hd, max(end))
        s["q_out"] = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=DEV)
    s["k_held"], s["v_held"] = (torch.empty((rows, kv, hd), device=DEV) for _ in "kv")
    return s


# ---------------------------------------------------------------- plain forms
def _hold(x):
    """Rows [..., hd] of 32 bits as they are held: bytes [..., hd / 2], scale and low [..., hd / 64, 2]."""
    hd = x.shape[-1]
    group = x.unflatten(-1, (hd // GROUP, GROUP))
    low, high = (f(-1).clamp(-MOST, MOST).half() for f in (group.amin, group.amax))
    scale = ((high.double() - low.double()) / 15.0).half()
    unit = scale.double()[..., None]
    n = torch.where(unit > 0, (group.double() - low.double()[..., None]) / unit, 0.0).round().clamp(0, 15).to(torch.uint8)
    n = n.unflatten(-1, (8, 8)).transpose(-3, -2).flatten(-3)  # the groups' words take turns
    return n[..., 0::2] | n[..., 1::2] << 4, torch.stack([scale, low], -1)


def _values(held, scale):
    """What held rows stand for, in 32 bits."""
    groups = scale.shape[-2]
    n = torch.stack([held & 15, held >> 4], -1).flatten(-2)
    n = n.unflatten(-1, (8, groups, 8)).transpose(-3, -2).flatten(-2).float()
    scale = scale.float()
    return (scale[..., 1:] + scale[..., :1] * n).flatten(-2)


def _rotate(x, cos, sin):
    """x [rows, heads, hd] in 32 bits, its interleaved pairs rotated."""
    a, b, c, z = x[..., 0::2], x[..., 1::2], cos[:, None], sin[:, None]
    return torch.stack([a * c - b * z, a * z + b * c], -1).flatten(-2)


def _plain_append(s):
    r, k, block = {}, s["k"].float(), s["case"]["block"]
    slots = s["slots"].long()
    if s["case"]["rope"]:
        at = s["positions"].long()
        cos, sin = s["cos"][at], s["sin"][at]
        k = _rotate(k, cos, sin)
        r["q"] = _rotate(s["q"].float(), cos, sin).to(s["q"].dtype)
    for name, x in (("k", k), ("v", s["v"].float())):
        held, scale = s[name + "_cache"], s[name + "_scale"]
        held[slots // block, :, slots % block], scale[slots // block, :, slots % block] = _hold(x)
        r[name] = _values(held[slots // block, :, slots % block], scale[slots // block, :, slots % block])
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

    def whole(held, scale):
        x = _values(held[table], scale[table]).permute(0, 2, 1, 3, 4).reshape(n, kv, width, hd)
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


def _plain_logprobs(s):
    x, top, n = s["logits"].float(), s["case"]["top"], s["case"]["vocabulary"]
    index = torch.arange(n, device=DEV)
    token = s["tokens"].long()[:, None]
    peak = x.amax(1, keepdim=True)
    shifted = x - peak
    e = shifted.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    given = x.gather(1, token)
    before = (x > given) | ((x == given) & (index[None] < token))
    r = {"logprob": (given - peak - log_total)[:, 0],
         "entropy": (log_total - torch.where(e > 0, e * shifted, 0.0).sum(1, keepdim=True) / total)[:, 0],
         "rank": before.sum(1).to(torch.int32)}
    # greatest first, of equal ones the first: keys of 64 bits, no two alike
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32 | (n - 1 - index)[None]
    best = n - 1 - (key.topk(min(top, n), 1).values & 0xFFFFFFFF)
    values = x.gather(1, best)
    r["top_tokens"] = torch.where(values > -torch.inf, best, -1).to(torch.int32)
    r["top_logprobs"] = values - peak - log_total
    return r


# ---------------------------------------------------------------- the framework's operators
def _cache(s):
    """The cache handle that a serving program keeps."""
    if "cache" not in s:
        import fyodor_b200 as F
        s["cache"] = F.KV4Cache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    return s["cache"]


def _own_append(s):
    cache, r = _cache(s), {}
    if s["case"]["rope"]:
        cache.append(s["k"], s["v"], s["slots"], positions=s["positions"], cos=s["cos"], sin=s["sin"],
                     layout="interleaved", q=s["q"], q_out=s["q_out"])
        r["q"] = s["q_out"]
    else:
        cache.append(s["k"], s["v"], s["slots"])
    cache.read(s["slots"], s["k_held"], s["v_held"])
    return r | {"k": s["k_held"], "v": s["v_held"]}


def _own_attention(s):
    cache = _cache(s)
    if "workspace" not in s:
        s["workspace"] = cache.attention_workspace(len(s["lengths"]), s["most_rows"], s["q"].shape[1])
    cache.attention(s["q"], s["lengths"], s["table"], s["out"], s["workspace"], row_start=s["row_start"],
                    most_rows=s["most_rows"], scale=s["scale"])
    return s["out"]


def _own_logprobs(s):
    import fyodor_b200 as F
    if "workspace" not in s:
        s["workspace"] = F.logprobs_workspace(s["case"]["rows"], s["case"]["vocabulary"], s["case"]["top"])
    F.logprobs(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["rank"], s["top_tokens"], s["top_logprobs"],
               s["workspace"])
    return {x: s[x] for x in ("logprob", "entropy", "rank", "top_tokens", "top_logprobs")}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "logprobs": _own_logprobs}[op](state)
    return {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[op](state)


# ---------------------------------------------------------------- in 64 bits
def _exact_turn(x, cos, sin):
    y = x.double().clone()
    z = torch.complex(y[..., 0::2].contiguous(), y[..., 1::2].contiguous()) * torch.complex(cos.double(), sin.double())[:, None]
    y[..., 0::2], y[..., 1::2] = z.real, z.imag
    return y


def _exact_held(x):
    """The values that rows [rows, heads, hd] are held as: by counting the borders below each."""
    x = x.double().cpu().numpy()
    out = np.empty_like(x)
    for h in range(0, x.shape[-1], GROUP):
        part = x[..., h:h + GROUP]
        low = np.clip(part.min(-1), -MOST, MOST).astype(np.float16).astype(np.float64)[..., None]
        high = np.clip(part.max(-1), -MOST, MOST).astype(np.float16).astype(np.float64)[..., None]
        unit = ((high - low) / 15).astype(np.float16).astype(np.float64)
        above, n = part - low, np.zeros(part.shape)
        for k in range(15):
            border = (2 * k + 1) * unit / 2
            n += (above > border) | ((above == border) & (k % 2 == 1))
        out[..., h:h + GROUP] = low + unit * np.where(unit > 0, n, 0)
    return torch.from_numpy(out)


def _exact_append(s):
    out, k = {}, s["k"].double()
    if s["case"]["rope"]:
        at = s["positions"].long()
        # what is held is K as rotated in 32 bits, each product and sum rounded: numbers of 4 bits follow from it
        k, cos, sin = (t.float().cpu().numpy() for t in (s["k"], s["cos"][at], s["sin"][at]))
        x, y, turned = k[..., 0::2], k[..., 1::2], np.empty_like(k)
        turned[..., 0::2] = x * cos[:, None] - y * sin[:, None]
        turned[..., 1::2] = x * sin[:, None] + y * cos[:, None]
        k = torch.from_numpy(turned)
        out["q"] = _exact_turn(s["q"], s["cos"][at], s["sin"][at])
    return out | {"k": _exact_held(k), "v": _exact_held(s["v"])}


def _exact_rows(s, name, r, blocks):
    """K or V of the first `blocks` blocks of request r in 64 bits: [kv, tokens, hd], word by word."""
    use = s["table"][r, :blocks].long()
    held, scale = s[name + "_cache"][use].transpose(0, 1).flatten(1, 2), s[name + "_scale"][use].transpose(0, 1).flatten(1, 2)
    groups = scale.shape[2]
    x = torch.empty((*held.shape[:2], 2 * held.shape[2]), dtype=torch.float64, device=DEV)
    for word in range(held.shape[2] // 4):
        h, j = word % groups, word // groups
        for byte in range(4):
            b = held[..., 4 * word + byte].int()
            e = GROUP * h + 8 * j + 2 * byte
            x[..., e] = scale[:, :, h, 1].double() + scale[:, :, h, 0].double() * (b % 16)
            x[..., e + 1] = scale[:, :, h, 1].double() + scale[:, :, h, 0].double() * (b // 16)
    return x


def _exact_attention(s):
    block = s["case"]["block"]
    heads, kv, hd = GEOMETRY[s["case"]["geometry"]]
    n = len(s["lengths"])
    start = list(range(n + 1)) if s["row_start"] is None else s["row_start"].tolist()
    out = torch.zeros((len(s["q"]), heads, hd), dtype=torch.float64, device=DEV)
    for r, length in enumerate(s["lengths"].tolist()):
        k, v = (_exact_rows(s, x, r, _ceil(length, block))[:, :length] for x in "kv")
        rows = start[r + 1] - start[r]
        last = length - rows + torch.arange(rows, device=DEV)
        hidden = torch.arange(length, device=DEV)[None] > last[:, None]
        for h in range(heads):
            score = (s["q"][start[r]:start[r + 1], h].double() @ k[h // (heads // kv)].t()) * s["scale"]
            p = torch.softmax(score.masked_fill(hidden, -torch.inf), -1)
            out[start[r]:start[r + 1], h] = torch.nan_to_num(p, nan=0.0) @ v[h // (heads // kv)]
    return out


def _exact_logprobs(s):
    r = {"logprob": [], "entropy": [], "rank": None, "top_tokens": None, "top_logprobs": []}
    for row, token in zip(s["logits"], s["tokens"].tolist()):
        log_p = torch.log_softmax(row.double(), 0)
        p = log_p.exp()
        r["logprob"].append(log_p[token])
        r["entropy"].append(-torch.where(p > 0, p * log_p, 0.0).sum())
        r["top_logprobs"].append(log_p.sort(descending=True).values[:s["case"]["top"]])
    return {name: v if v is None else torch.stack(v) for name, v in r.items()}


def exact(case, seed):
    """run()'s outputs from the operators' definitions in 64 bits; None in the place of whole numbers."""
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["op"]](s)
