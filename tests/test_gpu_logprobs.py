"""GPU tests of the log probabilities against their definition in 64 bits; whole
numbers (ranks, alternatives) exactly.

Tolerances: with d = x - max, an exponential of F32 is within 2 units (2^-22)
and moves by |d| 2^-24 with the rounding of d, a sum of n of them in 256 parts or
more by (n / 256 + 32) 2^-24: the sum S is off by r = 2^-21 + E|d| 2^-24 + (n /
256 + 32) 2^-24 of itself. ln S then by r + |ln S| 2^-22, a log probability by
that and |d| 2^-23; the entropy ln S - E d by r (1 + 2 E|d|) + E(d^2) 2^-24 + (|ln
S| + E|d|) 2^-22."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(v):
    return torch.tensor(np.asarray(v, np.int64).astype(np.int32), device="cuda")


def outputs(rows, top):
    return dict(logprob=torch.full((rows,), 77.0, device="cuda"), entropy=torch.full((rows,), 77.0, device="cuda"),
                rank=i32([77] * rows), top_tokens=torch.full((rows, top), 77, dtype=torch.int32, device="cuda"),
                top_logprobs=torch.full((rows, top), 77.0, device="cuda"))


def check(x, tokens, top, error=0, ws=None):
    """One call against the definition; x [rows][n] on the GPU."""
    rows, n = x.shape
    out, err = outputs(rows, top), i32([0])
    ws = F.logprobs_workspace(rows, n, top) if ws is None else ws
    F.logprobs(x, i32(tokens), workspace=ws, error=err, **out)
    assert err.item() == error
    again = outputs(rows, top)
    F.logprobs(x, i32(tokens), workspace=ws, **again)  # the workspace is left as it has to be
    assert all(torch.equal(out[k].view(torch.int32), again[k].view(torch.int32)) for k in out)
    got = {k: v.cpu().numpy() for k, v in out.items()}
    for r in range(rows):
        v = x[r].double().cpu().numpy()
        bad, t = bool(np.isnan(v).any() or (v == np.inf).any()), tokens[r]
        fine = np.where(np.isnan(v), -np.inf, v)
        order = np.argsort(-fine, kind="stable")[:top]
        order = [int(i) for i in order if fine[i] > -np.inf]
        assert got["top_tokens"][r].tolist() == order + [-1] * (top - len(order)), r
        if not 0 <= t < n:
            assert got["logprob"][r] == 0 and got["rank"][r] == -1
        elif not np.isnan(v[t]):
            assert got["rank"][r] == (fine > v[t]).sum() + ((v == v[t]) & (np.arange(n) < t)).sum()
        if bad:
            assert np.isnan(got["entropy"][r]) and np.isnan(got["top_logprobs"][r]).all()
            assert not 0 <= t < n or np.isnan(got["logprob"][r])
            continue
        if (v == -np.inf).all():
            assert got["entropy"][r] == 0 and (got["top_logprobs"][r] == -np.inf).all()
            assert not 0 <= t < n or got["logprob"][r] == -np.inf
            continue
        d = v - v.max()
        e = np.exp(d)
        s = e.sum()
        near = np.where(e > 0, d, 0.0)
        mean, square = (e * np.abs(near)).sum() / s, (e * near * near).sum() / s
        rel = 2.0 ** -21 + mean * 2.0 ** -24 + (n / 256 + 32) * 2.0 ** -24
        ln = np.log(s)
        far = lambda d: rel + ln * 2.0 ** -22 + np.abs(d) * 2.0 ** -23  # noqa: E731
        if 0 <= t < n:
            assert got["logprob"][r] == -np.inf if v[t] == -np.inf else abs(got["logprob"][r] - (d[t] - ln)) <= far(d[t]), r
        assert abs(got["entropy"][r] - (ln + mean)) <= rel * (1 + 2 * mean) + square * 2.0 ** -24 + (ln + mean) * 2.0 ** -22, r
        assert (np.abs(got["top_logprobs"][r][:len(order)] - (d[order] - ln)) <= far(d[order])).all(), r
        assert (got["top_logprobs"][r][len(order):] == -np.inf).all()
    return got


def some(rows, n, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = spread * torch.randn(rows, n, generator=g, device="cuda")
    t = torch.randint(0, n, (rows,), generator=g, device="cuda").tolist()
    return x, t


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("rows,n,top", [(1, 1, 0), (2, 1, 3), (1, 2, 1), (3, 7, 32), (5, 31, 5), (4, 33, 32), (1, 255, 1),
                                        (7, 1000, 20), (2, 4097, 8), (1, 128256, 5), (16, 128256, 20), (37, 32003, 2),
                                        (300, 513, 32), (1500, 129, 1), (149, 9001, 0)])
def test_shapes(kind, rows, n, top):
    x, t = some(rows, n, rows + n)
    check(x.to(TYPES[kind]), t, top)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("pad,off", [(1, 0), (3, 1), (8, 2), (5, 3), (64, 0)])
def test_strides_and_alignment(kind, pad, off):
    """Rows that begin on any element; what lies between them (NaN, the largest number) is not looked at."""
    rows, n = 9, 5003
    x, t = some(rows, n, pad)
    wide = torch.full((rows, n + pad + off), float("nan"), dtype=TYPES[kind], device="cuda")
    wide[:, ::2] = torch.finfo(TYPES[kind]).max
    wide[:, off:off + n] = x.to(TYPES[kind])
    check(wide[:, off:off + n], t, 5)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_masks(kind):
    """Suppressed tokens: some, all but one, all; as the given token; the type's lowest value as a mask."""
    rows, n = 12, 3001
    x, t = some(rows, n, 5)
    x = x.to(TYPES[kind])
    x[0, ::3] = -torch.inf
    x[1] = -torch.inf
    x[2] = -torch.inf
    x[2, 17] = -3.0
    t[2] = 17
    x[3, :2999] = -torch.inf
    t[3] = 5
    x[4] = torch.finfo(x.dtype).min
    x[5, 1:] = torch.finfo(x.dtype).min
    t[5] = 0
    x[6, 100:] = -torch.inf
    x[7, :-1] = -torch.inf
    x[8] = 0.0
    x[8, ::2] = -0.0  # all equal, whatever the zero's sign
    x[9] = torch.finfo(x.dtype).max
    x[10, 5] = torch.finfo(x.dtype).max
    check(x, t, 20)
    check(x, t, 0)
    check(x[:, :1], [0] * rows, 2)


def test_values_that_are_no_numbers():
    for kind in TYPES:
        x, t = some(6, 2500, 8)
        x = x.to(TYPES[kind])
        x[0, 2000] = torch.nan
        x[1, 3] = torch.inf
        x[2] = torch.nan
        x[3, t[3]] = torch.nan
        x[4, 7], x[4, 9] = -torch.inf, torch.inf
        check(x, t, 4, error=2)


def test_ties_and_order():
    """Many equal logits: the first of them come first, at every place of the row."""
    x, t = some(8, 20011, 3)
    check(x.round(), t, 32)
    check(torch.zeros_like(x), t, 32)
    check((x * 40).round().to(torch.float16), t, 7)
    y = torch.arange(20011, device="cuda", dtype=torch.float32)[None].repeat(3, 1)
    check(y * 0.01, [0, 20010, 77], 32)       # rising: every logit is the best so far
    check(-y * 0.01, [0, 20010, 77], 32)
    check(y.remainder(3), [0, 1, 2], 32)
    x[:, -1] = 50.0
    x[:, 0] = 50.0
    check(x, t, 3)


def test_peaked_and_far_rows():
    x, t = some(6, 30000, 4)
    x[0, 9] = 60.0
    x[1] *= 100
    x[2] += 1e4
    x[3] -= 3e38
    x[4] *= 1e-6
    check(x, [9, 5, 0, 3, 1, 7], 5)


def test_tokens_left_out():
    """Negative tokens ask for nothing; one past the vocabulary is taken so and raises 4."""
    x, t = some(5, 700, 2)
    check(x, [3, -1, -2 ** 31, 699, 0], 2)
    check(x, [3, 700, 2 ** 31 - 1, 699, 0], 2, error=4)


def test_outputs_left_out_and_refusals():
    x, t = some(4, 900, 6)
    full, ws = outputs(4, 3), F.logprobs_workspace(4, 900, 3)
    F.logprobs(x, i32(t), workspace=ws, **full)
    for drop in (["rank"], ["entropy"], ["top_tokens", "top_logprobs"], ["rank", "entropy"]):
        out = {k: None if k in drop else v for k, v in outputs(4, 3).items()}
        F.logprobs(x, i32(t), workspace=ws, **out)
        assert all(v is None or torch.equal(v, full[k]) for k, v in out.items())
    out = outputs(4, 3)
    F.logprobs(x, None, None, out["entropy"], None, out["top_tokens"], out["top_logprobs"], ws)
    assert torch.equal(out["entropy"], full["entropy"]) and torch.equal(out["top_tokens"], full["top_tokens"])
    assert (out["logprob"] == 77).all()
    good = dict(logits=x, tokens=i32(t), workspace=ws) | outputs(4, 3)
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.t()), dict(tokens=i32(t[:3])),
                dict(tokens=i32(t).long()), dict(tokens=None), dict(logprob=None), dict(logprob=good["logprob"][:3]),
                dict(entropy=good["entropy"].half()), dict(top_logprobs=None), dict(top_logprobs=good["top_logprobs"][:, :2]),
                dict(workspace=ws[:16]), dict(workspace=ws[1:]), dict(logits=x.cpu()), dict(logits=x[:1].expand(4, 900)),
                dict(top_tokens=torch.zeros((4, 33), dtype=torch.int32, device="cuda"),
                     top_logprobs=torch.zeros((4, 33), device="cuda"))):
        with pytest.raises(ValueError):
            F.logprobs(**(good | bad))
    none = {k: v[:0] for k, v in outputs(1, 3).items()}
    F.logprobs(x[:0], i32([]), workspace=ws, **none)


@pytest.mark.parametrize("rows,n,top", [(1, 140000, 3), (1, 300001, 8), (1, 300001, 9), (2, 200001, 32), (1, 2000000, 5)])
def test_rows_of_many_ctas(rows, n, top):
    """More than 32 CTAs hold a part of a row, with alternatives of both forms of the join; then a row whose largest
    logits ascend to its end, so every batch holds new ones."""
    x, t = some(rows, n, rows + n)
    check(x, t, top)
    check(x.sort(1).values, t, top)


def test_streams_and_graph():
    """On another stream behind work of its own, twice at once with a workspace each, and captured."""
    x, t = some(16, 50000, 7)
    t = i32(t)
    want, ws = outputs(16, 5), F.logprobs_workspace(16, 50000, 5)
    F.logprobs(x, t, workspace=ws, **want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = outputs(16, 5)
    with torch.cuda.stream(s):
        y = torch.zeros_like(x)
        for _ in range(50):
            y.add_(1.0)
        y.copy_(x)
        F.logprobs(y, t, workspace=ws, **out)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(out[k], want[k]) for k in out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces, outs = [F.logprobs_workspace(16, 50000, 5) for _ in streams], [outputs(16, 5) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, w, o in zip(streams, spaces, outs):
            F.logprobs(x, t, workspace=w, stream=st.cuda_stream, **o)
    torch.cuda.synchronize()
    assert all(torch.equal(o[k], want[k]) for o in outs for k in o)
    graph, out = torch.cuda.CUDAGraph(), outputs(16, 5)
    with torch.cuda.graph(graph):
        F.logprobs(y, t, workspace=ws, **out)
    y.zero_()
    graph.replay()
    y.copy_(x)
    graph.replay()
    assert all(torch.equal(out[k], want[k]) for k in out)
