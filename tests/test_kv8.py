"""The paged 8-bit KV cache on the host side: rotary frequencies against their
formulas in 64 bits, and the refusals of every entry point (arguments are
checked before anything reaches a device, so no GPU is needed)."""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

BUF = np.zeros(4096, np.float32)
P = C.c_void_p((BUF.ctypes.data + 255) // 256 * 256)  # never read: every call below is refused or empty
ODD = C.c_void_p(P.value + 4)


def plain(dims, base):
    return base ** (-np.arange(dims // 2) / (dims // 2))


# F32 powf is within 2 ulp; everything else is rounded once from 64 bits
def close(a, b):
    return np.all(np.abs(a - b) <= 3e-7 * np.abs(b))


def test_frequencies_plain_linear_ntk():
    assert close(F.rope_frequencies(128, 500000.0)[0], plain(128, 500000.0))
    assert F.rope_frequencies(128, 500000.0)[1] == 1.0
    assert close(F.rope_frequencies(64, 10000.0, "linear", 4.0)[0], plain(64, 10000.0) / 4)
    assert close(F.rope_frequencies(64, 10000.0, "ntk", 8.0)[0], plain(64, 10000.0 * 8 ** (64 / 62)))
    factors = np.linspace(1, 8, 32).astype(np.float32)
    assert close(F.rope_frequencies(64, 10000.0, factors=factors)[0], plain(64, 10000.0) / factors)


def test_frequencies_plain_are_the_engines():
    """Bit for bit powf(base, -j / pairs), what a plan's own tables are made of."""
    libm = C.CDLL("libm.so.6")
    libm.powf.restype, libm.powf.argtypes = C.c_float, [C.c_float, C.c_float]
    want = [libm.powf(500000.0, -float(np.float32(j) / np.float32(64))) for j in range(64)]
    assert (F.rope_frequencies(128, 500000.0)[0] == np.array(want, np.float32)).all()


def test_frequencies_yarn():
    dims, base, factor, ctx = 128, 10000.0, 16.0, 4096.0
    got, mag = F.rope_frequencies(dims, base, "yarn", factor, ctx)
    f, j = plain(dims, base), np.arange(64)
    pair = lambda turns: 64 * np.log(ctx / (turns * 2 * np.pi)) / np.log(base)  # noqa: E731
    lo, hi = np.floor(pair(32.0)), np.ceil(pair(1.0))
    ramp = np.clip((j - lo) / (hi - lo), 0, 1)
    assert close(got, f / factor * ramp + f * (1 - ramp))
    assert abs(mag - (0.1 * np.log(factor) + 1)) < 1e-6
    assert got[0] == 1.0 and abs(got[-1] * factor / f[-1] - 1) < 1e-6  # fast pairs kept, slow ones divided


def test_frequencies_bands():
    base, factor, ctx, low, high = 500000.0, 8.0, 8192.0, 1.0, 4.0
    got = F.rope_frequencies(128, base, "bands", factor, ctx, low_freq=low, high_freq=high)[0]
    f = plain(128, base)
    wave = 2 * np.pi / f
    want = np.where(wave < ctx / high, f, f / factor)
    smooth = (ctx / wave - low) / (high - low)
    mid = (wave >= ctx / high) & (wave <= ctx / low)
    want = np.where(mid, (1 - smooth) * f / factor + smooth * f, want)
    assert mid.any() and close(got, want)


@pytest.mark.parametrize("bad", [dict(dims=63), dict(dims=0), dict(base=0.0), dict(base=float("nan")),
                                 dict(kind="linear", factor=0.5), dict(kind="yarn", factor=4.0),
                                 dict(kind="bands", factor=4.0, original_context=8192.0, low_freq=4.0, high_freq=1.0),
                                 dict(dims=2, kind="ntk", factor=2.0), dict(kind="other"),
                                 dict(factors=np.zeros(32)), dict(factors=np.ones(31))])
def test_frequencies_refuse(bad):
    with pytest.raises(ValueError):
        F.rope_frequencies(**{"dims": 64, "base": 10000.0, **bad})


def desc(**kw):
    d = dict(k=P.value, v=P.value, k_scale=P.value, v_scale=P.value, blocks=4, kv_heads=2, block_size=16, head_dim=64,
             format=0) | kw
    return F.KV8CacheDesc(**d)


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=ODD.value), dict(blocks=0),
              dict(kv_heads=0), dict(block_size=8), dict(block_size=48), dict(block_size=512), dict(head_dim=96),
              dict(format=2), dict(blocks=1 << 27)]


def rope_desc(**kw):
    return F.RopeDesc(**(dict(cos_table=P.value, sin_table=P.value, table_rows=8, dims=64, layout=0) | kw))


BAD_ROPES = [dict(cos_table=None), dict(sin_table=None), dict(table_rows=0), dict(dims=0), dict(dims=7),
             dict(dims=66), dict(layout=2)]


def append(cache, rows=1, type_=0, k=P, ks=128, v=P, vs=128, rope=None, pos=P, q=None, qs=0, qo=None, qos=0, heads=0,
           slots=P):
    return F.lib.fyb_kv8_append(C.byref(cache) if cache else None, slots, rows, type_, k, ks, v, vs,
                                C.byref(rope) if rope else None, pos, q, qs, qo, qos, heads, None, None)


def attention(cache, n=1, most=1, rows=1, stride=1, type_=0, q=P, qs=256, out=P, os_=256, heads=4, ws=P, wb=1 << 40,
              lengths=P, table=P, starts=None):
    return F.lib.fyb_kv8_attention(C.byref(cache) if cache else None, lengths, starts, n, most, rows, table, stride,
                                   type_, q, qs, out, os_, heads, 0.1, ws, wb, None, None)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_cache_refused(bad):
    c = desc(**bad)
    assert append(c) == -1
    assert attention(c) == -1
    assert F.lib.fyb_kv8_read(C.byref(c), P, 1, P, P, None, None) == -1


def test_append_refuses():
    c = desc()
    assert append(None) == -1
    for kw in (dict(k=None), dict(v=None), dict(ks=127), dict(vs=127), dict(type_=8), dict(type_=2), dict(slots=None),
               dict(heads=4), dict(rope=rope_desc(), pos=None), dict(rope=rope_desc(), heads=4, q=P, qs=256),
               dict(rope=rope_desc(), heads=4, q=P, qs=255, qo=P, qos=256),
               dict(rope=rope_desc(), heads=4, q=P, qs=256, qo=P, qos=512),
               dict(rope=rope_desc(dims=20, layout=1))):
        assert append(c, **kw) == -1, kw
    for bad in BAD_ROPES:
        assert append(c, rope=rope_desc(**bad)) == -1, bad
    assert append(c, rows=0) == 0  # nothing to do is no error


def test_read_refuses():
    c = desc()
    read = lambda slots=P, rows=1, k=P, v=P: F.lib.fyb_kv8_read(C.byref(c), slots, rows, k, v, None, None)  # noqa: E731
    assert read(slots=None) == read(k=None) == read(v=None) == read(k=ODD) == -1
    assert F.lib.fyb_kv8_read(None, P, 1, P, P, None, None) == -1
    assert read(rows=0) == 0


def test_attention_refuses():
    c = desc()
    assert attention(None) == -1
    for kw in (dict(n=0), dict(most=0), dict(rows=2), dict(stride=0), dict(type_=8), dict(q=None), dict(qs=255),
               dict(out=None), dict(os_=255), dict(heads=3), dict(heads=0), dict(heads=130), dict(ws=None),
               dict(wb=0), dict(lengths=None), dict(table=None)):
        assert attention(c, **kw) == -1, kw
    assert attention(c, rows=0, starts=P) == 0
    ws = F.lib.fyb_kv8_attention_workspace
    assert ws(1, 1, 4, 2, 64) > 0
    assert ws(0, 1, 4, 2, 64) == ws(1, 0, 4, 2, 64) == ws(1, 1, 3, 2, 64) == ws(1, 1, 4, 2, 96) == 0
    assert ws(1, 1, 130, 2, 64) == ws(1, 1, 4, 0, 64) == 0


def test_rope_refuses():
    def call(d, rows=1, hd=64, type_=0, pos=P, q=P, qs=128, qo=P, qos=128, h=2, k=None, ks=0, ko=None, kos=0, kv=0):
        return F.lib.fyb_rope(C.byref(d) if d else None, pos, rows, hd, type_, q, qs, qo, qos, h, k, ks, ko, kos, kv,
                              None, None)
    assert call(None) == -1
    for bad in BAD_ROPES:
        assert call(rope_desc(**bad)) == -1, bad
    for kw in (dict(hd=62), dict(hd=65), dict(type_=8), dict(pos=None), dict(q=None), dict(qo=None), dict(qs=127),
               dict(qos=127), dict(qos=256), dict(kv=1), dict(kv=1, k=P, ks=64), dict(kv=1, k=P, ks=63, ko=P, kos=64),
               dict(h=0)):
        assert call(rope_desc(), **kw) == -1, kw
    assert call(rope_desc(), rows=0) == 0
    assert F.lib.fyb_rope_tables(None, 64, 1.0, 0, 8, P, P, None) == -1
    assert F.lib.fyb_rope_tables(P, 63, 1.0, 0, 8, P, P, None) == -1
    assert F.lib.fyb_rope_tables(P, 64, 1.0, 1 << 31, 8, P, P, None) == -1
    assert F.lib.fyb_rope_tables(P, 64, 1.0, 0, 0, P, P, None) == 0


def test_blocks_refuse():
    names = ["lengths", "new", "n", "table", "stride", "block", "free", "count", "lengths_out", "count_out", "start",
             "slots", "positions", "who", "rows", "status", "stream"]
    other = C.c_void_p(P.value + 64)
    good = dict(zip(names, [P, P, 1, P, 1, 16, P, P, other, other, P, P, P, P, 4, P, None]))
    call = lambda **kw: F.lib.fyb_kv_blocks(*(good | kw).values())  # noqa: E731
    for k in ("lengths", "new", "table", "free", "count", "lengths_out", "count_out", "start", "slots", "positions",
              "who", "status"):
        assert call(**{k: None}) == -1, k
    for kw in (dict(n=0), dict(n=16385), dict(stride=0), dict(block=0), dict(block=24), dict(rows=1 << 30),
               dict(lengths_out=P), dict(count_out=P)):
        assert call(**kw) == -1, kw
    names = ["lengths", "keep", "n", "table", "stride", "block", "free", "count", "capacity", "stream"]
    good = dict(zip(names, [P, P, 1, P, 1, 16, P, P, 4, None]))
    call = lambda **kw: F.lib.fyb_kv_release(*(good | kw).values())  # noqa: E731
    for kw in (dict(lengths=None), dict(keep=None), dict(table=None), dict(free=None), dict(count=None), dict(n=0),
               dict(n=16385), dict(stride=0), dict(block=24), dict(capacity=1 << 30)):
        assert call(**kw) == -1, kw


def test_wrappers_refuse_host_tensors():
    import torch
    x = torch.zeros((4, 2, 16, 64), dtype=torch.int8)
    with pytest.raises(ValueError):
        F.KV8Cache(x, x, torch.zeros((4, 2)), torch.zeros((4, 2)))
    q = torch.zeros((1, 2, 64))
    with pytest.raises(ValueError):
        F.rope(q, None, torch.zeros(1, dtype=torch.int32), torch.zeros((4, 32)), torch.zeros((4, 32)), "half", q, None)


def test_batch_refuses():
    assert not F.lib.fyb_batch_create_kv8(None, 4, 16, 32, 0)
    assert F.lib.fyb_batch_free_blocks(None) == -1
