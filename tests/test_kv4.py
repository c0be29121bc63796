"""The paged 4-bit KV cache and the log probabilities on the host side: every
entry point refuses what it has to before anything reaches a device, so no GPU
is needed."""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

BUF = np.zeros(4096, np.float32)
P = C.c_void_p((BUF.ctypes.data + 255) // 256 * 256)  # never read: every call below is refused or empty
ODD = C.c_void_p(P.value + 4)


def desc(**kw):
    return F.KV4CacheDesc(**(dict(k=P.value, v=P.value, k_scale=P.value, v_scale=P.value, blocks=4, kv_heads=2,
                                  block_size=16, head_dim=64) | kw))


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=ODD.value), dict(v=ODD.value),
              dict(k_scale=ODD.value), dict(v_scale=ODD.value), dict(blocks=0), dict(kv_heads=0), dict(kv_heads=65537),
              dict(block_size=8), dict(block_size=48), dict(block_size=512), dict(head_dim=96), dict(head_dim=32),
              dict(blocks=1 << 27)]


def rope_desc(**kw):
    return F.RopeDesc(**(dict(cos_table=P.value, sin_table=P.value, table_rows=8, dims=64, layout=0) | kw))


def append(cache, rows=1, type_=0, k=P, ks=128, v=P, vs=128, rope=None, pos=P, q=None, qs=0, qo=None, qos=0, heads=0,
           slots=P):
    return F.lib.fyb_kv4_append(C.byref(cache) if cache else None, slots, rows, type_, k, ks, v, vs,
                                C.byref(rope) if rope else None, pos, q, qs, qo, qos, heads, None, None)


def attention(cache, n=1, most=1, rows=1, stride=1, type_=0, q=P, qs=256, out=P, os_=256, heads=4, ws=P, wb=1 << 40,
              lengths=P, table=P, starts=None):
    return F.lib.fyb_kv4_attention(C.byref(cache) if cache else None, lengths, starts, n, most, rows, table, stride,
                                   type_, q, qs, out, os_, heads, 0.1, ws, wb, None, None)


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_cache_refused(bad):
    c = desc(**bad)
    assert append(c) == -1
    assert attention(c) == -1
    assert F.lib.fyb_kv4_read(C.byref(c), P, 1, P, P, None, None) == -1


def test_append_refuses():
    c = desc()
    assert append(None) == -1
    for kw in (dict(k=None), dict(v=None), dict(ks=127), dict(vs=127), dict(type_=8), dict(type_=2), dict(slots=None),
               dict(heads=4), dict(rope=rope_desc(), pos=None), dict(rope=rope_desc(), heads=4, q=P, qs=256),
               dict(rope=rope_desc(), heads=4, q=P, qs=255, qo=P, qos=256),
               dict(rope=rope_desc(), heads=4, q=P, qs=256, qo=P, qos=512), dict(rows=1 << 31)):
        assert append(c, **kw) == -1, kw
    for bad in (dict(cos_table=None), dict(sin_table=None), dict(table_rows=0), dict(dims=0), dict(dims=7),
                dict(dims=66), dict(layout=2)):
        assert append(c, rope=rope_desc(**bad)) == -1, bad
    assert append(c, rows=0) == append(c, rows=0, k=None, v=None, slots=None) == 0  # nothing to do is no error


def test_read_refuses():
    c = desc()
    read = lambda slots=P, rows=1, k=P, v=P: F.lib.fyb_kv4_read(C.byref(c), slots, rows, k, v, None, None)  # noqa: E731
    assert read(slots=None) == read(k=None) == read(v=None) == read(k=ODD) == read(v=ODD) == read(rows=1 << 31) == -1
    assert F.lib.fyb_kv4_read(None, P, 1, P, P, None, None) == -1
    assert read(rows=0) == 0


def test_attention_refuses():
    c = desc()
    assert attention(None) == -1
    for kw in (dict(n=0), dict(most=0), dict(rows=2), dict(stride=0), dict(type_=8), dict(q=None), dict(qs=255),
               dict(out=None), dict(os_=255), dict(heads=3), dict(heads=0), dict(heads=130), dict(ws=None), dict(ws=ODD),
               dict(wb=0), dict(lengths=None), dict(table=None), dict(most=1 << 31), dict(stride=1 << 31)):
        assert attention(c, **kw) == -1, kw
    assert attention(c, rows=0, starts=P) == 0
    ws = F.lib.fyb_kv4_attention_workspace
    assert ws(1, 1, 4, 2, 64) > 0
    assert ws(0, 1, 4, 2, 64) == ws(1, 0, 4, 2, 64) == ws(1, 1, 3, 2, 64) == ws(1, 1, 4, 2, 96) == 0
    assert ws(1, 1, 130, 2, 64) == ws(1, 1, 4, 0, 64) == 0


def test_logprobs_refuse():
    names = ["type", "logits", "stride", "rows", "vocabulary", "tokens", "logprob", "rank", "entropy", "top",
             "top_tokens", "top_logprobs", "workspace", "bytes", "error", "stream"]
    good = dict(zip(names, [0, P, 100, 1, 100, P, P, P, P, 2, P, P, P, 1 << 40, None, None]))
    call = lambda **kw: F.lib.fyb_logprobs(*(good | kw).values())  # noqa: E731
    for kw in (dict(type=8), dict(logits=None), dict(stride=99), dict(vocabulary=0), dict(vocabulary=1 << 31),
               dict(rows=1 << 31), dict(tokens=None), dict(logprob=None), dict(tokens=None, logprob=None), dict(top=33),
               dict(top_tokens=None), dict(top_logprobs=None), dict(workspace=None), dict(workspace=ODD), dict(bytes=0),
               dict(logits=C.c_void_p(P.value + 2))):
        assert call(**kw) == -1, kw
    assert call(rows=0) == call(rows=0, logits=None, tokens=None) == 0
    need = F.lib.fyb_logprobs_workspace
    assert need(1, 1, 0) > 0 and need(1000, 128256, 32) > 0
    assert need(1, 0, 0) == need(1, 5, 33) == need(1 << 31, 5, 0) == need(1, 1 << 31, 0) == 0
    for bad in ((-1, 5), (1, -5), (1, 5, -1), (1, 5, 33)):
        with pytest.raises(ValueError):
            F.logprobs_workspace(*bad, device="cpu")


def test_wrappers_refuse_host_tensors():
    import torch
    k, s = torch.zeros((4, 2, 16, 32), dtype=torch.uint8), torch.zeros((4, 2, 16, 1, 2), dtype=torch.float16)
    for a in ((k, k, s, s), (k, k, s, s[..., :1]), (k[0], k[0], s[0], s[0]), (k, k[:2], s, s)):
        with pytest.raises(ValueError):
            F.KV4Cache(*a)
    x = torch.zeros((2, 7))
    with pytest.raises(ValueError):
        F.logprobs(x, None, None, None, None, None, None, torch.zeros(256, dtype=torch.uint8))


def test_batch_refuses():
    assert not F.lib.fyb_batch_create_kv4(None, 4, 16, 32)
    assert F.lib.fyb_batch_score(None, P, P, P, P, P, P, 0, None, None) == -1
