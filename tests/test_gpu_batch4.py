"""GPU tests of a plan's batched decode over the paged 4-bit cache, and of steps
that return log probabilities instead of logits: the step in 64 bits over the
same 4-bit cache, greedy runs, refusals, and the loss of a text by every cache."""
import ctypes as C

import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from .test_gpu_kv4 import hold  # noqa: E402
from .test_gpu_kv8 import RefModel  # noqa: E402

CFG = dict(layers=2, embedding=512, heads=8, kv_heads=2, feed_forward=1024, vocabulary=1024, context=64,
           matrix_type=F.Q4_K, seed=21, norm_mode=2)
CFG128 = dict(layers=2, embedding=512, heads=4, kv_heads=2, feed_forward=1024, vocabulary=1024, context=64,
              matrix_type=F.Q4_K, seed=22, norm_mode=2)


class Cache4:
    """K and V rows of one sequence as they are held, in the shape that RefModel's steps use."""

    def __init__(self, capacity):
        self.rows = {"k": {}, "v": {}}

    def append(self, name, rows, slots):
        n, scale, low = hold(rows.numpy())
        x = low.astype(np.float64)[..., None] + scale.astype(np.float64)[..., None] * n
        for r, slot in enumerate(slots):
            self.rows[name][slot] = x[r].reshape(x.shape[1], -1)

    def values(self, name, slots):
        return torch.from_numpy(np.stack([self.rows[name][s] for s in slots]))


class RefModel4(RefModel):
    def __init__(self, model):
        super().__init__(model, "uint4", 16)

    def session(self, capacity):
        return [Cache4(capacity) for _ in range(self.m.layers)]


@pytest.mark.parametrize("cfg", [CFG, CFG128])
@pytest.mark.parametrize("nseq", [1, 5, 12])
def test_batch_over_the_cache(provider, nseq, cfg):
    """Logits within 1e-3 of the logit scale of the same step in 64 bits, but for K and V that lie so near a border
    between two held numbers that the step's own rounding moves them: a step of the cache is a fifteenth of its group's
    range, and what a few of them move stays below 2e-2. Sequences go on at ragged positions, some going back."""
    m = F.SynthModel(**cfg)
    plan = provider.plan(m, cfg["context"])
    batch = F.Batch(plan, nseq, kv="uint4", blocks=4 * nseq, block_size=16)
    ref = RefModel4(m)
    refs = [ref.session(cfg["context"]) for _ in range(nseq)]
    rng = np.random.default_rng(nseq)
    pos = np.zeros(nseq, np.uint32)
    off = []
    for s in range(24):
        toks = rng.integers(0, m.vocabulary, nseq).astype(np.uint32)
        lg, am = batch.step(toks, pos)
        assert (am == lg.argmax(1)).all()
        for b in range(nseq):
            e = ref.step(refs[b], int(toks[b]), int(pos[b]))
            off.append(float(np.max(np.abs(lg[b] - e)) / (1 + np.max(np.abs(e)))))
        held = int(sum(-(-(int(p) + 1) // 16) for p in pos))
        assert batch.free_blocks() == 4 * nseq - held
        pos = np.where(rng.random(nseq) < 0.1, pos * 2 // 3, pos + 1).astype(np.uint32)
    assert np.max(off) <= 2e-2 and np.median(off) <= 1e-3, (np.max(off), np.median(off))
    batch.close()
    plan.close()
    m.close()


def test_batch_greedy_and_refusals(provider):
    m = F.SynthModel(**CFG)
    plan = provider.plan(m, CFG["context"])
    nseq = 3
    batch, other = (F.Batch(plan, nseq, kv="uint4", blocks=4 * nseq, block_size=16) for _ in range(2))
    rng = np.random.default_rng(3)
    for s in range(20):
        toks = rng.integers(0, m.vocabulary, nseq).astype(np.uint32)
        for x in (batch, other):
            x.step(toks, np.full(nseq, s, np.uint32))
    start, first = np.full(nseq, 17, np.uint32), rng.integers(0, m.vocabulary, nseq).astype(np.uint32)
    got = other.decode_greedy(first, start, 8)
    cur = first
    for i in range(8):
        _, cur = batch.step(cur, start + np.uint32(i))
        assert (cur == got[i]).all(), i
    with pytest.raises(RuntimeError):
        batch.step(cur, np.full(nseq, 26, np.uint32))  # a gap
    tight = F.Batch(plan, nseq, kv="uint4", blocks=nseq, block_size=16)
    assert tight.decode_greedy(cur, np.zeros(nseq, np.uint32), 16).shape == (16, nseq)
    with pytest.raises(RuntimeError):
        tight.step(cur, np.full(nseq, 16, np.uint32))
    assert tight.free_blocks() == 0 and tight.time_greedy(cur, np.full(nseq, 3, np.uint32), 4) > 0
    for bad in ((0, 16), (16, 24), (16, 8), (16, 512)):
        assert not F.lib.fyb_batch_create_kv4(C.c_void_p(plan.ptr), 4, *bad)
    assert not F.lib.fyb_batch_create_kv4(C.c_void_p(plan.ptr), 17, 16, 16) and not F.lib.fyb_batch_create_kv4(None, 4, 16, 16)
    for x in (tight, other, batch):
        x.close()
    plan.close()
    m.close()


@pytest.mark.parametrize("kv", [None, "int8", "uint4"])
def test_score(provider, kv):
    """A scored step is the step, its logits turned into log probabilities on the device."""
    m = F.SynthModel(**CFG)
    plan = provider.plan(m, CFG["context"])
    nseq, args = 5, {} if kv is None else dict(kv=kv, blocks=20, block_size=16)
    a, b = (F.Batch(plan, nseq, **args) for _ in range(2))
    rng = np.random.default_rng(4)
    for s in range(12):
        toks, pos = rng.integers(0, m.vocabulary, nseq).astype(np.uint32), np.full(nseq, s, np.uint32)
        targets = rng.integers(0, m.vocabulary, nseq).astype(np.int32)
        targets[s % nseq] = -1
        lg, am = a.step(toks, pos)
        got = b.score(toks, pos, targets, top=s)
        x = lg.astype(np.float64)
        ln = x - x.max(1, keepdims=True)
        ln -= np.log(np.exp(ln).sum(1, keepdims=True))
        # sums of 1024 terms in F32: the bound of the log probabilities' own tests
        tol = 2.0 ** -19 + np.abs(ln).max() * 2.0 ** -22
        for r in range(nseq):
            order = np.argsort(-lg[r], kind="stable")
            assert got["top_tokens"][r].tolist() == order[:s].tolist()
            assert (np.abs(got["top_logprobs"][r] - ln[r][order[:s]]) <= tol).all()
            if targets[r] < 0:
                assert got["logprob"][r] == 0 and got["rank"][r] == -1
            else:
                assert abs(got["logprob"][r] - ln[r][targets[r]]) <= tol and order[got["rank"][r]] == targets[r]
            assert abs(got["entropy"][r] + (np.exp(ln[r]) * ln[r]).sum()) <= 8 * tol
    only = b.score(toks, np.full(nseq, 12, np.uint32))
    assert "logprob" not in only and only["top_tokens"].shape == (nseq, 0) and np.isfinite(only["entropy"]).all()
    t, p = toks, np.full(nseq, 13, np.uint32)
    for bad in (dict(targets=[m.vocabulary] * nseq), dict(positions=np.full(nseq, 64, np.uint32))):
        with pytest.raises(RuntimeError):
            b.score(t, bad.get("positions", p), bad.get("targets"))
    for bad in (dict(top=33), dict(top=-1), dict(targets=[1, 2])):
        with pytest.raises(ValueError):
            b.score(t, p, **bad)
    b.score(t, p)  # and goes on
    for x in (a, b):
        x.close()
    plan.close()
    m.close()


def test_loss_of_a_text_by_cache(provider):
    """The same text scored over fp16, 8-bit and 4-bit caches: the loss moves by less with more bits, and by little."""
    m = F.SynthModel(**CFG128)
    plan = provider.plan(m, CFG128["context"])
    text = np.random.default_rng(7).integers(0, m.vocabulary, (4, 61)).astype(np.uint32)
    loss = {}
    for kv in (None, "int8", "uint4"):
        batch = F.Batch(plan, 4, **({} if kv is None else dict(kv=kv, blocks=16, block_size=16)))
        lp = [batch.score(text[:, i], np.full(4, i, np.uint32), text[:, i + 1])["logprob"] for i in range(60)]
        loss[kv] = np.stack(lp)
        batch.close()
    spread = np.std(loss[None])
    assert np.sqrt(np.mean((loss["int8"] - loss[None]) ** 2)) < np.sqrt(np.mean((loss["uint4"] - loss[None]) ** 2)) < 0.5 * spread
    plan.close()
    m.close()
