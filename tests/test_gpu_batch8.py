"""GPU tests of a plan's batched decode over the paged 8-bit cache beside
test_gpu_kv8.py: runs of several lengths, the ends of its capacity and of its
life, what it refuses."""
import numpy as np
import pytest

import fyodor_b200 as F

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

CFG = dict(layers=2, embedding=512, heads=8, kv_heads=2, feed_forward=1024, vocabulary=1024, context=64,
           matrix_type=F.Q4_K, seed=21, norm_mode=2)


@pytest.mark.parametrize("kv", ["int8", None])
def test_timing_ends_at_the_capacity(provider, kv):
    """Timing a single step at the last position of the plan, or of the pool, takes no step past it: the batch goes
    on after it. The capacity is no multiple of the block size, so the tables would hold more."""
    m, nseq, capacity = F.SynthModel(**CFG), 3, 40
    plan = provider.plan(m, capacity)
    batch = F.Batch(plan, nseq, **(dict(kv=kv, blocks=3 * nseq, block_size=16) if kv else {}))
    cur = np.arange(nseq, dtype=np.uint32)
    batch.decode_greedy(cur, np.zeros(nseq, np.uint32), capacity - 1)
    last = np.full(nseq, capacity - 1, np.uint32)
    want = batch.step(cur, last)[0]
    assert batch.time_greedy(cur, last, 1) > 0
    assert plan.error() == 0
    assert (batch.step(cur, last)[0] == want).all()
    assert batch.time_greedy(cur, last, 2) < 0
    if kv:
        assert batch.free_blocks() == 0
        tight = F.Batch(plan, nseq, kv=kv, blocks=nseq, block_size=16)
        tight.decode_greedy(cur, np.zeros(nseq, np.uint32), 15)
        assert tight.time_greedy(cur, np.full(nseq, 15, np.uint32), 1) > 0
        assert tight.free_blocks() == 0 and plan.error() == 0
        tight.step(cur, np.full(nseq, 15, np.uint32))
        tight.close()
    batch.close()
    plan.close()
    m.close()


@pytest.mark.parametrize("kv", ["int8", None])
def test_longer_runs_after_shorter_ones(provider, kv):
    """Greedy runs of growing length replay one captured step: each run's tokens are those of single steps."""
    m, nseq = F.SynthModel(**CFG), 3
    plan = provider.plan(m, CFG["context"])
    batch, other = (F.Batch(plan, nseq, **(dict(kv=kv, blocks=4 * nseq, block_size=16) if kv else {})) for _ in range(2))
    cur, at = np.arange(nseq, dtype=np.uint32), 0
    for steps in (1, 2, 5, 40):
        got = batch.decode_greedy(cur, np.full(nseq, at, np.uint32), steps)
        for i in range(steps):
            _, cur = other.step(cur, np.full(nseq, at + i, np.uint32), logits=False)
            assert (got[i] == cur).all(), (steps, i)
        at += steps
    with pytest.raises(RuntimeError):
        batch.decode_greedy(cur, np.full(nseq, at, np.uint32), CFG["context"])
    batch.close()
    other.close()
    plan.close()
    m.close()


def test_batches_end_with_their_plan(provider):
    """A plan that is closed closes its batches: their memory comes back, and they refuse further steps."""
    m = F.SynthModel(**CFG)
    plan = provider.plan(m, CFG["context"])
    zero = np.zeros(2, np.uint32)
    free = torch.cuda.mem_get_info()[0]
    paged, plain = F.Batch(plan, 2, kv="int8", blocks=1 << 18, block_size=16), F.Batch(plan, 2)
    held = free - torch.cuda.mem_get_info()[0]
    assert held >= 2 * 2 * (1 << 18) * 16 * 2 * 64  # layers, K and V, blocks, tokens, KV heads, dimensions
    paged.step(zero, zero)
    plan.close()
    assert torch.cuda.mem_get_info()[0] - free > -(64 << 20)
    for batch in (paged, plain):
        assert not batch.ptr
        with pytest.raises(RuntimeError):
            batch.step(zero, zero)
        batch.close()
    m.close()


def test_unknown_format_is_refused(provider):
    m = F.SynthModel(**CFG)
    plan = provider.plan(m, 64)
    with pytest.raises(ValueError):
        F.Batch(plan, 2, kv="int4", blocks=8)
    with pytest.raises(ValueError):
        F.KV8Cache.empty(4, 2, 16, 64, "int4")
    plan.close()
    m.close()
