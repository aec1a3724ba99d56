"""Rows of a batch that see nothing, and sequences that a plan cannot hold, through the plan and the attention."""
import numpy as np
import pytest

from test_batch_attention_gpu import Batch

pytestmark = pytest.mark.gpu


def _check(hlkv, b, heads, max_query, block_cap=None, window=0, sinks=0):
    """Rows of rejected sequences are zeros or as they were, everything else is the oracle's: a row that sees nothing is
    exactly zero (its bound is 0)."""
    import torch
    cap_b = b.plan.c.block_cap if block_cap is None else block_cap
    b.plan = hlkv.BatchPlan(len(b.q), cap_b, b.cap, max_query, window, sinks)
    b.window, b.sinks = window, sinks
    b.fill_plan()
    x, d_q = b.queries(heads, 1)
    got = b.run(d_q, b.D ** -0.5)
    torch.cuda.synchronize()
    want, tol, err = b.want(x, b.D ** -0.5)
    assert int(b.err.item()) == err == 1 << 13
    assert (got[sum(b.q):] == 0x1234).all()
    g = got.cpu().numpy().view(np.float16)
    blocks = at = 0
    for i, q in enumerate(b.q):
        n = int(b.wl.segs_host[i, 1])
        rows = slice(at, at + q)
        if q > max_query or blocks + n > cap_b:
            assert (np.isin(g[rows].view(np.int16), (0, 0x1234))).all(), i
        else:
            assert (np.abs(g[rows].astype(np.float64) - want[rows]) <= tol[rows]).all(), i
        blocks, at = blocks + n, at + q


@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 3)])
@pytest.mark.parametrize("q", [1, 5, 40])
def test_more_new_tokens_than_tokens(hlkv_lib, cuda_device, q, window, sinks):
    """A sequence without blocks, one whose blocks are empty, one of fewer tokens than new ones, and a long one."""
    vt = [[], [0, 0], [max(q // 2, 1)] if q > 1 else [0], [16] * 30]
    b = Batch(hlkv_lib, 64, 2, 64, vt, [q] * 4, window=window, sinks=sinks, seed=q, pad=3)
    _check(hlkv_lib, b, 8, q, window=window, sinks=sinks)


@pytest.mark.parametrize("q", [[40, 600], [9, 5], [600, 3]])
def test_more_new_tokens_than_tokens_when_split(hlkv_lib, cuda_device, q):
    """Row tiles split over the tokens: the first rows see nothing."""
    b = Batch(hlkv_lib, 16, 1, 128, [[16] * 30, [16] * 150], [480 + q[0], q[1]], seed=1, pad=2)
    _check(hlkv_lib, b, 4, 1200)


@pytest.mark.parametrize("nseq", [3, 140])
@pytest.mark.parametrize("max_query", [1, 4, 8])
def test_sequences_that_the_plan_cannot_hold(hlkv_lib, cuda_device, nseq, max_query):
    """Far more new tokens than max_query, beside sequences of max_query new tokens with and without blocks."""
    vt = [[16] * 2, [], [16] * 9] + [[16] * 3] * (nseq - 3)
    q = [5000, max_query, max_query] + [max_query] * (nseq - 3)
    b = Batch(hlkv_lib, 16, 8, 64, vt, q, seed=2, pad=4)
    _check(hlkv_lib, b, 32, max_query)


@pytest.mark.parametrize("q", [1, 40])
def test_blocks_that_do_not_fit(hlkv_lib, cuda_device, q):
    b = Batch(hlkv_lib, 16, 2, 64, [[16] * 9, [16] * 12, []], [q, q, q], seed=3)
    _check(hlkv_lib, b, 8, q, block_cap=15)


@pytest.mark.parametrize("nseq", [129, 600, 1200])
@pytest.mark.parametrize("q", ["one token", "some chunks", "all"])
def test_many_sequences_in_a_plan_for_long_prompts(hlkv_lib, cuda_device, nseq, q):
    """Past 128 sequences the tile kernel's grid goes by the batch's tokens where a plan holds more rows than they make."""
    import torch
    rng = np.random.default_rng(nseq)
    lens = [1] * nseq
    if q == "some chunks":
        for i in (0, 7, nseq // 2, nseq - 1):
            lens[i] = int(rng.integers(17, 700))
    elif q == "all":
        lens = [int(n) for n in rng.choice([0, 1, 5, 9, 40], nseq)]
    vt = [[16] * (n // 16) + [n % 16 or 16] for n in lens]
    b = Batch(hlkv_lib, 16, 1, 64, vt, lens, seed=nseq, pad=50)
    b.plan = hlkv_lib.BatchPlan(nseq, b.plan.c.block_cap, b.cap, 1 << 20)
    b.fill_plan()
    x, d_q = b.queries(4, 1)
    got = b.run(d_q, 0.125)
    torch.cuda.synchronize()
    want, tol, err = b.want(x, 0.125)
    assert int(b.err.item()) == err == 0
    n = sum(lens)
    assert (got[n:] == 0x1234).all()
    assert (np.abs(got.cpu().numpy().view(np.float16).astype(np.float64)[:n] - want[:n]) <= tol[:n]).all()


def test_few_tokens_of_many_sequences(hlkv_lib, cuda_device):
    """Fewer rows in the whole batch than a row tile needs, in a plan for long prompts of many sequences."""
    import torch
    lens = [0] * 200
    lens[3], lens[150] = 1, 2
    b = Batch(hlkv_lib, 16, 1, 64, [[16, 9]] * 200, lens, seed=1)
    b.plan = hlkv_lib.BatchPlan(200, b.plan.c.block_cap, b.cap, 8192)
    b.fill_plan()
    x, d_q = b.queries(4, 1)
    got = b.run(d_q, 0.125)
    torch.cuda.synchronize()
    want, tol, err = b.want(x, 0.125)
    assert int(b.err.item()) == err == 0
    assert (np.abs(got.cpu().numpy().view(np.float16).astype(np.float64) - want) <= tol).all()
