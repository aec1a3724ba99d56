"""hlkv_batch_plan against a plain implementation: every array, every word."""
import numpy as np
import pytest

from batch_helpers import PAD, plan_oracle

pytestmark = pytest.mark.gpu

LAYOUT = 1


def _tables(rng, lens, T, vt=None):
    """Scattered block ids and segments: (segs, arena, table), uint32."""
    total = int(sum(lens))
    size = total + 5
    ids = rng.permutation(size)[:total].astype(np.uint32)
    table = np.zeros((size, 4), np.uint32)
    table[:, 1], table[:, 3] = 15, np.arange(size)
    v = rng.integers(0, T + 1, total) if vt is None else np.asarray(vt)
    f = rng.integers(0, 4, total)
    table[ids, 0] = rng.integers(0, 1 << 20, total)
    table[ids, 1] = f | LAYOUT << 6 | v << 10
    segs = np.zeros((len(lens), 2), np.uint32)
    segs[:, 1] = lens
    order = rng.permutation(len(lens))
    off = 3
    for i in order:
        segs[i, 0] = off
        off += lens[i]
    arena = np.full(off + 2, 0xFFFFFFFF, np.uint32)
    at = 0
    for i, n in enumerate(lens):
        arena[segs[i, 0]:segs[i, 0] + n] = ids[at:at + n]
        at += n
    return segs, arena, table


def _dev(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.uint32).view(np.int32)).cuda()


def _check(hlkv, segs, arena, table, qlens, T, cap_b=None, cap_t=None, max_query=None, window=0, sinks=0, null_q=False,
           expect_err=None):
    import torch
    nseq = len(segs)
    cap_b = int(segs[:, 1].sum()) if cap_b is None else cap_b
    cap_t = int(sum(qlens)) if cap_t is None else cap_t
    max_query = max([1, *map(int, qlens)]) if max_query is None else max_query
    plan = hlkv.BatchPlan(nseq, cap_b, cap_t, max_query, window, sinks)
    for t in (plan.blocks, plan.targets, plan.positions, plan.block_first, plan.block_count, plan.token_first, plan.context,
              plan.block_cost, plan.cost):
        t.fill_(0x5A5A5A5A)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    d_table, d_arena = _dev(table), _dev(arena)
    args = (plan, hlkv.Layout(T, 2, 64, LAYOUT), d_table.data_ptr(), len(table), d_arena.data_ptr(), len(arena), _dev(segs),
            None if null_q else _dev(np.asarray(qlens)), err)
    seqs, targets, positions, tf, bf, want_err = plan_oracle(segs, qlens, arena, table, T, LAYOUT, cap_b, cap_t, max_query,
                                                             window, sinks)
    u = lambda t: t.cpu().numpy().view(np.uint32)  # noqa: E731
    for _ in range(2):  # a second call finds the first one's arrays
        hlkv.batch_plan(*args)
        torch.cuda.synchronize()
        assert int(err.item()) == want_err and (expect_err is None or want_err == expect_err)
        assert np.array_equal(u(plan.block_first), bf)
        assert np.array_equal(u(plan.token_first), tf)
        assert u(plan.context).tolist() == [s["context"] for s in seqs]
        assert u(plan.block_count).tolist() == [len(s["blocks"]) for s in seqs]
        blocks = np.full((cap_b, 4), 0x5A5A5A5A, np.uint32)
        for b, s in zip(bf, seqs):
            if s["blocks"]:
                blocks[b:b + len(s["blocks"])] = np.array(s["blocks"], np.uint32)
        assert np.array_equal(u(plan.blocks), blocks)
        cost = np.full(cap_b, 0x5A5A5A5A, np.uint32)
        for b, s in zip(bf, seqs):
            cost[b:b + len(s["cost"])] = s["cost"]
        assert np.array_equal(u(plan.block_cost), cost)
        assert u(plan.cost).tolist() == [s["cost"][-1] if s["cost"] else 0 for s in seqs]
        assert np.array_equal(u(plan.targets), targets)
        assert np.array_equal(u(plan.positions).view(np.int32), positions)


@pytest.mark.parametrize("T,lens,q", [
    (16, [1], [1]), (16, [4, 1, 7, 30], [1, 1, 1, 1]), (1, [5, 0, 9], [2, 0, 9]), (512, [3, 2], [700, 1]),
    (16, [0, 0], [0, 0]), (20, [40, 3, 0, 25, 1], [100, 0, 0, 1, 5]),
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (100, 0), (33, 500)])
def test_plan_matches_plain(hlkv_lib, cuda_device, T, lens, q, window, sinks):
    rng = np.random.default_rng(T + len(lens))
    segs, arena, table = _tables(rng, lens, T)
    v = {int(b): int(x[1]) >> 10 for b, x in enumerate(table)}
    ctx = [sum(v[int(a)] for a in arena[o:o + n]) for o, n in segs]
    _check(hlkv_lib, segs, arena, table, [min(a, b) for a, b in zip(q, ctx)], T, window=window, sinks=sinks)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4096, 8191, 8193, 20000])
@pytest.mark.parametrize("window", [0, 5000])
def test_long_sequences(hlkv_lib, cuda_device, n, window):
    """Around the blocks that a CTA, and the largest cluster, take at once."""
    rng = np.random.default_rng(n)
    segs, arena, table = _tables(rng, [n], 8, vt=np.where(rng.random(n) < 0.05, rng.integers(0, 8, n), 8))
    _check(hlkv_lib, segs, arena, table, [777], 8, window=window, sinks=9)


def test_one_long_among_short(hlkv_lib, cuda_device):
    """The cluster's size goes by the average: the long sequence takes rounds."""
    rng = np.random.default_rng(1)
    lens = [3] * 40 + [5000] + [2] * 60
    segs, arena, table = _tables(rng, lens, 16, vt=np.full(sum(lens), 16))
    for window in (0, 3000):
        _check(hlkv_lib, segs, arena, table, [1] * 40 + [900] + [3] * 60, 16, window=window, sinks=20)


@pytest.mark.parametrize("nseq", [257, 2048, 2049, 5000])
def test_many_sequences(hlkv_lib, cuda_device, nseq):
    rng = np.random.default_rng(nseq)
    lens = rng.integers(1, 4, nseq).tolist()
    segs, arena, table = _tables(rng, lens, 4, vt=rng.integers(1, 5, sum(lens)))
    _check(hlkv_lib, segs, arena, table, [1] * nseq, 4, null_q=True, cap_t=nseq + 9)


def test_padding_and_capacities(hlkv_lib, cuda_device):
    """Rows behind the last token are padding; sequences that do not fit are planned as empty."""
    rng = np.random.default_rng(5)
    lens = [3, 2, 6, 1]
    segs, arena, table = _tables(rng, lens, 16, vt=np.full(12, 16))
    q = [5, 1, 20, 2]
    _check(hlkv_lib, segs, arena, table, q, 16, cap_t=40)
    for kw in (dict(cap_b=10), dict(cap_b=0), dict(cap_t=26), dict(cap_t=5), dict(max_query=19), dict(cap_b=11, cap_t=27, max_query=4)):
        _check(hlkv_lib, segs, arena, table, q, 16, **kw, expect_err=1 << 13)
    _check(hlkv_lib, segs, arena, table, [5, 40, 97, 2], 16, expect_err=1 << 13)  # more new tokens than tokens


def test_capacities_of_many_sequences(hlkv_lib, cuda_device):
    rng = np.random.default_rng(6)
    lens = rng.integers(1, 4, 2500).tolist()
    segs, arena, table = _tables(rng, lens, 4, vt=rng.integers(1, 5, sum(lens)))
    _check(hlkv_lib, segs, arena, table, [1] * 2500, 4, cap_b=sum(lens) - 700, expect_err=1 << 13)
    _check(hlkv_lib, segs, arena, table, [1] * 2500, 4, cap_t=2000, expect_err=1 << 13)


def test_bad_blocks_are_left_out(hlkv_lib, cuda_device):
    rng = np.random.default_rng(8)
    segs, arena, table = _tables(rng, [12], 16, vt=np.full(12, 16))
    ids = arena[segs[0, 0]:segs[0, 0] + 12].copy()
    table[ids[1], 1] |= 15                                   # not executable
    table[ids[2], 1] = (int(table[ids[2], 1]) & ~15) | 7      # no such format
    table[ids[3], 3] ^= 1                                    # another block's record
    table[ids[4], 1] = (int(table[ids[4], 1]) & ~(15 << 6)) | 2 << 6  # another layout
    table[ids[5], 1] = 1 | 3 << 4 | LAYOUT << 6 | 16 << 10      # external parameters
    table[ids[6], 1] = 1 | LAYOUT << 6 | 17 << 10               # more tokens than the block has
    arena[segs[0, 0] + 7] = len(table)                       # no such block
    _check(hlkv_lib, segs, arena, table, [3], 16, expect_err=1 | 2 | 1 << 8 | 1 << 6 | 1 << 7 | 1 << 5 | 1 << 4)
    segs, arena, table = _tables(rng, [4], 16, vt=np.full(4, 16))
    segs[0, 0] = len(arena) - 2                              # runs off the arena
    arena[-2:] = [0, 1]
    table[:2, 1] = 1 | LAYOUT << 6 | 5 << 10
    _check(hlkv_lib, segs, arena, table, [3], 16, expect_err=1 << 3)
    segs[0] = (0xFFFFFFFE, 4)                                # an offset that passes 32 bits
    _check(hlkv_lib, segs, arena, table, [0], 16, cap_t=2, expect_err=1 << 3)
    segs[0] = (0, 0xFFFFFFFF)                                # a length beyond any array
    _check(hlkv_lib, segs, arena, table, [1], 16, cap_b=4, expect_err=1 << 13)


def test_plan_of_the_host_table(hlkv_lib, cuda_device):
    """The host's CSR build_exec_table and append_tokens' targets, for one new token per sequence."""
    import torch
    from hlkv.workload import build_workload, mixed_formats
    T = 16
    fm = mixed_formats(6, [3, 9, 1, 4, 12, 2], probs=(1, 1, 1, 1), seed=3)
    vt = [[T] * (len(r) - 1) + [T if i % 2 else 5] for i, r in enumerate(fm)]
    wl = build_workload(fm, T=T, H=2, D=64, seed=3, valid_tokens=vt, spare_slots=4)
    st, targets, done = wl.table.append_tokens(wl.seqs, [0, 1, 2, 3, 0, 1], 1)
    assert st == 0 and done == 6
    wl.dt.sync(wl.table)
    st, segs = wl.table.batch_segments(wl.seqs)
    st, indptr, blocks = wl.table.build_exec_table(wl.seqs)
    plan = hlkv_lib.BatchPlan(6, int(segs[:, 1].sum()), 6)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    hlkv_lib.batch_plan(plan, wl.layout, wl.dt.table_ptr, wl.dt.table_size, wl.dt.arena_ptr, wl.dt.arena_size, _dev(segs),
                        None, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    u = lambda t: t.cpu().numpy().view(np.uint32)  # noqa: E731
    assert np.array_equal(u(plan.block_first), indptr[:-1])
    assert np.array_equal(u(plan.blocks)[:, :3], blocks[:, :3])
    assert np.array_equal(u(plan.targets), targets)
    assert not (u(plan.targets) == PAD).any()
