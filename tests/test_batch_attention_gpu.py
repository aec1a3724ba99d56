"""hlkv_batch_attention against attention in 64 bits over the blocks' exact values; the error bound of
every value is counted in batch_helpers.attention_oracle."""
import numpy as np
import pytest

from batch_helpers import attention_oracle, plan_oracle
from helpers import device_arena, device_table_words, host_pools

pytestmark = pytest.mark.gpu


class Batch:
    """A cache with its plan, on the device and in plain form."""

    def __init__(self, hlkv, T, H, D, vt, q, probs=(1, 1, 1, 1), window=0, sinks=0, seed=0, pad=0, change=None):
        import torch
        from hlkv.workload import build_workload, mixed_formats
        fm = mixed_formats(len(vt), [len(v) for v in vt], probs=probs, seed=seed)
        self.hlkv, self.T, self.H, self.D, self.window, self.sinks = hlkv, T, H, D, window, sinks
        self.wl = build_workload(fm, T=T, H=H, D=D, seed=seed, valid_tokens=vt)
        if change is not None:
            change(self.wl)
        self.cap = sum(q) + pad
        self.plan = hlkv.BatchPlan(len(vt), sum(map(len, vt)), self.cap, max([1, *q]), window, sinks)
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.qlens = torch.tensor(q, dtype=torch.int32, device="cuda")
        self.q = q
        self.fill_plan()

    def fill_plan(self, stream=None):
        wl = self.wl
        self.hlkv.batch_plan(self.plan, wl.layout, wl.dt.table_ptr, wl.dt.table_size, wl.dt.arena_ptr, wl.dt.arena_size,
                             wl.segs, self.qlens, self.err, stream=stream)

    def queries(self, heads, seed):
        import torch
        x = np.random.default_rng(seed).standard_normal((self.cap, heads, self.D)).astype(np.float16)
        return x, torch.from_numpy(x.view(np.int16)).cuda()

    def workspace(self, heads):
        import torch
        n = self.hlkv.batch_attention_workspace_bytes(self.plan, self.wl.layout, heads)
        return torch.full((n,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten

    def run(self, d_q, scale, out=None, ws=None, stream=None):
        import torch
        out = torch.full_like(d_q, 0x1234) if out is None else out
        self.hlkv.batch_attention(self.wl.hlkv_pools(), self.wl.layout, self.plan, d_q, scale, out, self.err,
                                  workspace=self.workspace(d_q.shape[1]) if ws is None else ws, stream=stream)
        return out

    def want(self, x, scale):
        wl = self.wl
        seqs, _, _, tf, _, err = plan_oracle(wl.segs_host, self.q, device_arena(wl), device_table_words(wl), self.T, 1,
                                             self.plan.c.block_cap, self.cap, self.plan.c.max_query, self.window, self.sinks)
        out, tol = attention_oracle(seqs, tf, host_pools(wl), self.T, self.H, self.D, x.astype(np.float64), scale,
                                    self.window, self.sinks)
        return out, tol, err

    def check(self, heads, seed=0, scale=None):
        import torch
        scale = self.D ** -0.5 if scale is None else scale
        x, d_q = self.queries(heads, seed)
        got = self.run(d_q, scale)
        again = self.run(d_q, scale)
        torch.cuda.synchronize()
        assert torch.equal(got, again)  # no order of arrival in the result
        want, tol, err = self.want(x, scale)
        assert int(self.err.item()) == err
        n = sum(self.q)
        assert (got[n:] == 0x1234).all()  # rows behind the last new token
        close(got, want, tol, n)


def close(got, want, tol, n):
    g = got.cpu().numpy().view(np.float16).astype(np.float64)[:n]
    bad = ~(np.abs(g - want[:n]) <= tol[:n])
    assert not bad.any(), (int(bad.sum()), g[bad][:4], want[:n][bad][:4], tol[:n][bad][:4])


def _vt(rng, T, lens, partial=0.1):
    """Blocks of full and partly filled ones, some empty."""
    return [[int(rng.integers(0, T + 1)) if rng.random() < partial else T for _ in range(n - 1)] + [int(rng.integers(1, T + 1))]
            if n else [] for n in lens]


@pytest.mark.parametrize("T,H,D,group", [(16, 8, 128, 4), (16, 2, 64, 1), (4, 2, 128, 8), (32, 1, 64, 2), (512, 1, 64, 3),
                                         (1, 2, 64, 5), (20, 3, 128, 7), (16, 6, 64, 16), (16, 1, 128, 32), (128, 4, 128, 1),
                                         (16, 16, 128, 2), (16, 1, 128, 8)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 4)])
def test_decode(hlkv_lib, cuda_device, T, H, D, group, window, sinks):
    """One new token per sequence; an empty sequence, and one without a new token."""
    rng = np.random.default_rng(T + D + group)
    scale = max(1, 48 // T)
    vt = _vt(rng, T, [n * scale if T < 512 else min(n, 3) for n in (3, 1, 0, 17, 9, 40)])
    b = Batch(hlkv_lib, T, H, D, vt, [1, 1, 0, 1, 0, 1], window=window, sinks=sinks, seed=T)
    b.check(H * group, seed=group)


@pytest.mark.parametrize("probs", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q", [1, 40])
def test_each_format(hlkv_lib, cuda_device, probs, D, q):
    rng = np.random.default_rng(D)
    b = Batch(hlkv_lib, 16, 2, D, _vt(rng, 16, [70, 5], partial=0), [q, q], probs=probs, seed=3)
    b.check(8, seed=1)


@pytest.mark.parametrize("T,H,D,group,q", [(16, 2, 128, 4, [2, 1, 3, 4]), (16, 1, 64, 8, [2, 1, 2, 1]), (16, 2, 128, 1, [16, 3, 9, 1]),
                                           (16, 2, 128, 4, [33, 1, 0, 130]), (16, 2, 64, 7, [18, 100, 1, 19]),
                                           (4, 1, 128, 8, [64, 5, 16, 17]), (64, 4, 128, 2, [200, 1, 64, 129]),
                                           (1, 1, 64, 4, [20, 1, 40, 40]), (20, 2, 128, 5, [77, 1, 26, 300]),
                                           (512, 1, 128, 3, [300, 90, 86, 1]), (16, 1, 128, 32, [9, 1, 4, 5])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (50, 3), (200, 70)])
def test_several_new_tokens(hlkv_lib, cuda_device, T, H, D, group, q, window, sinks):
    """Chunks and proposed tokens, causal inside the chunk; padded rows behind them."""
    rng = np.random.default_rng(T * D + group)
    need = [n + e for n, e in zip(q, (0, 61, 300, 7))]
    vt = []
    for n in need:
        row, left = [], n
        while left > 0:
            v = min(left, int(rng.integers(0, T + 1)) if rng.random() < 0.1 else T)
            row.append(v)
            left -= v
        vt.append(row)
    b = Batch(hlkv_lib, T, H, D, vt, q, window=window, sinks=sinks, seed=D + T, pad=5)
    b.check(H * group, seed=group)


@pytest.mark.parametrize("H,D", [(33, 128), (58, 128), (41, 64), (100, 64), (128, 128)])
@pytest.mark.parametrize("probs", [(0, 0, 0, 1), (1, 1, 1, 1)])
def test_many_heads(hlkv_lib, cuda_device, H, D, probs):
    """A token's parameters of all heads next to the codes of the last few: the ring holds fewer tiles."""
    rng = np.random.default_rng(H)
    for q in ([1, 1], [20, 1]):
        b = Batch(hlkv_lib, 16, H, D, _vt(rng, 16, [20, 45]), q, probs=probs, seed=H)
        b.check(H, seed=1)


def test_long_context_and_few_rows(hlkv_lib, cuda_device):
    """The work of one sequence spread over the GPU, at decode and with a chunk."""
    rng = np.random.default_rng(0)
    for q in (1, 3, 40):
        b = Batch(hlkv_lib, 16, 1, 128, _vt(rng, 16, [700, 2], partial=0.02), [q, 1], seed=q)
        b.check(4, seed=q)


def test_uneven_batch(hlkv_lib, cuda_device):
    rng = np.random.default_rng(4)
    lens = [300, 1, 1, 0, 2, 90, 1, 1, 1, 33] + [1] * 30
    b = Batch(hlkv_lib, 16, 2, 128, _vt(rng, 16, lens, partial=0.02), [1 if n else 0 for n in lens], seed=6)
    b.check(8, seed=2)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 5), (130, 0)])
@pytest.mark.parametrize("q", [[60], [5, 70, 1], [260, 33]])
def test_few_row_tiles_over_long_contexts(hlkv_lib, cuda_device, D, window, sinks, q):
    """A row tile's tokens split over several CTAs and joined; short contexts next to them are not."""
    rng = np.random.default_rng(D + window)
    b = Batch(hlkv_lib, 16, 2, D, _vt(rng, 16, [150, 90, 40][:len(q)], partial=0.05), q, window=window, sinks=sinks, seed=D, pad=4)
    b.check(8, seed=1)


@pytest.mark.parametrize("value", [np.nan, np.inf, 65504.0])
def test_hidden_tokens_do_not_matter_when_split(hlkv_lib, cuda_device, value):
    import torch
    T, H, D = 16, 1, 128
    q, ctx = [40], [2400]
    b = Batch(hlkv_lib, T, H, D, [[16] * 150], q, probs=(1, 0, 0, 0), seed=9)
    _poke(b.wl, None, {(0, ctx[0] - q[0] + r): value for r in (20, 39)})
    x, d_q = b.queries(4, 1)
    got = b.run(d_q, D ** -0.5)
    torch.cuda.synchronize()
    g = got.cpu().numpy().view(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol, _ = b.want(x, D ** -0.5)
    assert np.isfinite(want[:20]).all() and (np.abs(g - want)[:20] <= tol[:20]).all()
    if not np.isfinite(value):
        assert not np.isfinite(g[20:]).all(-1).any()


@pytest.mark.parametrize("nseq", [128, 129])
@pytest.mark.parametrize("window", [0, 40])
def test_many_sequences_of_many_rows(hlkv_lib, cuda_device, nseq, window):
    """Both orders of the tiles' CTAs: every row of every sequence once, next to short ones and absent ones."""
    rng = np.random.default_rng(nseq)
    q = [int(rng.choice([0, 1, 5, 17, 40, 140])) for _ in range(nseq)]
    vt = [[16] * (n // 16 + int(rng.integers(0, 6))) + [n % 16 or 16] for n in q]
    b = Batch(hlkv_lib, 16, 1, 64, vt, q, window=window, sinks=3 if window else 0, seed=nseq, pad=3)
    b.check(3, seed=1)


@pytest.mark.parametrize("q", [[30], [200, 17], [17, 0, 20]])
def test_no_sequence_of_few_rows(hlkv_lib, cuda_device, q):
    """Nothing for the streaming kernel to do."""
    rng = np.random.default_rng(len(q))
    b = Batch(hlkv_lib, 16, 1, 128, _vt(rng, 16, [20] * len(q), partial=0), q, seed=2)
    b.check(32, seed=1)


@pytest.mark.parametrize("group", [4, 32])
def test_plan_larger_than_its_batch(hlkv_lib, cuda_device, group):
    """A plan made for prompts that holds a decode step, and one with room for many more tokens."""
    import torch
    rng = np.random.default_rng(3)
    for q in ([1, 1, 1], [1, 60, 2]):
        b = Batch(hlkv_lib, 16, 1, 64, _vt(rng, 16, [20, 9, 30], partial=0), q, seed=2, pad=500)
        b.plan = hlkv_lib.BatchPlan(3, b.plan.c.block_cap + 70, b.cap, 8192, 0, 0)
        b.fill_plan()
        x, d_q = b.queries(group, 1)
        got = b.run(d_q, 0.125)
        torch.cuda.synchronize()
        want, tol, err = b.want(x, 0.125)
        assert int(b.err.item()) == err == 0
        close(got, want, tol, sum(q))
        assert (got[sum(q):] == 0x1234).all()


def _poke(wl, rng, what):
    """Overwrites cached rows: what = {(seq, position): value} in FP16 blocks of full tokens."""
    buf, sb, _ = wl.pools[0]
    host = buf.cpu().numpy()
    T, H, D = wl.T, wl.H, wl.D
    for (i, pos), value in what.items():
        ids = wl.table.sequence_block_ids(wl.seqs[i])[1]
        slot = wl.table.device_descriptor(ids[pos // T])[0]
        rows = host[slot, :4 * T * H * D].view(np.float16).reshape(2, T, H, D)
        rows[:, pos % T] = value
    import torch
    buf.copy_(torch.from_numpy(host))


@pytest.mark.parametrize("q,group", [([1, 2], 2), ([4, 1], 4), ([40, 33], 4), ([3, 150], 8)])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf, 65504.0])
def test_hidden_tokens_do_not_matter(hlkv_lib, cuda_device, q, group, value):
    """NaN and infinities behind the window and behind the causal border: rows that do not see them are
    as if they were not there."""
    import torch
    T, H, D, window, sinks = 16, 2, 128, 24, 2
    vt = [[16] * 14, [16] * 15]
    b = Batch(hlkv_lib, T, H, D, vt, q, probs=(1, 0, 0, 0), window=window, sinks=sinks, seed=9)
    ctx = [224, 240]
    bad = {}
    for i in range(2):
        for r in {q[i] // 2, q[i] - 1} - {0}:
            bad[i, ctx[i] - q[i] + r] = value  # a new token: earlier ones do not see it
        bad[i, sinks] = value                     # between the sinks and every window
        bad[i, ctx[i] - q[i] - window] = value
        if q[i] > 8:
            bad[i, ctx[i] - q[i] - window + 2] = value  # the first new tokens see it, later ones do not
    _poke(b.wl, None, bad)
    x, d_q = b.queries(H * group, 1)
    got = b.run(d_q, D ** -0.5)
    torch.cuda.synchronize()
    g = got.cpu().numpy().view(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol, _ = b.want(x, D ** -0.5)
    row, clean, seen_bad = 0, np.zeros(len(x), bool), 0
    for i in range(2):
        for r in range(q[i]):
            p = ctx[i] - q[i] + r
            hit = [t for (s, t) in bad if s == i and t <= p and (p - t < window or t < sinks)]
            clean[row] = not hit
            seen_bad += bool(hit)
            row += 1
    assert clean.any()
    assert np.isfinite(want[clean]).all() and (np.abs(g - want)[clean] <= tol[clean]).all()
    if not np.isfinite(value) and seen_bad:
        assert not np.isfinite(g[~clean]).all(-1).any()  # and the others do see them


def test_unused_rows_of_blocks_do_not_matter(hlkv_lib, cuda_device):
    """Rows behind a block's valid tokens hold anything (here all bits set: NaN codes and parameters)."""
    import torch

    def change(wl):
        for f, (buf, sb, ns) in wl.pools.items():
            host = buf.cpu().numpy()
            T, H, D = wl.T, wl.H, wl.D
            rb, pb = {0: (2 * D, 0), 1: (D, 4), 2: (D, 4), 3: (D // 2, 8)}[f]
            for i in range(wl.table.max_blocks()):
                slot, info, _, _ = wl.table.device_descriptor(i)
                if info & 15 != f:
                    continue
                v = info >> 10
                codes = host[slot, :2 * T * H * rb].reshape(2, T, H * rb)
                codes[:, v:] = 0xFF
                par = host[slot, 2 * T * H * rb:2 * T * H * (rb + pb)].reshape(2, T, H * pb)
                par[:, v:] = 0xFF
            buf.copy_(torch.from_numpy(host))

    rng = np.random.default_rng(2)
    for q in ([1, 1, 1], [50, 2, 9]):
        b = Batch(hlkv_lib, 16, 2, 128, _vt(rng, 16, [9, 4, 30], partial=0.5), [min(a, 1) if a == 1 else a for a in q], seed=1,
                  change=change)
        b.check(8, seed=3)


def test_block_wide_scales(hlkv_lib, cuda_device):
    from helpers import block_wide_scale_refs
    rng = np.random.default_rng(12)

    def change(wl):
        ids = [b for s in wl.seqs for b in wl.table.sequence_block_ids(s)[1]]
        for k, (bid, ref) in enumerate(zip(ids, block_wide_scale_refs(rng, len(ids), moderate=True))):
            if k % 3 != 2:
                assert wl.table.set_scale(wl.table.handle_of(bid), *ref) == 0
        wl.dt.sync(wl.table)

    for q in ([1, 1, 1, 1], [60, 1, 30, 2]):
        b = Batch(hlkv_lib, 16, 2, 64, _vt(rng, 16, [6, 13, 2, 21]), q, probs=(0.2, 0.4, 0, 0.4), seed=8, change=change)
        b.check(8, seed=3)


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -6, 300.0])
def test_scales_far_from_one(hlkv_lib, cuda_device, size):
    """Keys and values much smaller or larger than 1: binary16 weights keep their precision."""
    def change(wl):
        import torch
        for f, (buf, sb, ns) in wl.pools.items():
            rows, D = 2 * wl.T * wl.H, wl.D
            if f == 0:
                v = buf[:, :rows * D * 2].contiguous().view(torch.float16)
                buf[:, :rows * D * 2] = (v.float() * size / 4).to(torch.float16).view(torch.uint8)
            else:
                at = rows * (D // 2 if f == 3 else D)
                n = rows * (8 if f == 3 else 4)
                p = buf[:, at:at + n].contiguous().view(torch.float32)
                buf[:, at:at + n] = (p * size).contiguous().view(torch.uint8)

    rng = np.random.default_rng(1)
    for q in ([1, 1], [70, 2]):
        for probs in ((0, 1, 1, 0), (0, 0, 0, 1), (0, 1, 1, 2)):
            b = Batch(hlkv_lib, 16, 1, 128, _vt(rng, 16, [30, 8]), q, probs=probs, seed=4, change=change)
            b.check(4, seed=3, scale=min(2.0, 0.09 / size))


def test_strided_rows_and_streams(hlkv_lib, cuda_device):
    """Q as a slice of a fused projection, out inside a wider array, and a stream of its own."""
    import torch
    rng = np.random.default_rng(3)
    for q in ([1, 1, 1], [30, 1, 70]):
        b = Batch(hlkv_lib, 16, 2, 64, _vt(rng, 16, [9, 3, 12], partial=0), q, seed=5)
        wide = torch.from_numpy(rng.standard_normal((b.cap, 14, 64)).astype(np.float16).view(np.int16)).cuda()
        out = torch.full((b.cap, 12, 64), 0x1234, dtype=torch.int16, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        b.fill_plan(stream=s)
        ws = b.workspace(8)
        torch.cuda.synchronize()
        b.run(wide[:, 2:10], 0.1, out=out[:, 1:9], ws=ws, stream=s)
        s.synchronize()
        want, tol, _ = b.want(wide[:, 2:10].cpu().numpy().view(np.float16), 0.1)
        close(out[:, 1:9].contiguous(), want, tol, b.cap)
        assert (out[:, :1] == 0x1234).all() and (out[:, 9:] == 0x1234).all()


def test_missing_pools_and_slots(hlkv_lib, cuda_device):
    """Listed blocks whose pool or slot does not exist are left out, with their bits."""
    import torch
    rng = np.random.default_rng(7)
    for q in ([1, 1], [40, 20]):
        b = Batch(hlkv_lib, 16, 2, 64, _vt(rng, 16, [12, 6], partial=0), q, seed=2)
        pools = b.wl.hlkv_pools()
        pools.pool[1].base = None
        pools.pool[3].num_slots = 1
        x, d_q = b.queries(4, 1)
        out = torch.zeros_like(d_q)
        b.hlkv.batch_attention(pools, b.wl.layout, b.plan, d_q, 0.1, out, b.err, workspace=b.workspace(4))
        torch.cuda.synchronize()
        assert int(b.err.item()) == (1 << 1 | 1 << 2)
        wl = b.wl
        seqs, _, _, tf, _, _ = plan_oracle(wl.segs_host, q, device_arena(wl), device_table_words(wl), 16, 1, 18, b.cap,
                                           max(q), 0, 0)
        for s in seqs:
            s["blocks"] = [r for r in s["blocks"] if r[1] & 15 in (0, 2) or (r[1] & 15 == 3 and r[0] == 0)]
        want, tol = attention_oracle(seqs, tf, host_pools(wl), 16, 2, 64, x.astype(np.float64), 0.1, 0, 0)
        close(out, want, tol, b.cap)


def test_a_layers_step_together_in_a_graph(hlkv_lib, cuda_device):
    """Plan, rotary append and attention as one captured step of a mixed batch, replayed after the batch
    has changed; against the plain forms of the same step, and equal to the eager calls."""
    import torch
    from batch_helpers import rotate
    T, H, D, heads = 16, 2, 64, 6
    rng = np.random.default_rng(11)
    vt = [[16] * 6 + [9], [16, 16, 3], [16] * 20]
    q = [25, 1, 7]
    b = Batch(hlkv_lib, T, H, D, vt, q, window=100, sinks=4, seed=5, pad=8)
    wl, cap = b.wl, b.cap
    qkv = torch.zeros((cap, heads + 2 * H, D), dtype=torch.int16, device="cuda")
    q_rot = torch.zeros((cap, heads, D), dtype=torch.int16, device="cuda")
    out = torch.full_like(q_rot, 0x1234)
    rope = hlkv_lib.make_rotary([float(np.float32(10000.0 ** (-j / 32))) for j in range(32)])
    ws = b.workspace(heads)
    pools = wl.hlkv_pools()

    def step():
        b.fill_plan()
        hlkv_lib.rotary_append(pools, wl.layout, wl.dt.table_ptr, wl.dt.table_size, b.plan.targets, rope, b.plan.positions,
                               qkv[:, :heads], qkv[:, heads:heads + H], qkv[:, heads + H:], q_rot, b.err)
        hlkv_lib.batch_attention(pools, wl.layout, b.plan, q_rot, D ** -0.5, out, b.err, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in (q, [1, 1, 33], [0, 2, 25]):
        b.q = lens
        b.qlens.copy_(torch.tensor(lens, dtype=torch.int32))
        b.plan.c.max_query  # the plan's bound stays what it was captured with
        x = rng.standard_normal((cap, heads + 2 * H, D)).astype(np.float16)
        qkv.copy_(torch.from_numpy(x.view(np.int16)))
        if max(lens) > b.plan.c.max_query:
            lens = [min(n, b.plan.c.max_query) for n in lens]
            b.q = lens
            b.qlens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(0x1234)
        graph.replay()
        torch.cuda.synchronize()
        assert int(b.err.item()) == 0
        replayed = out.clone()
        n = sum(lens)
        assert (replayed[n:] == 0x1234).all()
        pos = np.concatenate([np.arange(sum(v) - k, sum(v)) for v, k in zip(vt, lens)]).astype(np.float64)
        angle = pos[:, None] * np.array([rope.inv_freq[j] for j in range(32)])
        want_q = rotate(x[:n, :heads].astype(np.float64), angle, False)
        got_q = q_rot.cpu().numpy().view(np.float16).astype(np.float64)
        assert (np.abs(got_q[:n] - want_q) <= 2.0 ** -11 * np.abs(want_q) + 2.0 ** -20 * np.abs(x).max()).all()
        want, tol, _ = b.want(got_q.astype(np.float16), D ** -0.5)
        close(replayed, want, tol, n)
        out.fill_(0x1234)
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)
