"""hlkv_batch_attention on caches whose keys and values are chosen: scores that climb inside a tile of tokens.  The
error bound of every value is counted in batch_helpers.attention_oracle."""
import numpy as np
import pytest

from test_batch_attention_gpu import Batch, close

pytestmark = pytest.mark.gpu


def put_rows(wl, i, k, v):
    """Writes binary16 K and V rows [tokens, H, D] into sequence i's FP16 blocks of full tokens."""
    import torch
    buf = wl.pools[0][0]
    host = buf.cpu().numpy()
    T, H, D = wl.T, wl.H, wl.D
    for j, bid in enumerate(wl.table.sequence_block_ids(wl.seqs[i])[1]):
        slot = wl.table.device_descriptor(bid)[0]
        rows = host[slot, :4 * T * H * D].view(np.float16).reshape(2, T, H, D)
        rows[0], rows[1] = k[j * T:(j + 1) * T], v[j * T:(j + 1) * T]
    buf.copy_(torch.from_numpy(host))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", [9.0, 30.0])
@pytest.mark.parametrize("ctx", [128, 400])
def test_maximum_climbs_in_every_group_of_a_tile(hlkv_lib, cuda_device, D, step, ctx):
    """Every 32 tokens the scores rise by `step` powers of two: in the first tile, where there is no output yet, and in
    the later ones the weights made so far are scaled each time, some of them three times."""
    rng = np.random.default_rng(D)
    q, group = [40], 4
    b = Batch(hlkv_lib, 16, 1, D, [[16] * (ctx // 16)], q, probs=(1, 0, 0, 0), seed=1)
    x = (0.5 + rng.random((b.cap, group, D))).astype(np.float16)  # sums near D
    scale = step * np.log(2.0) / D
    k = np.repeat(np.arange(ctx) % 128 // 32 + rng.uniform(-0.05, 0.05, ctx), D).reshape(ctx, 1, D).astype(np.float16)
    put_rows(b.wl, 0, k, rng.standard_normal((ctx, 1, D)).astype(np.float16))
    import torch
    got = b.run(torch.from_numpy(x.view(np.int16)).cuda(), scale)
    torch.cuda.synchronize()
    want, tol, err = b.want(x, scale)
    assert int(b.err.item()) == err == 0
    close(got, want, tol, q[0])


@pytest.mark.parametrize("D", [64, 128])
def test_weights_keep_their_sum_when_the_maximum_moves(hlkv_lib, cuda_device, D):
    """64 tokens of exact weights (scores 0 and 7, values 1), then a token of value 0 whose score passes the maximum: the
    factor that scales the weights of this tile scales their sum, so all that is rounded is the result."""
    import torch
    y = np.arange(8 + 1 / 16, 9, 2.0 ** -7)  # binary16 values
    a = np.exp2(-y)
    y = y[np.argmax(np.abs(a.astype(np.float16).astype(np.float64) / a - 1))]  # the factor that binary16 holds worst
    ctx, q = 176, [40]
    b = Batch(hlkv_lib, 16, 1, D, [[16] * (ctx // 16)], q, probs=(1, 0, 0, 0), seed=1)
    k, v = np.zeros((ctx, 1, D), np.float16), np.ones((ctx, 1, D), np.float16)
    k[32:64, :, 0], k[64:, :, 0], k[70, :, 0], v[70] = 7, -60, y, 0
    put_rows(b.wl, 0, k, v)
    x = np.zeros((b.cap, 4, D), np.float16)
    x[..., 0] = 1
    got = b.run(torch.from_numpy(x.view(np.int16)).cuda(), np.log(2.0))
    torch.cuda.synchronize()
    g = got.cpu().numpy().view(np.float16).astype(np.float64)
    s = k[:, 0, 0].astype(np.float64)
    want = (np.exp2(s) * v[:, 0, 0]).sum() / np.exp2(s).sum()
    assert 0.5 < want < 1 and np.abs(g - want).max() <= 2.0 ** -12 + 2.0 ** -18


def _value_rows(wl, f):
    """(slots of all of format f, codes [slots, T, H, row bytes], parameters [slots, T, H, floats]) of the V rows, on the
    host; the arrays are views of what `_write` puts back."""
    T, H, D = wl.T, wl.H, wl.D
    rb, n = {1: (D, 1), 2: (D, 1), 3: (D // 2, 2)}[f]
    host = wl.pools[f][0].cpu().numpy()
    rows = T * H
    codes = host[:, rows * rb:2 * rows * rb].reshape(-1, T, H, rb)
    at = 2 * rows * rb + rows * n * 4
    par = host[:, at:at + rows * n * 4].view(np.float32).reshape(-1, T, H, n)
    return host, codes, par


def _write(wl, f, host):
    import torch
    wl.pools[f][0].copy_(torch.from_numpy(host))


def by_weight(b, x, scale):
    """(out, bound) as attention_oracle's, with the part of weights below binary16's normal range counted against the
    row's largest weighted value instead of its largest value.  A weight below the range is off by 2^-25 at most, its codes
    in their unit are 1.75 at most, and a row's largest value is half its scale's unit at least.  The streaming kernel
    keeps the largest weight at 2^6 or more: 2^-25 * 1.75 * 2 / 2^6 = 2^-29 of the largest weighted value.  The tile kernel keeps
    it at 2^5, and less by the 2^6 that 16 tokens' scales may lie apart without being told apart: 2^-22.  Both are
    below what is allowed, 2^-24 for each visible token, from 4 tokens on; and fewer tokens than 4 have no such weights
    in these caches."""
    from batch_helpers import block_rows, plan_oracle
    from helpers import device_arena, device_table_words, host_pools
    wl = b.wl
    seqs, _, _, tf, _, err = plan_oracle(wl.segs_host, b.q, device_arena(wl), device_table_words(wl), b.T, 1, b.plan.c.block_cap,
                                         b.cap, b.plan.c.max_query, b.window, b.sinks)
    assert err == 0
    pools, g = host_pools(wl), x.shape[1] // b.H
    out, tol = np.zeros(x.shape), np.zeros(x.shape)
    for i, s in enumerate(seqs):
        rows = [block_rows(pools[info & 15], info & 15, slot, b.T, b.H, b.D)[0][:, :info >> 10 & 0x3FF] for slot, info, _, _ in s["blocks"]]
        K, V = np.concatenate([r[0] for r in rows]), np.concatenate([r[1] for r in rows])
        t = np.concatenate([start + np.arange(info >> 10 & 0x3FF) for _, info, _, start in s["blocks"]])
        for r in range(s["q"]):
            p = s["context"] - s["q"] + r
            see = (t <= p) & ((b.window == 0) | (p - t < b.window) | (t < b.sinks))
            for qh in range(x.shape[1]):
                k, v, y = K[see, qh // g], V[see, qh // g], x[tf[i] + r, qh].astype(np.float64)
                sc = scale * (k @ y)
                w = np.exp(sc - sc.max())
                w /= w.sum()
                big = np.abs(v).max(1)
                ds = scale * b.D * 2.0 ** -23 * (np.abs(k) @ np.abs(y)).max()
                out[tf[i] + r, qh] = w @ v
                tol[tf[i] + r, qh] = (2.0 ** -11 * np.abs(w @ v) + (2.0 ** -11 + 2 * ds) * 16 / 15 * (w @ big)
                                      + len(v) * 2.0 ** -24 * (w * big).max() + 2.0 ** -25)
    return out, tol


def _attend(b, heads, scale):
    import torch
    x, d_q = b.queries(heads, 1)
    got = b.run(d_q, scale)
    again = b.run(d_q, scale)
    torch.cuda.synchronize()
    assert torch.equal(got, again) and int(b.err.item()) == 0
    want, tol = by_weight(b, x, scale)
    close(got, want, tol, sum(b.q))


ROWS = [[1, 1], [3, 4], [70, 40]]  # new tokens: up to 8 rows, up to 16, row tiles


@pytest.mark.parametrize("sigma", [1.0, 0.1, 0.01])
@pytest.mark.parametrize("f", [1, 2])
@pytest.mark.parametrize("q", ROWS)
@pytest.mark.parametrize("zeros", ["one of 16", "tiles"])
def test_value_rows_of_zeros(hlkv_lib, cuda_device, sigma, f, q, zeros):
    """Encoders give a row of zeros the scale 1, far above its neighbours'."""
    def change(wl):
        host, codes, par = _value_rows(wl, f)
        par *= np.float32(sigma)
        which = (slice(None), slice(5, 6)) if zeros == "one of 16" else (slice(0, None, 3), slice(None))
        codes[which], par[which] = 0, 1.0
        codes[which][..., ::2] = 0x80  # of both signs
        _write(wl, f, host)

    probs = [0, 0, 0, 0]
    probs[f] = 1
    b = Batch(hlkv_lib, 16, 2, 128, [[16] * 40, [16] * 21 + [9]], q, probs=probs, seed=5, change=change)
    _attend(b, 8, 128 ** -0.5)


@pytest.mark.parametrize("probs", [(0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 1, 1)])
@pytest.mark.parametrize("q", ROWS)
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("by", ["token", "block"])
def test_value_scales_far_apart(hlkv_lib, cuda_device, probs, q, window, by):
    """Value rows of 2^-14 to 2^6 side by side, and blocks of them, under flat scores and steep ones: the rows with much
    weight may be the small ones."""
    rng = np.random.default_rng(sum(q))

    def change(wl):
        for f in (1, 2, 3):
            if not probs[f]:
                continue
            host, _, par = _value_rows(wl, f)
            size = rng.uniform(-14, 6, par.shape[:3] if by == "token" else (par.shape[0], 1, 1))
            par *= np.float32(2.0) ** size[..., None].astype(np.float32)
            par[rng.random(par.shape[:3]) < 0.02] = 0  # constant rows of 0
            _write(wl, f, host)

    for D, scale in ((128, 128 ** -0.5), (64, 0.5)):
        b = Batch(hlkv_lib, 16, 2, D, [[16] * 40, [16] * 21 + [9]], q, probs=probs, window=window, sinks=5 if window else 0, seed=7,
                  change=change)
        _attend(b, 8, scale)


@pytest.mark.parametrize("q", [[1], [3], [40]])
@pytest.mark.parametrize("hidden", [16, 48, 200])
def test_scores_of_minus_infinity(hlkv_lib, cuda_device, q, hidden):
    """Keys whose scores are minus infinity, from the first token on: weights of 0, as if they were hidden."""
    import torch
    ctx, D = 256, 64
    b = Batch(hlkv_lib, 16, 1, D, [[16] * (ctx // 16)], q, probs=(1, 0, 0, 0), seed=1)
    rng = np.random.default_rng(hidden)
    k, v = np.zeros((ctx, 1, D), np.float16), rng.standard_normal((ctx, 1, D)).astype(np.float16)
    k[:hidden, :, 0] = -np.inf
    put_rows(b.wl, 0, k, v)
    x = np.zeros((b.cap, 4, D), np.float16)
    x[..., 0] = 1
    got = b.run(torch.from_numpy(x.view(np.int16)).cuda(), 1.0)
    torch.cuda.synchronize()
    g = got.cpu().numpy().view(np.float16).astype(np.float64)
    for r in range(q[0]):
        seen = v[hidden:ctx - q[0] + r + 1, 0].astype(np.float64)  # of equal weight
        # the weights are powers of two; the result's rounding, and the sums'
        assert (np.abs(g[r] - seen.mean(0)) <= 2.0 ** -11 * np.abs(seen.mean(0)) + 2.0 ** -16 * np.abs(seen).mean(0)).all()


@pytest.mark.parametrize("probs", [(0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 1, 1)])
@pytest.mark.parametrize("window", [0, 1500])
@pytest.mark.parametrize("q", [[1], [40]])
def test_value_scales_far_apart_when_split(hlkv_lib, cuda_device, probs, window, q):
    """Parts of a row's tokens on several CTAs, some of them with nothing but zeros, joined."""
    rng = np.random.default_rng(window)

    def change(wl):
        ids = wl.table.sequence_block_ids(wl.seqs[0])[1]
        where = {f: [] for f in (1, 2, 3)}
        for j, bid in enumerate(ids):
            slot, info, _, _ = wl.table.device_descriptor(bid)
            where[info & 15].append((slot, j))
        for f, slots in where.items():
            if not slots:
                continue
            host, codes, par = _value_rows(wl, f)
            for slot, j in slots:
                par[slot] *= np.float32(2.0) ** np.float32(rng.uniform(-12, 4))
                if 60 <= j < 110:  # 800 tokens of zeros
                    codes[slot], par[slot] = 0, 0.0 if f == 3 else 1.0
            _write(wl, f, host)

    b = Batch(hlkv_lib, 16, 1, 128, [[16] * 150], q, probs=probs, window=window, sinks=5 if window else 0, seed=7, change=change)
    _attend(b, 4, 128 ** -0.5)
