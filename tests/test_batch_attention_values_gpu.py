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
