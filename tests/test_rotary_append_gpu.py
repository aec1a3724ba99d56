"""hlkv_rotary_append: rotated Q against 64 bits, and every byte of the pools against a plain encoding
of the rotated K (binary32) and of V."""
import numpy as np
import pytest

from batch_helpers import E4M3, E5M2, FP16, INT4, PAD, rotate
from helpers import device_table_words, host_pools

pytestmark = pytest.mark.gpu


def _freqs(n, base=10000.0):
    return np.array([base ** (-j / n) for j in range(n)], np.float32)


def _rotated32(x, angle, interleaved):
    """The same in binary32, operation by operation (x float32)."""
    r = angle.shape[1]
    c, s = np.cos(angle).astype(np.float32)[:, None], np.sin(angle).astype(np.float32)[:, None]
    y = x.copy()
    ia, ib = (np.arange(0, 2 * r, 2), np.arange(1, 2 * r, 2)) if interleaved else (np.arange(r), np.arange(r, 2 * r))
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def _encode_row(x, f):
    """(code bytes, parameter bytes) of one binary32 row."""
    import torch
    if f == FP16:
        return x.astype(np.float16).view(np.uint8), np.empty(0, np.uint8)
    if f == INT4:
        lo, hi = x.min(), x.max()
        scale = np.float32((hi - lo) * (np.float32(1) / np.float32(15)))
        q = np.clip(np.rint((x - lo) / scale), 0, 15).astype(np.uint8) if scale > 0 else np.zeros(x.size, np.uint8)
        return q[0::2] | q[1::2] << 4, np.array([scale, lo], np.float32).view(np.uint8)
    top = np.float32(448 if f == E4M3 else 57344)
    amax = np.abs(x).max()
    scale = max(np.float32(amax * (np.float32(1) / top)), np.finfo(np.float32).tiny) if amax > 0 else np.float32(1)
    y = torch.from_numpy((x / scale).astype(np.float32)).to(torch.float8_e4m3fn if f == E4M3 else torch.float8_e5m2)
    return y.view(torch.uint8).numpy(), np.array([scale], np.float32).view(np.uint8)


def _store(pools, table, T, H, D, target, rows):
    """rows: binary32 [2, H, D] into the host pools."""
    bid, tok = int(target[0]), int(target[1])
    f, slot = int(table[bid, 1]) & 15, int(table[bid, 0])
    buf, sb, _ = pools[f]
    rb = {FP16: 2 * D, E4M3: D, E5M2: D, INT4: D // 2}[f]
    pb = {FP16: 0, E4M3: 4, E5M2: 4, INT4: 8}[f]
    cb = 2 * T * H * rb
    for kv in range(2):
        for h in range(H):
            if not np.isfinite(rows[kv, h]).all() and f != FP16:
                continue
            row = (kv * T + tok) * H + h
            codes, par = _encode_row(rows[kv, h], f)
            buf[slot * sb + row * rb:slot * sb + (row + 1) * rb] = codes
            buf[slot * sb + cb + row * pb:slot * sb + cb + (row + 1) * pb] = par


def _setup(T, H, D, n, seed):
    from hlkv.workload import build_workload
    rng = np.random.default_rng(seed)
    fm = [list(rng.permutation([0, 1, 2, 3] * 3)), [3, 1, 2, 0]]
    wl = build_workload(fm, T=T, H=H, D=D, seed=seed, valid_tokens=[[T] * 12, [T] * 4], outlier_channels=0)
    ids = [b for s in wl.seqs for b in wl.table.sequence_block_ids(s)[1]]
    pairs = [(b, t) for b in ids for t in range(T)]
    pick = rng.permutation(len(pairs))[:n]
    return wl, rng, np.array([pairs[k] for k in pick], np.uint32)


@pytest.mark.parametrize("T,H,D,heads,n,rot,interleaved,axes", [
    (16, 8, 128, 32, 37, 128, False, 1), (16, 2, 64, 2, 5, 64, False, 3), (4, 3, 128, 21, 16, 128, True, 1),
    (16, 1, 256, 4, 33, 256, False, 2), (5, 2, 64, 6, 13, 32, True, 3), (16, 2, 128, 8, 9, 64, False, 1),
    (16, 2, 256, 2, 8, 48, False, 4), (16, 4, 64, 4, 1, 16, False, 1), (2, 2, 256, 6, 20, 96, True, 1),
    (16, 4, 128, 0, 21, 128, False, 1), (16, 2, 128, 2, 200, 128, False, 2),
])
def test_rotary_append(hlkv_lib, cuda_device, T, H, D, heads, n, rot, interleaved, axes):
    import torch
    wl, rng, targets = _setup(T, H, D, n, seed=T + D + n)
    n = len(targets)
    table = np.array([wl.table.device_descriptor(i) for i in range(wl.table.max_blocks())], np.uint32)
    pair_axis = rng.integers(0, axes, rot // 2)
    pair_axis[:axes] = np.arange(axes)
    freq = _freqs(rot // 2)
    pos = rng.integers(0, 1 << 20, (axes, n)).astype(np.int32)
    pos[:, 0] = 0
    pos[-1, -1] = -5
    if n > 4:
        pos[:, 1:3] = [[(1 << 29) - 1], ] * axes
    x = (rng.standard_normal((n, heads + 2 * H + 1, D)) * rng.choice([0.01, 1, 40], (n, heads + 2 * H + 1, 1))).astype(np.float16)
    d = torch.from_numpy(x.view(np.int16)).cuda()
    q, k, v = d[:, :heads], d[:, heads:heads + H], d[:, heads + H:heads + 2 * H]  # one row of the projection is not ours
    q_out = torch.full((n, heads + 1, D), 0x1234, dtype=torch.int16, device="cuda")
    d_pos = torch.from_numpy(pos).cuda().t()  # axis-major: strided
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    rope = hlkv_lib.make_rotary(freq, axes=axes, pair_axis=pair_axis, interleaved=interleaved)
    before = host_pools(wl)
    d_targets = torch.from_numpy(targets.view(np.int32)).cuda()
    for _ in range(2):
        hlkv_lib.rotary_append(wl.hlkv_pools(), wl.layout, wl.dt.table_ptr, wl.dt.table_size, d_targets, rope,
                               d_pos, q if heads else None, k, v, q_out[:, :heads] if heads else None, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    angle = np.stack([pos[a].astype(np.float64) * float(f) for a, f in zip(pair_axis, freq)], 1)
    x64 = x.astype(np.float64)
    want = rotate(x64[:, :heads + H], angle, interleaved)
    got = q_out.cpu().numpy()
    assert (got[:, heads] == 0x1234).all()
    # three binary32 roundings per product sum (cos or sin, the product, the sum), then binary16's
    size = rotate(np.abs(x64[:, :heads + H]), np.zeros_like(angle), interleaved)
    mag = np.abs(size) + np.abs(x64[:, :heads + H]).max(-1, keepdims=True)
    tol = 2.0 ** -11 * np.abs(want) + 3 * 2.0 ** -24 * 2 * mag + 2.0 ** -25
    if heads:
        diff = np.abs(got[:, :heads].view(np.float16).astype(np.float64) - want[:, :heads])
        assert (diff <= tol[:, :heads]).all()
    k32 = _rotated32(x[:, heads:heads + H].astype(np.float32), angle, interleaved)
    v32 = x[:, heads + H:heads + 2 * H].astype(np.float32)
    for i in range(n):
        _store(before, table, T, H, D, targets[i], np.stack((k32[i], v32[i])))
    after = host_pools(wl)
    for f in before:
        bad = np.nonzero(after[f][0] != before[f][0])[0]
        assert bad.size == 0, (f, bad.size, bad[:4])


def test_in_place_and_padding(hlkv_lib, cuda_device):
    """d_q_out == d_q, with and without partners in other lanes; padding rows are left as they were."""
    import torch
    T, H, D, heads, n = 16, 2, 128, 6, 30
    for rot, interleaved in ((128, False), (64, False), (96, False), (64, True)):
        wl, rng, targets = _setup(T, H, D, n, seed=rot)
        targets[[3, n - 1]] = PAD
        before = host_pools(wl)
        x = rng.standard_normal((n, heads + 2 * H, D)).astype(np.float16)
        d = torch.from_numpy(x.view(np.int16)).cuda()
        pos = torch.arange(n, dtype=torch.int32, device="cuda") + 7
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        rope = hlkv_lib.make_rotary(_freqs(rot // 2), interleaved=interleaved)
        args = (wl.hlkv_pools(), wl.layout, wl.dt.table_ptr, wl.dt.table_size, torch.from_numpy(targets.view(np.int32)).cuda(),
                rope, pos)
        out = torch.zeros((n, heads, D), dtype=torch.int16, device="cuda")
        q, k, v = d.split((heads, H, H), 1)
        hlkv_lib.rotary_append(*args, q, k, v, out, err)
        once = host_pools(wl)
        hlkv_lib.rotary_append(*args, q, k, v, q, err)
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        out[[3, n - 1]] = torch.from_numpy(x[[3, n - 1], :heads].view(np.int16)).cuda()
        assert torch.equal(d[:, :heads], out)
        changed = sum(int((once[f][0] != before[f][0]).sum()) for f in once)
        assert changed > 0 and all(np.array_equal(once[f][0], host_pools(wl)[f][0]) for f in once)


def test_bad_targets_and_values(hlkv_lib, cuda_device):
    import torch
    T, H, D = 16, 2, 64
    wl, rng, targets = _setup(T, H, D, 8, seed=1)
    table = np.array([wl.table.device_descriptor(i) for i in range(wl.table.max_blocks())], np.uint32)
    targets[0] = (wl.dt.table_size, 0)           # no such block
    targets[1, 1] = T                            # no such token
    targets[2] = (PAD, 3)                        # half a padding target is no padding
    x = rng.standard_normal((8, 3 * H, D)).astype(np.float16)
    x[4, H, 7] = np.inf                          # a K row and a V row that no quantized block takes
    x[5, 2 * H + 1, 0] = np.nan
    d = torch.from_numpy(x.view(np.int16)).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = host_pools(wl)
    q, k, v = d.split((H, H, H), 1)
    out = torch.zeros((8, H, D), dtype=torch.int16, device="cuda")
    fr = _freqs(D // 2)
    hlkv_lib.rotary_append(wl.hlkv_pools(), wl.layout, wl.dt.table_ptr, wl.dt.table_size,
                           torch.from_numpy(targets.view(np.int32)).cuda(), hlkv_lib.make_rotary(fr),
                           torch.arange(8, dtype=torch.int32, device="cuda"), q, k, v, out, err)
    torch.cuda.synchronize()
    quantized = any(int(table[int(t[0]), 1]) & 15 for t in targets[4:6])
    assert int(err.item()) == (1 << 4 | 1 << 10 | (1 << 9 if quantized else 0))
    angle = np.arange(8.0)[:, None] * fr.astype(np.float64)
    k32 = _rotated32(x[:, H:2 * H].astype(np.float32), angle, False)
    for i in range(3, 8):
        if i in (4, 5) and int(table[int(targets[i, 0]), 1]) & 15 == 0:
            continue
        _store(before, table, T, H, D, targets[i], np.stack((k32[i], x[i, 2 * H:].astype(np.float32))))
    after = host_pools(wl)
    for f in before:
        if f != 0:
            assert np.array_equal(after[f][0], before[f][0]), f
    assert (out.cpu().numpy()[0] != 0).any()  # Q is written all the same


def test_factor_scales_the_rotation(hlkv_lib, cuda_device):
    import torch
    T, H, D = 16, 2, 64
    wl, rng, targets = _setup(T, H, D, 4, seed=2)
    x = rng.standard_normal((4, 3 * H, D)).astype(np.float16)
    d = torch.from_numpy(x.view(np.int16)).cuda()
    q, k, v = d.split((H, H, H), 1)
    out = torch.zeros((4, H, D), dtype=torch.int16, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    fr = _freqs(16)
    hlkv_lib.rotary_append(wl.hlkv_pools(), wl.layout, wl.dt.table_ptr, wl.dt.table_size,
                           torch.from_numpy(targets.view(np.int32)).cuda(), hlkv_lib.make_rotary(fr, factor=1.5),
                           torch.full((4,), 123456, dtype=torch.int32, device="cuda"), q, k, v, out, err)
    torch.cuda.synchronize()
    want = rotate(x[:, :H].astype(np.float64), np.full((4, 1), 123456.0) * fr.astype(np.float64), False)
    want[..., :32] *= 1.5
    got = out.cpu().numpy().view(np.float16).astype(np.float64)
    assert (np.abs(got - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -20 * 1.5 * np.abs(x).max()).all()


@pytest.mark.parametrize("factor", [2.0 ** -136, 2.0 ** -128, 1e34])
def test_scales_whose_reciprocal_is_not_normal(hlkv_lib, cuda_device, factor):
    """At position 0 K is x times the factor: rows so small or large that the scale's reciprocal overflows or is
    subnormal still get the quotients' codes."""
    import torch
    T, H, D, n = 16, 2, 64, 40
    wl, rng, targets = _setup(T, H, D, n, seed=3)
    x = rng.standard_normal((n, 3 * H, D)).astype(np.float16)
    d = torch.from_numpy(x.view(np.int16)).cuda()
    q, k, v = d.split((H, H, H), 1)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want, table = host_pools(wl), device_table_words(wl)
    hlkv_lib.rotary_append(wl.hlkv_pools(), wl.layout, wl.dt.table_ptr, wl.dt.table_size,
                           torch.from_numpy(targets.view(np.int32)).cuda(), hlkv_lib.make_rotary(_freqs(32), factor=factor),
                           torch.zeros(n, dtype=torch.int32, device="cuda"), q, k, v, torch.zeros_like(q.contiguous()), err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    with np.errstate(over="ignore"):
        for i in range(n):
            rows = np.stack([x[i, H:2 * H].astype(np.float32) * np.float32(factor), x[i, 2 * H:].astype(np.float32)])
            _store(want, table, T, H, D, targets[i], rows)
    got = host_pools(wl)
    for f in want:
        assert np.array_equal(got[f][0], want[f][0]), f
