"""Plain implementations, in 64 bits, of the batch plan, the rotary append and the batch attention, on
host copies of the tables and the pools' bytes."""
from __future__ import annotations

import numpy as np

FP16, E4M3, E5M2, INT4 = 0, 1, 2, 3
PAD = 0xFFFFFFFF
ERR_PLAN_RANGE = 1 << 13


def fp8_values(fmt: int) -> np.ndarray:
    """Value of every FP8 code from its fields."""
    out = np.empty(256)
    ebits, mbits, bias = (4, 3, 7) if fmt == E4M3 else (5, 2, 15)
    for c in range(256):
        e, m = (c >> mbits) & ((1 << ebits) - 1), c & ((1 << mbits) - 1)
        v = m * 2.0 ** (1 - bias - mbits) if e == 0 else (1 + m / 2.0 ** mbits) * 2.0 ** (e - bias)
        if fmt == E4M3 and (c & 127) == 127:
            v = np.nan
        if fmt == E5M2 and e == 31:
            v = np.inf if m == 0 else np.nan
        out[c] = -v if c & 128 else v
    return out


def block_rows(pool, fmt, slot, T, H, D, mode=0, ref=0):
    """(values [2, T, H, D] float64: code * scale (+ bias), {scale, bias} [2, T, H, 2]) of one slot.
    pool: (uint8 array, slot_bytes, num_slots)."""
    buf, sb, _ = pool
    raw = buf[slot * sb:(slot + 1) * sb]
    n = 2 * T * H
    cb = {FP16: 2 * D, E4M3: D, E5M2: D, INT4: D // 2}[fmt]
    codes = raw[:n * cb].reshape(n, cb)
    if fmt == FP16:
        v = codes.copy().view(np.float16).astype(np.float64)
        par = np.tile([1.0, 0.0], (n, 1))
    else:
        if fmt == INT4:
            v = np.empty((n, D))
            v[:, 0::2], v[:, 1::2] = codes & 15, codes >> 4
            par = raw[n * cb:n * (cb + 8)].copy().view(np.float32).astype(np.float64).reshape(n, 2)
        else:
            v = fp8_values(fmt)[codes]
            par = np.zeros((n, 2))
            par[:, 0] = raw[n * cb:n * (cb + 4)].copy().view(np.float32)
        if mode == 1:
            par = np.tile([np.array([ref], np.uint32).view(np.float32)[0].astype(np.float64), 0.0], (n, 1))
        elif mode == 2:
            h = np.array([ref & 0xFFFF, ref >> 16], np.uint16).view(np.float16).astype(np.float64)
            par = np.tile(h, (n, 1))
        v = v * par[:, :1] + par[:, 1:]
    return v.reshape(2, T, H, D), par.reshape(2, T, H, 2)


def plan_oracle(segs, qlens, arena, table, T, layout_id, block_cap, token_cap, max_query, window, sinks):
    """The plan's arrays as dicts per sequence: (sequences, targets, positions, token_first, block_first, err).
    Each sequence: {"context", "q", "blocks": [(slot, info, ref, start)]}."""
    err, seqs = 0, []
    targets = np.full((token_cap, 2), PAD, np.uint32)
    positions = np.zeros(token_cap, np.int32)
    bfirst, tfirst, bf, tf = 0, 0, [], []
    for (off, n), q in zip(segs.tolist(), qlens):
        q = int(q)
        bf.append(min(bfirst, block_cap))
        tf.append(min(tfirst, token_cap))
        fits = bfirst + n <= block_cap and tfirst + q <= token_cap and q <= max_query
        if not fits:
            err |= ERR_PLAN_RANGE
            seqs.append({"context": 0, "q": q, "blocks": [], "cost": []})
            bfirst, tfirst = bfirst + n, tfirst + q
            continue
        rows, start = [], 0
        for j in range(n):
            pos, bad, v = off + j, 0, 0
            if pos >= arena.size:
                bad = 1 << 3
            elif arena[pos] >= table.shape[0]:
                bad = 1 << 4
            else:
                slot, info, ref, bid = (int(x) for x in table[arena[pos]])
                f, mode, lay, v = info & 15, (info >> 4) & 3, (info >> 6) & 15, (info >> 10) & 0x3FF
                if bid != arena[pos]:
                    bad = 1 << 8
                elif f == 15:
                    bad = 1
                elif f > 3:
                    bad = 2
                elif lay != layout_id:
                    bad = 1 << 6
                elif f != 0 and mode == 3:
                    bad = 1 << 7
                elif v > T:
                    bad = 1 << 5
            err |= bad
            if bad or v == 0:
                continue
            rows.append((slot, info, ref, start, bid, v))
            start += v
        ctx, from_ = start, max(0, start - q)
        if q > ctx:
            err |= ERR_PLAN_RANGE
        keep = [r for r in rows if window == 0 or r[3] < sinks or r[3] + r[5] > from_ - window + 1]
        for r in rows:
            for t in range(max(r[3], from_), r[3] + r[5]):
                row = tfirst + max(0, q - ctx) + t - from_
                targets[row] = (r[4], t - r[3])
                positions[row] = t
        cost = [(r[5] + 15) // 16 * (14, 7, 7, 7)[r[1] & 15] for r in keep]
        seqs.append({"context": ctx, "q": q, "blocks": [r[:4] for r in keep], "cost": np.cumsum(cost).tolist()})
        bfirst, tfirst = bfirst + n, tfirst + q
    tf.append(min(tfirst, token_cap))
    return seqs, targets, positions, np.array(tf, np.uint32), np.array(bf, np.uint32), err


def attention_oracle(seqs, tf, pools, T, H, D, q, scale, window, sinks):
    """out [tokens, heads, D] and the error bound of each value, both float64.  q: [tokens, heads, D].

    The bound counts, for a kernel that multiplies binary16 codes and binary16 weights with binary32 sums:
    the result's rounding (2^-11 of it); every weight's rounding (2^-11 of p times the row's codes under
    their scale: 8/15 of an INT4 row's range, at most 16/15 of its largest value, is the widest); a
    weight below binary16's normal range (2^-25 of the largest value, doubled for the codes' own scale);
    and the score's rounding, D products and sums at 2^-23 of the sum of their magnitudes, which is
    the relative error of p, in the weights and in their sum."""
    heads = q.shape[1]
    g = heads // H
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i, s in enumerate(seqs):
        if s["q"] == 0 or not s["blocks"]:
            continue
        ks, vs, at = [], [], []
        for slot, info, ref, start in s["blocks"]:
            f, mode, v = info & 15, (info >> 4) & 3, (info >> 10) & 0x3FF
            rows, _ = block_rows(pools[f], f, slot, T, H, D, mode if f else 0, ref)
            ks.append(rows[0, :v])
            vs.append(rows[1, :v])
            at.append(start + np.arange(v))
        K, V, at = np.concatenate(ks), np.concatenate(vs), np.concatenate(at)
        for r in range(s["q"]):
            p = s["context"] - s["q"] + r
            see = at <= p
            if window:
                see &= (p - at < window) | (at < sinks)
            if not see.any():
                continue
            for qh in range(heads):
                h, x = qh // g, q[int(tf[i]) + r, qh]
                k, v = K[see, h], V[see, h]
                sc = scale * (k @ x)
                w = np.exp(sc - sc.max())
                w /= w.sum()
                o = w @ v
                big = np.abs(v).max(1)
                ds = scale * D * 2.0 ** -23 * (np.abs(k) @ np.abs(x)).max()
                out[int(tf[i]) + r, qh] = o
                tol[int(tf[i]) + r, qh] = (2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 2 * ds) * 16 / 15 * (w @ big)
                                           + len(v) * 2.0 ** -24 * big.max() + 2.0 ** -24)
    return out, tol


def rotate(x, angle, interleaved):
    """x: float64 [n, heads, D]; angle: [n, pairs]."""
    r = angle.shape[1]
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y = x.copy()
    ia, ib = (np.arange(0, 2 * r, 2), np.arange(1, 2 * r, 2)) if interleaved else (np.arange(r), np.arange(r, 2 * r))
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y
