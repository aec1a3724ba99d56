"""The serving-step operators over the quantized KV cache, as cases that can be measured.

Three operators make one layer's step of a ragged batch: the batch plan (block tables, slot map
and positions from the request lengths), the rotary append (rotate Q and K, store K and V in the
blocks' formats) and the batch attention (causal, with a sliding window and visible first tokens).
``run`` computes them in elementary torch operations, or, where ``own`` is true, through the
``hlkv`` package.

The cache is the package's own layout: a block holds 2 (K, V) x T tokens x H heads rows of D
elements in one of four formats (FP16, FP8 E4M3, FP8 E5M2, INT4); a slot holds the codes of all
rows, then one parameter group per row (none, a binary32 scale, or a {scale, bias} pair).
"""
import os
import sys

import numpy as np
import torch

own = False

FP16, E4M3, E5M2, INT4 = 0, 1, 2, 3
LAYOUT_ID = 1
MAX_FINITE = {E4M3: 448.0, E5M2: 57344.0}
F8 = {E4M3: torch.float8_e4m3fn, E5M2: torch.float8_e5m2}


def _package():
    root = os.path.join(os.getcwd(), "hl-kv_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import hlkv
    return hlkv


# ---- cases -----------------------------------------------------------------------------------

def _case(op, nseq, ctx_min, ctx_max, q_min, q_max, T=16, H=8, G=4, D=128, mix="mixed", partial=0.0,
          window=0, sinks=0, axes=1, rotary=0, interleaved=False, pad=0, lens=1):
    return dict(op=op, nseq=nseq, ctx_min=ctx_min, ctx_max=ctx_max, q_min=q_min, q_max=q_max, T=T, H=H, G=G,
                D=D, mix=mix, partial=partial, window=window, sinks=sinks, axes=axes, rotary=rotary,
                interleaved=interleaved, pad=pad, lens=lens)


def listed():
    return [
        # The plan of the smallest decode step: a few short chats.
        {"name": "plan_few", **_case("plan", 8, 100, 900, 1, 1)},
        # The plan of the default workload's decode step (64 sequences of 8192 tokens).
        {"name": "plan_decode", **_case("plan", 64, 8192, 8192, 1, 1)},
        # Long contexts with a window and sinks, mixed chunk sizes, a few partly filled blocks and
        # a token array padded for a captured graph.
        {"name": "plan_long_window", **_case("plan", 48, 1000, 131072, 0, 512, partial=0.02, window=4096, sinks=4,
                                             pad=100, lens=2)},
        # One decode step's append: a token for each of 64 sequences (32 query, 8 KV heads).
        {"name": "rotary_decode", **_case("rotary", 64, 500, 8192, 1, 1, lens=3)},
        # Prompt ingestion: 8192 tokens of four prompts.
        {"name": "rotary_prefill", **_case("rotary", 4, 2048, 2048, 2048, 2048)},
        # Video tokens with time, height and width positions, 64 query heads.
        {"name": "rotary_video", **_case("rotary", 3, 1100, 1500, 1100, 1500, G=8, axes=3, mix="int4", lens=4)},
        # Half-rotated heads of 64 in adjacent pairs, odd lengths, small KV head count.
        {"name": "rotary_partial", **_case("rotary", 7, 1, 333, 1, 333, T=32, H=2, G=6, D=64, rotary=32,
                                           interleaved=True, mix="even", pad=19, lens=5)},
        # Decode of a few short sequences, where latency counts.
        {"name": "attention_few", **_case("attention", 4, 300, 1100, 1, 1, lens=6)},
        # The default workload's decode step: age tiers over 64 sequences of 8192 tokens.
        {"name": "attention_decode", **_case("attention", 64, 8192, 8192, 1, 1, mix="tiers")},
        # Long contexts with a sliding window and sinks, INT4 mostly, four proposed tokens each.
        {"name": "attention_window", **_case("attention", 32, 3000, 30000, 1, 4, mix="int4", partial=0.02,
                                             window=4096, sinks=4, lens=7)},
        # Chunked prefill over mixed-format contexts of up to 8192 tokens, next to decoding sequences.
        {"name": "attention_chunks", **_case("attention", 6, 200, 8192, 1, 2048, lens=8)},
        # Prompts of heads of 64 with a window, odd lengths, seven query heads per KV head.
        {"name": "attention_prompt64", **_case("attention", 5, 700, 3001, 700, 3001, T=32, H=2, G=7, D=64, mix="even",
                                               window=1024, sinks=1, lens=9)},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("plan", "rotary", "attention", "attention"))
    D = rng.choice((64, 128, 128))
    G = rng.choice((1, 2, 3, 4, 5, 7, 8))
    H = rng.choice((1, 2, 4, 6, 8))
    T = rng.choice((8, 16, 16, 32, 64))
    mix = rng.choice(("mixed", "tiers", "int4", "even", "fp16", "e4m3"))
    partial = rng.choice((0.0, 0.0, 0.02))
    lens = rng.randrange(10, 1 << 30)
    window, sinks = (0, 0) if rng.random() < 0.5 else (_log(rng, 64, 8192), rng.randrange(0, 9))
    if op == "plan":
        hi = _log(rng, 50, 60000)
        return _case(op, _log(rng, 1, max(1, min(300, 2000000 // hi))), max(1, hi // 4), hi, 0, _log(rng, 1, 300), T=T,
                     partial=partial, window=window, sinks=sinks, pad=rng.randrange(0, 40), lens=lens)
    if op == "rotary":
        D = rng.choice((64, 128, 256))
        n = _log(rng, 1, 4000)
        nseq = _log(rng, 1, 64)
        q = max(1, n // nseq)
        return _case(op, nseq, q, q + _log(rng, 1, 400), max(1, q // 2), q, T=T, H=H, G=G, D=D, mix=mix,
                     partial=partial, axes=rng.choice((1, 1, 2, 3)), rotary=rng.choice((0, 0, 32, D // 2)),
                     interleaved=rng.random() < 0.4, pad=rng.randrange(0, 20), lens=lens)
    if rng.random() < 0.5:  # decode, or a few proposed tokens
        hi = _log(rng, 30, 8192)
        return _case(op, _log(rng, 1, max(1, min(64, 300000 // hi))), max(1, hi // 3), hi, 1, rng.choice((1, 1, 2, 5)),
                     T=T, H=H, G=G, D=D, mix=mix, partial=partial, window=window, sinks=sinks, lens=lens)
    hi = _log(rng, 40, 5000)  # chunks of prompts
    return _case(op, _log(rng, 1, max(1, min(8, 12000 // hi))), max(1, hi // 3), hi, 1, _log(rng, 20, min(hi + 1, 1500)), T=T,
                 H=H, G=G, D=D, mix=mix, partial=partial, window=window, sinks=sinks, lens=lens)


# ---- the batch of a case: lengths, blocks and formats, from the case alone --------------------

_MIX = {"mixed": (0.25, 0.5, 0.0, 0.25), "int4": (0.05, 0.10, 0.0, 0.85), "even": (0.25, 0.25, 0.25, 0.25),
        "fp16": (1.0, 0.0, 0.0, 0.0), "e4m3": (0.0, 1.0, 0.0, 0.0)}


def _batch(case):
    """Per sequence: (valid tokens of each block, format of each block, new tokens), as numpy arrays."""
    rng, T = np.random.RandomState(case["lens"] % (1 << 31)), case["T"]
    out = []
    for _ in range(case["nseq"]):
        ctx = int(rng.randint(case["ctx_min"], case["ctx_max"] + 1))
        q = min(ctx, int(rng.randint(case["q_min"], case["q_max"] + 1)))
        if case["q_min"] == case["ctx_min"] and case["q_max"] == case["ctx_max"]:
            q = ctx  # a whole prompt
        vt = []
        if case["partial"] == 0.0:
            vt = [T] * (ctx // T) + ([ctx % T] if ctx % T else [])
        else:  # some blocks were closed early (a shared prefix that ended inside a block)
            left = ctx
            early = rng.random_sample(ctx // T * 2 + 2) < case["partial"]
            k = 0
            while left > 0:
                n = int(rng.randint(0, T)) if early[k % early.size] else T
                n = min(n, left)
                vt.append(n)
                left -= n
                k += 1
        nb = len(vt)
        if case["mix"] == "tiers":  # the newest 512 tokens FP16, 2048 before them E4M3, older INT4
            n16, n8 = 512 // T, 2048 // T
            fm = np.full(nb, INT4)
            fm[max(0, nb - n16 - n8):] = E4M3
            fm[max(0, nb - n16):] = FP16
        else:
            fm = rng.choice(4, size=nb, p=_MIX[case["mix"]])
        out.append((np.asarray(vt, np.int64), fm.astype(np.int64), q))
    return out


def _row_bytes(f, D):
    return (2 * D, D, D, D // 2)[f]


def _param_bytes(f):
    return (0, 4, 4, 8)[f]


def _visible(case, vt, q):
    """The blocks that some new token sees."""
    ctx, start = int(vt.sum()), np.cumsum(vt) - vt
    if not case["window"]:
        return vt > 0
    return (vt > 0) & ((start < case["sinks"]) | (start + vt > ctx - q - case["window"] + 1))


def work(case):
    T, H, G, D = case["T"], case["H"], case["G"], case["D"]
    by, fl = 0, 0
    for vt, fm, q in _batch(case):
        ctx = int(vt.sum())
        if case["op"] == "plan":
            by += len(vt) * 20 + int(_visible(case, vt, q).sum()) * 16 + q * 12 + 28
            fl += len(vt)
        elif case["op"] == "rotary":
            end = np.cumsum(vt)
            new = np.clip(end - np.maximum(end - vt, ctx - q), 0, None)
            by += q * (2 * D * (2 * G * H + 2 * H) + 8 + 4 * case["axes"])
            by += int(sum(int(n) * 2 * H * (_row_bytes(f, D) + _param_bytes(f)) for n, f in zip(new, fm)))
            fl += q * (G + 1) * H * D * 3
            # the touched blocks' values, which the run returns
            hit = new > 0
            by += int(hit.sum()) * 2 * T * H * D * 2 + int(sum(int(n) * 2 * H * (_row_bytes(f, D) + _param_bytes(f))
                                                              for n, f in zip(vt[hit], fm[hit])))
        else:
            w, s = case["window"] or ctx + 1, case["sinks"]
            keep = _visible(case, vt, q)
            by += int(sum(int(n) * 2 * H * (_row_bytes(f, D) + _param_bytes(f)) for n, f in zip(vt[keep], fm[keep])))
            by += int(keep.sum()) * 16 + 2 * 2 * q * H * G * D
            p = np.arange(ctx - q, ctx)
            seen = np.minimum(p + 1, w) + np.minimum(np.clip(p + 1 - w, 0, None), s)
            fl += int(seen.sum()) * 4 * H * G * D
    return {"bytes": by, "flops": fl}


# ---- quantization, as the package's blocks hold it ---------------------------------------------

def _encode(x, f):
    """Rows of x (binary32, [..., D]) -> (codes as uint8 [..., bytes], parameters binary32 [..., 0, 1 or 2])."""
    if f == FP16:
        h = x.to(torch.float16).contiguous()
        return h.view(torch.uint8), x.new_empty(x.shape[:-1] + (0,))
    if f == INT4:
        lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        scale = (hi - lo) / 15.0
        q = torch.where(scale > 0, torch.round((x - lo) / scale), torch.zeros_like(x)).clamp(0, 15).to(torch.uint8)
        return q[..., 0::2] | (q[..., 1::2] << 4), torch.cat((scale, lo), -1)
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, (amax / MAX_FINITE[f]).clamp_min(torch.finfo(torch.float32).tiny), torch.ones_like(amax))
    return (x / scale).to(F8[f]).view(torch.uint8), scale


def _decode(codes, params, f):
    """What the codes stand for, in binary32."""
    if f == FP16:
        return codes.contiguous().view(torch.float16).float()
    if f == INT4:
        q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
        return torch.addcmul(params[..., 1:2], q, params[..., 0:1])
    return codes.contiguous().view(F8[f]).float() * params


def _views(state, f):
    """The codes [slots, 2, T, H, bytes] and parameters [slots, 2, T, H, n] of a pool, as views."""
    c = state["case"]
    pool, rows, rb, pb = state["pool"][f], 2 * c["T"] * c["H"], _row_bytes(f, c["D"]), _param_bytes(f)
    shape = (2, c["T"], c["H"])
    codes = pool[:, :rows * rb].unflatten(1, shape + (rb,))
    params = pool.view(torch.float32)[:, rows * rb // 4:rows * (rb + pb) // 4].unflatten(1, shape + (pb // 4,))
    return codes, params


def _fill(n, f, T, H, D, gen, device):
    """n slots of format f with keys and values as a model makes them: some channels are outliers."""
    rb, pb = _row_bytes(f, D), _param_bytes(f)
    rows = 2 * T * H
    size = (rows * (rb + pb) + 15) // 16 * 16
    pool = torch.zeros((n, size), dtype=torch.uint8, device=device)
    loud = torch.ones((2, 1, H, D), device=device)
    loud[0, 0, :, :3] = 6.0
    step = max(1, (1 << 27) // (rows * D))
    for a in range(0, n, step):
        m = min(step, n - a)
        x = (torch.randn((m, 2, T, H, D), generator=gen, device=device) * loud).to(torch.float16).float()
        codes, params = _encode(x, f)
        pool[a:a + m, :rows * rb] = codes.reshape(m, -1)
        if pb:
            pool[a:a + m, rows * rb:rows * (rb + pb)] = params.contiguous().view(torch.uint8).reshape(m, -1)
    return pool


# ---- inputs ------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = "cuda"
    T, H, G, D = case["T"], case["H"], case["G"], case["D"]
    batch, rng = _batch(case), np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    lens = np.array([len(b[0]) for b in batch])
    total, ntok = int(lens.sum()), int(sum(b[2] for b in batch))
    vt = np.concatenate([b[0] for b in batch])
    fm = np.concatenate([b[1] for b in batch])
    # Block ids, slots and segments scattered as a running engine leaves them.
    size = total + 7
    ids = rng.permutation(size)[:total]
    slot = np.zeros(total, np.int64)
    count = {}
    for f in range(4):
        at = np.nonzero(fm == f)[0]
        slot[at] = rng.permutation(at.size)
        count[f] = int(at.size)
    table = np.zeros((size, 4), np.int64)
    table[:, 1], table[:, 3] = 15, np.arange(size)
    table[ids, 0] = slot
    table[ids, 1] = fm | LAYOUT_ID << 6 | vt << 10
    order = rng.permutation(case["nseq"])
    off = np.zeros(case["nseq"], np.int64)
    off[order] = np.cumsum(lens[order]) - lens[order]
    first = np.cumsum(lens) - lens
    arena = np.full(total + 1, size, np.int64)
    arena[np.repeat(off - first, lens) + np.arange(total)] = ids
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a).astype(np.uint32).view(np.int32)).to(dev)  # noqa: E731
    state = {"case": case, "total": total, "ntok": ntok, "cap": ntok + case["pad"], "table": i32(table), "arena": i32(arena),
             "segs": i32(np.stack((off, lens), 1)), "query_lens": i32(np.array([b[2] for b in batch])),
             "width": int(lens.max()), "max_query": max(1, max(b[2] for b in batch)), "err": torch.zeros(1, dtype=torch.int32, device=dev)}
    if case["op"] != "plan":
        # One slot more than the blocks need: the plain form writes there what belongs to no block.
        state["pool"] = {f: _fill(count[f] + 1, f, T, H, D, gen, dev) for f in range(4) if count[f]}
        state["slots"] = {f: count[f] for f in state["pool"]}
        state["first_slot"] = {}
        for f in state["pool"]:
            state["first_slot"][f] = sum(state["slots"][g] + 1 for g in state["first_slot"])
    if case["op"] == "rotary":
        R = case["rotary"] or D
        heads = (G + 2) * H
        state["qkv"] = torch.randn((state["cap"], heads * D), generator=gen, device=dev).to(torch.float16)
        state["inv_freq"] = [float(np.float32(500000.0 ** (-2.0 * j / R))) for j in range(R // 2)]
        # equal runs of the pairs for time, height and width
        state["pair_axis"] = [j * case["axes"] // (R // 2) for j in range(R // 2)]
        pos = []
        for v, _, q in batch:
            p = np.arange(int(v.sum()) - q, int(v.sum()))
            pos.append(np.stack([p] + [p // 7 % (23 + a) + p // 400 for a in range(1, case["axes"])], 1))
        pos.append(np.zeros((case["pad"], case["axes"])))
        state["rope_pos"] = i32(np.concatenate(pos))
        state["freq64"] = torch.tensor(state["inv_freq"], dtype=torch.float64, device=dev)
        state["axis"] = torch.tensor(state["pair_axis"], device=dev)
        state["q_out"] = torch.zeros((state["cap"], G * H, D), dtype=torch.float16, device=dev)
        # the blocks that take new tokens: the last ones of each sequence
        seg, blocks = [], []
        for i, (v, _, q) in enumerate(batch):
            j0 = int(np.searchsorted(np.cumsum(v), int(v.sum()) - q, side="right"))
            seg.append((off[i] + j0, lens[i] - j0))
            blocks.append(np.arange(first[i] + j0, first[i] + lens[i]))
        blocks = np.concatenate(blocks)
        state["touched"], state["touched_segs"] = i32(ids[blocks]), i32(np.array(seg))
        state["values"] = torch.empty((blocks.size, 2, T, H, D), dtype=torch.float16, device=dev)
        state["targets"] = _plan(state)["targets"]
    if case["op"] == "attention":
        state["q"] = torch.randn((state["cap"], G * H, D), generator=gen, device=dev).to(torch.float16)
        state["out"] = torch.zeros_like(state["q"])
        state["scale"] = D ** -0.5
    if own:
        hlkv = _package()
        state["layout"] = hlkv.Layout(T, H, D, LAYOUT_ID)
        if case["op"] != "plan":
            state["pools"] = hlkv.make_pools({f: (p, p.shape[1], state["slots"][f]) for f, p in state["pool"].items()})
        if case["op"] == "rotary":
            state["rope"] = hlkv.make_rotary(state["inv_freq"], pair_axis=state["pair_axis"], interleaved=case["interleaved"])
            q, k, v = state["qkv"].unflatten(1, (-1, D)).split((G * H, H, H), 1)
            state["q"], state["k"], state["v"] = q, k, v
        else:
            state["plan"] = hlkv.BatchPlan(case["nseq"], total, state["cap"], max_query=state["max_query"],
                                           window=case["window"], sinks=case["sinks"], device=dev)
        if case["op"] == "attention":
            _call_plan(hlkv, state)
            n = hlkv.batch_attention_workspace_bytes(state["plan"], state["layout"], G * H)
            state["workspace"] = torch.empty(n, dtype=torch.uint8, device=dev)
    elif case["op"] == "attention":
        state["plan"] = _plan(state)
    return state


# ---- the operators in plain form ---------------------------------------------------------------

def _plan(state):
    """Block table, slot map and positions from the segments, the descriptors and the new tokens' counts."""
    c = state["case"]
    nseq, total, ntok, cap, T = c["nseq"], state["total"], state["ntok"], state["cap"], c["T"]
    dev = state["segs"].device
    off, lens = state["segs"].long().unbind(1)
    q = state["query_lens"].long()
    seqs = torch.arange(nseq, device=dev)
    first = lens.cumsum(0) - lens
    seq = torch.repeat_interleave(seqs, lens, output_size=total)
    ids = state["arena"][off[seq] + torch.arange(total, device=dev) - first[seq]].long()
    desc = state["table"][ids]
    vt = (desc[:, 1].long() >> 10) & 0x3FF
    upto = torch.cat((vt.new_zeros(1), vt.cumsum(0)))
    start = upto[:-1] - upto[first][seq]
    context = upto[first + lens] - upto[first]
    keep = vt > 0
    if c["window"]:
        keep &= (start < c["sinks"]) | (start + vt > (context - q)[seq] - c["window"] + 1)
    kept = torch.cat((keep.new_zeros(1).long(), keep.long().cumsum(0)))
    count = kept[first + lens] - kept[first]
    to = torch.where(keep, first[seq] + kept[:-1] - kept[first][seq], total)
    blocks = torch.zeros((total + 1, 4), dtype=torch.int32, device=dev)
    blocks[to] = torch.cat((desc[:, :3], start[:, None].int()), 1)
    token_first = torch.cat((q.new_zeros(1), q.cumsum(0)))
    tseq = torch.repeat_interleave(seqs, q, output_size=ntok)
    pos = (context - q)[tseq] + torch.arange(ntok, device=dev) - token_first[tseq]
    held = torch.searchsorted(upto[1:], upto[first][tseq] + pos, right=True)
    targets = torch.full((cap, 2), -1, dtype=torch.int32, device=dev)
    targets[:ntok] = torch.stack((ids[held], pos - start[held]), 1).int()
    positions = torch.zeros(cap, dtype=torch.int32, device=dev)
    positions[:ntok] = pos.int()
    return {"block_first": first.int(), "block_count": count.int(), "token_first": token_first.int(), "context": context.int(),
            "blocks": blocks[:total], "targets": targets, "positions": positions}


def _rotate(x, cos, sin, interleaved):
    """x: binary32 [n, heads, D]; cos, sin: [n, 1, R / 2]."""
    half = cos.shape[-1]
    rot, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((rot, rest), -1)


def _rotary(state):
    c = state["case"]
    T, H, G, D, n = c["T"], c["H"], c["G"], c["D"], state["ntok"]
    q, k, v = state["qkv"][:n].unflatten(1, (-1, D)).float().split((G * H, H, H), 1)
    angle = state["rope_pos"][:n].double()[:, state["axis"]] * state["freq64"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    q_out = state["q_out"].clone()
    q_out[:n] = _rotate(q, cos, sin, c["interleaved"]).to(torch.float16)
    rows = torch.stack((_rotate(k, cos, sin, c["interleaved"]), v), 1)
    block, token = state["targets"][:n].long().unbind(1)
    desc = state["table"][block].long()
    seen = state["table"][state["touched"].long()].long()
    live = (torch.arange(T, device=q.device) < ((seen[:, 1] >> 10) & 0x3FF)[:, None])[:, None, :, None, None]
    values = torch.zeros((seen.shape[0], 2, T, H, D), device=q.device)
    for f, slots in state["slots"].items():
        codes, params = _views(state, f)
        new_codes, new_params = _encode(rows, f)
        slot = torch.where(desc[:, 1] % 16 == f, desc[:, 0], slots)
        codes[slot, :, token] = new_codes
        params[slot, :, token] = new_params
        is_f = seen[:, 1] % 16 == f
        at = torch.where(is_f, seen[:, 0], slots)
        values = torch.where(is_f[:, None, None, None, None] & live, _decode(codes[at], params[at], f), values)
    return {"q_out": q_out, "values": values.to(torch.float16)}


def _attention(state):
    c, plan = state["case"], state["plan"]
    nseq, T, H, G, D, L = c["nseq"], c["T"], c["H"], c["G"], c["D"], state["max_query"]
    dev = state["q"].device
    # every slot's values, formats one behind the other
    cache = torch.cat([_decode(*_views(state, f), f) for f in state["pool"]])
    shift = torch.zeros(4, dtype=torch.long, device=dev)
    for f, s in state["first_slot"].items():
        shift[f:f + 1].fill_(s)
    j = torch.arange(state["width"], device=dev)
    have = j < plan["block_count"][:, None]
    entry = plan["blocks"][torch.where(have, plan["block_first"][:, None] + j, 0)].long()
    start, vt = entry[..., 3], (entry[..., 1] >> 10) & 0x3FF
    kv = cache[torch.where(have, shift[entry[..., 1] % 16] + entry[..., 0], 0)]  # [nseq, width, 2, T, H, D]
    t = torch.arange(T, device=dev)
    pos = (start[..., None] + t).flatten(1)
    live = (have[..., None] & (t < vt[..., None])).flatten(1)
    k = kv[:, :, 0].permute(0, 3, 4, 1, 2).flatten(3)  # [nseq, H, D, width * T]
    v = torch.where(live[:, None, :, None], kv[:, :, 1].permute(0, 3, 1, 2, 4).flatten(2, 3), 0.0)
    r = torch.arange(L, device=dev)
    lens = state["query_lens"].long()
    own_row = r < lens[:, None]
    row = torch.where(own_row, plan["token_first"][:-1, None].long() + r, 0)
    q = state["q"][row].float().unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [nseq, H, L * G, D]
    at = plan["context"].long()[:, None] - lens[:, None] + r
    see = live[:, None] & (pos[:, None] <= at[..., None])
    if c["window"]:
        see &= (at[..., None] - pos[:, None] < c["window"]) | (pos[:, None] < c["sinks"])
    see = see.repeat_interleave(G, 1)[:, None]  # [nseq, 1, L * G, width * T]
    s = torch.where(see, torch.matmul(q, k) * state["scale"], -torch.inf)
    p = torch.where(see, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, torch.matmul(p, v) / total, 0.0)
    o = o.unflatten(2, (L, G)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(torch.float16)
    out = torch.zeros((state["cap"] + 1, G * H, D), dtype=torch.float16, device=dev)
    out[torch.where(own_row, row, state["cap"]).flatten()] = o.flatten(0, 1)
    return out[:state["cap"]]


# ---- a pass ------------------------------------------------------------------------------------

def _call_plan(hlkv, state):
    hlkv.batch_plan(state["plan"], state["layout"], state["table"].data_ptr(), state["table"].shape[0],
                    state["arena"].data_ptr(), state["arena"].shape[0], state["segs"], state["query_lens"], state["err"])


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plan, "rotary": _rotary, "attention": _attention}[op](state)
    hlkv = _package()
    if op == "plan":
        _call_plan(hlkv, state)
        p = state["plan"]
        return {"block_first": p.block_first, "block_count": p.block_count, "token_first": p.token_first, "context": p.context,
                "blocks": p.blocks, "targets": p.targets, "positions": p.positions}
    if op == "rotary":
        hlkv.rotary_append(state["pools"], state["layout"], state["table"].data_ptr(), state["table"].shape[0],
                           state["targets"], state["rope"], state["rope_pos"], state["q"], state["k"], state["v"],
                           state["q_out"], state["err"])
        # What the touched blocks hold now, through the package's gather: the values that the codes stand for.
        hlkv.gather_dequant(state["pools"], state["layout"], state["table"].data_ptr(), state["table"].shape[0],
                            state["arena"].data_ptr(), state["arena"].shape[0], state["touched_segs"], state["values"],
                            state["err"])
        return {"q_out": state["q_out"], "values": state["values"]}
    hlkv.batch_attention(state["pools"], state["layout"], state["plan"], state["q"], state["scale"], state["out"], state["err"],
                         workspace=state["workspace"])
    return state["out"]


# ---- the definition in 64 bits -----------------------------------------------------------------

def _code_values(f):
    """The value of every code of an FP8 format, from its sign, exponent and mantissa fields."""
    ebits, mbits, bias = (4, 3, 7) if f == E4M3 else (5, 2, 15)
    code = np.arange(256)
    e, m = (code >> mbits) & ((1 << ebits) - 1), code & ((1 << mbits) - 1)
    mag = np.where(e == 0, m * 2.0 ** (1 - bias - mbits), (1 + m / 2.0 ** mbits) * 2.0 ** (e - bias * 1.0))
    if f == E4M3:
        mag = np.where((code & 127) == 127, np.nan, mag)
    else:
        mag = np.where(e == 31, np.where(m == 0, np.inf, np.nan), mag)
    return np.where(code >= 128, -mag, mag)


def _slot_values(state, f, slot):
    """[n, 2, T, H, D] binary64 values of the given slots, from the slots' bytes."""
    c = state["case"]
    T, H, D = c["T"], c["H"], c["D"]
    rows, rb = 2 * T * H, _row_bytes(f, D)
    raw = state["pool"][f][slot]
    codes = raw[:, :rows * rb].reshape(-1, rows, rb)
    if f == FP16:
        return codes.contiguous().view(torch.float16).double().view(-1, 2, T, H, D)
    par = raw[:, rows * rb:rows * (rb + _param_bytes(f))].contiguous().view(torch.float32).double().view(-1, rows, _param_bytes(f) // 4)
    if f == INT4:
        b = codes.long()
        val = torch.empty((raw.shape[0], rows, D), dtype=torch.float64, device=raw.device)
        val[:, :, 0::2], val[:, :, 1::2] = (b % 16).double(), (b // 16).double()
        val = val * par[:, :, :1] + par[:, :, 1:]
    else:
        val = torch.from_numpy(_code_values(f)).to(raw.device)[codes.long()] * par
    return val.view(-1, 2, T, H, D)


def _quantize_exact(x, f):
    """What rows of x (binary64) are after being stored in format f, to the nearest code."""
    if f == FP16:
        return x
    if f == INT4:
        lo, hi = x.min(-1, True).values, x.max(-1, True).values
        step = (hi - lo) / 15
        return torch.where(step > 0, ((x - lo) / step).round() * step + lo, lo)
    scale = x.abs().max(-1, True).values / MAX_FINITE[f]
    y = x / scale
    mbits, emin = (3, -6) if f == E4M3 else (2, -14)
    ulp = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -60))).clamp_min(emin) - mbits)
    return (y / ulp).round() * ulp * scale


def exact(case, seed):
    if case["op"] == "plan":
        return None
    state = prepare(case, seed)
    T, H, G, D = case["T"], case["H"], case["G"], case["D"]
    batch = _batch(case)
    table, arena, segs = (state[k].cpu().numpy().astype(np.int64) for k in ("table", "arena", "segs"))
    dev = state["segs"].device
    if case["op"] == "rotary":
        R = case["rotary"] or D
        x = state["qkv"].double().view(state["cap"], -1, D)
        pos = state["rope_pos"].cpu().numpy().astype(np.float64)
        turn = np.stack([pos[:, a] * f for a, f in zip(state["pair_axis"], state["inv_freq"])], 1)
        z = torch.polar(torch.ones(turn.shape, dtype=torch.float64), torch.from_numpy(turn)).to(dev)[:, None]
        i = torch.arange(R // 2, device=dev)
        ia, ib = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2)
        y = x[:, :(G + 1) * H].clone()
        turned = torch.complex(y[..., ia], y[..., ib]) * z
        y[..., ia], y[..., ib] = turned.real, turned.imag
        q_out = torch.zeros_like(x[:, :G * H])
        q_out[:state["ntok"]] = y[:state["ntok"], :G * H]
        rows = torch.stack((y[:, G * H:], x[:, (G + 1) * H:]), 1)
        values, at = [], 0
        for (vt, fm, q), (o, n) in zip(batch, segs):
            end, ctx = np.cumsum(vt), int(vt.sum())
            for j in range(int(np.searchsorted(end, ctx - q, side="right")), len(vt)):
                f, slot = int(fm[j]), int(table[arena[o + j], 0])
                val = _slot_values(state, f, slice(slot, slot + 1))[0]
                lo = max(0, ctx - q - int(end[j] - vt[j]))
                new = rows[at:at + int(vt[j]) - lo]
                at += int(vt[j]) - lo
                val[:, lo:int(vt[j])] = _quantize_exact(new, f).transpose(0, 1)
                val[:, int(vt[j]):] = 0
                values.append(val)
            if len(values) > 20000:
                return None
        return {"q_out": q_out, "values": torch.stack(values)}
    out = torch.zeros((state["cap"], G * H, D), dtype=torch.float64, device=dev)
    at = 0
    for (vt, fm, q), (o, n) in zip(batch, segs):
        if not q:
            continue
        keep = np.nonzero(_visible(case, vt, q))[0]
        start, ctx = np.cumsum(vt) - vt, int(vt.sum())
        val = torch.empty((keep.size, 2, T, H, D), dtype=torch.float64, device=dev)
        for f in range(4):
            mine = np.nonzero(fm[keep] == f)[0]
            if mine.size:
                val[torch.from_numpy(mine).to(dev)] = _slot_values(state, f, torch.from_numpy(table[arena[o + keep[mine]], 0]).to(dev))
        place = (start[keep][:, None] + np.arange(T)).reshape(-1)
        has = (np.arange(T) < vt[keep][:, None]).reshape(-1)
        sel = torch.from_numpy(np.nonzero(has)[0]).to(dev)
        t = torch.from_numpy(place[has]).to(dev)
        k, v = val.transpose(0, 1).reshape(2, -1, H, D)[:, sel].permute(0, 2, 1, 3)  # [H, tokens, D] each
        x = state["q"][at:at + q].double().view(q, H, G, D).permute(1, 0, 2, 3)
        for a in range(0, q, 256):
            p = torch.arange(ctx - q + a, ctx - q + min(q, a + 256), device=dev)[:, None]
            dark = t > p
            if case["window"]:
                dark = dark | ((p - t >= case["window"]) & (t >= case["sinks"]))
            s = torch.einsum("hrgd,htd->hrgt", x[:, a:a + 256], k) * state["scale"]
            w = torch.softmax(s.masked_fill(dark[None, :, None], -torch.inf), -1)
            out[at + a:at + min(q, a + 256)] = torch.einsum("hrgt,htd->rhgd", w, v).flatten(1, 2)
        at += q
    return out
