"""Argument checks of the batch plan, the rotary append and the batch attention: refused before any
CUDA call (the pointers below are never dereferenced)."""
import ctypes as C

import pytest

P = C.c_void_p(4096)
ODD = C.c_void_p(4100)


def _plan(hlkv, **kw):
    d = dict(nseq=2, max_query=4, window=0, sinks=0, block_cap=8, token_cap=8, block_first=4096, block_count=4096,
             token_first=4096, context=4096, blocks=4096, targets=4096, positions=4096, block_cost=4096, cost=4096)
    d.update(kw)
    return hlkv.PlanArrays(*d.values())


def test_plan_arguments(hlkv_lib):
    L, INV = hlkv_lib.lib(), hlkv_lib.INVALID_ARGUMENT

    def call(plan, layout=hlkv_lib.Layout(16, 8, 128, 1), table=P, arena=P, segs=P, err=P):
        return L.hlkv_batch_plan(C.byref(plan), C.byref(layout), table, 4, arena, 4, segs, None, err, None)

    assert call(_plan(hlkv_lib, nseq=0)) == hlkv_lib.OK
    for kw in (dict(max_query=0), dict(block_first=None), dict(block_count=None), dict(token_first=None), dict(context=None),
               dict(blocks=None), dict(targets=None), dict(positions=None), dict(blocks=4104), dict(targets=4100),
               dict(nseq=1 << 29), dict(block_cap=1 << 28), dict(block_cost=None), dict(cost=None)):
        assert call(_plan(hlkv_lib, **kw)) == INV, kw
    assert call(_plan(hlkv_lib), err=None) == INV
    assert call(_plan(hlkv_lib), segs=None) == INV
    assert call(_plan(hlkv_lib), table=None) == INV
    assert call(_plan(hlkv_lib), arena=None) == INV
    assert call(_plan(hlkv_lib), layout=hlkv_lib.Layout(16, 8, 100, 1)) == INV
    assert L.hlkv_batch_plan(None, C.byref(hlkv_lib.Layout(16, 8, 128, 1)), P, 4, P, 4, P, None, P, None) == INV
    assert L.hlkv_last_cuda_error() == 0


def test_rotary_arguments(hlkv_lib):
    L, INV = hlkv_lib.lib(), hlkv_lib.INVALID_ARGUMENT
    pools = hlkv_lib.Pools()
    good = hlkv_lib.make_rotary([1.0] * 64)

    def call(rope=good, layout=hlkv_lib.Layout(16, 8, 128, 1), n=3, targets=P, pos=P, q=P, heads=32, qs=4096, k=P, ks=1024, v=P,
             vs=1024, out=C.c_void_p(8192), os=4096, err=P, table=P):
        return L.hlkv_rotary_append(C.byref(pools), C.byref(layout), table, 4, targets, n, C.byref(rope), pos, 1, 0, q, heads, qs,
                                    k, ks, v, vs, out, os, err, None)

    assert call(n=0) == hlkv_lib.OK
    for kw in (dict(err=None), dict(targets=None), dict(pos=None), dict(q=None), dict(out=None), dict(k=None), dict(v=None),
               dict(table=None), dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(out=ODD), dict(targets=C.c_void_p(4100)),
               dict(qs=4095), dict(qs=4100), dict(ks=1016), dict(vs=1020), dict(os=4088),
               dict(out=P, os=8192),                       # in place with another stride
               dict(n=1 << 27), dict(layout=hlkv_lib.Layout(16, 8, 96, 1)),
               dict(layout=hlkv_lib.Layout(16, 8, 64, 1))):  # more rotated elements than a head has
        assert call(**kw) == INV, kw
    for field, value in (("rotary_dim", 0), ("rotary_dim", 24), ("rotary_dim", 144), ("interleaved", 2), ("axes", 0), ("axes", 5),
                         ("factor", float("nan")), ("factor", float("inf"))):
        r = hlkv_lib.make_rotary([1.0] * 64)
        setattr(r, field, value)
        assert call(rope=r) == INV, field
    for value in (float("nan"), float("inf"), 1e6):
        r = hlkv_lib.make_rotary([1.0] * 64)
        r.inv_freq[63] = value
        assert call(rope=r) == INV
    r = hlkv_lib.make_rotary([1.0] * 64, axes=3)
    r.pair_axis[5] = 3
    assert call(rope=r) == INV
    with pytest.raises(hlkv_lib.HlkvError):
        hlkv_lib.make_rotary([1.0] * 129)
    with pytest.raises(hlkv_lib.HlkvError):
        hlkv_lib.make_rotary([1.0] * 16, pair_axis=[0] * 15)
    assert L.hlkv_last_cuda_error() == 0


def test_attention_arguments(hlkv_lib):
    L, INV = hlkv_lib.lib(), hlkv_lib.INVALID_ARGUMENT
    pools = hlkv_lib.Pools()

    def call(plan=None, layout=hlkv_lib.Layout(16, 8, 128, 1), q=P, heads=32, qs=4096, scale=0.1, ws=P, ws_bytes=1 << 40, out=P,
             os=4096, err=P):
        plan = _plan(hlkv_lib) if plan is None else plan
        return L.hlkv_batch_attention(C.byref(pools), C.byref(layout), C.byref(plan), q, heads, qs, scale, ws, ws_bytes, out, os, err,
                                      None)

    assert call(plan=_plan(hlkv_lib, nseq=0)) == hlkv_lib.OK
    assert call(plan=_plan(hlkv_lib, token_cap=0)) == hlkv_lib.OK
    for kw in (dict(err=None), dict(q=None), dict(out=None), dict(q=ODD), dict(out=ODD), dict(qs=4088), dict(os=4092),
               dict(heads=12), dict(heads=0), dict(heads=8 * 33), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
               dict(scale=float("nan")), dict(scale=2.0 ** 61), dict(layout=hlkv_lib.Layout(16, 8, 256, 1)), dict(layout=hlkv_lib.Layout(1024, 8, 128, 1)),
               dict(plan=_plan(hlkv_lib, blocks=None)), dict(plan=_plan(hlkv_lib, blocks=4104)),
               dict(plan=_plan(hlkv_lib, context=None)), dict(plan=_plan(hlkv_lib, token_first=None)),
               dict(ws=None), dict(ws=ODD), dict(plan=_plan(hlkv_lib, max_query=0)), dict(plan=_plan(hlkv_lib, block_cost=None)), dict(plan=_plan(hlkv_lib, cost=None)), dict(plan=_plan(hlkv_lib, token_cap=1 << 30)),
               dict(layout=hlkv_lib.Layout(16, 129, 128, 1), heads=129, qs=129 * 128, os=129 * 128),
               dict(plan=_plan(hlkv_lib, nseq=1 << 20, max_query=1 << 20))):
        assert call(**kw) == INV, kw
    assert L.hlkv_last_cuda_error() == 0
    need = L.hlkv_batch_attention_workspace_bytes(C.byref(_plan(hlkv_lib)), C.byref(hlkv_lib.Layout(16, 8, 128, 1)), 32)
    assert need > 0 and call(ws_bytes=need - 1) == hlkv_lib.BUFFER_TOO_SMALL
