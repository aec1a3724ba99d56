"""Calls of the batch plan, the rotary append and the batch attention that are refused: pointers off their records'
alignment, and tensors of another type.  Refused before any CUDA call (the pointers below are never dereferenced)."""
import ctypes as C

import pytest

from test_batch_step_args import P, _plan

OFF = {n: C.c_void_p(4096 + n) for n in (4, 8)}


def test_records_off_their_alignment(hlkv_lib):
    """A segment is read as 8 bytes, a descriptor as 16."""
    L, INV = hlkv_lib.lib(), hlkv_lib.INVALID_ARGUMENT
    layout = C.byref(hlkv_lib.Layout(16, 8, 128, 1))
    plan = C.byref(_plan(hlkv_lib))
    assert L.hlkv_batch_plan(plan, layout, P, 4, P, 4, OFF[4], None, P, None) == INV
    rope, pools = hlkv_lib.make_rotary([1.0] * 64), hlkv_lib.Pools()
    for n in (4, 8):
        assert L.hlkv_batch_plan(plan, layout, OFF[n], 4, P, 4, P, None, P, None) == INV
        assert L.hlkv_rotary_append(C.byref(pools), layout, OFF[n], 4, P, 3, C.byref(rope), P, 1, 0, P, 32, 4096, P, 1024, P,
                                    1024, C.c_void_p(8192), 4096, P, None) == INV
    assert L.hlkv_last_cuda_error() == 0


class _OnDevice:
    """A tensor that says it lies on device 0: the binding's checks, without a GPU."""

    def __init__(self, t):
        self.t = t

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.fixture
def device0(hlkv_lib, monkeypatch):
    """The calls on a machine without a GPU, up to the C entry point, which takes nothing here."""
    import torch
    monkeypatch.setattr(hlkv_lib, "_elsewhere", lambda index: hlkv_lib._cuda() is None)
    monkeypatch.setattr(hlkv_lib, "_stream_handle", lambda stream: 0)

    class Taken(Exception):
        pass

    class Entry:
        def __getattr__(self, name):
            def call(*args):
                raise Taken
            return call

    monkeypatch.setattr(hlkv_lib, "lib", Entry)
    return lambda *shape, dtype=torch.int32: _OnDevice(torch.zeros(shape, dtype=dtype)), Taken


def test_tensors_of_another_type(hlkv_lib, device0):
    """bfloat16 is no binary16, and float32 no int32, though their sizes are equal."""
    import torch
    zeros, Taken = device0
    layout, n, H, heads, D = hlkv_lib.Layout(16, 2, 64, 1), 3, 2, 4, 64
    rope = hlkv_lib.make_rotary([1.0] * 32)
    plan = hlkv_lib.BatchPlan(2, 4, n, device="cpu")
    plan.index = 0
    half, bf, f32 = torch.float16, torch.bfloat16, torch.float32

    def append(**other):
        t = dict(targets=zeros(n, 2), positions=zeros(n), q=zeros(n, heads, D, dtype=half), k=zeros(n, H, D, dtype=half),
                 v=zeros(n, H, D, dtype=half), q_out=zeros(n, heads, D, dtype=half), err=zeros(1))
        t.update(other)
        return hlkv_lib.rotary_append(None, layout, 16, 4, t["targets"], rope, t["positions"], t["q"], t["k"], t["v"], t["q_out"],
                                      t["err"])

    def fill(segs=zeros(2, 2), query_lens=zeros(2), err=zeros(1)):
        return hlkv_lib.batch_plan(plan, layout, 16, 4, 16, 4, segs, query_lens, err)

    def attend(q=zeros(n, heads, D, dtype=half), out=zeros(n, heads, D, dtype=half), err=zeros(1)):
        return hlkv_lib.batch_attention(None, layout, plan, q, 0.1, out, err, workspace=zeros(16, dtype=torch.uint8))

    for call in (append, fill, attend):
        with pytest.raises(Taken):
            call()
    for bits in (torch.int16, torch.uint16):
        with pytest.raises(Taken):
            append(k=zeros(n, H, D, dtype=bits), q=zeros(n, heads, D, dtype=bits))
    wrong = [(append, {name: zeros(n, H if name in "kv" else heads, D, dtype=bf)}) for name in ("q", "k", "v", "q_out")]
    wrong += [(append, dict(targets=zeros(n, 2, dtype=f32))), (append, dict(positions=zeros(n, dtype=f32))),
              (append, dict(err=zeros(1, dtype=f32))), (fill, dict(segs=zeros(2, 2, dtype=f32))),
              (fill, dict(query_lens=zeros(2, dtype=f32))), (fill, dict(err=zeros(1, dtype=f32))),
              (attend, dict(q=zeros(n, heads, D, dtype=bf))), (attend, dict(out=zeros(n, heads, D, dtype=bf))),
              (attend, dict(err=zeros(1, dtype=f32)))]
    for call, other in wrong:
        with pytest.raises(hlkv_lib.HlkvError):
            call(**other)


def test_a_plan_begins_as_padding(hlkv_lib):
    """A plan that was not filled, or of no sequence (which batch_plan leaves as it is), appends nothing: a target of
    zeros would be token 0 of block 0."""
    for nseq in (0, 2):
        plan = hlkv_lib.BatchPlan(nseq, 4, 5, device="cpu")
        assert (plan.targets == -1).all() and (plan.positions == 0).all() and (plan.token_first == 0).all()
