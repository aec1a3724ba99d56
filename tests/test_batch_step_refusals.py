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
