"""Calls of the rotary and paged entry points beside what else a program does."""
import ctypes as C

import pytest
import torch

from tests.paged_ref import Case

pytestmark = pytest.mark.gpu


def test_an_error_of_another_call_is_not_theirs():
    """An error that another HIP call of the thread has left is neither reported by a call of this library nor taken away."""
    from kore_amd import hip, rope
    c = Case([(2, 40), (20, 90)], 4, 2, 64, 16, "f32", "f16", seed=1).up()
    L = hip.lib()
    L.hipPeekAtLastError.restype = L.hipGetLastError.restype = C.c_int
    with c.handle(rope.Config(64)) as kv, rope.Rope(rope.Config(64)) as r:
        pos = torch.arange(22, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        calls = [lambda: kv.append_dev(0, c.batch(), "f32", c.ptr("k"), c.ptr("v")),
                 lambda: kv.attend_dev(0, c.batch(), "f32", c.ptr("q"), c.ptr("out")),
                 lambda: kv.attend_dev(0, c.batch(1), "f32", c.ptr("q"), c.ptr("out")),
                 lambda: r.apply_dev("f32", 22, 4, 64, c.ptr("q"), pos.data_ptr(), c.ptr("out"))]
        for call in calls:
            assert L.hipSetDevice(1 << 20) != 0      # no such device
            left = L.hipPeekAtLastError()
            try:
                call()
                assert L.hipPeekAtLastError() == left
            finally:
                L.hipGetLastError()
        kv.sync()
        r.sync()
