"""Refusals of the training operators' later entry points and calls (no GPU)."""
import ctypes as C

import numpy as np
import pytest


@pytest.mark.parametrize("args", [(-1, 4, 1, 1000), (4096, 4, 1, 1000), (0, 0, 1, 1000), (0, 65, 1, 1000),
                                  (0, 4, -1, 1000), (0, 4, 1, 0), (0, 4, 1, 1000001)])
def test_walk_selftest_refuses(boa, args):
    out = np.zeros((65, 128), np.float32).ctypes.data_as(C.POINTER(C.c_float))
    assert boa.lib().boa_selftest_walk_timeout(*args, out) == boa.BOA_E_INVALID
    assert boa.lib().boa_last_error(None).startswith(b"boa_selftest_walk_timeout")
