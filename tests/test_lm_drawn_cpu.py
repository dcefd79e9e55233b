"""Steps that draw, over a device in host memory."""
import ctypes as C

import numpy as np
import pytest

from test_lm_device_errors_cpu import Model, lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("temperatures", [False, True])
def test_a_step_that_wants_nothing_needs_no_random_numbers(lib, pkg, temperatures):  # noqa: F811
    """A prompt's first portions draw no tokens."""
    lib.cml_lm_step_sampled.argtypes, lib.cml_lm_step_sampled.restype = pkg.lib.cml_lm_step_sampled.argtypes, C.c_int
    m = Model(lib, pkg)
    s, t, out, heat = m.open([1, 2, 3]), np.arange(1, 20, dtype=np.int32), np.zeros(1, np.int32), np.ones(1, np.float32)
    entry = pkg.LMEntry(s, t.ctypes.data, len(t), None, 0)
    assert lib.cml_lm_step_sampled(m.h, entry, 1, heat.ctypes.data if temperatures else None, None, out.ctypes.data) == 0
    m.lines[s] += t.tolist()
    m.check()
    want = np.zeros(1, np.int32)                        # one row that is drawn does need one
    entry.want, entry.num_want = want.ctypes.data, 1
    assert lib.cml_lm_step_sampled(m.h, entry, 1, heat.ctypes.data if temperatures else None, None, out.ctypes.data) == -1
    m.check()
    lib.cml_lm_free(m.h)
