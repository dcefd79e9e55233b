"""Places that a step asks for, over a device in host memory."""
import numpy as np
import pytest

from test_lm_device_errors_cpu import Model, lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("room,tokens,places", [(800, 3, 801), (800, 100, 900), (48, 3, 65), (64, 1, 65)])
def test_more_places_than_a_step_has_room_for(lib, pkg, room, tokens, places):  # noqa: F811
    """A place asked for again and again: refused where there is no room for it, in front of anything else that a step does."""
    m = Model(lib, pkg, tokens=room)
    s, other = m.open([1, 2, 3]), m.open([4])
    t, want, logits = np.full(tokens, 7, np.int32), np.zeros(places, np.int32), np.zeros((places + 1, 1000), np.float32)
    entry = pkg.LMEntry(s, t.ctypes.data, tokens, want.ctypes.data, places)
    one = np.full(1, 9, np.int32)
    both = (pkg.LMEntry * 2)(pkg.LMEntry(other, one.ctypes.data, 1, want.ctypes.data, 1), entry)
    assert lib.cml_lm_step(m.h, entry, 1, logits.ctypes.data) == -1 and lib.cml_lm_step(m.h, both, 2, logits.ctypes.data) == -1
    m.check()
    entry.num_want = places - 1
    if places - 1 <= max(room, 64):
        assert lib.cml_lm_step(m.h, entry, 1, logits.ctypes.data) == 0
        m.lines[s] += t.tolist()
        m.check()
    lib.cml_lm_free(m.h)
