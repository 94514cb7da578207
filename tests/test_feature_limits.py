"""How large the feature operators' calls may be: a launch has fewer than 2^32 threads, and what would pass that is refused on the host, before
anything is launched (no pointer is followed here)."""
import ctypes as C

import pytest

ESHAPE, EWORKSPACE = -2, -4
FAKE = 0x10000


@pytest.mark.parametrize("n_neg,segments", [(1025, 1), (2048, 1), (2049, 2), (40943, 20)])
def test_preference_batches(n_neg, segments):
    from cuke_amd import _lib
    L = _lib.lib()
    most = (2 ** 32 - 1) // (256 * segments)
    for type in range(3):
        pref = lambda batch: _lib.Preference(type, 0, batch, n_neg, FAKE, FAKE, n_neg, None, None, 0, None, 0, 1.0, 1.0, 0.0, 0.0)
        for batch in (most + 1, 2 ** 24, 2 ** 31):
            d = pref(batch)
            assert L.kge_preference_loss(C.byref(d), FAKE, FAKE, FAKE, FAKE, 1 << 62, None) == ESHAPE and L.kge_preference_workspace(C.byref(d)) == 0
        d = pref(most)                                   # taken, as far as a workspace that is too small
        need = L.kge_preference_workspace(C.byref(d))
        assert need >= most * segments * 8
        assert L.kge_preference_loss(C.byref(d), FAKE, FAKE, FAKE, FAKE, need - 1, None) == EWORKSPACE
    # rows that a wave holds are walked by a bounded grid
    d = _lib.Preference(0, 0, 2 ** 33, 1024, FAKE, FAKE, 1024, None, None, 0, None, 0, 1.0, 1.0, 0.0, 0.0)
    assert L.kge_preference_loss(C.byref(d), FAKE, FAKE, FAKE, FAKE, 0, None) == EWORKSPACE
