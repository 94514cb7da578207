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


def linear(type, rows, fin, fout):
    from cuke_amd import _lib
    return _lib.Linear(type, type, 0, 0, rows, fin, fout, FAKE, fin, FAKE, fin, None, None, 0, 0.0, 0, 0, None)


# (type, rows, in, out) beyond what tiles of any shape cover with fewer than 2^32 threads
@pytest.mark.parametrize("size", [(0, 2 ** 30, 8, 1), (0, 2 ** 31 - 1, 8, 64), (1, 2 ** 31 - 1, 8, 1), (2, 2 ** 31 - 1, 8, 200), (1, 2 ** 24, 8, 2 ** 16)])
def test_linear_sizes_that_no_launch_takes(size):
    from cuke_amd import _lib
    L = _lib.lib()
    d = linear(*size)
    assert L.kge_linear_fwd(C.byref(d), FAKE, 1 << 31, 0, None, 0, FAKE, 1 << 62, None) == ESHAPE
    assert L.kge_linear_bwd(C.byref(d), FAKE, 1 << 31, FAKE, 1 << 62, FAKE, FAKE, FAKE, FAKE, 1 << 62, None) == ESHAPE
    assert L.kge_linear_saved_bytes(C.byref(d)) == 0 and L.kge_linear_bwd_workspace(C.byref(d)) == 0


@pytest.mark.parametrize("size", [(0, 2 ** 30 - 2 ** 16, 8, 1), (1, 2 ** 30, 8, 1), (2, 2 ** 31 - 2 ** 16, 8, 64),
                                  (1, 2 ** 20, 8, 2 ** 16)])
def test_linear_sizes_that_are_taken(size):
    """As far as a saved block and a workspace that are too small.  (2^16 rows fewer leave the backward pass room for at least 256 tiles of dW.)"""
    from cuke_amd import _lib
    L = _lib.lib()
    d = linear(*size)
    d.act = 2
    saved = L.kge_linear_saved_bytes(C.byref(d))
    assert saved >= size[1] * size[3] * 2
    assert L.kge_linear_fwd(C.byref(d), FAKE, 1 << 31, 1, FAKE, saved - 1, FAKE, 1 << 62, None) == EWORKSPACE
    need = L.kge_linear_bwd_workspace(C.byref(d))
    assert need > 0
    assert L.kge_linear_bwd(C.byref(d), FAKE, 1 << 31, FAKE, saved, FAKE, FAKE, FAKE, FAKE, need - 1, None) == EWORKSPACE


def test_a_gradient_of_x_too_large_beside_that_of_the_weight():
    """dx of 2^30 columns takes more tiles than a launch holds; the weight's gradient alone does not."""
    from cuke_amd import _lib
    L = _lib.lib()
    d = linear(0, 2 ** 29, 600, 8)
    need = L.kge_linear_bwd_workspace(C.byref(d))
    assert need > 0
    assert L.kge_linear_bwd(C.byref(d), FAKE, 8, None, 0, FAKE, FAKE, None, FAKE, need, None) == ESHAPE
    assert L.kge_linear_bwd(C.byref(d), FAKE, 8, None, 0, None, FAKE, None, FAKE, need - 1, None) == EWORKSPACE
