"""What layers on rows in 8 bits refuse for the sizes of their launches, without a GPU (no pointer is followed, and what is refused is not launched)."""
import ctypes as C

import pytest

ESHAPE = -2
FAKE = 0x10000


def both(rows, out, x_stride, w_stride):
    from cuke_amd import _lib
    d = _lib.Linear(1, 1, 0, 0, rows, 32, out, None, 0, None, 0, None, None, 0, 0.0, 0, 0, None)
    x, w = _lib.Rows8(FAKE, x_stride, FAKE, 4), _lib.Rows8(FAKE, w_stride, FAKE, 4)
    return _lib.lib().kge_linear8_fwd(C.byref(d), C.byref(x), C.byref(w), FAKE, out, 0, None, 0, None, 0, None)


@pytest.mark.parametrize("rows,out,x_stride,w_stride", [(64, 1 << 30, 1 << 27, 32), (1, 1 << 30, 1 << 24, 32), (65, 1 << 30, 32, 1 << 24)])
def test_far_rows_that_only_the_largest_tiles_take(rows, out, x_stride, w_stride):
    """Those address a tile's rows with 32 bits; a launch of the others does not hold so many."""
    assert both(rows, out, x_stride, w_stride) == ESHAPE
