"""Tables whose rows are as wide as an int counts: 2^31 - 1 columns."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
D = 2**31 - 1


def ends(dev, buf, off=0, n=4096):
    out = np.empty((2, n), np.float32)
    dev.d2h_raw(out[0].ctypes.data, buf.ptr + 4 * off, 4 * n)
    dev.d2h_raw(out[1].ctypes.data, buf.ptr + 4 * (off + D - n), 4 * n)
    return out


def test_a_row_of_2_31_less_one_columns(dev):
    # one row out of two, and one position: 17 GB of table, 9 of results
    W, y = dev.empty(2 * D), dev.empty(D)
    dev.fill_f32(W, 1.5, 2 * D)
    dev.fill_f32(y, 7.0, D)
    ids = dev.to_device(np.array([1], np.int32))
    dev.embedding_fwd_f32(W, 2, D, ids, 1, y, scale=2.0)
    assert (ends(dev, y) == 3.0).all()
    dev.fill_f32(W, 7.0, 2 * D)  # now the gradient: the row met, and the other one
    dev.embedding_bwd_f32(y, ids, 1, 2, D, W, scale=0.5)
    assert (ends(dev, W) == 0.0).all() and (ends(dev, W, D) == 1.5).all()
    dev.embedding_bwd_f32(y, ids, 1, 2, D, W, scale=0.5, accumulate=True)
    assert (ends(dev, W) == 0.0).all() and (ends(dev, W, D) == 3.0).all()
    for b in (W, y, ids):
        b.free()
