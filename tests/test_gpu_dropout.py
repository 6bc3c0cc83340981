"""vtlb_dropout_*: the mask is the generator's, element by element, and the kept values are the one rounded product."""
import numpy as np
import pytest

import token_ops_ref as ref

pytestmark = pytest.mark.gpu


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 31, 128, 1023, 16384, 100003, 2**21 + 1])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_matches_the_definition_bit_for_bit(dev, n, p):
    x = np.random.default_rng(n).standard_normal(n).astype(np.float32)
    dx, dy = dev.to_device(x), dev.zeros(n)
    for call in (dev.dropout_fwd_f32, dev.dropout_bwd_f32):
        call(dx, dy, n, p, 0x123456789ABCDEF0, 2**40 + 5)
        assert same(dy.numpy(), ref.dropout_f32(x, p, 0x123456789ABCDEF0, 2**40 + 5))
    dev.dropout_fwd_f32(dx, dx, n, p, 1, 0)  # in place
    assert same(dx.numpy(), ref.dropout_f32(x, p, 1, 0))
    dx.free(); dy.free()


@pytest.mark.parametrize("p", [0.0, 1e-12, 2.0**-32, 0.999999, 1.0])
def test_edges_of_p(dev, p):
    x = np.random.default_rng(1).standard_normal(4099).astype(np.float32)
    x[:4] = [np.nan, np.inf, -np.inf, -0.0]
    dx, dy = dev.to_device(x), dev.to_device(np.full(4099, 7, np.float32))
    dev.dropout_fwd_f32(dx, dy, 4099, p, 3, 4)
    got, want = dy.numpy(), ref.dropout_f32(x, p, 3, 4)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert same(got[ok], want[ok])
    dx.free(); dy.free()


@pytest.mark.parametrize("off_x,off_y", [(1, 0), (0, 3), (2, 2)])
def test_pointers_off_the_16_byte_grid(dev, off_x, off_y):
    n = 1001
    x = np.random.default_rng(2).standard_normal(n + 4).astype(np.float32)
    dx, dy = dev.to_device(x), dev.to_device(np.full(n + 8, 7, np.float32))
    dev.dropout_fwd_f32(dx.ptr + 4 * off_x, dy.ptr + 4 * off_y, n, 0.3, 5, 6)
    y = dy.numpy()
    assert same(y[off_y:off_y + n], ref.dropout_f32(x[off_x:off_x + n], 0.3, 5, 6))
    assert (y[:off_y] == 7).all() and (y[off_y + n:] == 7).all()
    dx.free(); dy.free()


def test_dropped_elements_are_zero_whatever_they_held(dev):
    n = 512
    x = np.full(n, np.nan, np.float32)
    x[::2] = np.inf
    dx, dy = dev.to_device(x), dev.zeros(n)
    dev.dropout_fwd_f32(dx, dy, n, 0.5, 11, 12)
    y, keep = dy.numpy(), ref.kept(n, 0.5, 11, 12)
    assert (y[~keep] == 0).all() and not np.isfinite(y[keep]).any()
    dx.free(); dy.free()


def test_elements_beyond_32_bits_of_index(dev):
    """4 G elements and some: the counter's upper word and the 64-bit offsets."""
    n = 2**32 + 1029
    buf = dev.empty(n)
    dev.fill_f32(buf, 1.0, n)
    dev.dropout_fwd_f32(buf, buf, n, 0.5, 21, 1)
    for start in (0, 2**31 - 512, 2**32 - 512, n - 1024):
        part = np.empty(1024, np.float32)
        dev.d2h_raw(part.ctypes.data, buf.ptr + 4 * start, part.nbytes)
        block = np.arange(start // 4, (start + 1024 + 3) // 4 + 1, dtype=np.uint64)
        w = ref.philox4x32(np.stack([block & ref.MASK32, block >> np.uint64(32), np.full_like(block, 1),
                                     np.zeros_like(block)], 1), (21, 0)).reshape(-1)
        w = w[start - 4 * (start // 4):][:1024]
        assert same(part, np.where(w >= 2**31, np.float32(2), np.float32(0)))
    buf.free()


def test_nothing_and_refusals(dev):
    from vtl_b200.capi import VtlbError, EINVAL
    d = dev.to_device(np.ones(64, np.float32))
    dev.dropout_fwd_f32(None, None, 0, 0.5, 1, 1)
    for bad in (-0.1, 1.1, float("nan"), float("inf")):
        with pytest.raises(VtlbError, match=r"p must be in \[0, 1\]") as e:
            dev.dropout_fwd_f32(d, d, 64, bad, 1, 1)
        assert e.value.code == EINVAL
    with pytest.raises(VtlbError, match="null pointer"):
        dev.dropout_bwd_f32(d, None, 64, 0.5, 1, 1)
    with pytest.raises(VtlbError, match="overlap in part"):
        dev.dropout_fwd_f32(d, d.ptr + 16, 32, 0.5, 1, 1)
    assert (d.numpy() == 1).all()
    d.free()
