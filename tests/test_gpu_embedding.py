"""vtlb_embedding_*: the lookup bit for bit, the gradient within the rounding of its sums."""
import numpy as np
import pytest

import token_ops_ref as ref

pytestmark = pytest.mark.gpu


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


def tokens(rng, n, V, how):
    if how == "uniform":
        return rng.integers(0, V, n).astype(np.int32)
    if how == "skewed":
        w = 1 / (np.arange(V) + 2.7)
        return rng.choice(V, n, p=w / w.sum()).astype(np.int32)
    if how == "one":
        return np.full(n, V // 2, np.int32)
    if how == "distinct":
        return rng.permutation(V)[:n].astype(np.int32) if n <= V else (np.arange(n) % V).astype(np.int32)
    ids = rng.integers(-2, V + 2, n).astype(np.int32)  # padded: -2, -1 and V, V + 1 lie outside
    ids[rng.random(n) < 0.3] = -1
    ids[rng.random(n) < 0.05] = np.iinfo(np.int32).min
    ids[rng.random(n) < 0.05] = np.iinfo(np.int32).max
    return ids


SHAPES = [(1, 1, 1), (1, 8, 5), (3, 4, 2), (8, 256, 100), (33, 7, 3), (257, 130, 1000), (512, 96, 40), (513, 97, 40), (600, 640, 7), (150, 1027, 9), (999, 2047, 61), (1024, 64, 17),
          (4097, 12, 5000), (8192, 20, 70000), (20011, 5, 300)]
HOW = ["uniform", "skewed", "one", "distinct", "padded"]


@pytest.mark.parametrize("n,D,V", SHAPES)
@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("p", [0.0, 0.25])
def test_lookup_and_gradient(dev, n, D, V, how, p):
    rng = np.random.default_rng(n * 7 + D)
    W, g = rng.standard_normal((V, D)).astype(np.float32), rng.standard_normal((n, D)).astype(np.float32)
    ids = tokens(rng, n, V, how)
    dW_, dids, dg = dev.to_device(W), dev.to_device(ids), dev.to_device(g)
    dy, dd = dev.to_device(np.full((n, D), 7, np.float32)), dev.to_device(np.full((V, D), 7, np.float32))
    dev.embedding_fwd_f32(dW_, V, D, dids, n, dy, scale=0.37, p=p, seed=99, step=5, check=False)
    assert same(dy.numpy(), ref.embedding_f32(W, ids, 0.37, p, 99, 5))
    if p:  # the same as the two operators one after the other
        dev.embedding_fwd_f32(dW_, V, D, dids, n, dy, scale=0.37, check=False)
        dev.dropout_fwd_f32(dy, dy, n * D, p, 99, 5)
        assert same(dy.numpy(), ref.embedding_f32(W, ids, 0.37, p, 99, 5))
    want, tol = ref.embedding_bwd(g, ids, V, 0.37, p, 99, 5)
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.37, p=p, seed=99, step=5)
    got = dd.numpy()
    assert (np.abs(got - want) <= tol).all()
    absent = np.setdiff1d(np.arange(V), ids)
    assert same(got[absent], np.zeros((absent.size, D)))
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.37, p=p, seed=99, step=5)
    assert same(dd.numpy(), got)  # the same call, the same bits
    # added to what is there: one rounding more, of the sum
    base = rng.standard_normal((V, D)).astype(np.float32)
    dev.h2d_raw(dd.ptr, base.ctypes.data, base.nbytes)
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.37, p=p, seed=99, step=5, accumulate=True)
    acc = dd.numpy()
    assert (np.abs(acc - (base + want)) <= 1.01 * tol + 2.0**-24 * np.abs(base + want)).all()
    assert same(acc[absent], base[absent])
    for b in (dW_, dids, dg, dy, dd):
        b.free()


def test_known_answer(dev):
    W = np.arange(12, dtype=np.float32).reshape(4, 3)
    ids = np.array([2, -1, 2, 0, 4], np.int32)
    g = np.arange(15, dtype=np.float32).reshape(5, 3)
    dW_, dids, dg, dy, dd = dev.to_device(W), dev.to_device(ids), dev.to_device(g), dev.zeros((5, 3)), dev.zeros((4, 3))
    dev.embedding_fwd_f32(dW_, 4, 3, dids, 5, dy, scale=2.0, check=False)
    assert dy.numpy().tolist() == [[12, 14, 16], [0, 0, 0], [12, 14, 16], [0, 2, 4], [0, 0, 0]]
    dev.embedding_bwd_f32(dg, dids, 5, 4, 3, dd, scale=2.0)
    assert dd.numpy().tolist() == [[18, 20, 22], [0, 0, 0], [12, 16, 20], [0, 0, 0]]
    for b in (dW_, dids, dg, dy, dd):
        b.free()


def test_gradient_of_one_position_is_one_product(dev):
    rng = np.random.default_rng(8)
    n, D, V = 700, 36, 900
    ids, g = rng.permutation(V)[:n].astype(np.int32), rng.standard_normal((n, D)).astype(np.float32)
    dids, dg, dd = dev.to_device(ids), dev.to_device(g), dev.zeros((V, D))
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.7)
    want = np.zeros((V, D), np.float32)
    want[ids] = g * np.float32(0.7)
    assert same(dd.numpy(), want)
    for b in (dids, dg, dd):
        b.free()


@pytest.mark.parametrize("n", [40, 700])
def test_infinities_and_nan_stay_in_their_rows(dev, n):
    D, V = 9, 6
    rng = np.random.default_rng(9)
    ids = rng.integers(0, V, n).astype(np.int32)
    ids[5], ids[6], ids[7] = 1, 2, -1
    g = rng.standard_normal((n, D)).astype(np.float32)
    g[5, 3], g[6, 4], g[7] = np.nan, np.inf, np.nan  # position 7 is padding: what it holds is never read
    dids, dg, dd = dev.to_device(ids), dev.to_device(g), dev.zeros((V, D))
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd)
    got = dd.numpy()
    assert np.isnan(got[1, 3]) and np.isinf(got[2, 4]) and np.isfinite(got).sum() == V * D - 2
    W = np.ones((V, D), np.float32)
    W[3] = np.inf
    dW_, dy = dev.to_device(W), dev.zeros((n, D))
    dev.embedding_fwd_f32(dW_, V, D, dids, n, dy, check=False)
    y = dy.numpy()
    assert (np.isinf(y).all(1) == (ids == 3)).all() and (y[7] == 0).all()
    for b in (dids, dg, dd, dW_, dy):
        b.free()


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("D", [64, 21])
@pytest.mark.parametrize("n", [130, 900])
def test_pointers_off_the_16_byte_grid(dev, off, D, n):
    rng = np.random.default_rng(off)
    V = 40
    W, g, ids = rng.standard_normal(V * D + 4).astype(np.float32), rng.standard_normal(n * D + 4).astype(np.float32), \
        rng.integers(-1, V, n + 4).astype(np.int32)
    dW_, dg, dids = dev.to_device(W), dev.to_device(g), dev.to_device(ids)
    dy, dd = dev.to_device(np.full(n * D + 8, 7, np.float32)), dev.to_device(np.full(V * D + 8, 7, np.float32))
    w0, g0, i0 = W[off:off + V * D].reshape(V, D), g[off:off + n * D].reshape(n, D), ids[off:off + n]
    dev.embedding_fwd_f32(dW_.ptr + 4 * off, V, D, dids.ptr + 4 * off, n, dy.ptr + 4 * off, p=0.2, seed=1, step=2, check=False)
    y = dy.numpy()
    assert same(y[off:off + n * D].reshape(n, D), ref.embedding_f32(w0, i0, 1.0, 0.2, 1, 2))
    assert (y[:off] == 7).all() and (y[off + n * D:] == 7).all()
    dev.embedding_bwd_f32(dg.ptr + 4 * off, dids.ptr + 4 * off, n, V, D, dd.ptr + 4 * off, p=0.2, seed=1, step=2)
    d = dd.numpy()
    want, tol = ref.embedding_bwd(g0, i0, V, 1.0, 0.2, 1, 2)
    assert (np.abs(d[off:off + V * D].reshape(V, D) - want) <= tol).all()
    assert (d[:off] == 7).all() and (d[off + V * D:] == 7).all()
    for b in (dW_, dg, dids, dy, dd):
        b.free()


@pytest.mark.parametrize("n,V", [(200000, 37), (150000, 150000), (300001, 1 << 20)])
def test_many_positions(dev, n, V):
    rng = np.random.default_rng(n)
    D = 4
    ids, g = tokens(rng, n, V, "padded" if V < 100 else "skewed"), rng.standard_normal((n, D)).astype(np.float32)
    dids, dg, dd = dev.to_device(ids), dev.to_device(g), dev.zeros((V, D))
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd)
    want, tol = ref.embedding_bwd(g, ids, V, 1.0)
    assert (np.abs(dd.numpy() - want) <= tol).all()
    for b in (dids, dg, dd):
        b.free()


def test_offsets_beyond_32_bits(dev):
    """A table of 2^32 and more elements, read and written at its end."""
    V, D = (1 << 20) + 3, 4100
    W, dd = dev.empty((V, D)), dev.empty((V, D))
    dev.fill_f32(W, 1.5, V * D)
    ids = np.array([V - 1, 0, V - 2, V - 1], np.int32)
    g = np.random.default_rng(1).standard_normal((4, D)).astype(np.float32)
    dids, dg, dy = dev.to_device(ids), dev.to_device(g), dev.zeros((4, D))
    dev.embedding_fwd_f32(W, V, D, dids, 4, dy, scale=2.0)
    assert (dy.numpy() == 3.0).all()
    dev.fill_f32(dd, 7.0, V * D)
    dev.embedding_bwd_f32(dg, dids, 4, V, D, dd)
    rows = np.empty((3, D), np.float32)
    dev.d2h_raw(rows.ctypes.data, dd.ptr + 4 * (V - 3) * D, rows.nbytes)
    assert same(rows[0], np.zeros(D)) and same(rows[1], g[2]) and same(rows[2], g[0] + g[3])
    for b in (W, dd, dids, dg, dy):
        b.free()


def test_nothing(dev):
    dd = dev.to_device(np.full((3, 5), 7, np.float32))
    dev.embedding_fwd_f32(dd, 3, 5, None, 0, None)
    dev.embedding_bwd_f32(None, None, 0, 3, 5, dd, accumulate=True)
    assert (dd.numpy() == 7).all()
    dev.embedding_bwd_f32(None, None, 0, 3, 5, dd)
    assert (dd.numpy() == 0).all()
    ids = dev.to_device(np.full(4, -1, np.int32))  # nothing but padding
    g = dev.to_device(np.full((4, 5), np.nan, np.float32))
    dev.fill_f32(dd, 7.0, 15)
    dev.embedding_bwd_f32(g, ids, 4, 3, 5, dd)
    assert (dd.numpy() == 0).all()
    for b in (dd, ids, g):
        b.free()


def test_check_reports_tokens_outside_the_table(dev):
    from vtl_b200.capi import VtlbError, EINVAL
    W, y = dev.to_device(np.ones((3, 2), np.float32)), dev.zeros((2, 2))
    good, bad = dev.to_device(np.array([0, 2], np.int32)), dev.to_device(np.array([1, 3], np.int32))
    dev.embedding_fwd_f32(W, 3, 2, good, 2, y)
    with pytest.raises(VtlbError, match=r"outside \[0, 3\)") as e:
        dev.embedding_fwd_f32(W, 3, 2, bad, 2, y)
    assert e.value.code == EINVAL and y.numpy().tolist() == [[1, 1], [0, 0]]
    for b in (W, y, good, bad):
        b.free()


def test_refusals(dev):
    from vtl_b200.capi import VtlbError
    d = dev.to_device(np.ones(64, np.float32))
    ids = dev.to_device(np.zeros(4, np.int32))
    out = dev.zeros(64)
    for V, D in ((0, 4), (4, 0), (-1, 4)):
        with pytest.raises(VtlbError, match="bad table"):
            dev.embedding_fwd_f32(d, V, D, ids, 4, out)
        with pytest.raises(VtlbError, match="bad table"):
            dev.embedding_bwd_f32(d, ids, 4, V, D, out)
    with pytest.raises(VtlbError, match=r"2\^31 - 1"):
        dev.embedding_fwd_f32(d, 4, 4, ids, 2**31, out)
    with pytest.raises(VtlbError, match=r"p must be in"):
        dev.embedding_bwd_f32(d, ids, 4, 4, 4, out, p=1.5)
    with pytest.raises(VtlbError, match="null pointer"):
        dev.embedding_fwd_f32(d, 4, 4, ids, 4, None)
    with pytest.raises(VtlbError, match="null pointer"):
        dev.embedding_bwd_f32(None, ids, 4, 4, 4, out)
    with pytest.raises(VtlbError, match="overlaps"):
        dev.embedding_fwd_f32(d, 4, 4, ids, 4, d.ptr + 32)
    with pytest.raises(VtlbError, match="overlaps"):
        dev.embedding_bwd_f32(d, ids, 4, 4, 4, d)
    assert (d.numpy() == 1).all() and (out.numpy() == 0).all()
    for b in (d, ids, out):
        b.free()


def test_ids_from_f32(dev):
    src = np.array([0, -0.0, 1, 2.5, -1, np.nan, np.inf, -np.inf, 16777216, 2147483520, 2147483648, 1e30, 0.999], np.float32)
    want = [0, 0, 1, -1, -1, -1, -1, -1, 16777216, 2147483520, -1, -1, -1]
    a, b = dev.to_device(src), dev.zeros(src.size, np.int32)
    dev.ids_from_f32(a, src.size, b)
    assert b.numpy().tolist() == want
    from vtl_b200.capi import VtlbError
    with pytest.raises(VtlbError, match="overlap"):
        dev.ids_from_f32(a, src.size - 1, a.ptr + 4)
    dev.ids_from_f32(a, src.size, a)  # in place
    assert a.numpy().view(np.int32).tolist() == want
    a.free(); b.free()
