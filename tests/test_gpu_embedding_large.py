"""Embedding at the sizes whose kernels the small tests do not reach.  At 148 SMs: lookups of four loads a thread (from
4.85 million elements on); tiles of 8 to 64 positions; rows of several slabs of columns, aligned and odd; the one-launch
kernel with several pieces of columns to a CTA; a mask in the second and third batch of positions (of 131072)."""
import numpy as np
import pytest

import token_ops_ref as ref
from test_gpu_embedding import same, tokens

pytestmark = pytest.mark.gpu


def sums_by_token(g, ids, V):
    """(sums, sums of absolute values) of the rows of each token in 64 bits, and how many there are."""
    inside = np.flatnonzero((ids >= 0) & (ids < V))
    order = inside[np.argsort(ids[inside], kind="stable")]
    met, first = np.unique(ids[order], return_index=True)
    rows = g[order].astype(np.float64)
    out, mag, count = np.zeros((V, g.shape[1])), np.zeros((V, g.shape[1])), np.zeros((V, 1))
    if met.size:
        out[met] = np.add.reduceat(rows, first, 0)
        mag[met] = np.add.reduceat(np.abs(rows, out=rows), first, 0)
        count[met, 0] = np.diff(np.append(first, order.size))
    return out, mag, count


CASES = [  # n, D, V, p, tokens;   what is new in it
    (512, 4096, 300, 0.0, "skewed"),      # one launch, two pieces of columns to a CTA
    (512, 4095, 300, 0.0, "padded"),
    (250, 8192, 90, 0.25, "skewed"),
    (256, 8190, 90, 0.25, "one"),
    (600, 4097, 50, 0.0, "padded"),       # five slabs of an odd row
    (2049, 8200, 400, 0.25, "skewed"),    # nine slabs
    (3000, 4100, 700, 0.25, "padded"),    # five slabs, tiles of eight
    (1300, 4096, 700, 0.25, "uniform"),   # four loads a thread, aligned
    (1300, 4095, 700, 0.25, "uniform"),   # and odd
    (4100, 4096, 600, 0.0, "skewed"),     # four slabs, tiles of eight
    (8191, 1023, 3001, 0.25, "skewed"),
    (8191, 1023, 3001, 0.25, "one"),
    (8191, 1023, 500, 0.0, "padded"),
    (20000, 516, 900, 0.25, "skewed"),    # tiles of 16
    (20000, 516, 1300, 0.0, "distinct"),
    (20000, 516, 900, 0.0, "one"),
    (40000, 497, 50, 0.25, "padded"),     # of 32
    (76000, 497, 700, 0.25, "skewed"),    # of 64, odd with a mask
    (76000, 516, 1200, 0.0, "distinct"),  # runs of 63 and 64 positions in tiles of 64
    (76000, 516, 40, 0.0, "uniform"),
    (140000, 7, 300, 0.25, "padded"),     # a mask in the second batch
    (140000, 12, 300, 0.25, "skewed"),
    (262149, 33, 5000, 0.25, "skewed"),   # and in the third
]


@pytest.mark.parametrize("n,D,V,p,how", CASES)
def test_lookup_and_gradient(dev, n, D, V, p, how):
    rng = np.random.default_rng(n + D)
    W, g = rng.standard_normal((V, D), dtype=np.float32), rng.standard_normal((n, D), dtype=np.float32)
    ids = tokens(rng, n, V, how)
    kept = ref.kept(n * D, p, 99, 5).reshape(n, D) if p else None
    factor = np.float32(1.0 / (1.0 - p))
    dW_, dids, dg = dev.to_device(W), dev.to_device(ids), dev.to_device(g)
    dy, dd = dev.to_device(np.full((n, D), 7, np.float32)), dev.to_device(np.full((V, D), 7, np.float32))
    dev.embedding_fwd_f32(dW_, V, D, dids, n, dy, scale=0.37, p=p, seed=99, step=5, check=False)
    want = ref.embedding_f32(W, ids, 0.37)
    if p:
        want = np.where(kept, want * factor, np.float32(0))
    assert same(dy.numpy(), want)
    if p:
        g = np.where(kept, g * factor, np.float32(0))  # the product is rounded as the kernels round it
    sums, mag, count = sums_by_token(g, ids, V)
    scale = float(np.float32(0.37))
    # at most count - 1 additions in f32 one after the other and the product with the scale
    want, tol = sums * scale, 1.01 * (count + 1) * 2.0**-24 * mag * scale + 1e-40
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.37, p=p, seed=99, step=5)
    got = dd.numpy()
    assert (np.abs(got - want) <= tol).all()
    absent = count[:, 0] == 0
    assert same(got[absent], np.zeros((int(absent.sum()), D)))
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.37, p=p, seed=99, step=5)
    assert same(dd.numpy(), got)
    base = rng.standard_normal((V, D), dtype=np.float32)
    dev.h2d_raw(dd.ptr, base.ctypes.data, base.nbytes)
    dev.embedding_bwd_f32(dg, dids, n, V, D, dd, scale=0.37, p=p, seed=99, step=5, accumulate=True)
    acc = dd.numpy()
    batches = -(-n // 131072)  # each is added to what is there, and what is there in between is no larger than mag
    assert (np.abs(acc - (base + want)) <= 1.01 * tol + batches * 2.0**-24 * (np.abs(base) + mag * scale)).all()
    assert same(acc[absent], base[absent])
    for b in (dW_, dids, dg, dy, dd):
        b.free()
