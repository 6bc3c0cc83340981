"""The mean and rstd of vtlb_groupnorm_fwd_f32 where the spread of a group is far below its mean, or one value far from the
others.  Half steps u = 2^-24; every bound is counted where it is used."""
import numpy as np
import pytest

import token_ops_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0**-24

# one position (odd and aligned rows), a cluster with and without TMA, a group no cluster holds (aligned and odd)
SHAPES = [(3, 1, 64, 2), (2, 1, 33, 1), (2, 40, 16, 4), (1, 30, 33, 3), (300, 17, 64, 64), (4, 1024, 256, 32), (2, 20000, 8, 1),
          (2, 20000, 33, 1), (1, 5, 40000, 2), (2, 515, 96, 3)]


@pytest.mark.parametrize("B,S,C,G", SHAPES)
@pytest.mark.parametrize("at", [3.0, 1e4, 1000003.0, 1e8])
def test_statistics_of_groups_that_hardly_vary(dev, B, S, C, G, at):
    """Constant groups, and groups of four neighbouring f32 values: the variance is what the definition says, however
    far the mean.  The distances between such values, or from a mean within 16 steps of them, are exact in f32 and so are
    the sums of their few bits; what rounds is the join in 64 bits (2^-50 of the squared distances, at most 400 steps
    squared), the sum with eps and the root: 3 half steps, and one for the result."""
    rng = np.random.default_rng(C)
    step = np.spacing(np.float32(at))
    steps = rng.integers(0, 4, (B, S, C))
    steps[0, :, :C // G if B == 1 else C] = 0  # constant groups
    x = (np.float32(at) + steps.astype(np.float32) * step).astype(np.float32)
    assert (x.astype(np.float64) == float(np.float32(at)) + steps * float(step)).all()
    d = dev.to_device(x)
    y, mean, rstd = dev.zeros(x.shape), dev.zeros((B, G)), dev.zeros((B, G))
    dev.groupnorm_fwd_f32(d, B, S, C, G, None, None, 1e-5, ref.NONE, y, mean, rstd)
    # (from the steps, whose variance numpy gets right in 64 bits)
    sg = steps.reshape(B, S, G, C // G).astype(np.float64)
    var = sg.var((1, 3)) * float(step)**2
    want = 1 / np.sqrt(var + 1e-5)
    lost = 2.0**-50 * 400 * float(step)**2
    tol = want * (4 * U + 0.5 * lost / (var + 1e-5))
    assert (np.abs(rstd.numpy() - want) <= tol).all()
    m = float(np.float32(at)) + sg.mean((1, 3)) * float(step)
    assert (np.abs(mean.numpy() - m) <= U * m * 1.01).all()
    assert (y.numpy()[0, :, :C // G if B == 1 else C] == 0).all()
    # the same in place: the statistics are read before the first result is written
    dev.groupnorm_fwd_f32(d, B, S, C, G, None, None, 1e-5, ref.NONE, d, mean, rstd)
    assert (np.abs(rstd.numpy() - want) <= tol).all()
    assert np.array_equal(d.numpy(), y.numpy())
    for b in (d, y, mean, rstd):
        b.free()


@pytest.mark.parametrize("B,S,C,G", [s for s in SHAPES if s[1] > 1])
def test_eps_below_the_smallest_f32_with_several_positions(dev, B, S, C, G):
    """rstd = 1 / sqrt(1e-60) of constant groups: the variance is exactly zero, the root in 64 bits rounds once."""
    x = dev.to_device(np.full((B, S, C), 3, np.float32))
    y, mean, rstd = dev.zeros((B, S, C)), dev.zeros((B, G)), dev.zeros((B, G))
    dev.groupnorm_fwd_f32(x, B, S, C, G, None, None, 1e-60, ref.NONE, y, mean, rstd)
    assert (y.numpy() == 0).all() and (mean.numpy() == 3).all()
    assert (np.abs(rstd.numpy().astype(np.float64) - 1e30) <= 2 * U * 1e30).all()
    for b in (x, y, mean, rstd):
        b.free()


@pytest.mark.parametrize("first", [1e6, -3e4])
@pytest.mark.parametrize("B,S,C,G", [(2, 40, 16, 4), (4, 1024, 256, 32), (1, 40000, 32, 1), (1, 30, 33, 3), (3, 1, 64, 2)])
def test_a_first_value_far_from_all_others(dev, B, S, C, G, first):
    """The first value of a group is far out: neither its own distance nor the others' lose anything by it."""
    rng = np.random.default_rng(S)
    x = (rng.standard_normal((B, S, C)) + 2).astype(np.float32)
    x[:, 0, ::C // G] = first
    d = dev.to_device(x)
    y, mean, rstd = dev.zeros(x.shape), dev.zeros((B, G)), dev.zeros((B, G))
    dev.groupnorm_fwd_f32(d, B, S, C, G, None, None, 1e-5, ref.NONE, y, mean, rstd)
    _, wm, wr = ref.groupnorm(x, G, None, None, 1e-5, ref.NONE)
    # chains of at most 128 additions in f32, each term of which is rounded twice, and squares twice as often
    mag = np.abs(x.astype(np.float64)).reshape(B, S, G, C // G).mean((1, 3))
    assert (np.abs(mean.numpy() - wm) <= 128 * U * mag + U * np.abs(wm)).all()
    assert (np.abs(rstd.numpy() - wr) <= 140 * U * wr).all()
    for b in (d, y, mean, rstd):
        b.free()


@pytest.mark.parametrize("B,S,C,G", SHAPES)
@pytest.mark.parametrize("kind", [ref.NONE, ref.RELU, ref.SILU])
def test_groups_that_hardly_vary_beside_others(dev, B, S, C, G, kind):
    """Every third group of every second sample lies at a million and takes four neighbouring values, the others are drawn
    from N(1, 1): y, in place and not."""
    rng = np.random.default_rng(B * S + C)
    w = C // G
    x = (rng.standard_normal((B, S, G, w)) + 1).astype(np.float32)
    far = np.add.outer(2 * np.arange(B), np.arange(G)) % 3 == 0
    far[1::2] = False
    near = np.float32(1000003.0) + rng.integers(0, 4, (B, S, G, w)).astype(np.float32) * np.float32(0.0625)
    x = np.ascontiguousarray(np.where(far[:, None, :, None], near, x), np.float32).reshape(B, S, C)
    gamma, beta = rng.uniform(0.5, 1.5, C).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    d, dga, dbe = dev.to_device(x), dev.to_device(gamma), dev.to_device(beta)
    y, mean, rstd = dev.zeros(x.shape), dev.zeros((B, G)), dev.zeros((B, G))
    args = (B, S, C, G, dga, dbe, 1e-5, kind)
    dev.groupnorm_fwd_f32(d, *args, y, mean, rstd)
    want, wm, wr = ref.groupnorm(x, G, gamma, beta, 1e-5, kind)
    per = lambda t: np.repeat(t, w, 1)[:, None, :]  # noqa: E731
    # the mean: rounded once, and chains of 128 additions of the distances of the groups near zero (below 2 in the mean);
    # rstd: half of what the variance carries, 128 additions and three roundings a term, and three roundings
    d_mean = np.where(far, 1.01 * U * np.abs(wm), 2 * 128 * U)
    d_rstd = wr * np.where(far, 4 * U, 70 * U)
    assert (np.abs(mean.numpy() - wm) <= d_mean).all() and (np.abs(rstd.numpy() - wr) <= d_rstd).all()
    x64 = x.astype(np.float64)
    h = (x64 - per(wm)) * per(wr)
    z = h * gamma + beta
    d_z = np.abs(gamma) * (per(wr * d_mean) + np.abs(h) * (per(d_rstd / wr) + 3 * U)) + U * (2 * np.abs(gamma * h) + np.abs(beta))
    tol = 1.01 * (1.1 * d_z + (8 + np.abs(z)) * U * np.abs(want)) + 1e-37
    got = y.numpy()
    assert (np.abs(got - want) <= tol).all()
    stats = mean.numpy(), rstd.numpy()
    dev.groupnorm_fwd_f32(d, *args, d, mean, rstd)
    assert np.array_equal(d.numpy(), got)
    assert np.array_equal(mean.numpy(), stats[0]) and np.array_equal(rstd.numpy(), stats[1])
    for b in (d, dga, dbe, y, mean, rstd):
        b.free()


@pytest.mark.parametrize("B,S,C,G", SHAPES)
@pytest.mark.parametrize("size", [1e-18, 1.0, 1e17])
def test_the_range_of_distances(dev, B, S, C, G, size):
    """x = +-size in turn, eps = 0: y is the sign of x, or close to it where there is one more of either."""
    sign = np.where(np.add.outer(np.arange(S), np.arange(C)) % 2, 1, -1)
    x = np.ascontiguousarray(np.broadcast_to(sign, (B, S, C)), np.float32) * np.float32(size)
    d = dev.to_device(x)
    y, mean, rstd = dev.zeros(x.shape), dev.zeros((B, G)), dev.zeros((B, G))
    dev.groupnorm_fwd_f32(d, B, S, C, G, None, None, 0.0, ref.NONE, y, mean, rstd)
    want, wm, wr = ref.groupnorm(x, G, None, None, 0.0, ref.NONE)
    # chains of at most 128 additions, each term rounded twice, its square three times; h three more
    assert (np.abs(mean.numpy() - wm) <= 130 * U * size).all()
    assert (np.abs(rstd.numpy() - wr) <= 70 * U * wr).all()
    assert np.abs(y.numpy() - want).max() <= 210 * U
    for b in (d, y, mean, rstd):
        b.free()
