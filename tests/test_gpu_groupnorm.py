"""vtlb_groupnorm_* against the 64-bit definition.  Tolerances are bounds on the rounding of f32 arithmetic, worked out
below with half steps u = 2^-24 and CHAIN, a bound on the additions that one sum in f32 passes through one after the
other (a thread's own rows, then threads, warps and blocks: at most 32 + 64 + 16 + 16)."""
import numpy as np
import pytest

import token_ops_ref as ref

pytestmark = pytest.mark.gpu
U, CHAIN, D53 = 2.0**-24, 128, 2.0**-53


def same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


def forward_bounds(x, G, gamma, beta, eps, kind, y, mean, rstd):
    """Bounds for y, mean and rstd."""
    B, S, C = x.shape
    per = lambda t: np.repeat(t, C // G, 1)[:, None, :]  # noqa: E731
    x = np.asarray(x, np.float64)
    mag = np.abs(x).reshape(B, S, G, C // G).mean((1, 3))
    d_mean = CHAIN * U * mag + U * np.abs(mean)
    # variance from squared distances (three roundings each, a shifted mean adds the square of its error) or from sums
    # in 64 bits, whose cancellation costs 2^-53 of the mean square
    d_rstd = rstd * (0.5 * ((CHAIN + 4) * U + (d_mean * rstd)**2 + 512 * D53 * (mean**2 + 1 / rstd**2) * rstd**2) + 3 * U)
    h = (x - per(mean)) * per(rstd)
    d_h = per(rstd * d_mean) + np.abs(h) * (per(d_rstd / rstd) + 2 * U)
    ga, be = (1.0 if gamma is None else np.abs(gamma.astype(np.float64))), (0.0 if beta is None else np.abs(beta.astype(np.float64)))
    d_z = ga * d_h + U * (2 * ga * np.abs(h) + be)
    # the logistic function of SiLU is evaluated within |z| + 7 half steps (the argument of its power is rounded: |z|; the
    # power 4, the sum 1, the reciprocal 2), its product with z rounds once more
    z = np.abs(h * (1.0 if gamma is None else gamma) + (0.0 if beta is None else beta))
    return 1.01 * (1.1 * d_z + (8 + z) * U * np.abs(y)) + 1e-37, 1.01 * d_mean + 1e-37, 1.01 * d_rstd


def backward_bounds(r, g, gamma, kind, S):
    g, h, dz, dh, z = np.abs(g.astype(np.float64)), np.abs(r["h"]), np.abs(r["dz"]), np.abs(r["dh"]), np.abs(r["z"])
    ga = 1.0 if gamma is None else np.abs(gamma.astype(np.float64))
    d_h = 2 * U * h
    d_z = ga * d_h + U * (2 * ga * h + z)
    d_dz = (g * (0.5 * d_z + 9 * U) if kind == ref.SILU else 0.0) + 2 * U * dz
    d_dh = ga * d_dz + U * dh
    over, per = r["over"], r["per"]
    m1, m2 = np.abs(per(over(r["dh"]))), np.abs(per(over(r["dh"] * r["h"])))
    d_m1 = per(over(d_dh) + CHAIN * U * over(dh))
    d_m2 = per(over(h * d_dh + dh * d_h) + (CHAIN + 2) * U * over(dh * h))
    dx = r["rstd"] * (d_dh + d_m1 + h * d_m2 + m2 * d_h + 4 * U * (dh + m1 + h * m2))
    dgamma = (h * d_dz + dz * d_h + (CHAIN + 2) * U * dz * h).sum((0, 1))
    dbeta = (d_dz + CHAIN * U * dz).sum((0, 1))
    return 1.01 * dx + 1e-37, 1.01 * dgamma + 1e-37, 1.01 * dbeta + 1e-37


SHAPES = [(1, 1, 1, 1), (2, 1, 8, 2), (1, 2, 4, 4), (3, 5, 6, 3), (2, 64, 128, 32), (1, 1000, 33, 11), (3, 323, 330, 30),
          (4, 1024, 256, 32), (1, 4097, 40, 5), (2, 7, 4096, 1), (65, 3, 20, 4), (1, 20001, 8, 2), (5, 1, 1000, 1),
          (2, 130, 36, 3), (300, 17, 64, 64), (1, 300, 1028, 2), (2, 2048, 24, 24), (1, 9000, 72, 1), (3, 33, 130, 13),
          (2, 515, 96, 3), (1, 1, 20000, 1), (1, 5, 40000, 2), (37, 1, 4096, 1), (9, 1, 16384, 2), (3, 1, 8196, 1), (50, 1, 130, 10),
          (1000, 1, 640, 5), (33, 1, 2047, 1), (200, 1, 300, 1), (7, 1, 513, 1), (65, 1, 96, 32), (20000, 1, 600, 1)]


@pytest.mark.parametrize("B,S,C,G", SHAPES)
@pytest.mark.parametrize("kind", [ref.NONE, ref.RELU, ref.SILU])
def test_forward_and_backward(dev, B, S, C, G, kind):
    rng = np.random.default_rng(B + S + C + G)
    x = (rng.standard_normal((B, S, C)) * 2 + 0.5).astype(np.float32)
    g = rng.standard_normal((B, S, C)).astype(np.float32)
    gamma, beta = rng.uniform(-1.5, 1.5, C).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    d = {k: dev.to_device(v) for k, v in dict(x=x, g=g, gamma=gamma, beta=beta).items()}
    out = {k: dev.to_device(np.full(s, 7, np.float32)) for k, s in
           dict(y=x.shape, mean=(B, G), rstd=(B, G), dx=x.shape, dgamma=C, dbeta=C).items()}
    dev.groupnorm_fwd_f32(d["x"], B, S, C, G, d["gamma"], d["beta"], 1e-3, kind, out["y"], out["mean"], out["rstd"])
    got = {k: out[k].numpy() for k in ("y", "mean", "rstd")}
    y, mean, rstd = ref.groupnorm(x, G, gamma, beta, float(1e-3), kind)
    tol = forward_bounds(x, G, gamma, beta, 1e-3, kind, y, mean, rstd)
    for name, want, t in zip(("y", "mean", "rstd"), (y, mean, rstd), tol):
        assert (np.abs(got[name] - want) <= t).all(), name
    dev.groupnorm_fwd_f32(d["x"], B, S, C, G, d["gamma"], d["beta"], 1e-3, kind, out["y"], out["mean"], out["rstd"])
    assert all(same(out[k].numpy(), got[k]) for k in got)
    r = ref.groupnorm_bwd(g, x, G, gamma, beta, got["mean"], got["rstd"], kind)
    tol = backward_bounds(r, g, gamma, kind, S)
    args = (d["g"], d["x"], B, S, C, G, d["gamma"], d["beta"], out["mean"], out["rstd"], kind)
    dev.groupnorm_bwd_f32(*args, out["dx"], out["dgamma"], out["dbeta"])
    first = {}
    for name, t in zip(("dx", "dgamma", "dbeta"), tol):
        first[name] = out[name].numpy()
        assert (np.abs(first[name] - r[name]) <= t).all(), name
    # each output by itself, and in place, gives the same bits
    for name in first:
        one = dev.to_device(np.full(first[name].shape, 7, np.float32))
        dev.groupnorm_bwd_f32(*args, **{name: one})
        assert same(one.numpy(), first[name]), name
        one.free()
    dev.groupnorm_bwd_f32(*args, dx=d["g"])
    assert same(d["g"].numpy(), first["dx"])
    dev.h2d_raw(d["g"].ptr, g.ctypes.data, g.nbytes)
    dev.groupnorm_bwd_f32(*args, dx=d["x"])
    assert same(d["x"].numpy(), first["dx"])
    dev.h2d_raw(d["x"].ptr, x.ctypes.data, x.nbytes)
    dev.groupnorm_fwd_f32(d["x"], B, S, C, G, d["gamma"], d["beta"], 1e-3, kind, d["x"], out["mean"], out["rstd"])
    assert same(d["x"].numpy(), got["y"])
    for b in list(d.values()) + list(out.values()):
        b.free()


@pytest.mark.parametrize("B,S,C,G", [(2, 9, 12, 3), (1, 700, 64, 8)])
def test_without_weights_or_biases(dev, B, S, C, G):
    rng = np.random.default_rng(5)
    x, g = rng.standard_normal((B, S, C)).astype(np.float32), rng.standard_normal((B, S, C)).astype(np.float32)
    gamma, beta = rng.uniform(0.5, 1.5, C).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    dx_, dg, dga, dbe = (dev.to_device(a) for a in (x, g, gamma, beta))
    y, mean, rstd, dx, dgamma, dbeta = (dev.zeros(s) for s in (x.shape, (B, G), (B, G), x.shape, C, C))
    for ga, be in ((None, None), (gamma, None), (None, beta)):
        pa, pb = (dga if ga is not None else None), (dbe if be is not None else None)
        dev.groupnorm_fwd_f32(dx_, B, S, C, G, pa, pb, 1e-5, ref.SILU, y, mean, rstd)
        want = ref.groupnorm(x, G, ga, be, 1e-5, ref.SILU)
        tol = forward_bounds(x, G, ga, be, 1e-5, ref.SILU, *want)
        assert (np.abs(y.numpy() - want[0]) <= tol[0]).all()
        dev.groupnorm_bwd_f32(dg, dx_, B, S, C, G, pa, pb, mean, rstd, ref.SILU, dx, dgamma, dbeta)
        r = ref.groupnorm_bwd(g, x, G, ga, be, mean.numpy(), rstd.numpy(), ref.SILU)
        for out, name, t in zip((dx, dgamma, dbeta), ("dx", "dgamma", "dbeta"), backward_bounds(r, g, ga, ref.SILU, S)):
            assert (np.abs(out.numpy() - r[name]) <= t).all(), name
    for b in (dx_, dg, dga, dbe, y, mean, rstd, dx, dgamma, dbeta):
        b.free()


@pytest.mark.parametrize("B,S,C,G", [(2, 50, 16, 4), (1, 3000, 64, 2), (1, 40000, 32, 1)])
def test_values_far_from_zero_and_constant_groups(dev, B, S, C, G):
    """A mean of ten thousand deviations keeps what its rounding leaves; a group without spread gives beta."""
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((B, S, C)) + 1e4).astype(np.float32)
    x[0, :, :C // G] = 3.25
    gamma, beta = rng.uniform(0.5, 1.5, C).astype(np.float32), rng.standard_normal(C).astype(np.float32)
    dx_, dga, dbe = dev.to_device(x), dev.to_device(gamma), dev.to_device(beta)
    y, mean, rstd = dev.zeros(x.shape), dev.zeros((B, G)), dev.zeros((B, G))
    dev.groupnorm_fwd_f32(dx_, B, S, C, G, dga, dbe, 1e-5, ref.NONE, y, mean, rstd)
    want = ref.groupnorm(x, G, gamma, beta, 1e-5, ref.NONE)
    for out, w, t in zip((y, mean, rstd), want, forward_bounds(x, G, gamma, beta, 1e-5, ref.NONE, *want)):
        assert (np.abs(out.numpy() - w) <= t).all()
    assert same(mean.numpy()[0, 0], np.float32(3.25))
    assert same(y.numpy()[0, :, :C // G], np.broadcast_to(beta[:C // G], (S, C // G)))
    for b in (dx_, dga, dbe, y, mean, rstd):
        b.free()


@pytest.mark.parametrize("B,S,C,G", [(2, 50, 16, 4), (2, 3000, 64, 4)])
def test_nan_and_infinities_stay_in_their_group(dev, B, S, C, G):
    rng = np.random.default_rng(7)
    x, g = rng.standard_normal((B, S, C)).astype(np.float32), rng.standard_normal((B, S, C)).astype(np.float32)
    w = C // G
    x[0, 3, w] = np.nan
    x[1, 4, 2 * w + 1] = np.inf
    dx_, dg = dev.to_device(x), dev.to_device(g)
    y, mean, rstd, dx = dev.zeros(x.shape), dev.zeros((B, G)), dev.zeros((B, G)), dev.zeros(x.shape)
    dev.groupnorm_fwd_f32(dx_, B, S, C, G, None, None, 1e-5, ref.SILU, y, mean, rstd)
    dev.groupnorm_bwd_f32(dg, dx_, B, S, C, G, None, None, mean, rstd, ref.SILU, dx)
    bad = np.zeros((B, G), bool)
    bad[0, 1] = bad[1, 2] = True
    for out in (y, dx):
        finite = np.isfinite(out.numpy()).reshape(B, S, G, w)
        assert finite.all((1, 3))[~bad].all() and not finite.any((1, 3))[bad].any()
    for b in (dx_, dg, y, mean, rstd, dx):
        b.free()


def test_relu_passes_its_gradient_by_the_sign_in_64_bits(dev):
    """Values whose z is zero but for rounding: x = mean, beta = 0, and its neighbours."""
    S, C = 64, 4
    x = np.zeros((1, S, C), np.float32)
    x[0, :, 0] = np.float32(0.1)
    x[0, ::2, 0] = np.nextafter(np.float32(0.1), np.float32(1))
    x[0, :, 1:] = np.random.default_rng(8).standard_normal((S, C - 1)).astype(np.float32)
    g = np.ones((1, S, C), np.float32)
    gamma, beta = np.array([1, 0.5, -1, 2], np.float32), np.array([0, 0, 0, 0.25], np.float32)
    mean, rstd = np.array([[0.1]], np.float32), np.array([[1.7]], np.float32)
    d = [dev.to_device(a) for a in (g, x, gamma, beta, mean, rstd)]
    dbeta = dev.zeros(C)
    dev.groupnorm_bwd_f32(d[0], d[1], 1, S, C, 1, d[2], d[3], d[4], d[5], ref.RELU, dbeta=dbeta)
    want = ref.groupnorm_bwd(g, x, 1, gamma, beta, mean, rstd, ref.RELU)["dbeta"]
    assert (dbeta.numpy() == want).all()  # counts
    for b in d + [dbeta]:
        b.free()


@pytest.mark.parametrize("B,S,C,G", [(2, 40, 16, 4), (1, 30, 33, 3), (1, 20000, 8, 1)])
def test_silu_of_large_values(dev, B, S, C, G):
    """z to a few hundred on both sides: 0 and z, slopes 0 and 1, no infinities."""
    rng = np.random.default_rng(11)
    x, g = rng.standard_normal((B, S, C)).astype(np.float32), rng.standard_normal((B, S, C)).astype(np.float32)
    gamma = np.full(C, 100, np.float32)
    dx_, dg, dga = dev.to_device(x), dev.to_device(g), dev.to_device(gamma)
    y, mean, rstd, dx, dgamma, dbeta = (dev.zeros(s) for s in (x.shape, (B, G), (B, G), x.shape, C, C))
    dev.groupnorm_fwd_f32(dx_, B, S, C, G, dga, None, 1e-5, ref.SILU, y, mean, rstd)
    want = ref.groupnorm(x, G, gamma, None, 1e-5, ref.SILU)
    # (below z = -87.3 the logistic function is held at 2^-126)
    assert (np.abs(y.numpy() - want[0]) <= forward_bounds(x, G, gamma, None, 1e-5, ref.SILU, *want)[0] + 1e-35).all()
    dev.groupnorm_bwd_f32(dg, dx_, B, S, C, G, dga, None, mean, rstd, ref.SILU, dx, dgamma, dbeta)
    r = ref.groupnorm_bwd(g, x, G, gamma, None, mean.numpy(), rstd.numpy(), ref.SILU)
    for out, name, t in zip((dx, dgamma, dbeta), ("dx", "dgamma", "dbeta"), backward_bounds(r, g, gamma, ref.SILU, S)):
        assert (np.abs(out.numpy() - r[name]) <= t + 1e-33).all(), name
    for b in (dx_, dg, dga, y, mean, rstd, dx, dgamma, dbeta):
        b.free()


@pytest.mark.parametrize("C,G", [(64, 8), (33, 3)])
def test_pointers_off_the_16_byte_grid(dev, C, G):
    rng = np.random.default_rng(9)
    B, S, n = 2, 45, 2 * 45 * C
    x, g = rng.standard_normal(n + 4).astype(np.float32), rng.standard_normal(n + 4).astype(np.float32)
    dx_, dg = dev.to_device(x), dev.to_device(g)
    gamma = rng.uniform(0.5, 1.5, C + 4).astype(np.float32)
    dga = dev.to_device(gamma)
    y, dx = dev.to_device(np.full(n + 8, 7, np.float32)), dev.to_device(np.full(n + 8, 7, np.float32))
    mean, rstd = dev.zeros((B, G)), dev.zeros((B, G))
    x0, g0, ga0 = x[1:n + 1].reshape(B, S, C), g[3:n + 3].reshape(B, S, C), gamma[2:C + 2]
    dev.groupnorm_fwd_f32(dx_.ptr + 4, B, S, C, G, dga.ptr + 8, None, 1e-5, ref.SILU, y.ptr + 8, mean, rstd)
    want = ref.groupnorm(x0, G, ga0, None, 1e-5, ref.SILU)
    got = y.numpy()
    assert (np.abs(got[2:n + 2].reshape(B, S, C) - want[0]) <= forward_bounds(x0, G, ga0, None, 1e-5, ref.SILU, *want)[0]).all()
    assert (got[:2] == 7).all() and (got[n + 2:] == 7).all()
    dev.groupnorm_bwd_f32(dg.ptr + 12, dx_.ptr + 4, B, S, C, G, dga.ptr + 8, None, mean, rstd, ref.SILU, dx.ptr + 4)
    r = ref.groupnorm_bwd(g0, x0, G, ga0, None, mean.numpy(), rstd.numpy(), ref.SILU)
    got = dx.numpy()
    assert (np.abs(got[1:n + 1].reshape(B, S, C) - r["dx"]) <= backward_bounds(r, g0, ga0, ref.SILU, S)[0]).all()
    assert (got[:1] == 7).all() and (got[n + 1:] == 7).all()
    for b in (dx_, dg, dga, y, dx, mean, rstd):
        b.free()


@pytest.mark.parametrize("B,S,C,G", [(3, 1, 64, 2), (2, 5, 8, 1)])
def test_eps_below_the_smallest_f32(dev, B, S, C, G):
    """rstd = 1 / sqrt(eps) of constant groups, where eps itself is no f32.  With several positions the variance comes from
    sums in 64 bits, of which it loses some 2^-53 of the mean square, 9: more than this eps, so there only the bound that
    counts it (512 * D53 * mean^2 in forward_bounds) can hold."""
    h = np.full((B, S, C), 3, np.float32)
    x = dev.to_device(h)
    y, mean, rstd = dev.zeros((B, S, C)), dev.zeros((B, G)), dev.zeros((B, G))
    dev.groupnorm_fwd_f32(x, B, S, C, G, None, None, 1e-60, ref.NONE, y, mean, rstd)
    assert (y.numpy() == 0).all() and (mean.numpy() == 3).all()
    want = ref.groupnorm(h, G, None, None, 1e-60, ref.NONE)
    t = 1e30 * 2 * U if S == 1 else forward_bounds(h, G, None, None, 1e-60, ref.NONE, *want)[2]
    assert (np.abs(rstd.numpy().astype(np.float64) - 1e30) <= t).all()
    for b in (x, y, mean, rstd):
        b.free()


def test_layer_norm_is_one_group_of_one_position(dev):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((70, 1, 256)).astype(np.float32)
    dx_, y, mean, rstd = dev.to_device(x), dev.zeros(x.shape), dev.zeros(70), dev.zeros(70)
    dev.groupnorm_fwd_f32(dx_, 70, 1, 256, 1, None, None, 1e-5, ref.NONE, y, mean, rstd)
    v = x.astype(np.float64)
    want = (v - v.mean(2, keepdims=True)) / np.sqrt(v.var(2, keepdims=True) + 1e-5)
    assert np.abs(y.numpy() - want).max() <= 200 * U * np.abs(want).max()
    for b in (dx_, y, mean, rstd):
        b.free()


def test_refusals(dev):
    from vtl_b200.capi import VtlbError
    d = dev.to_device(np.ones(256, np.float32))
    o = dev.zeros(256)
    for B, S, C, G in ((0, 1, 4, 2), (1, 0, 4, 2), (1, 1, 0, 1), (1, 1, 4, 0), (1, 1, 4, 3), (-1, 1, 4, 2)):
        with pytest.raises(VtlbError, match="bad shape"):
            dev.groupnorm_fwd_f32(d, B, S, C, G, None, None, 1e-5, 0, o, o, o)
        with pytest.raises(VtlbError, match="bad shape"):
            dev.groupnorm_bwd_f32(d, d, B, S, C, G, None, None, d, d, 0, o)
    with pytest.raises(VtlbError, match="unknown activation"):
        dev.groupnorm_fwd_f32(d, 1, 4, 4, 2, None, None, 1e-5, 3, o, o, o)
    for B, S, C, G in ((1 << 30, 1, 4, 4), (1 << 16, 1 << 15, 1, 1), (1, 65535 * 256 + 1, 4, 1)):
        with pytest.raises(VtlbError, match="go to"):
            dev.groupnorm_fwd_f32(d, B, S, C, G, None, None, 1e-5, 0, o, o, o)
    for eps in (-1e-5, float("nan")):
        with pytest.raises(VtlbError, match="eps"):
            dev.groupnorm_fwd_f32(d, 1, 4, 4, 2, None, None, eps, 0, o, o, o)
    with pytest.raises(VtlbError, match="null pointer"):
        dev.groupnorm_fwd_f32(d, 1, 4, 4, 2, None, None, 1e-5, 0, o, None, o)
    with pytest.raises(VtlbError, match="null pointer"):
        dev.groupnorm_bwd_f32(d, None, 1, 4, 4, 2, None, None, d, d, 0, o)
    with pytest.raises(VtlbError, match="overlap in part"):
        dev.groupnorm_fwd_f32(d, 1, 4, 4, 2, None, None, 1e-5, 0, d.ptr + 16, o, o)
    with pytest.raises(VtlbError, match="overlap in part"):
        dev.groupnorm_bwd_f32(d, o, 1, 4, 4, 2, None, None, o, o, 0, d.ptr + 32)
    assert (d.numpy() == 1).all()
    d.free(); o.free()


@pytest.mark.parametrize("B,S,C,G", [(70001, 1, 32, 1), (66000, 2, 6, 3), (70000, 1, 40, 40)])
def test_many_samples(dev, B, S, C, G):
    rng = np.random.default_rng(12)
    x, g = rng.standard_normal((B, S, C)).astype(np.float32), rng.standard_normal((B, S, C)).astype(np.float32)
    dx_, dg = dev.to_device(x), dev.to_device(g)
    y, mean, rstd, dx, dgamma, dbeta = (dev.zeros(s) for s in (x.shape, (B, G), (B, G), x.shape, C, C))
    dev.groupnorm_fwd_f32(dx_, B, S, C, G, None, None, 0.1, ref.SILU, y, mean, rstd)
    want = ref.groupnorm(x, G, None, None, 0.1, ref.SILU)
    for out, w, t in zip((y, mean, rstd), want, forward_bounds(x, G, None, None, 0.1, ref.SILU, *want)):
        assert (np.abs(out.numpy() - w) <= t).all()
    dev.groupnorm_bwd_f32(dg, dx_, B, S, C, G, None, None, mean, rstd, ref.SILU, dx, dgamma, dbeta)
    r = ref.groupnorm_bwd(g, x, G, None, None, mean.numpy(), rstd.numpy(), ref.SILU)
    for out, name, t in zip((dx, dgamma, dbeta), ("dx", "dgamma", "dbeta"), backward_bounds(r, g, None, ref.SILU, S)):
        assert (np.abs(out.numpy() - r[name]) <= t).all(), name
    for b in (dx_, dg, y, mean, rstd, dx, dgamma, dbeta):
        b.free()


def test_many_samples_whose_groups_are_read_twice(dev):
    """More samples than a grid has rows: the last ones get what they get in a call of their own."""
    B, S, C, last = 65600, 257, 33, 70
    n = S * C
    x, g, dx = (dev.empty(B * n) for _ in range(3))
    dev.init_normal_f32(x, B * n, 0.5, 2.0, 1)
    dev.init_normal_f32(g, B * n, 0.0, 1.0, 2)
    mean, rstd, part = dev.empty(B), dev.empty(B), dev.empty(last * n)
    dev.init_normal_f32(mean, B, 0.5, 0.1, 3)
    dev.init_uniform_f32(rstd, B, 0.4, 0.6, 4)
    dev.groupnorm_bwd_f32(g, x, B, S, C, 1, None, None, mean, rstd, ref.SILU, dx)
    at, st = 4 * (B - last) * n, 4 * (B - last)
    dev.groupnorm_bwd_f32(g.ptr + at, x.ptr + at, last, S, C, 1, None, None, mean.ptr + st, rstd.ptr + st, ref.SILU, part)
    got = np.empty(last * n, np.float32)
    dev.d2h_raw(got.ctypes.data, dx.ptr + at, got.nbytes)
    # dx is of the order of 1; its two means differ by the order of their sums (64 bits) and one rounding
    assert np.abs(got - part.numpy()).max() <= 2.0**-20
    xs, gs = np.empty((1, S, C), np.float32), np.empty((1, S, C), np.float32)
    dev.d2h_raw(xs.ctypes.data, x.ptr + 4 * (B - 1) * n, xs.nbytes)
    dev.d2h_raw(gs.ctypes.data, g.ptr + 4 * (B - 1) * n, gs.nbytes)
    r = ref.groupnorm_bwd(gs, xs, 1, None, None, mean.numpy()[-1:, None], rstd.numpy()[-1:, None], ref.SILU)
    t = backward_bounds(r, gs, None, ref.SILU, S)[0]
    assert (np.abs(got[-n:].reshape(1, S, C) - r["dx"]) <= t).all()
    for b in (x, g, dx, mean, rstd, part):
        b.free()
