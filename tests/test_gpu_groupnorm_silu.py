"""SiLU in group norm where the logistic function is zero or one.  Half steps u = 2^-24."""
import numpy as np
import pytest

import token_ops_ref as ref

pytestmark = pytest.mark.gpu
U = 2.0**-24

# one position (odd and aligned rows), a cluster with and without TMA, a group no cluster holds (aligned and odd)
SHAPES = [(3, 1, 64, 2), (2, 1, 33, 1), (2, 40, 16, 4), (1, 30, 33, 3), (300, 17, 64, 64), (4, 1024, 256, 32), (2, 20000, 8, 1),
          (2, 20000, 33, 1), (1, 5, 40000, 2), (2, 515, 96, 3)]


@pytest.mark.parametrize("B,S,C,G", SHAPES)
def test_silu_where_the_logistic_function_is_zero_or_one(dev, B, S, C, G):
    """x = +1 and -1 in turn, gamma = 1e36: z is near +-1e36, so y is z or zero and the slope one or zero."""
    sign = np.where(np.add.outer(np.arange(S), np.arange(C)) % 2, 1, -1)
    x = np.ascontiguousarray(np.broadcast_to(sign, (B, S, C)), np.float32)
    g = np.random.default_rng(B + S + C).standard_normal((B, S, C)).astype(np.float32)
    gamma = np.full(C, 1e36, np.float32)
    d = {k: dev.to_device(v) for k, v in dict(x=x, g=g, gamma=gamma).items()}
    y, mean, rstd, dx, dgamma, dbeta = (dev.zeros(s) for s in (x.shape, (B, G), (B, G), x.shape, C, C))
    dev.groupnorm_fwd_f32(d["x"], B, S, C, G, d["gamma"], None, 1e-5, ref.SILU, y, mean, rstd)
    want, wm, wr = ref.groupnorm(x, G, gamma, None, 1e-5, ref.SILU)
    # h: the mean and rstd of values of size one, chains of at most 128 additions, and four roundings
    got = y.numpy()
    assert (got[x < 0] == 0).all()
    assert (np.abs(got - want) <= 300 * U * np.abs(want)).all()
    dev.groupnorm_bwd_f32(d["g"], d["x"], B, S, C, G, d["gamma"], None, mean, rstd, ref.SILU, dx, dgamma, dbeta)
    r = ref.groupnorm_bwd(g, x, G, gamma, None, mean.numpy(), rstd.numpy(), ref.SILU)
    # slopes are exactly 0 and 1, so dz is g or zero; sums of at most S * B terms in chains of fewer than 128 additions in
    # f32 with three roundings a term, joined in 64 bits
    size = np.abs(r["dz"])
    assert (np.abs(dbeta.numpy() - r["dbeta"]) <= 140 * U * size.sum((0, 1)) + 1e-37).all()
    assert (np.abs(dgamma.numpy() - r["dgamma"]) <= 140 * U * (size * np.abs(r["h"])).sum((0, 1)) + 1e-37).all()
    over, per = r["over"], r["per"]
    scale = r["rstd"] * (np.abs(r["dh"]) + per(over(np.abs(r["dh"]))) + np.abs(r["h"]) * per(over(np.abs(r["dh"] * r["h"]))))
    assert (np.abs(dx.numpy() - r["dx"]) <= 140 * U * scale).all()
    for b in list(d.values()) + [y, mean, rstd, dx, dgamma, dbeta]:
        b.free()
