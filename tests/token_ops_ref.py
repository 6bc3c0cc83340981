"""The operators of token models (embedding, dropout, group norm) in 64 bits, from their definitions."""
import numpy as np

MASK32 = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=10):
    """Philox4x32 (Salmon, Moraes, Dror, Shaw, SC 2011): counter [n, 4], key [2] of 32-bit words -> [n, 4] words."""
    c = [np.asarray(counter, np.uint64).reshape(-1, 4)[:, k].copy() for k in range(4)]
    k0, k1 = np.uint64(key[0]), np.uint64(key[1])
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & MASK32, (a >> np.uint64(32)) ^ c[3] ^ k1, a & MASK32]
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & MASK32, (k1 + np.uint64(0xBB67AE85)) & MASK32
    return np.stack(c, 1)


def words(n, seed, step):
    """The generator's words of elements 0 .. n-1."""
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    counter = np.stack([block & MASK32, block >> np.uint64(32), np.full_like(block, step & 0xFFFFFFFF),
                        np.full_like(block, step >> 32)], 1)
    return philox4x32(counter, (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF)).reshape(-1)[:n]


def kept(n, p, seed, step):
    return words(n, seed, step) >= np.uint64(int(p * 2.0**32))


def dropout_f32(x, p, seed, step):
    """In f32, as defined: one product with the rounded 1 / (1 - p), or zero."""
    x = np.asarray(x, np.float32)
    if p == 1.0:
        return np.zeros_like(x)
    with np.errstate(all="ignore"):
        return np.where(kept(x.size, p, seed, step).reshape(x.shape), x * np.float32(1.0 / (1.0 - p)), np.float32(0))


def embedding_f32(W, ids, scale, p=0.0, seed=0, step=0):
    W, ids = np.asarray(W, np.float32), np.asarray(ids)
    inside = (ids >= 0) & (ids < W.shape[0])
    y = np.zeros((ids.size, W.shape[1]), np.float32)
    with np.errstate(all="ignore"):
        y[inside] = W[ids[inside]] * np.float32(scale)
    return dropout_f32(y, p, seed, step) if p else y


def embedding_bwd(g, ids, V, scale, p=0.0, seed=0, step=0):
    """-> (dW in 64 bits, a bound on the error of sums in f32 taken in any order).

    A sum of m terms, each of which carries the rounding of the mask's product, takes at most m - 1 additions; its
    product with the scale rounds once more: (m + 1) half steps of the sum of the terms' absolute values, and second
    order terms (1 %)."""
    g, ids = np.asarray(g, np.float64), np.asarray(ids)
    if p == 1.0:
        g = np.zeros_like(g)
    elif p:
        g = np.where(kept(g.size, p, seed, step).reshape(g.shape), g * (1.0 / (1.0 - p)), 0.0)
    inside = (ids >= 0) & (ids < V)
    dW, mag = np.zeros((V, g.shape[1])), np.zeros((V, g.shape[1]))
    np.add.at(dW, ids[inside], g[inside])
    np.add.at(mag, ids[inside], np.abs(g[inside]))
    m = np.bincount(ids[inside], minlength=V)[:, None]
    scale = float(np.float32(scale))
    # (the mask's factor is rounded once, the product with it once)
    return dW * scale, 1.01 * (m + (3 if p else 1)) * 2.0**-24 * mag * abs(scale) + 1e-40


# The activations by the numbers of the C interface.
NONE, RELU, SILU = 0, 1, 2


def act(z, kind):
    with np.errstate(over="ignore"):
        return z if kind == NONE else np.where(z < 0, 0.0, z) if kind == RELU else z / (1 + np.exp(-z))


def act_slope(z, kind):
    if kind == NONE:
        return np.ones_like(z)
    if kind == RELU:
        return (~(z < 0)).astype(np.float64)
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-z))
    return s * (1 + z * (1 - s))


def groupnorm(x, groups, gamma, beta, eps, kind):
    """x [B, S, C] -> (y, mean [B, groups], rstd [B, groups]) in 64 bits."""
    B, S, C = x.shape
    xg = np.asarray(x, np.float64).reshape(B, S, groups, C // groups)
    mean, var = xg.mean((1, 3)), xg.var((1, 3))
    rstd = 1 / np.sqrt(var + eps)
    h = (xg - mean[:, None, :, None]) * rstd[:, None, :, None]
    z = h.reshape(B, S, C) * (1.0 if gamma is None else np.asarray(gamma, np.float64)) + \
        (0.0 if beta is None else np.asarray(beta, np.float64))
    return act(z, kind), mean, rstd


def groupnorm_bwd(g, x, groups, gamma, beta, mean, rstd, kind):
    """-> dict of dx, dgamma, dbeta and what the sums are made of, in 64 bits, from the given statistics."""
    B, S, C = x.shape
    width = C // groups
    per = lambda t: np.repeat(np.asarray(t, np.float64), width, 1)[:, None, :]  # noqa: E731
    ga = np.ones(C) if gamma is None else np.asarray(gamma, np.float64)
    be = np.zeros(C) if beta is None else np.asarray(beta, np.float64)
    h = (np.asarray(x, np.float64) - per(mean)) * per(rstd)
    z = ga * h + be
    dz = np.asarray(g, np.float64) * act_slope(z, kind)
    dh = ga * dz
    over = lambda t: t.reshape(B, S, groups, width).mean((1, 3))  # noqa: E731
    dx = per(rstd) * (dh - per(over(dh)) - h * per(over(dh * h)))
    return {"dx": dx, "dgamma": (dz * h).sum((0, 1)), "dbeta": dz.sum((0, 1)), "h": h, "dz": dz, "dh": dh, "z": z,
            "rstd": per(rstd), "over": over, "per": per}
