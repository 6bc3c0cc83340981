"""The 64-bit definitions that the GPU tests of embedding, dropout and group norm compare with: the generator against
the known answers that its authors publish with it, the gradients against differences."""
import numpy as np
import pytest

import token_ops_ref as ref


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
    ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
    ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
     (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))])
def test_philox_known_answers(counter, key, want):
    assert tuple(int(w) for w in ref.philox4x32([counter], key)[0]) == want


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_share_of_dropped_elements(p):
    """n draws of probability p: within five standard deviations."""
    n = 200000
    dropped = 1 - ref.kept(n, p, 7, 3).mean()
    assert abs(dropped - p) <= 5 * np.sqrt(p * (1 - p) / n)


def test_masks_of_steps_and_seeds_are_unrelated():
    a = ref.kept(100000, 0.5, 1, 0)
    for other in (ref.kept(100000, 0.5, 1, 1), ref.kept(100000, 0.5, 2, 0), np.roll(ref.kept(100000, 0.5, 2, 0), 1)):
        assert abs((a == other).mean() - 0.5) < 5 * 0.5 / np.sqrt(100000)


@pytest.mark.parametrize("kind", [ref.NONE, ref.RELU, ref.SILU])
def test_groupnorm_gradient_against_differences(kind):
    """Central differences of sum(y * g) with h = 1e-5 in 64 bits: an error of h^2 times the third derivative, of order
    1, and of 1e-16 / h from rounding: 1e-8, and a factor of a hundred for the sizes of the values."""
    rng = np.random.default_rng(3)
    B, S, C, G = 2, 3, 6, 3
    x, g = rng.standard_normal((B, S, C)), rng.standard_normal((B, S, C))
    gamma, beta = rng.uniform(0.5, 1.5, C), rng.standard_normal(C) * 0.3
    value = lambda x_, ga, be: (ref.groupnorm(x_, G, ga, be, 1e-2, kind)[0] * g).sum()  # noqa: E731
    _, mean, rstd = ref.groupnorm(x, G, gamma, beta, 1e-2, kind)
    got = ref.groupnorm_bwd(g, x, G, gamma, beta, mean, rstd, kind)
    step = 1e-5

    def differences(a, f):
        out = np.zeros_like(a)
        for i in np.ndindex(a.shape):
            up, down = a.copy(), a.copy()
            up[i] += step
            down[i] -= step
            out[i] = (f(up) - f(down)) / (2 * step)
        return out

    assert np.abs(got["z"]).min() > 10 * step  # no kink of ReLU between the two points
    assert np.abs(got["dx"] - differences(x, lambda a: value(a, gamma, beta))).max() < 1e-6
    assert np.abs(got["dgamma"] - differences(gamma, lambda a: value(x, a, beta))).max() < 1e-6
    assert np.abs(got["dbeta"] - differences(beta, lambda a: value(x, gamma, a))).max() < 1e-6


def test_embedding_gradient_against_differences():
    rng = np.random.default_rng(4)
    V, D, ids = 5, 3, np.array([4, 0, -1, 4, 2, 5])
    W, g = rng.standard_normal((V, D)), rng.standard_normal((ids.size, D))
    keep = ref.kept(g.size, 0.4, 9, 2).reshape(g.shape) / 0.6

    def value(w):
        inside = (ids >= 0) & (ids < V)
        return (np.where(inside[:, None], w[np.where(inside, ids, 0)], 0) * 1.5 * keep * g).sum()

    got, _ = ref.embedding_bwd(g, ids, V, 1.5, 0.4, 9, 2)
    for i in np.ndindex(W.shape):  # linear: the difference is exact but for rounding
        up = W.copy()
        up[i] += 1.0
        assert abs((value(up) - value(W)) - got[i]) < 1e-12
