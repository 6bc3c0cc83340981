"""Embedding, dropout and group norm as layers of a model: training steps through the host mirror against the same steps
in 64 bits, from the same masks."""
import numpy as np
import pytest

import token_ops_ref as ref

pytestmark = pytest.mark.gpu

B, T, V, D, G, OUT, P, SCALE, EPS = 6, 5, 40, 8, 2, 4, 0.3, 1.5, 1e-3


@pytest.fixture(scope="module")
def sess():
    from vtl_b200 import capi, host
    if capi.device_count() == 0:
        pytest.skip("no CUDA device")
    s = host.Session(0)
    yield s
    s.dev.sync()
    assert s.dev.check_status() == 0
    s.close()


def build(sess, params=None, fuse=True, second_dropout=True):
    from vtl_b200 import host
    sess.set_seed(5)
    m = host.Model(sess)
    m.input([T])
    m.embedding(V, D, SCALE)
    m.dropout(P)
    m.groupnorm(G, EPS, "silu")
    m.flatten()
    if second_dropout:
        m.dropout(0.5)
    m.linear(OUT)
    m.softmax_cross_entropy_loss()
    m.sgd(lr=0.1)
    m.set_fuse_relu(fuse)
    if params:
        for i, p in enumerate(params):
            m.set_param(i, p)
    return m


def parameters(rng):
    return [rng.standard_normal((V, D)), rng.uniform(0.5, 1.5, D), rng.standard_normal(D) * 0.2,
            rng.standard_normal((OUT, T * D)) * 0.2, rng.standard_normal(OUT) * 0.1]


def forward(params, ids, target, masks):
    """-> loss and what the backward pass needs, in 64 bits; masks: (seed, step) of both dropouts or None."""
    E, gamma, beta, W, b = params
    inside = (ids >= 0) & (ids < V)
    e = np.where(inside[..., None], E[np.where(inside, ids, 0)], 0.0) * SCALE
    k1 = ref.kept(e.size, P, *masks[0]).reshape(e.shape) / (1 - P)
    k2 = ref.kept(B * T * D, 0.5, *masks[1]).reshape(B, T * D) / 0.5
    x = e * k1
    y, mean, rstd = ref.groupnorm(x, G, gamma, beta, EPS, ref.SILU)
    f = y.reshape(B, T * D) * k2
    z = f @ W.T + b
    lse = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1, keepdims=True)) + z.max(1, keepdims=True)
    return (lse - (z * target).sum(1, keepdims=True)).mean(), (inside, k1, k2, x, mean, rstd, f, np.exp(z - lse))


def gradients(params, ids, target, masks):
    E, gamma, beta, W, b = params
    loss, (inside, k1, k2, x, mean, rstd, f, soft) = forward(params, ids, target, masks)
    dz = (soft - target) / B
    dy = ((dz @ W) * k2).reshape(B, T, D)
    r = ref.groupnorm_bwd(dy, x, G, gamma, beta, mean, rstd, ref.SILU)
    dE = np.zeros_like(E)
    np.add.at(dE, ids[inside], (r["dx"] * k1 * SCALE)[inside])
    return loss, [dE, r["dgamma"], r["dbeta"], dz.T @ f, dz.sum(0)]


def data(rng):
    ids = rng.integers(0, V, (B, T))
    ids[0, 3:] = -1   # a padded sample
    ids[1] = 7        # one token all over
    return ids, np.eye(OUT)[rng.integers(0, OUT, B)]


def test_gradients_against_differences():
    """The step that the device is compared with, by central differences (h = 1e-5: an error of order 1e-9)."""
    rng = np.random.default_rng(1)
    params, (ids, target), masks = parameters(rng), data(rng), ((11, 0), (12, 0))
    _, grads = gradients(params, ids, target, masks)
    for k, p in enumerate(params):
        for i in [np.unravel_index(j, p.shape) for j in rng.integers(0, p.size, 12)]:
            up, down = [q.copy() for q in params], [q.copy() for q in params]
            up[k][i] += 1e-5
            down[k][i] -= 1e-5
            diff = (forward(up, ids, target, masks)[0] - forward(down, ids, target, masks)[0]) / 2e-5
            assert abs(diff - grads[k][i]) < 1e-7


@pytest.mark.parametrize("fuse", [True, False])
def test_training_steps(sess, fuse):
    """Four SGD steps.  Every value passes fewer than 200 f32 roundings per step at sizes of a few units: 200 * 2^-24 *
    10 = 1.2e-4 per step bounds the parameters, four steps 5e-4 (a wrong mask or gradient is off by 1e-2 and more)."""
    rng = np.random.default_rng(2)
    params = [p.astype(np.float32) for p in parameters(rng)]
    ids, target = data(rng)
    m = build(sess, params, fuse)
    assert m.num_params() == 5
    want = [p.astype(np.float64) for p in params]
    seeds = [m.dropout_state(0)[0], m.dropout_state(1)[0]]
    assert seeds[0] != seeds[1] and m.dropout_state(0)[1] == 0
    dX, dT = sess.dev.to_device(ids.astype(np.float32)), sess.dev.to_device(target.astype(np.float32))
    for step in range(4):
        loss = m.train_step(dX, ids.shape, dT, target.shape)
        ref_loss, grads = gradients(want, ids, target, [(s, step) for s in seeds])
        want = [p - np.float32(0.1) * g for p, g in zip(want, grads)]
        assert abs(loss - ref_loss) <= 5e-4
        for i, p in enumerate(want):
            assert np.abs(m.get_param(i) - p.reshape(-1)).max() <= 5e-4, (step, i)
    assert m.dropout_state(0)[1] == 4
    m.close(); dX.free(); dT.free()


def test_fused_and_separate_layers_give_the_same_bits(sess):
    rng = np.random.default_rng(3)
    params = [p.astype(np.float32) for p in parameters(rng)]
    ids, target = data(rng)
    dX, dT = sess.dev.to_device(ids.astype(np.float32)), sess.dev.to_device(target.astype(np.float32))
    got = []
    for fuse in (True, False):
        m = build(sess, params, fuse)
        loss = m.train_step(dX, ids.shape, dT, target.shape, update=False)
        got.append([loss] + [m.get_grad(i) for i in range(5)])
        m.close()
    assert got[0][0] == got[1][0]
    for a, b in zip(got[0][1:], got[1][1:]):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
    dX.free(); dT.free()


def test_masks_change_from_step_to_step_and_can_be_repeated(sess):
    rng = np.random.default_rng(4)
    params = [p.astype(np.float32) for p in parameters(rng)]
    ids, target = data(rng)
    dX, dT = sess.dev.to_device(ids.astype(np.float32)), sess.dev.to_device(target.astype(np.float32))
    m = build(sess, params)
    run = lambda: m.train_step(dX, ids.shape, dT, target.shape, update=False)  # noqa: E731
    first, second = run(), run()
    assert first != second
    for k in range(2):
        seed, step = m.dropout_state(k)
        assert step == 2
        m.set_dropout_state(k, seed, 0)
    m.zero_grad()
    assert run() == first and run() == second
    m.close(); dX.free(); dT.free()


def test_inference_drops_nothing(sess):
    rng = np.random.default_rng(5)
    params = [p.astype(np.float32) for p in parameters(rng)]
    ids, _ = data(rng)
    m = build(sess, params)
    dX, dY = sess.dev.to_device(ids.astype(np.float32)), sess.dev.zeros((B, OUT))
    m.forward(dX, ids.shape, dY)
    E, gamma, beta, W, b = [p.astype(np.float64) for p in params]
    e = np.where((ids >= 0)[..., None], E[np.maximum(ids, 0)], 0.0) * SCALE
    y, _, _ = ref.groupnorm(e, G, gamma, beta, EPS, ref.SILU)
    z = y.reshape(B, T * D) @ W.T + b
    assert np.abs(dY.numpy() - z).max() <= 200 * 2.0**-24 * 10
    assert m.dropout_state(0)[1] == 0
    first = dY.numpy()
    m.forward(dX, ids.shape, dY)
    assert np.array_equal(first, dY.numpy())
    m.close(); dX.free(); dY.free()


def test_checkpoint_round_trip(sess, tmp_path):
    rng = np.random.default_rng(6)
    params = [p.astype(np.float32) for p in parameters(rng)]
    m, other = build(sess, params), build(sess)
    path = str(tmp_path / "tokens.json")
    m.save_checkpoint(path, 3, 0.25)
    assert not np.array_equal(other.get_param(0), params[0].reshape(-1))
    other.load_weights(path)
    for i, p in enumerate(params):
        assert np.array_equal(other.get_param(i), p.reshape(-1))
    m.close(); other.close()


def test_builder_refusals(sess):
    from vtl_b200 import host
    from vtl_b200.capi import VtlbError
    m = host.Model(sess)
    with pytest.raises(VtlbError, match="input"):
        m.dropout(0.5)
    m.input([3, 4, 4])
    for bad in (-0.1, 1.5, float("nan")):
        with pytest.raises(VtlbError, match="probability"):
            m.dropout(bad)
    with pytest.raises(VtlbError, match="divide"):
        m.groupnorm(3)
    with pytest.raises(VtlbError, match="eps"):
        m.groupnorm(2, eps=-1.0)
    with pytest.raises(VtlbError, match="positive"):
        m.embedding(0, 8)
    with pytest.raises(VtlbError, match="2\\^24"):
        m.embedding((1 << 24) + 2, 1)
    m.groupnorm(2)
    with pytest.raises(VtlbError, match="follows the input"):
        m.embedding(5, 8)
    d = sess.dev.zeros(64)
    with pytest.raises(VtlbError, match="batch"):
        m.forward(d, (0, 3, 4, 4), d)
    with pytest.raises(VtlbError, match="channels"):
        m.forward(d, (1, 3, 4, 5), d)
    d.free()
    m.close()
    m = host.Model(sess)
    m.input([3, 4, 4])
    m.conv2d(3, 4, (3, 3), padding=(1, 1))
    with pytest.raises(VtlbError, match="convolutions"):
        m.groupnorm(2)
    m.close()
