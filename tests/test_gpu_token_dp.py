"""Embedding, dropout and group norm in a data-parallel session of one rank: its collectives are identities, so that gradients
and parameters have to be those of a plain session bit for bit, and a second pass adds to gradients under way."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, T, V, OUT = 12, 7, 60, 5


@pytest.mark.parametrize("D,G", [(24, 3), (128, 32)])  # dgamma and dbeta with a gap between them, and without one
def test_single_rank_communicator_equals_plain_session(D, G):
    from vtl_b200 import capi, host
    if capi.device_count() == 0:
        pytest.skip("no CUDA device")
    rng = np.random.default_rng(D)
    ids = rng.integers(-1, V, (B, T)).astype(np.float32)
    target = np.eye(OUT, dtype=np.float32)[rng.integers(0, OUT, B)]
    params = [rng.standard_normal((V, D)), rng.uniform(0.5, 1.5, D), rng.standard_normal(D) * 0.2,
              rng.standard_normal((OUT, T * D)) * 0.2, rng.standard_normal(OUT) * 0.1]
    results = []
    for with_comm in (False, True):
        s = host.Session(0)
        s.set_seed(3)
        if with_comm:
            s.comm_init(1, 0, s.dev.comm_unique_id())
        m = host.Model(s)
        m.input([T])
        m.embedding(V, D, 1.5)
        m.dropout(0.25)
        m.groupnorm(G, activation="silu")
        m.flatten()
        m.linear(OUT)
        m.softmax_cross_entropy_loss()
        m.adam(lr=1e-2)
        for i, p in enumerate(params):
            m.set_param(i, p.astype(np.float32))
        dX, dT = s.dev.to_device(ids), s.dev.to_device(target)
        step = lambda **kw: m.train_step(dX, ids.shape, dT, target.shape, global_rows=B, **kw)  # noqa: E731
        losses = [step(update=False)]
        once = [m.get_grad(i) for i in range(5)]
        losses += [step(), step(), step()]
        results.append((losses, once + [m.get_param(i) for i in range(5)] + [m.get_moment(i) for i in range(5)],
                        m.dropout_state(0)))
        assert s.dev.check_status() == 0
        m.close()
        dX.free(); dT.free()
        s.close()
    (l0, a0, d0), (l1, a1, d1) = results
    assert l0 == l1 and d0 == d1
    for a, b in zip(a0, a1):
        assert np.array_equal(a.view(np.uint32), b.view(np.uint32))
