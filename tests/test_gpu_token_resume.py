"""A training run with dropout that is saved, loaded into another session and continued gives the bits of the run that
was not interrupted: a checkpoint holds the key and the next step of every dropout layer."""
import json

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

B, T, V, D, OUT = 6, 5, 40, 8, 4


def model(session):
    from vtl_b200 import host
    m = host.Model(session)
    m.input([T])
    m.embedding(V, D, 1.5)
    m.dropout(0.3)
    m.groupnorm(2, 1e-3, "silu")
    m.flatten()
    m.dropout(0.123456789)
    m.linear(OUT)
    m.softmax_cross_entropy_loss()
    m.sgd(lr=0.1)
    return m


def session(seed):
    from vtl_b200 import capi, host
    if capi.device_count() == 0:
        pytest.skip("no CUDA device")
    s = host.Session(0)
    s.set_seed(seed)
    return s


def steps(s, m, n):
    rng = np.random.default_rng(1)
    ids, target = rng.integers(-1, V, (B, T)).astype(np.float32), np.eye(OUT, dtype=np.float32)[rng.integers(0, OUT, B)]
    dX, dT = s.dev.to_device(ids), s.dev.to_device(target)
    losses = [m.train_step(dX, ids.shape, dT, target.shape) for _ in range(n)]
    dX.free(); dT.free()
    return losses


def bits(m):
    return [m.get_param(i).view(np.uint32) for i in range(m.num_params())]


def test_a_resumed_run_continues_with_the_same_masks(tmp_path):
    path = str(tmp_path / "c.json")
    one = session(5)
    m = model(one)
    first = steps(one, m, 3)
    m.save_checkpoint(path, 1, first[-1])
    last, want, state = steps(one, m, 2), bits(m), [m.dropout_state(k) for k in range(2)]
    m.close()
    one.close()
    two = session(77)  # other initial weights, other keys
    m = model(two)
    m.load_weights(path)
    assert [m.dropout_state(k)[1] for k in range(2)] == [3, 3]
    assert steps(two, m, 2) == last
    assert all(np.array_equal(a, b) for a, b in zip(bits(m), want))
    assert [m.dropout_state(k) for k in range(2)] == state
    m.close()
    two.close()


def test_keys_and_steps_of_64_bits(tmp_path):
    path = str(tmp_path / "c.json")
    s = session(5)
    m = model(s)
    m.set_dropout_state(0, 2**64 - 1, 2**63 + 1)
    m.set_dropout_state(1, 0, 2**53 + 1)
    m.save_checkpoint(path, 0, 0.0)
    m.set_dropout_state(0, 1, 2)
    m.set_dropout_state(1, 3, 4)
    m.load_weights(path)
    assert m.dropout_state(0) == (2**64 - 1, 2**63 + 1) and m.dropout_state(1) == (0, 2**53 + 1)
    # a file without them (an older one) leaves them; a malformed one is refused
    file = json.load(open(path))
    entry = file["layer_data"][2]
    state = entry.pop("state")
    json.dump(file, open(path, "w"))
    m.set_dropout_state(0, 1, 2)
    m.load_weights(path)
    assert m.dropout_state(0) == (1, 2) and m.dropout_state(1) == (0, 2**53 + 1)
    from vtl_b200.capi import VtlbError
    for bad in ({"seed": "1"}, {"seed": "1", "step": "-1"}, {"seed": "1", "step": ""}, {"seed": "x", "step": "1"},
                {"seed": str(2**64), "step": "1"}, {"seed": 1, "step": 2}):
        entry["state"] = bad
        json.dump(file, open(path, "w"))
        with pytest.raises(VtlbError, match="state"):
            m.load_weights(path)
        assert m.dropout_state(0) == (1, 2)
    entry["state"] = state
    json.dump(file, open(path, "w"))
    m.load_weights(path)
    assert m.dropout_state(0) == (2**64 - 1, 2**63 + 1)
    m.close()
    s.close()


def test_a_checkpoint_tells_scale_eps_and_probability(tmp_path):
    path = str(tmp_path / "c.json")
    s = session(5)
    m = model(s)
    m.save_checkpoint(path, 0, 0.0)
    config = [layer["config"] for layer in json.load(open(path))["layers"]]
    assert config[1]["scale"] == 1.5 and config[1]["vocabulary"] == V and config[1]["dim"] == D
    assert config[2]["prob"] == 0.3 and config[5]["prob"] == 0.123456789
    assert config[3]["eps"] == 1e-3 and config[3]["num_groups"] == 2 and config[3]["activation"] == 2
    m.close()
    s.close()
