"""States of a GatedRecurrence beside recordings of its predictions: a recording reads and writes the tensor that it was made with, so that stays, and
reset_states() zeroes it."""
import numpy as np
import pytest

import sequence_model as sm
from test_host_logic_cpu import host  # noqa: F401  (fixture)


def build(S):
    np.random.seed(0)
    rec = S.GatedRecurrence(sm.IN, sm.U, stateful=True)
    return rec, S.Sequential([S.Input((1, sm.IN)), rec])


def test_reset_keeps_what_a_recording_goes_on_from(host, monkeypatch):
    S = host.seera
    rec, model = build(S)
    X, _ = sm.data()
    step = lambda n, t: model.predict(X[:n, t:t + 1]).to_numpy()  # noqa: E731
    first = step(sm.N, 0)
    monkeypatch.setattr(host.fake, "is_capturing", lambda: True)
    step(sm.N, 1)
    monkeypatch.setattr(host.fake, "is_capturing", lambda: False)
    held = rec._state
    value = lambda: host.fake.to_host_f32(held.main_ptr, (sm.N, sm.U))  # noqa: E731
    assert value().any()
    rec.reset_states()
    assert not value().any()
    assert np.array_equal(step(sm.N, 0), first) and rec._state is held
    # other numbers of sequences come and go beside it
    rec.reset_states()
    at = held.main_ptr
    few = step(2, 0)
    assert np.array_equal(few, first[:2]) and rec._state is not held
    assert not value().any() and held.main_ptr == at
    with pytest.raises(ValueError):
        step(sm.N, 1)
    rec.reset_states()
    assert np.array_equal(step(sm.N, 0), first) and rec._state is held
    with pytest.raises(ValueError):
        step(2, 1)


def test_states_that_no_recording_holds_are_given_back(host):
    S = host.seera
    rec, model = build(S)
    X, _ = sm.data()
    for n in (1, 2, 3):
        rec.reset_states()
        model.predict(X[:n, :1])
    assert not rec._recorded and rec._state.shape == (3, sm.U)


@pytest.mark.gpu
def test_replays_after_a_reset():
    """Replay, reset, replay against fresh sequences; the memory is another tensor's neighbour and not another tensor."""
    from ml_framework_b200 import seera as S, seera_cuda as sc
    from ml_framework_b200.cuTen import cuten
    sc.init(0)
    sc.set_precision(3)
    rec, model = build(S)
    X, _ = sm.data()
    want = [model.predict(X[:, t:t + 1]).to_numpy() for t in range(6)]
    x = S.Tensor(X[:, :1], is_leaf=True)
    sc.graph_begin()
    out = model.predict(x)
    g = sc.graph_end()

    def replay(t):
        sc.upload_f32(x.value.main_ptr, np.ascontiguousarray(X[:, t:t + 1]))
        sc.graph_launch(g)
        return out.to_numpy()
    try:
        for _ in range(2):
            rec.reset_states()
            others = [cuten(np.full((sm.N, sm.U), 7, np.float32)) for _ in range(32)]
            got = [replay(t) for t in range(6)]
            assert all(np.array_equal(a, b) for a, b in zip(want, got))
            assert all((o.to_host_f32() == 7).all() for o in others)
        # an eager prediction of fewer sequences in between, then the recording again from zeros, and on by an eager step
        rec.reset_states()
        assert np.allclose(model.predict(X[:2, :1]).to_numpy(), want[0][:2], rtol=1e-6, atol=1e-6)
        assert np.array_equal(replay(0), want[0])
        rec.reset_states()
        assert np.array_equal(replay(0), want[0]) and np.array_equal(replay(1), want[1])
        assert np.array_equal(model.predict(X[:, 2:3]).to_numpy(), want[2])
    finally:
        sc.graph_destroy(g)
