"""Host logic of the sequence layers, the norms and AdamW on the host-memory stand-in for the binding: what is called with what, whose gradient goes
where, states, lengths, checkpoints, refusals."""
import numpy as np
import pytest

import sequence_model as sm
import sequence_np as ref
from test_host_logic_cpu import host  # noqa: F401  (fixture)

# a handful of float32 matrix products of inner size up to 36 and roundings of stored values: far below this
TOL = 2e-5


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("head,norm,gate", [("softmax", "rms", "silu"), ("mse", "layer", "sigmoid"), ("mse", "rms", None)])
def test_step_against_64_bits(host, monkeypatch, fused, head, norm, gate):
    monkeypatch.setattr(host.seera, "FUSE_NORM", fused)
    before = dict(host.fake.CALLS)
    sm.check_step(host.seera, TOL, head, norm, gate)
    calls = lambda k: host.fake.CALLS.get(k, 0) - before.get(k, 0)  # noqa: E731
    assert calls("gated_residual_fwd") == calls("gated_residual_bwd") == 2
    assert calls("norm_fwd") == calls("norm_bwd") == (1 if fused else 3)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("head", ["softmax", "mse"])
def test_ragged_step_against_64_bits(host, monkeypatch, fused, head):
    monkeypatch.setattr(host.seera, "FUSE_NORM", fused)
    sm.check_step(host.seera, TOL, head, lengths=np.array([21, 1, 0, 13, 20]), passes=2)


def test_lengths_belong_to_one_pass(host):
    S = host.seera
    model = sm.build(S)
    X, _ = sm.data()
    whole = model.forward(X).to_numpy()
    short = model.forward(X, lengths=[3] * sm.N).to_numpy()
    assert not np.allclose(whole, short)
    assert np.array_equal(model.forward(X).to_numpy(), whole)
    assert np.array_equal(model.forward(X[:, :3]).to_numpy(), short)
    on_device = host.cuTen.cuten(np.full(sm.N, 3, np.int32), "int32")
    assert np.array_equal(model.predict(X, lengths=on_device).to_numpy(), short)
    for bad in ([3] * (sm.N - 1), [[3] * sm.N], [0.5] * sm.N):
        with pytest.raises(ValueError):
            model.forward(X, lengths=bad)


def test_state_goes_from_prediction_to_prediction(host):
    S = host.seera
    np.random.seed(0)
    rec = S.GatedRecurrence(sm.IN, sm.U, stateful=True)
    last = S.GatedRecurrence(sm.U, sm.U, stateful=True, return_sequences=False)
    model = S.Sequential([S.Input((sm.T, sm.IN)), rec, last])
    X, _ = sm.data()
    want = model.forward(X).to_numpy()                     # training passes start from zeros and leave no state
    assert rec._state is None
    for cut in ((0, 1, 2, 20, 21), (0, 21)):
        rec.reset_states(), last.reset_states()
        outs = [model.predict(X[:, a:b]) for a, b in zip(cut, cut[1:])]
        first = outs[0].to_numpy()
        assert np.allclose(outs[-1].to_numpy(), want, atol=1e-6)
        assert np.array_equal(outs[0].to_numpy(), first)   # an output is not the state that the next call writes
    assert np.allclose(model.forward(X).to_numpy(), want, atol=0)
    with pytest.raises(ValueError):
        model.predict(X[:2])
    rec.reset_states(), last.reset_states()
    model.predict(X[:2])
    with pytest.raises(RuntimeError):
        S.autograd4nn(S.Loss().mse(model.predict(X[:2]), S.Tensor(np.zeros((2, sm.U), np.float32), is_leaf=True)))


def test_an_output_gate_that_nobody_takes_has_no_gradient(host):
    S = host.seera
    np.random.seed(1)
    rec = S.GatedRecurrence(sm.IN, sm.U, output_gate=True)
    model = S.Sequential([S.Input((sm.T, sm.IN)), rec])
    X, Y = sm.data(classes=False)
    S.autograd4nn(S.Loss().mse(model.forward(X), S.Tensor(Y, is_leaf=True)))
    assert (rec.weights.grad.to_host_f32()[:, 2 * sm.U:] == 0).all() and (rec.bais.grad.to_host_f32()[:, 2 * sm.U:] == 0).all()
    assert (rec.weights.grad.to_host_f32()[:, :2 * sm.U] != 0).any()


def test_residual_end_without_residual_and_gate_in_a_plain_network(host):
    """Between Dense layers: rows instead of sequences, no gate, no residual, and a residual that is the input itself."""
    S = host.seera
    np.random.seed(2)
    inp = S.Input((sm.IN,))
    end = S.GatedResidual(sm.IN, residual=inp, norm="layer")
    alone = S.GatedResidual(sm.IN)
    model = S.Sequential([inp, S.LayerNorm(sm.IN), S.Dense(sm.IN, sm.IN, "tanh"), end, S.Dense(sm.IN, sm.IN, "sigmoid"), alone])
    r = np.random.RandomState(0)
    X, Y = r.standard_normal((7, sm.IN)).astype(np.float32), r.standard_normal((7, sm.IN)).astype(np.float32)
    S.autograd4nn(S.Loss().mse(model.forward(X), S.Tensor(Y, is_leaf=True)))
    assert (alone.scale.grad.to_host_f32() == 0).all()
    import torch
    P = sm.params64(model)
    x = torch.tensor(X, dtype=torch.float64)
    n = lambda a, k, e: (a - (a.mean(-1, keepdim=True) if k else 0)) / torch.sqrt(((a - (a.mean(-1, keepdim=True) if k else 0)) ** 2).mean(-1, keepdim=True) + e)  # noqa: E731
    h = torch.tanh((n(x, 1, 1e-5) * P[0][0] + P[0][1]) @ P[1][0] + P[1][1])
    h = P[2][1] * x + P[2][0] * n(h, 1, 1e-6)
    h = P[4][0] * n(torch.sigmoid(h @ P[3][0] + P[3][1]), 0, 1e-6)
    ((h - torch.tensor(Y, dtype=torch.float64)) ** 2).mean().backward()
    for l, p in zip(model.param_layers, P):
        for t, q in zip((l.weights, l.bais), p):
            if q.grad is not None:
                g = t.grad.to_host_f32().reshape(q.shape)
                assert np.linalg.norm(g - q.grad.numpy()) < TOL * max(1e-3, np.linalg.norm(q.grad.numpy())), l


def test_refusals(host):
    S = host.seera
    for bad in (lambda: S.GatedResidual(4, activation="softmax"), lambda: S.GatedResidual(4, norm="batch"), lambda: S.GatedRecurrence(4, 4, True, False),
                lambda: S.GatedRecurrence(4, 4, kernel_initializer="none"), lambda: S.GatedRecurrence(4, 4, bias_initializer="none")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        S.GatedResidual(4, residual=3)
    with pytest.raises(ValueError):                          # a residual of another model, and one that comes later
        S.Sequential([S.Input((4,)), S.GatedResidual(4, residual=S.Input((4,)))])
    late = S.RMSNorm(4)
    with pytest.raises(ValueError):
        S.Sequential([S.Input((4,)), S.GatedResidual(4, residual=late), late])
    x3 = np.zeros((2, 3, 4), np.float32)
    for layer, x in ((S.RMSNorm(5), x3), (S.RMSNorm(4), np.zeros(4, np.float32)), (S.GatedRecurrence(5, 4), x3), (S.GatedRecurrence(4, 4), x3[0]),
                     (S.GatedResidual(5), x3)):
        with pytest.raises(ValueError):
            S.Sequential([S.Input((3, 4)), layer]).forward(x)
    inp = S.Input((3, 4))
    with pytest.raises(ValueError):                          # shapes that differ
        S.Sequential([inp, S.GatedRecurrence(4, 6), S.GatedResidual(6, residual=inp)]).forward(x3)
    m = S.Sequential([S.Input((4,)), S.Dense(4, 4, "tanh")])
    with pytest.raises(ValueError):
        S.AdamW(m, state_bits=16)
    with pytest.raises(TypeError):
        S.AdamW(None)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_step_decays_matrices_alone(host, bits):
    S = host.seera
    model = sm.build(S)
    opt = S.AdamW(model, lr=1e-2, weight_decay=0.2, state_bits=bits)
    X, Y = sm.data()
    w0, m, v = {}, {}, {}
    for step in range(3):
        loss = S.Loss().categorical_cross_entropy(model.forward(X), S.Tensor(Y, is_leaf=True))
        model.zero_grad()
        S.autograd4nn(loss)
        before = [[t.to_numpy() for t in (l.weights, l.bais)] for l in model.param_layers]
        grads = [[t.grad.to_host_f32().copy() for t in (l.weights, l.bais)] for l in model.param_layers]
        opt.step()
        t = step + 1
        for k, (l, b, g) in enumerate(zip(model.param_layers, before, grads)):
            for j, p in enumerate((l.weights, l.bais)):
                decay = 0.2 if j == 0 and l.__class__.__name__ in ("Dense", "GatedRecurrence") else 0.0
                z = np.zeros(p.value.size, np.float32)
                W, M, V, bound = ref.adamw(b[j].ravel(), g[j].ravel(), m.get((k, j), z), v.get((k, j), z), decay, 1e-2, 0.9, 1 - 0.9, 0.999, 1 - 0.999, 1e-8,
                                           1 - 0.9 ** t, 1 - 0.999 ** t, 1.0)
                assert (np.abs(p.to_numpy().ravel() - W) <= bound).all(), (l, j)
                if bits == 8:
                    M, V = ref.unpack8(ref.pack8(M, V, t, p._arena_off), M.size)
                m[k, j], v[k, j] = M, V
    assert opt.t == 4


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_by_ranges_is_the_whole_update(host, bits):
    """As the bucket hooks of a data-parallel run update, with the scalars on the device."""
    S = host.seera
    out = []
    for parts in (1, 3):
        model = sm.build(S)
        opt = S.AdamW(model, lr=1e-2, state_bits=bits)
        X, Y = sm.data()
        for _ in range(2):
            S.autograd4nn(S.Loss().categorical_cross_entropy(model.forward(X), S.Tensor(Y, is_leaf=True)))
            model.gather_grads()
            if parts == 1:
                opt.step()
            else:
                opt._advanced = False
                cuts = [0] + [model.parameters()[i]._arena_off for i in (5, 11)] + [model.n_arena]
                for a, b in reversed(list(zip(cuts, cuts[1:]))):
                    opt.update_range(a, b)
            model.zero_grad()
        out.append(model.params.to_host_f32().copy())
    assert np.array_equal(*out)


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_resumes_exactly(host, tmp_path, bits):
    S = host.seera
    X, Y = sm.data()

    def step(m, o):
        loss = S.Loss().categorical_cross_entropy(m.forward(X), S.Tensor(Y, is_leaf=True))
        m.zero_grad()
        S.autograd4nn(loss)
        o.step()
    a = sm.build(S, norm="layer", gate="tanh")
    oa = S.AdamW(a, lr=1e-2, weight_decay=0.1, state_bits=bits)
    step(a, oa), step(a, oa)
    path = str(tmp_path / "c.pkl")
    a.save(path, optimizer=oa)
    b, ob = S.Sequential.load(path, with_optimizer=True)
    assert ob.state_bits == bits and ob.t == 3 and ob.weight_decay == 0.1
    assert [type(l) for l in a.model] == [type(l) for l in b.model]
    assert b.model[4].residual is b.model[1] and b.model[4].activation == "tanh" and b.model[4].norm == "layer"
    step(a, oa), step(b, ob)
    assert np.array_equal(a.params.to_host_f32(), b.params.to_host_f32())


def test_fit_trains_sequences(host):
    S = host.seera
    model = sm.build(S)
    X, Y = sm.data()
    w = model.params.to_host_f32().copy()
    hist = model.fit(X, Y, S.AdamW(model, lr=1e-2, state_bits=8), S.Loss().categorical_cross_entropy, 2, batch_size=2)
    assert len(hist) == 2 and np.isfinite(hist).all() and not np.array_equal(w, model.params.to_host_f32())


def test_two_norms_of_one_residual_end_keep_apart(host):
    """Put together by hand: only the norm that was linked last is taken in the residual's launch."""
    S = host.seera
    inp = S.Input((4,))
    end = S.GatedResidual(4, residual=inp)(S.Dense(4, 4, "tanh")(inp))
    one, two = S.RMSNorm(4)(end), S.RMSNorm(4)(end)
    one.set_weights(np.full(4, 2, np.float32), np.zeros(4, np.float32))
    inp.inputs = S.Tensor(np.random.RandomState(0).standard_normal((3, 4)).astype(np.float32), is_leaf=True)
    inp.forward(), end.inpobj.forward(), end.forward()
    a, b = one.forward().to_numpy(), two.forward().to_numpy()
    assert np.allclose(a, 2 * b)
