"""Gated recurrent blocks, their norms and AdamW as a user has them: whole steps against 64 bits in the precision modes, in batches, recorded and replayed, on
another stream, through fit, and token by token."""
import numpy as np
import pytest

import sequence_model as sm
import sequence_np as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def E():
    from ml_framework_b200 import seera as S, seera_cuda as sc
    sc.init(0)
    yield S, sc
    sc.set_precision(3)


# products of at most 36 terms: fp32 and the fp32-class splits stay at float32's rounding, mode 4's weight gradients are formed from one fp16 copy each
# (2^-12 of an entry, 2.4e-4), mode 5 and its data gradients likewise; gradients pass five such products at most
@pytest.mark.parametrize("mode,tol", [(0, 2e-5), (3, 2e-5), (4, 2e-3)])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("head,norm,gate,lengths", [("softmax", "rms", "silu", None), ("mse", "layer", "sigmoid", [21, 1, 0, 13, 20]), ("softmax", "layer", "tanh", [1, 2, 3, 4, 5])])
def test_step_against_64_bits(E, monkeypatch, mode, tol, fused, head, norm, gate, lengths):
    S, sc = E
    monkeypatch.setattr(S, "FUSE_NORM", fused)
    sc.set_precision(mode)
    sm.check_step(S, tol, head, norm, gate, lengths=lengths, passes=4)        # from the second on in batches


def steps(S, model, opt, X, Y, n):
    for _ in range(n):
        loss = S.Loss().categorical_cross_entropy(model.forward(X), Y)
        model.zero_grad()
        S.autograd4nn(loss)
        opt.step()
    return loss


@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_steps_are_the_eager_ones(E, bits):
    """Two recordings alive at once, replayed in turn with eager steps between them, against eager steps alone: the same bits.  The learning rate changes
    on the way and the 8-bit rounding draws anew each step."""
    S, sc = E
    sc.set_precision(3)
    out = []
    for recorded in (False, True):
        X, Y = (S.Tensor(a, is_leaf=True) for a in sm.data())
        models = [sm.build(S, seed=k) for k in (0, 1)]
        opts = [S.AdamW(m, lr=1e-2, weight_decay=0.1, state_bits=bits) for m in models]
        for m, o in zip(models, opts):
            steps(S, m, o, X, Y, 2)
        graphs, keep = [], []
        if recorded:
            for m, o in zip(models, opts):
                o._scalars_in_graph = True
                sc.graph_begin()
                keep.append(steps(S, m, o, X, Y, 1))
                o._scalars_in_graph = False
                graphs.append(sc.graph_end())
        for k in range(6):
            for i, (m, o) in enumerate(zip(models, opts)):
                o.lr = 1e-2 / (k + 1)
                if recorded and k != 3:
                    sc.graph_set_scalars(graphs[i], o._scalars())
                    sc.graph_launch(graphs[i])
                else:
                    steps(S, m, o, X, Y, 1)
        out.append([m.params.to_host_f32().copy() for m in models])
        for g in graphs:
            sc.graph_destroy(g)
    assert all(np.array_equal(a, b) for a, b in zip(*out))


def test_recorded_prediction_carries_its_state(E):
    S, sc = E
    sc.set_precision(3)
    np.random.seed(0)
    rec = S.GatedRecurrence(sm.IN, sm.U, stateful=True)
    model = S.Sequential([S.Input((1, sm.IN)), S.RMSNorm(sm.IN), rec])
    X, _ = sm.data()
    x = S.Tensor(X[:, :1], is_leaf=True)
    sc.graph_begin()
    try:
        with pytest.raises(RuntimeError):                 # the state's zeros would be part of the recording
            model.predict(x)
    finally:
        sc.graph_destroy(sc.graph_end())
    want = [model.predict(X[:, t:t + 1]).to_numpy() for t in range(sm.T)]
    rec.reset_states()
    got = [model.predict(x).to_numpy()]
    sc.graph_begin()
    out = model.predict(x)
    g = sc.graph_end()
    for t in range(1, sm.T):
        sc.upload_f32(x.value.main_ptr, np.ascontiguousarray(X[:, t:t + 1]))
        sc.graph_launch(g)
        got.append(out.to_numpy())
    sc.graph_destroy(g)
    assert all(np.array_equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("bits", [8, 32])
def test_fit_records_the_same_steps(E, bits):
    """fit, whose full batches are replays, against the unpipelined loop."""
    S, sc = E
    sc.set_precision(3)
    r = np.random.RandomState(3)
    X = r.standard_normal((38, sm.T, sm.IN)).astype(np.float32)
    Y = np.eye(sm.CLASSES, dtype=np.float32)[r.randint(0, sm.CLASSES, 38)]
    out = []
    for loop in ("fit", "_fit_unpipelined"):
        model = sm.build(S)
        opt = S.AdamW(model, lr=1e-2, state_bits=bits)
        np.random.seed(4)
        hist = getattr(model, loop)(X, Y, opt, S.Loss().categorical_cross_entropy, 3, batch_size=6)
        out.append((np.asarray(hist), model.params.to_host_f32().copy(), opt.t))
    assert out[0][2] == out[1][2]
    assert np.array_equal(out[0][1], out[1][1])
    assert np.allclose(out[0][0], out[1][0], rtol=1e-6, atol=0)


def test_on_a_stream_of_the_caller(E):
    import torch
    S, sc = E
    sc.set_precision(3)
    model = sm.build(S)
    X, Y = sm.data()
    opt = S.AdamW(model, state_bits=8)
    x, y = S.Tensor(X, is_leaf=True), S.Tensor(Y, is_leaf=True)
    steps(S, model, opt, x, y, 3)
    want = model.params.to_host_f32().copy()
    side = torch.cuda.Stream()
    model = sm.build(S)
    opt = S.AdamW(model, state_bits=8)
    sc.stream_synchronize()
    sc.set_stream(side.cuda_stream)
    try:
        steps(S, model, opt, x, y, 3)
        got = model.params.to_host_f32().copy()
    finally:
        sc.stream_synchronize()
        sc.set_stream(0)
    assert np.array_equal(want, got)


def test_more_tensors_than_one_launch_takes(E):
    """A recorded update of 200 tensors in several launches: all of them get the new scalars."""
    S, sc = E
    from ml_framework_b200.cuTen import cuten
    r = np.random.RandomState(0)
    sizes = [1 + 13 * i % 97 for i in range(200)]
    host = {k: [r.standard_normal(n).astype(np.float32) for n in sizes] for k in "wg"}
    dev = {k: [cuten(a) for a in host[k]] for k in "wg"}
    st = [cuten._wrap(sc.cuda_zeros_f(sc.adamw8_state_bytes(n) // 4), (sc.adamw8_state_bytes(n) // 4,)) for n in sizes]
    at = lambda ts: np.array([t.main_ptr for t in ts], np.uint64)  # noqa: E731
    table = (at(dev["w"]), at(dev["g"]), at(st), np.array(sizes, np.int64), np.full(200, 0.1, np.float32))
    hp = lambda t: [1e-2 / t, 0.9, 1 - 0.9, 0.99, 1 - 0.99, 1e-8, 1 - 0.9 ** t, 1 - 0.99 ** t, 1.0, float(t)]  # noqa: E731
    sc.graph_begin()
    sc.adamw8_step(*table, *hp(1))
    g = sc.graph_end()
    for t in (1, 2, 3):
        sc.graph_set_scalars(g, hp(t))
        sc.graph_launch(g)
    sc.stream_synchronize()
    first = 0
    for i, n in enumerate(sizes):
        w, m, v = host["w"][i].astype(np.float64), np.zeros(n, np.float32), np.zeros(n, np.float32)
        off = np.zeros(n)
        for t in (1, 2, 3):
            w32 = w.astype(np.float32)
            w, M, V, bound = ref.adamw(w32, host["g"][i], m, v, 0.1, *hp(t)[:9])
            m, v = ref.unpack8(ref.pack8(M, V, t, first), n)
            off += bound + ref.U * np.abs(w)
        assert (np.abs(dev["w"][i].to_host_f32() - w) <= off).all()
        want = ref.pack8(M, V, 3, first)
        assert np.array_equal(st[i].to_host_f32().view(np.uint8), want)
        first += -(-n // 64) * 64
    sc.graph_destroy(g)


def test_binding_refuses(E):
    """Bad arguments are errors of the host, before anything is enqueued."""
    S, sc = E
    p = sc.cuda_malloc_f32(4096)
    launches = sc.launch_count()
    for bad in [(0, p, 8, 0, 0, p, 0, 2, 3, 8), (p, p, 7, 0, 0, p, 0, 2, 3, 8), (p, p, 8, 0, 0, 0, 0, 2, 3, 8), (p, p, 8, 0, 0, p, 0, -1, 3, 8),
                (p, p, 8, 0, 0, p, 0, 2, -3, 8), (p, p, 8, 0, 0, p, 0, 2, 3, 0), (p, p, 1 << 30, 0, 0, p, 0, 1 << 20, 1, 1 << 12),
                (p, p, 8, 0, 0, p, 0, 1, (1 << 30) + 1, 8)]:
        with pytest.raises(RuntimeError):
            sc.gated_scan_fwd(*bad)
    for bad in [(p, p, 8, 0, 0, 0, p, 0, p, p, 8, 0, 2, 3, 8), (p, p, 8, 0, 0, p, 0, 0, p, p, 8, 0, 2, 3, 8), (p, p, 8, 0, 0, p, p, 0, p, 0, 8, 0, 2, 3, 8),
                (p, p, 8, 0, 0, p, p, 0, p, p, 7, 0, 2, 3, 8)]:
        with pytest.raises(RuntimeError):
            sc.gated_scan_bwd(*bad)
    for bad in [(0, p, p, p, p, 2, 8, 0, 1e-5), (p, 0, p, p, p, 2, 8, 0, 1e-5), (p, p, p, 0, p, 2, 8, 0, 1e-5), (p, p, p, p, p, -2, 8, 0, 1e-5), (p, p, p, p, p, 2, 0, 0, 1e-5),
                (p, p, p, p, p, 2, 8193, 0, 1e-5), (p, p, p, p, p, 2, 8, 2, 1e-5), (p, p, p, p, p, 2, 8, 0, -1.0), (p, p, p, p, p, 2, 8, 0, float("nan")),
                (p, p, p, p, p + 4, 2, 8, 0, 1e-5)]:
        with pytest.raises(RuntimeError):
            sc.norm_fwd(*bad)
    for bad in [(p, p, p, 0, p, p, p, 2, 8, 0), (p, p, p, p, p, p, p, 0, 8, 0), (p, p, p, p, p, p, p, 2, 8193, 0), (p, p, p, p, p, p, p, 2, 8, 7)]:
        with pytest.raises(RuntimeError):
            sc.norm_bwd(*bad)
    good = [p, p, 8, p, p, p, p, p, p, p, p, 2, 8, 0, 4, 0, 1e-5, 1e-5]
    for at, v in [(0, 0), (2, 7), (4, 0), (5, 0), (7, 0), (10, p + 4), (11, -1), (12, 0), (12, 8193), (13, 2), (14, 5), (14, -1), (15, 2), (16, -1.0), (17, float("nan"))]:
        with pytest.raises(RuntimeError):
            sc.gated_residual_fwd(*good[:at], v, *good[at + 1:])
    good = [p, p, p, p, 8, p, p, p, p, p, p, p, 8, p, p, p, p, p, 2, 8, 0, 4, 0]
    for at, v in [(2, 0), (3, 0), (4, 7), (5, 0), (6, 0), (7, 0), (8, 0), (9, 0), (9, p + 4), (12, 7), (18, 0), (19, 0), (19, 8193), (20, 3), (21, 9), (22, -1)]:
        with pytest.raises(RuntimeError):
            sc.gated_residual_bwd(*good[:at], v, *good[at + 1:])
    one, n, dec, s = np.array([p], np.uint64), np.array([8], np.int64), np.array([0.0], np.float32), [1e-3, 0.9, 0.1, 0.9, 0.1, 1e-8, 0.1, 0.1, 1.0]
    for at, v in [(0, one * 0), (1, one * 0), (2, one * 0), (3, one * 0), (4, -n), (4, n * (1 << 41)), (4, np.array([8, 8]))]:
        args = [one, one, one, one, n, dec]
        args[at] = v
        with pytest.raises(RuntimeError):
            sc.adamw_step(*args, *s)
    for at, v, t in [(2, one + np.uint64(4), 1.0), (0, one, -1.0), (0, one, float("nan")), (0, one, 2.0 ** 32)]:
        args = [one, one, one, n, dec]
        args[at] = v
        with pytest.raises(RuntimeError):
            sc.adamw8_step(*args, *s, t)
    with pytest.raises(RuntimeError):
        sc.adamw8_step(one, one, one, n, dec, *s, 1.0, first=-64)
    for bad in [(0, p, p, 4), (p, 0, p, 4), (p + 4, p, p, 4), (p, p, p, -1)]:
        with pytest.raises(RuntimeError):
            sc.adamw8_read(*bad)
    assert sc.launch_count() == launches
    sc.cuda_free(p)


def test_long_ragged_sequences_recorded(E):
    """Sequences long enough for clusters of blocks, with their lengths on the device, an odd width and one of whole vectors: recorded steps, replayed with the
    lengths of another batch, against eager ones."""
    S, sc = E
    from ml_framework_b200.cuTen import cuten
    sc.set_precision(3)
    N, T, IN, U = 2, 1500, 20, 36
    r = np.random.RandomState(6)
    X = S.Tensor(r.standard_normal((N, T, IN)).astype(np.float32), is_leaf=True)
    Y = S.Tensor(np.eye(3, dtype=np.float32)[r.randint(0, 3, N)], is_leaf=True)
    lengths = [np.array(k, np.int32) for k in ([1500, 1203], [17, 0], [1499, 1500], [1, 700])]
    out = []
    for recorded in (False, True):
        np.random.seed(2)
        layers = [S.Input((T, IN)), S.GatedRecurrence(IN, U)]
        layers += [S.RMSNorm(U), S.GatedRecurrence(U, U, output_gate=True), S.GatedResidual(U, residual=layers[1]), S.LayerNorm(U),
                   S.GatedRecurrence(U, 33, return_sequences=False), S.Dense(33, 3, activation="softmax")]
        model = S.Sequential(layers)
        opt = S.AdamW(model, lr=1e-3)
        at = cuten(lengths[0], "int32")

        def step():
            loss = S.Loss().categorical_cross_entropy(model.forward(X, lengths=at), Y)
            model.zero_grad()
            S.autograd4nn(loss)
            opt.step()
            return loss
        step(), step()
        if recorded:
            opt._scalars_in_graph = True
            sc.graph_begin()
            kept = step()
            opt._scalars_in_graph = False
            g = sc.graph_end()
        for k in range(1, 8):
            other = cuten(lengths[k % 4], "int32")
            sc.cuda_memcopy_devicetodevice(at.main_ptr, other.main_ptr, N)
            if recorded:
                sc.graph_set_scalars(g, opt._scalars())
                sc.graph_launch(g)
            else:
                step()
            sc.stream_synchronize()
        assert sc.tc_device_status() == 0
        out.append(model.params.to_host_f32().copy())
        if recorded:
            sc.graph_destroy(g)
            del kept
    assert np.isfinite(out[0]).all() and np.array_equal(out[0], out[1])
