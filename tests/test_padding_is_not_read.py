"""A padded batch whose padding holds NaNs, infinities and the largest numbers: outputs and gradients are the bits of the same batch padded with zeros."""
import numpy as np
import pytest

import sequence_model as sm
from test_host_logic_cpu import host  # noqa: F401  (fixture)

LENGTHS = np.array([21, 1, 0, 13, 20], np.int32)


def batches():
    X, Y = sm.data()
    zeros, rough = X.copy(), X.copy()
    for n, k in enumerate(LENGTHS):
        zeros[n, k:] = 0
        rough[n, k:] = np.resize(np.array([np.nan, np.inf, -np.inf, 3e38, -3e38, 1e-40, 7], np.float32), rough[n, k:].shape)
    return X, zeros, rough, Y


def build(S, first):
    """What the input meets first: a recurrence, or a norm with a block around the input itself."""
    if first == "recurrence":
        return sm.build(S)
    np.random.seed(3)
    inp = S.Input((sm.T, sm.IN))
    return S.Sequential([inp, S.LayerNorm(sm.IN), S.GatedRecurrence(sm.IN, sm.IN, output_gate=True), S.GatedResidual(sm.IN, residual=inp), S.RMSNorm(sm.IN),
                         S.GatedRecurrence(sm.IN, sm.U, return_sequences=False), S.Dense(sm.U, sm.CLASSES, activation="softmax")])


def step(S, model, x, Y, lengths):
    out = model.forward(x, lengths=lengths)
    loss = S.Loss().categorical_cross_entropy(out, S.Tensor(Y, is_leaf=True))
    model.zero_grad()
    S.autograd4nn(loss)
    return [out.to_numpy()] + [t.grad.to_host_f32().copy() for l in model.param_layers for t in (l.weights, l.bais)]


def compare(S, first, device_lengths=None):
    _, zeros, rough, Y = batches()
    model = build(S, first)
    lengths = LENGTHS if device_lengths is None else device_lengths
    for _ in range(3):                                     # from the second on in batches
        for make in (lambda a: a, lambda a: S.Tensor(a, is_leaf=True), S.Tensor):
            want, got = (step(S, model, make(a), Y, lengths) for a in (zeros, rough))
            assert all(np.isfinite(a).all() for a in want)
            assert all(np.array_equal(a, b) for a, b in zip(want, got))
    assert np.array_equal(model.predict(rough, lengths=lengths).to_numpy(), want[0])


@pytest.mark.parametrize("first", ["recurrence", "norm"])
def test_steps(host, first):
    compare(host.seera, first)
    compare(host.seera, first, host.cuTen.cuten(LENGTHS, "int32"))


def test_the_callers_batch_and_its_gradient(host):
    """The batch stays as it is; a batch that was computed gets zeros as the gradient of its padding."""
    S = host.seera
    X, zeros, _, Y = batches()
    x = S.Tensor(X, is_leaf=True)
    model = build(S, "norm")
    step(S, model, x, Y, LENGTHS)
    assert np.array_equal(x.to_numpy(), X)
    whole = step(S, model, x, Y, None)
    assert not np.allclose(whole[0], step(S, model, x, Y, LENGTHS)[0])
    assert np.array_equal(step(S, model, x, Y, [sm.T] * sm.N)[0], whole[0])
    got = []
    x = S.Tensor(X)
    x._backward = lambda g: got.append(g.to_host_f32().copy())
    step(S, model, x, Y, LENGTHS)
    for n, k in enumerate(LENGTHS):
        assert (got[0][n, k:] == 0).all() and (k == 0 or got[0][n, :k].any())


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [0, 3, 4])
@pytest.mark.parametrize("first", ["recurrence", "norm"])
def test_steps_on_the_device(mode, first):
    from ml_framework_b200 import seera as S, seera_cuda as sc
    from ml_framework_b200.cuTen import cuten
    sc.init(0)
    sc.set_precision(mode)
    try:
        compare(S, first)
        compare(S, first, cuten(LENGTHS, "int32"))
    finally:
        sc.set_precision(3)


@pytest.mark.gpu
def test_recorded_step():
    """Replays with another batch's lengths and padding."""
    from ml_framework_b200 import seera as S, seera_cuda as sc
    from ml_framework_b200.cuTen import cuten
    sc.init(0)
    sc.set_precision(3)
    X, _, rough, Y = batches()
    model = build(S, "norm")
    at, x = cuten(LENGTHS, "int32"), S.Tensor(rough, is_leaf=True)
    want = {}
    for k in (0, 2):
        other = np.roll(LENGTHS, k)
        a = X.copy()
        for n, m in enumerate(other):
            a[n, m:] = 0
        want[k] = step(S, model, a, Y, other)
    step(S, model, x, Y, at)
    sc.graph_begin()
    out = model.forward(x, lengths=at)
    loss = S.Loss().categorical_cross_entropy(out, S.Tensor(Y, is_leaf=True))
    model.zero_grad()
    S.autograd4nn(loss)
    grads = [t.grad for l in model.param_layers for t in (l.weights, l.bais)]
    g = sc.graph_end()
    try:
        for k in (0, 2, 0):
            other, a = np.roll(LENGTHS, k), X.copy()
            for n, m in enumerate(other):
                a[n, m:] = np.nan
            sc.upload_f32(x.value.main_ptr, a)
            fresh = cuten(other.astype(np.int32), "int32")
            sc.cuda_memcopy_devicetodevice(at.main_ptr, fresh.main_ptr, sm.N)
            sc.graph_launch(g)
            got = [out.to_numpy()] + [t.to_host_f32() for t in grads]
            assert all(np.array_equal(p, q) for p, q in zip(want[k], got))
    finally:
        sc.graph_destroy(g)


@pytest.mark.gpu
@pytest.mark.parametrize("N,T,C", [(1, 1, 1), (3, 5, 1), (2, 7, 3), (4, 9, 4), (5, 333, 20), (70000, 2, 3), (3, 1000, 1000), (2, 40000, 33)])
@pytest.mark.parametrize("shift", [0, 1])
def test_entry(N, T, C, shift):
    from ml_framework_b200 import capi
    import engine_np
    r = np.random.RandomState(N + T + C)
    x = r.standard_normal((N, T, C)).astype(np.float32)
    lengths = r.randint(-1, T + 3, N).astype(np.int32)
    for n in range(min(N, 64)):
        x[n, max(lengths[n], 0):] = np.nan
    want = np.where((np.arange(T) < lengths[:, None])[..., None], x, np.float32(0))
    with engine_np._Dev() as d:
        guard = np.full(x.size + 16 + shift, 5.5, np.float32)
        guard[8 + shift:8 + shift + x.size] = x.ravel()
        px, py, pl = d.up(guard), d.up(np.full(guard.size, 2.5, np.float32)), d.up(lengths, np.int32)
        at = 4 * (8 + shift)
        capi.check(d.L.seera_pad_steps(px + at, pl, py + at, N, T, C))
        y = d.down(py, guard.shape)
        assert np.array_equal(y[8 + shift:8 + shift + x.size], want.ravel()) and (y[:8 + shift] == 2.5).all() and (y[8 + shift + x.size:] == 2.5).all()
        assert np.array_equal(d.down(px, guard.shape), guard, equal_nan=True)
        capi.check(d.L.seera_pad_steps(px + at, pl, px + at, N, T, C))
        y = d.down(px, guard.shape)
        assert np.array_equal(y[8 + shift:8 + shift + x.size], want.ravel()) and (y[:8 + shift] == 5.5).all() and (y[8 + shift + x.size:] == 5.5).all()


@pytest.mark.gpu
def test_entry_refuses():
    from ml_framework_b200 import capi
    import engine_np
    with engine_np._Dev() as d:
        x, pl = d.up(np.ones(24, np.float32)), d.up(np.ones(2, np.int32), np.int32)
        before = d.L.seera_launch_count()
        for bad in ((None, pl, x, 2, 3, 4), (x, None, x, 2, 3, 4), (x, pl, None, 2, 3, 4), (x, pl, x, -1, 3, 4), (x, pl, x, 2, -3, 4), (x, pl, x, 2, 3, 0)):
            assert d.L.seera_pad_steps(*bad) != 0
        for empty in ((None, None, None, 0, 3, 4), (None, None, None, 2, 0, 4)):
            assert d.L.seera_pad_steps(*empty) == 0
        assert d.L.seera_launch_count() == before
        assert (d.down(x, (24,)) == 1).all()
