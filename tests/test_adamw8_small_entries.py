"""AdamW in 8 bits where the entries of a block of 64 are far apart: the averages of the small ones end below the smallest codes, and the weights' steps have to
stay near what 32 bits make of the same gradients.

How large a step may be, with m and v as the corrections leave them (the largest of a block about 1).  Exact averages: by Cauchy and Schwarz
|m| <= (1 - b1) / sqrt((1 - b2) (1 - b1^2 / b2)) sqrt(v), 7.3 lr for 0.9 and 0.999.  The rounding of m, where 2^-17 is its smallest code: up to half of that off with
the standard deviation each step, fading by b1, 1.15 x 2^-17 in all, 7 x 2^-17 at six deviations; over the root of v's smallest code, 2^-16.5, 5 lr.  The rms of
the steps: that of 32 bits (below 1) and 1.15 x 2^-17 / 2^-16.5 = 0.82 beside it."""
import ctypes

import numpy as np
import pytest

import adamw8_np
import sequence_np as ref
from test_host_logic_cpu import host  # noqa: F401  (fixture)

LARGEST, RMS = 7.3 + 5.0, 1.3
B1, B2, STEPS, BLOCKS = 0.9, 0.999, 300, 16


def gradients(e, scale, mean, seed=0):
    """One entry in 64 of size `scale`, the others 2^-e of it."""
    r = np.random.RandomState(seed)
    n = 64 * BLOCKS
    size = np.full(n, 2.0 ** -e * scale)
    size[::64] = scale
    return [((r.choice([-1, 1], n) + mean) / (1 + mean) * size).astype(np.float32) for _ in range(STEPS)]


def hp(t):
    return 1.0, B1, 1 - B1, B2, 1 - B2, 1e-8, 1 - B1 ** t, 1 - B2 ** t, 1.0


def model(g, eight):
    """The weights' moves of each step, by the formulas."""
    n = g[0].size
    m, v, w, moves = np.zeros(n, np.float32), np.zeros(n, np.float32), np.zeros(n, np.float32), []
    for t, x in enumerate(g, 1):
        move, m, v, _ = ref.adamw(w, x, m, v, 0.0, *hp(t))
        if eight:
            m, v = ref.unpack8(adamw8_np.pack8_bounded(m, v, t), n)
        moves.append(move)
    return np.array(moves)


def small(moves):
    return moves[:, np.arange(moves.shape[1]) % 64 != 0]


CASES = [(e, s, mean) for e in (14, 16, 17, 19, 24, 30) for s, mean in ((1.0, 0.0), (0.01, 0.0), (1.0, 1.0))]


@pytest.mark.parametrize("e,scale,mean", CASES)
def test_rule_keeps_the_steps(e, scale, mean):
    g = gradients(e, scale, mean)
    a, b = small(model(g, True)), small(model(g, False))
    assert np.abs(a).max() <= LARGEST and np.sqrt((a ** 2).mean()) <= RMS
    # not by leaving steps out: where the averages have codes of their own the steps are those of 32 bits
    if e == 14:
        assert abs(np.sqrt((a ** 2).mean()) / np.sqrt((b ** 2).mean()) - 1) < 0.1


def test_what_the_rule_leaves_zero():
    """A v of 0, and all of a block whose largest is held as 0 or is not finite."""
    m = np.ones(64, np.float32)
    code = lambda v: adamw8_np.pack8_bounded(m, v, 5)[:128].reshape(16, 2, 4)[:, 1].reshape(-1)  # noqa: E731
    v = np.full(64, 1e-30, np.float32)
    v[0], v[1] = 1.0, 0.0
    assert code(v)[0] == 0xF8 and code(v)[1] == 0 and (code(v)[2:] == 1).all()
    assert (code(np.full(64, 1e-40, np.float32)) == 0).all()
    v[0] = np.inf
    assert (code(v)[1:] == 0).all()


def test_optimizer_takes_bounded_steps(host, monkeypatch):
    """A model whose gradients have entries 2^-17 and 2^-20 of their neighbours, through AdamW itself."""
    S = host.seera
    monkeypatch.setattr(host.fake, "adamw8_step", None)
    model = S.Sequential([S.Input((64,)), S.Dense(64, 8, "tanh"), S.Dense(8, 4, "tanh")])
    r = np.random.RandomState(2)
    X = r.standard_normal((16, 64)).astype(np.float32) * np.float32(2.0) ** -np.array([0, 17, 17, 20] * 16, np.float32)
    w = model.param_layers[0].weights
    moves = {}
    for bits in (32, 8):
        model.param_layers[0].set_weights(np.zeros((64, 8), np.float32), np.zeros((1, 8), np.float32))
        opt, moves[bits] = S.AdamW(model, lr=2.0 ** -20, weight_decay=0.0, state_bits=bits), []
        for _ in range(120):
            Y = r.standard_normal((16, 4)).astype(np.float32) * 30
            S.autograd4nn(S.Loss().mse(model.forward(X), S.Tensor(Y, is_leaf=True)))
            before = w.to_numpy().astype(np.float64)
            opt.step()
            model.zero_grad()
            moves[bits].append((w.to_numpy() - before) * 2.0 ** 20)
    assert np.abs(moves[32]).max() < 7.4
    assert np.abs(moves[8]).max() <= LARGEST


@pytest.mark.gpu
@pytest.mark.parametrize("e,scale,mean", CASES)
def test_kernel_keeps_the_steps(e, scale, mean):
    from ml_framework_b200 import capi
    import engine_np
    g = gradients(e, scale, mean)
    n = g[0].size
    with engine_np._Dev() as d:
        one = lambda q: (ctypes.c_void_p * 1)(q)  # noqa: E731
        st = d.up(np.zeros(d.L.seera_adamw8_state_bytes(n), np.uint8), np.uint8)
        pw, pg = [d.up(np.zeros(n, np.float32)) for _ in g], [d.up(x) for x in g]
        for t in range(1, STEPS + 1):
            capi.check(d.L.seera_adamw8_bounded_step(1, one(pw[t - 1]), one(pg[t - 1]), one(st), (ctypes.c_longlong * 1)(n), (ctypes.c_float * 1)(0.0), *hp(t), float(t),
                                             None, 0))
        moves = np.array([d.down(p, (n,)) for p in pw], np.float64)
    a = small(moves)
    assert np.abs(a).max() <= LARGEST and np.sqrt((a ** 2).mean()) <= RMS
    # the averages are the rule's bit for bit (the other tests), so the steps are the model's within a few roundings
    want = model(g, True)
    assert (np.abs(moves - want) <= 16 * ref.U * np.abs(want) + 1e-37).all()


@pytest.mark.gpu
def test_kernel_leaves_zero_what_the_rule_does():
    """Blocks with zeros, with values below the smallest code, with a largest that is held as 0 and with infinities, bit for bit."""
    from ml_framework_b200 import capi
    import engine_np
    n, lr = 64 * 5 + 3, 0.0
    r = np.random.RandomState(1)
    g = (r.standard_normal(n) * 2.0 ** -r.randint(0, 40, n)).astype(np.float32)
    g[5:20] = 0
    g[64:128] = (r.standard_normal(64) * 1e-21).astype(np.float32)
    g[200] = np.inf
    g[256:320] *= np.float32(1e-12)
    with engine_np._Dev() as d:
        one = lambda q: (ctypes.c_void_p * 1)(q)  # noqa: E731
        nb = d.L.seera_adamw8_state_bytes(n)
        st, pw, pg = d.up(np.zeros(nb, np.uint8), np.uint8), d.up(np.zeros(n, np.float32)), d.up(g)
        m, v = np.zeros(n, np.float32), np.zeros(n, np.float32)
        for t in (1, 2, 3):
            h = (lr,) + hp(t)[1:]
            capi.check(d.L.seera_adamw8_bounded_step(1, one(pw), one(pg), one(st), (ctypes.c_longlong * 1)(n), (ctypes.c_float * 1)(0.0), *h, float(t), None, 0))
            _, m, v, _ = ref.adamw(np.zeros(n, np.float32), g, m, v, 0.0, *h)
            packed = adamw8_np.pack8_bounded(m, v, t)
            got = d.down(st, (nb,), np.uint8)
            top = lambda s: np.ascontiguousarray(s.reshape(-1, 136)[:, 128:]).view(np.float32)  # noqa: E731
            finite = np.isfinite(top(packed)).all(1)
            assert np.array_equal(got.reshape(-1, 136)[finite], packed.reshape(-1, 136)[finite])
            assert np.array_equal(np.isfinite(top(got)).all(1), finite) and finite.sum() == 5
            m, v = ref.unpack8(packed, n)


@pytest.mark.gpu
def test_refusals():
    from ml_framework_b200 import capi
    import engine_np
    n = 100
    with engine_np._Dev() as d:
        w, g, st = d.up(np.arange(n, dtype=np.float32)), d.up(np.ones(n, np.float32)), d.up(np.zeros(2 * 136, np.uint8), np.uint8)
        one = lambda q: (ctypes.c_void_p * 1)(q)  # noqa: E731
        call = lambda w, g, s, k, step, first: d.L.seera_adamw8_bounded_step(1, one(w), one(g), one(s), (ctypes.c_longlong * 1)(k), (ctypes.c_float * 1)(0.0), *hp(1),  # noqa: E731
                                                                             step, None, first)
        launches = d.L.seera_launch_count()
        for bad in ((None, g, st, n, 1.0, 0), (w, None, st, n, 1.0, 0), (w, g, None, n, 1.0, 0), (w, g, st + 4, n, 1.0, 0), (w, g, st, -1, 1.0, 0),
                    (w, g, st, n, -1.0, 0), (w, g, st, n, float("nan"), 0), (w, g, st, n, 1.0, -64), (w, g, st, n, 1.0, 32), (w, g, st, (1 << 40) + 1, 1.0, 0)):
            assert call(*bad) != 0
        assert call(w, g, st, 0, 1.0, 0) == 0
        assert d.L.seera_launch_count() == launches and np.array_equal(d.down(w, (n,)), np.arange(n))
