"""AdamW over many tensors through the C ABI: the averages bit for bit, in 32 bits and in 8, the weights within a few roundings of 64 bits."""
import ctypes

import numpy as np
import pytest

import sequence_np as ref

pytestmark = pytest.mark.gpu
HP = (1e-2, 0.9, 1 - 0.9, 0.95, 1 - 0.95, 1e-8, 1 - 0.9 ** 3, 1 - 0.95 ** 3, 0.5)
SIZES = {"one": [1], "few": [5, 64, 0, 63, 65, 2048, 2049], "edges": [2047, 4096, 4095, 1, 0, 128], "many": [17 * i % 301 for i in range(200)],
         "large": [300000, 3, 1 << 20]}


@pytest.fixture(scope="module")
def D():
    from ml_framework_b200 import capi
    import engine_np
    capi.check(capi.load().seera_init(capi.default_device()))
    return engine_np._Dev, capi


def arr(xs, t):
    return (t * max(1, len(xs)))(*xs)


def place(d, values, shift):
    """The tensors in one block with guards of 16 floats between them, each `shift` floats past a 16-byte boundary."""
    starts, at = [], 16 + shift
    for v in values:
        starts.append(at)
        at = (at + v.size + 16 + 15) // 16 * 16 + shift
    host = np.full(at + 16, 5.5, np.float32)
    for s, v in zip(starts, values):
        host[s:s + v.size] = v
    return d.up(host), starts, host


def make(sizes, seed):
    r = np.random.RandomState(seed)
    mag = [np.exp(r.standard_normal(n) * 2).astype(np.float32) for n in sizes]
    w = [r.standard_normal(n).astype(np.float32) for n in sizes]
    g = [(r.standard_normal(n) * 1e-3).astype(np.float32) * k for n, k in zip(sizes, mag)]
    m = [(r.standard_normal(n) * 1e-4).astype(np.float32) * k for n, k in zip(sizes, mag)]
    v = [(r.standard_normal(n) ** 2 * 1e-7).astype(np.float32) * k * k for n, k in zip(sizes, mag)]
    decay = np.array([0.1 if i % 2 else 0.0 for i in range(len(sizes))], np.float32)
    return w, g, m, v, decay


def check_place(host, starts, values, got):
    want = host.copy()
    for s, v in zip(starts, values):
        want[s:s + v.size] = got[s:s + v.size]
    assert np.array_equal(want, got), "written outside the tensors"


@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("device_scalars", [False, True])
def test_32_bits(D, sizes, shift, device_scalars):
    Dev, capi = D
    sizes = SIZES[sizes]
    w, g, m, v, decay = make(sizes, len(sizes))
    with Dev() as d:
        placed = [place(d, x, shift) for x in (w, g, m, v)]
        at = [arr([p + 4 * s for s in st], ctypes.c_void_p) for p, st, _ in placed]
        hyper = d.up(np.array(HP, np.float32)) if device_scalars else None
        scal = (0.0,) * 9 if device_scalars else HP
        capi.check(d.L.seera_adamw_step(len(sizes), *at, arr(sizes, ctypes.c_longlong), arr(decay.tolist(), ctypes.c_float), *scal, hyper))
        got = [d.down(p, h.shape) for p, _, h in placed]
    for (p, st, host), vals, x in zip(placed, (w, g, m, v), got):
        check_place(host, st, vals, x)
    assert np.array_equal(got[1], placed[1][2])
    for i, n in enumerate(sizes):
        W, M, V, bound = ref.adamw(w[i], g[i], m[i], v[i], decay[i], *HP)
        cut = lambda k: got[k][placed[k][1][i]:placed[k][1][i] + n]  # noqa: E731
        assert np.array_equal(cut(2), M) and np.array_equal(cut(3), V)
        assert (np.abs(cut(0) - W) <= bound).all()


@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("shift", [0, 3])
@pytest.mark.parametrize("step", [1, 77])
def test_8_bits(D, sizes, shift, step):
    Dev, capi = D
    sizes = SIZES[sizes]
    w, g, m, v, decay = make(sizes, len(sizes) + step)
    state = [ref.pack8(a, b, 1000) if n else np.zeros(0, np.uint8) for a, b, n in zip(m, v, sizes)]
    first = 1 << 33 if step == 77 else 0
    with Dev() as d:
        assert [d.L.seera_adamw8_state_bytes(n) for n in sizes] == [s.size for s in state]
        placed = [place(d, x, shift) for x in (w, g)]
        at = [arr([p + 4 * s for s in st], ctypes.c_void_p) for p, st, _ in placed]
        ends = np.cumsum([0] + [s.size + 24 for s in state])                                    # 24 bytes between the states
        host = np.full(int(ends[-1]) + 24, 0xAB, np.uint8)
        for e, s in zip(ends, state):
            host[e:e + s.size] = s
        ps = d.up(host, np.uint8)
        capi.check(d.L.seera_adamw8_step(len(sizes), *at, arr([ps + int(e) for e in ends[:-1]], ctypes.c_void_p), arr(sizes, ctypes.c_longlong),
                                         arr(decay.tolist(), ctypes.c_float), *HP, float(step), None, first))
        gw, gs = d.down(placed[0][0], placed[0][2].shape), d.down(ps, host.shape, np.uint8)
        want, k = host.copy(), first
        for i, n in enumerate(sizes):
            if not n:
                continue
            m0, v0 = ref.unpack8(state[i], n)
            W, M, V, bound = ref.adamw(w[i], g[i], m0, v0, decay[i], *HP)
            s = placed[0][1][i]
            assert (np.abs(gw[s:s + n] - W) <= bound).all()
            packed = ref.pack8(M, V, step, k)
            want[ends[i]:ends[i] + packed.size] = packed
            k += -(-n // 64) * 64
            pm, pv = d.new(n), d.new(n)
            capi.check(d.L.seera_adamw8_read(ps + int(ends[i]), pm, pv, n))
            um, uv = ref.unpack8(packed, n)
            assert np.array_equal(d.down(pm, (n,)), um) and np.array_equal(d.down(pv, (n,)), uv)
        assert np.array_equal(gs, want)
        check_place(placed[0][2], placed[0][1], w, gw)


def test_rounding_keeps_the_mean(D):
    """m and v of constant gradients in 8 bits, over many entries: their means follow the averages in 32 bits.  v moves by 0.1 % a step, less than half a code.
    An entry's v is a product of steps whose roundings have variance at most (1/8)^2 / 6 of its square each, and the old ones fade: after 300 steps with
    beta2 = 0.999 the variance is below 300 x 0.0027 < 0.9 of the square, the mean over 65536 entries off by 0.004 of itself with the standard deviation."""
    Dev, capi = D
    n, steps, b1, b2 = 65536, 300, 0.9, 0.999
    r = np.random.RandomState(0)
    g = (np.exp(r.standard_normal(n) * 0.5) * r.choice([-1, 1], n)).astype(np.float32)
    with Dev() as d:
        nb = d.L.seera_adamw8_state_bytes(n)
        st, w, pg = d.up(np.zeros(nb, np.uint8), np.uint8), d.up(np.zeros(n, np.float32)), d.up(g)
        for t in range(1, steps + 1):
            capi.check(d.L.seera_adamw8_step(1, arr([w], ctypes.c_void_p), arr([pg], ctypes.c_void_p), arr([st], ctypes.c_void_p), arr([n], ctypes.c_longlong),
                                             arr([0.0], ctypes.c_float), 0.0, b1, 1 - b1, b2, 1 - b2, 1e-8, 1 - b1 ** t, 1 - b2 ** t, 1.0, float(t), None, 0))
        pm, pv = d.new(n), d.new(n)
        capi.check(d.L.seera_adamw8_read(st, pm, pv, n))
        m, v = d.down(pm, (n,)).astype(np.float64), d.down(pv, (n,)).astype(np.float64)
    g = g.astype(np.float64)
    assert abs((v / (g * g)).mean() / (1 - b2 ** steps) - 1) < 6 * 0.004
    # m: the sum of fading roundings of variance at most (1/8)^2 / 6 each, 0.0027 / (1 - 0.81) = 0.014 of the square: 0.0005 for the mean
    assert abs((m / g).mean() / (1 - b1 ** steps) - 1) < 6 * 0.0005


def test_what_is_not_finite(D):
    """32 bits: the entry alone.  8 bits: the weight of the entry, the averages of its 64: the block's largest is what is not finite, a code of 0 times
    infinity is a NaN, and the entry's own code of 1 times infinity is infinity."""
    Dev, capi = D
    n = 300
    w, g, m, v, _ = make([n], 3)
    w, g, m, v = w[0], g[0], m[0], v[0]
    g[70], g[200] = np.nan, np.inf
    bad = np.zeros(n, bool)
    bad[[70, 200]] = True
    with Dev() as d:
        p = [d.up(x) for x in (w, g, m, v)]
        one = lambda q: arr([q], ctypes.c_void_p)  # noqa: E731
        capi.check(d.L.seera_adamw_step(1, *map(one, p), arr([n], ctypes.c_longlong), arr([0.1], ctypes.c_float), *HP, None))
        for q in (p[0], p[2], p[3]):
            assert np.isfinite(d.down(q, (n,))[~bad]).all()
        assert np.isnan(d.down(p[0], (n,))[70]) and np.isnan(d.down(p[0], (n,))[200])
        pw, st = d.up(w), d.up(ref.pack8(m, v, 1), np.uint8)
        capi.check(d.L.seera_adamw8_step(1, one(pw), one(p[1]), one(st), arr([n], ctypes.c_longlong), arr([0.1], ctypes.c_float), *HP, 2.0, None, 0))
        got = d.down(pw, (n,))
        assert np.isfinite(got[~bad]).all() and np.isnan(got[bad]).all()
        pm, pv = d.new(n), d.new(n)
        capi.check(d.L.seera_adamw8_read(st, pm, pv, n))
        block = np.zeros(n, bool)
        block[64:128] = block[192:256] = True
        for q in (pm, pv):
            a = d.down(q, (n,))
            assert np.isnan(a[64:128]).all() and np.isnan(np.delete(a[192:256], 8)).all() and a[200] == np.inf and np.isfinite(a[~block]).all()


def test_refusals(D):
    """Bad arguments are errors of the host: nothing is launched and nothing written."""
    Dev, capi = D
    n = 100
    w = np.arange(n, dtype=np.float32)
    with Dev() as d:
        pw, pg, st = d.up(w), d.up(w), d.up(np.zeros(2 * 136, np.uint8), np.uint8)
        one = lambda q: arr([q], ctypes.c_void_p)  # noqa: E731
        call = lambda w, g, s, k, step, first: d.L.seera_adamw8_step(1, one(w), one(g), one(s), arr([k], ctypes.c_longlong),  # noqa: E731
                                                                     arr([0.1], ctypes.c_float), *HP, step, None, first)
        launches = d.L.seera_launch_count()
        for bad in ((None, pg, st, n, 1.0, 0), (pw, None, st, n, 1.0, 0), (pw, pg, None, n, 1.0, 0), (pw, pg, st + 4, n, 1.0, 0), (pw, pg, st, -1, 1.0, 0),
                    (pw, pg, st, n, -1.0, 0), (pw, pg, st, n, float("nan"), 0), (pw, pg, st, n, 1.0, -64), (pw, pg, st, n, 1.0, 32), (pw, pg, st, (1 << 40) + 1, 1.0, 0)):
            assert call(*bad) != 0
        assert d.L.seera_adamw8_read(st, pw, None, n) != 0 and d.L.seera_adamw8_read(st + 4, pw, pg, n) != 0 and d.L.seera_adamw8_read(st, pw, pg, -1) != 0
        assert d.L.seera_launch_count() == launches
        assert np.array_equal(d.down(pw, (n,)), w)
        assert call(pw, pg, st, 0, 1.0, 0) == 0 and d.L.seera_launch_count() == launches
