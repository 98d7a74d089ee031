"""The gated scan and its gradients through the C ABI against 64 bits, with bounds that count the roundings (tests/sequence_np.py)."""
import numpy as np
import pytest

import sequence_np as ref

pytestmark = pytest.mark.gpu
GUARD = 128          # floats on both sides of an output that no call may touch


@pytest.fixture(scope="module")
def D():
    from ml_framework_b200 import capi
    import engine_np
    capi.check(capi.load().seera_init(capi.default_device()))
    return engine_np._Dev, capi


class Guarded:
    def __init__(self, d, n):
        self.d, self.n = d, n
        self.p = d.up(np.full(n + 2 * GUARD, 7.5, np.float32))
        self.at = self.p + 4 * GUARD

    def get(self, shape):
        a = self.d.down(self.p, (self.n + 2 * GUARD,))
        assert (a[:GUARD] == 7.5).all() and (a[GUARD + self.n:] == 7.5).all()
        return a[GUARD:GUARD + self.n].reshape(shape)


def inputs(N, T, C, seed, ragged, bias=2.0):
    r = np.random.RandomState(seed)
    f = (r.standard_normal((N, T, C)) * 1.5 + bias).astype(np.float32)
    v, dh = (r.standard_normal((N, T, C)).astype(np.float32) for _ in range(2))
    h0, dlast = (r.standard_normal((N, C)).astype(np.float32) for _ in range(2))
    lengths = None
    if ragged:
        lengths = r.randint(0, T + 1, N).astype(np.int32)
        lengths[:3] = [0, T, min(1, T)][:N] if N < 3 else [0, T, min(1, T)]
    return f, v, h0, dh, dlast, lengths


def joined(f, v, extra=0):
    """Gate logits and candidates as column ranges of one array, as a projection leaves them."""
    N, T, C = f.shape
    z = np.full((N, T, 2 * C + extra), np.nan, np.float32)
    z[..., :C], z[..., C:2 * C] = f, v
    return z


def poison(z, lengths):
    """What lies behind a sequence's length is not read."""
    if lengths is not None:
        for n, k in enumerate(lengths):
            z[n, k:] = np.array([np.nan, np.inf, -np.inf, np.finfo(np.float32).min], np.float32)[np.arange(z[n, k:].size) % 4].reshape(z[n, k:].shape)
    return z


SHAPES = [(1, 1, 1), (3, 1, 2048), (2, 2, 33), (4, 16, 64), (3, 17, 5), (5, 64, 31), (2, 127, 32), (2, 129, 100), (7, 255, 65), (1, 1025, 32), (3, 2049, 40),
          (300, 40, 33), (1, 5000, 1), (40, 300, 130)]


@pytest.mark.parametrize("N,T,C", SHAPES)
@pytest.mark.parametrize("state,ragged", [(False, False), (True, True)])
def test_forward(D, N, T, C, state, ragged):
    Dev, capi = D
    f, v, h0, _, _, lengths = inputs(N, T, C, N + T + C, ragged)
    want, last, eh, elast = ref.scan_fwd(f, v, h0 if state else None, lengths)
    with Dev() as d:
        ld = 2 * C + 3
        z = d.up(poison(joined(f, v, 3), lengths))
        h, hl = Guarded(d, N * T * C), Guarded(d, N * C)
        args = (z, z + 4 * C, ld, d.up(h0) if state else None, d.up(lengths, np.int32) if ragged else None)
        capi.check(d.L.seera_gated_scan_fwd(*args, h.at, hl.at, N, T, C))
        got, gl = h.get((N, T, C)), hl.get((N, C))
        assert (np.abs(got - want) <= eh).all() and (np.abs(gl - last) <= elast).all()
        if ragged:
            for n, k in enumerate(lengths):
                assert (got[n, k:] == 0).all()
        capi.check(d.L.seera_gated_scan_fwd(*args, h.at, None, N, T, C))               # the same bits again, each output alone
        assert np.array_equal(h.get((N, T, C)), got)
        capi.check(d.L.seera_gated_scan_fwd(*args, None, hl.at, N, T, C))
        assert np.array_equal(hl.get((N, C)), gl)
        if state:                                                                       # in place of the state that it began with
            s = d.up(h0)
            capi.check(d.L.seera_gated_scan_fwd(*args[:3], s, args[4], None, s, N, T, C))
            assert np.array_equal(d.down(s, (N, C)), gl)


@pytest.mark.parametrize("N,T,C", SHAPES)
@pytest.mark.parametrize("state,ragged,given", [(False, False, "dh"), (True, True, "both"), (True, False, "dlast")])
def test_backward(D, N, T, C, state, ragged, given):
    Dev, capi = D
    f, v, h0, dh, dlast, lengths = inputs(N, T, C, N + 2 * T + C, ragged)
    h = ref.scan_fwd(f, v, h0 if state else None, lengths)[0].astype(np.float32)
    use_dh, use_last = given != "dlast", given != "dh"
    df, dv, dh0, edf, edv, edh0 = ref.scan_bwd(f, v, h, dh if use_dh else None, dlast if use_last else None, h0 if state else None, lengths)
    with Dev() as d:
        z = d.up(poison(joined(f, v), lengths))
        ldg = 2 * C + 1
        out, o0 = Guarded(d, N * T * ldg), Guarded(d, N * C)
        args = (z, z + 4 * C, 2 * C, d.up(h0) if state else None, d.up(lengths, np.int32) if ragged else None, d.up(poison(h.copy(), lengths)),
                d.up(poison(dh.copy(), lengths)) if use_dh else None, d.up(dlast) if use_last else None)
        capi.check(d.L.seera_gated_scan_bwd(*args, out.at, out.at + 4 * C, ldg, o0.at, N, T, C))
        got, g0 = out.get((N, T, ldg)), o0.get((N, C))
        assert (got[..., 2 * C] == 7.5).all()                                           # between the rows of the gradient
        assert (np.abs(got[..., :C] - df) <= edf).all() and (np.abs(got[..., C:2 * C] - dv) <= edv).all() and (np.abs(g0 - dh0) <= edh0).all()
        capi.check(d.L.seera_gated_scan_bwd(*args, out.at, out.at + 4 * C, ldg, None, N, T, C))
        assert np.array_equal(out.get((N, T, ldg)), got)


def test_gradients_against_differences(D):
    """The derivative of a weighted sum of all outputs, by central differences of the forward formula in 64 bits."""
    Dev, capi = D
    N, T, C = 2, 37, 3
    f, v, h0, dh, dlast, lengths = inputs(N, T, C, 5, False, bias=0.5)
    lengths = np.array([37, 20], np.int32)

    def value(f, v, h0):
        h, last, _, _ = ref.scan_fwd(f, v, h0, lengths)
        return (h * dh).sum() + (last * dlast).sum()
    with Dev() as d:
        pf, pv, p0, pl = d.up(f), d.up(v), d.up(h0), d.up(lengths, np.int32)
        h, df, dv, o0 = d.new(N * T * C), d.new(N * T * C), d.new(N * T * C), d.new(N * C)
        capi.check(d.L.seera_gated_scan_fwd(pf, pv, C, p0, pl, h, None, N, T, C))
        capi.check(d.L.seera_gated_scan_bwd(pf, pv, C, p0, pl, h, d.up(dh), d.up(dlast), df, dv, C, o0, N, T, C))
        got = [d.down(df, (N, T, C)), d.down(dv, (N, T, C)), d.down(o0, (N, C))]
    x = [f.astype(np.float64), v.astype(np.float64), h0.astype(np.float64)]
    r = np.random.RandomState(1)
    for k, g in enumerate(got):
        for _ in range(25):
            at = tuple(r.randint(0, s) for s in g.shape)
            step = 1e-4
            y = [a.copy() for a in x]
            y[k][at] += step
            up = value(*y)
            y[k][at] -= 2 * step
            diff = (up - value(*y)) / (2 * step)
            # the difference itself is off by step^2 / 6 of a third derivative and by the sum's rounding in 64 bits over the step
            assert abs(diff - g[at]) <= 1e-6 + 2e-5 * abs(diff)


@pytest.mark.parametrize("bias", [-60.0, -9.0, 9.0, 60.0, 200.0])
def test_gates_at_their_ends(D, bias):
    """States that are replaced at once and states that hardly move: 1 - a of 1e-26 and a of 1e-26 keep their digits."""
    Dev, capi = D
    N, T, C = 2, 300, 33
    f, v, h0, dh, dlast, _ = inputs(N, T, C, 3, False, bias)
    want, last, eh, elast = ref.scan_fwd(f, v, h0)
    h32 = want.astype(np.float32)
    df, dv, dh0, edf, edv, edh0 = ref.scan_bwd(f, v, h32, dh, dlast, h0)
    with Dev() as d:
        pf, pv, p0 = d.up(f), d.up(v), d.up(h0)
        h, hl, a, b, c = d.new(N * T * C), d.new(N * C), d.new(N * T * C), d.new(N * T * C), d.new(N * C)
        capi.check(d.L.seera_gated_scan_fwd(pf, pv, C, p0, None, h, hl, N, T, C))
        assert (np.abs(d.down(h, (N, T, C)) - want) <= eh).all() and (np.abs(d.down(hl, (N, C)) - last) <= elast).all()
        capi.check(d.L.seera_gated_scan_bwd(pf, pv, C, p0, None, d.up(h32), d.up(dh), d.up(dlast), a, b, C, c, N, T, C))
        for p, w, e in ((a, df, edf), (b, dv, edv)):
            assert (np.abs(d.down(p, (N, T, C)) - w) <= e).all()
        assert (np.abs(d.down(c, (N, C)) - dh0) <= edh0).all()


def test_what_is_not_finite_stays_in_its_channel_and_its_future(D):
    Dev, capi = D
    N, T, C = 2, 200, 40
    f, v, h0, _, _, _ = inputs(N, T, C, 9, False)
    want, _, eh, _ = ref.scan_fwd(f, v, h0)
    f2, v2 = f.copy(), v.copy()
    v2[0, 50, 3], f2[1, 70, 7], v2[1, 90, 33] = np.inf, np.nan, np.nan
    with Dev() as d:
        h = d.new(N * T * C)
        capi.check(d.L.seera_gated_scan_fwd(d.up(f2), d.up(v2), C, d.up(h0), None, h, None, N, T, C))
        got = d.down(h, (N, T, C))
    bad = np.zeros((N, T, C), bool)
    bad[0, 50:, 3] = bad[1, 70:, 7] = bad[1, 90:, 33] = True
    assert not np.isfinite(got[bad]).any()
    assert (np.abs(got - want) <= eh)[~bad].all()


def test_no_steps_and_no_sequences(D):
    Dev, capi = D
    with Dev() as d:
        s, o = d.up(np.arange(6, dtype=np.float32)), d.up(np.full(6, 9, np.float32))
        capi.check(d.L.seera_gated_scan_fwd(None, None, 3, s, None, None, o, 2, 0, 3))
        assert np.array_equal(d.down(o, (6,)), np.arange(6))
        capi.check(d.L.seera_gated_scan_fwd(None, None, 3, None, None, None, o, 2, 0, 3))
        assert (d.down(o, (6,)) == 0).all()
        capi.check(d.L.seera_gated_scan_bwd(None, None, 3, None, None, None, None, s, None, None, 3, o, 2, 0, 3))
        assert np.array_equal(d.down(o, (6,)), np.arange(6))
        capi.check(d.L.seera_gated_scan_fwd(None, None, 3, None, None, None, o, 0, 5, 3))


def test_time_in_parts_is_the_whole(D):
    """A sequence in three calls, the state handed on, as a program does that answers token by token."""
    Dev, capi = D
    N, T, C = 3, 150, 70
    f, v, h0, _, _, _ = inputs(N, T, C, 2, False)
    want, last, eh, elast = ref.scan_fwd(f, v, h0)
    with Dev() as d:
        s = d.up(h0)
        got = []
        for a, b in ((0, 1), (1, 2), (2, 149), (149, 150)):
            h = d.new(N * (b - a) * C)
            capi.check(d.L.seera_gated_scan_fwd(d.up(f[:, a:b]), d.up(v[:, a:b]), C, s, None, h, s, N, b - a, C))
            got.append(d.down(h, (N, b - a, C)))
        assert (np.abs(np.concatenate(got, 1) - want) <= eh).all() and (np.abs(d.down(s, (N, C)) - last) <= elast).all()


def test_offsets_past_32_bits(D):
    """Rows so far apart that the last one starts behind 2^31 floats."""
    Dev, capi = D
    N, T, C, ld = 1, 19, 4, 1 << 27
    f, v, h0, dh, _, _ = inputs(N, T, C, 8, False)
    want, _, eh, _ = ref.scan_fwd(f, v, h0)
    with Dev() as d:
        big = d.new(T * ld, 4)
        pf, pv = d.up(f), d.up(v)
        for t in range(T):
            at = big + 4 * t * ld
            capi.check(d.L.seera_cuda_memcopy_devicetodevice(at, pf + 4 * t * C, C))
            capi.check(d.L.seera_cuda_memcopy_devicetodevice(at + 64, pv + 4 * t * C, C))
        h = d.new(T * C)
        capi.check(d.L.seera_gated_scan_fwd(big, big + 64, ld, d.up(h0), None, h, None, N, T, C))
        assert (np.abs(d.down(h, (N, T, C)) - want) <= eh).all()
    capi.check(capi.load().seera_pool_trim())


# Channels and rows of whole vectors, which are copied 16 bytes at a time: one block a tile, clusters of a few blocks and of as many as there are
WIDE = [(3, 17, 64), (1, 129, 4), (5, 64, 32), (2, 300, 100), (7, 255, 68), (300, 40, 36), (40, 300, 128), (3, 2049, 40), (1, 5000, 256), (1, 12000, 64), (2, 3001, 512)]


@pytest.mark.parametrize("N,T,C", WIDE)
@pytest.mark.parametrize("state,ragged,given", [(False, False, "dh"), (True, True, "both"), (True, False, "dlast")])
def test_whole_vectors(D, N, T, C, state, ragged, given):
    Dev, capi = D
    f, v, h0, dh, dlast, lengths = inputs(N, T, C, N + 3 * T + C, ragged)
    want, last, eh, elast = ref.scan_fwd(f, v, h0 if state else None, lengths)
    h32 = want.astype(np.float32)
    use_dh, use_last = given != "dlast", given != "dh"
    df, dv, dh0, edf, edv, edh0 = ref.scan_bwd(f, v, h32, dh if use_dh else None, dlast if use_last else None, h0 if state else None, lengths)
    with Dev() as d:
        ld, ldg = 2 * C + 4, 2 * C + 2
        z = d.up(poison(joined(f, v, 4), lengths))
        h, hl = Guarded(d, N * T * C), Guarded(d, N * C)
        args = (z, z + 4 * C, ld, d.up(h0) if state else None, d.up(lengths, np.int32) if ragged else None)
        capi.check(d.L.seera_gated_scan_fwd(*args, h.at, hl.at, N, T, C))
        got, gl = h.get((N, T, C)), hl.get((N, C))
        assert (np.abs(got - want) <= eh).all() and (np.abs(gl - last) <= elast).all()
        if ragged:
            assert all((got[n, k:] == 0).all() for n, k in enumerate(lengths))
        out, o0 = Guarded(d, N * T * ldg), Guarded(d, N * C)
        args += (d.up(poison(h32.copy(), lengths)), d.up(poison(dh.copy(), lengths)) if use_dh else None, d.up(dlast) if use_last else None)
        capi.check(d.L.seera_gated_scan_bwd(*args, out.at, out.at + 4 * C, ldg, o0.at, N, T, C))
        got, g0 = out.get((N, T, ldg)), o0.get((N, C))
        assert (got[..., 2 * C:] == 7.5).all()                                          # between the rows of the gradient
        assert (np.abs(got[..., :C] - df) <= edf).all() and (np.abs(got[..., C:2 * C] - dv) <= edv).all() and (np.abs(g0 - dh0) <= edh0).all()
        if ragged:
            assert all((got[n, k:, :2 * C] == 0).all() for n, k in enumerate(lengths))
        capi.check(d.L.seera_gated_scan_bwd(*args, out.at, out.at + 4 * C, ldg, None, N, T, C))
        assert np.array_equal(out.get((N, T, ldg)), got)
        assert d.L.seera_tc_device_status() == 0


@pytest.mark.parametrize("N,T,C", [(1, 4000, 64), (2, 777, 33)])
def test_two_recordings_share_nothing(D, N, T, C):
    """Two recordings of forward and backward calls of clusters, replayed in turn with other inputs in place of their own."""
    Dev, capi = D
    with Dev() as d:
        runs = []
        for seed in (1, 2):
            f, v, h0, dh, dlast, lengths = inputs(N, T, C, seed, True)
            a = {"f": d.up(f), "v": d.up(v), "h0": d.up(h0), "dh": d.up(dh), "len": d.up(lengths, np.int32)}
            a.update(h=d.new(N * T * C), last=d.new(N * C), df=d.new(N * T * C), dv=d.new(N * T * C), dh0=d.new(N * C))
            capi.check(d.L.seera_graph_begin())
            capi.check(d.L.seera_gated_scan_fwd(a["f"], a["v"], C, a["h0"], a["len"], a["h"], a["last"], N, T, C))
            capi.check(d.L.seera_gated_scan_bwd(a["f"], a["v"], C, a["h0"], a["len"], a["h"], a["dh"], a["last"], a["df"], a["dv"], C, a["dh0"], N, T, C))
            g = d.L.seera_graph_end()
            assert g
            runs.append((a, g))
        for seed in (3, 4, 5):
            data = [inputs(N, T, C, 10 * seed + i, True) for i in range(2)]
            for (a, g), (f, v, h0, dh, _, lengths) in zip(runs, data):
                for k, x in (("f", f), ("v", v), ("h0", h0), ("dh", dh)):
                    capi.check(d.L.seera_cuda_memcopy_devicetodevice(a[k], d.up(x), x.size))
                capi.check(d.L.seera_cuda_memcopy_devicetodevice(a["len"], d.up(lengths, np.int32), N))
            for _, g in runs:
                capi.check(d.L.seera_graph_launch(g))
            for (a, g), (f, v, h0, dh, _, lengths) in zip(runs, data):
                want, last, eh, elast = ref.scan_fwd(f, v, h0, lengths)
                got, gl = d.down(a["h"], (N, T, C)), d.down(a["last"], (N, C))
                assert (np.abs(got - want) <= eh).all() and (np.abs(gl - last) <= elast).all()
                df, dv, dh0, edf, edv, edh0 = ref.scan_bwd(f, v, got, dh, gl, h0, lengths)
                for k, w, e in (("df", df, edf), ("dv", dv, edv), ("dh0", dh0, edh0)):
                    assert (np.abs(d.down(a[k], w.shape) - w) <= e).all()
        for _, g in runs:
            capi.check(d.L.seera_graph_destroy(g))
        assert d.L.seera_tc_device_status() == 0
