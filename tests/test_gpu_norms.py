"""Norms over features and the fused end of a block through the C ABI against 64 bits, with bounds that count the roundings."""
import numpy as np
import pytest

import sequence_np as ref

pytestmark = pytest.mark.gpu
GUARD = 64
EPS = 1e-5


@pytest.fixture(scope="module")
def D():
    from ml_framework_b200 import capi
    import engine_np
    capi.check(capi.load().seera_init(capi.default_device()))
    return engine_np._Dev, capi


class Out:
    """An output with untouched places around it; `pad`: floats between its rows."""

    def __init__(self, d, rows, C, pad=0):
        self.d, self.rows, self.C, self.pad = d, rows, C, pad
        self.n = rows * (C + pad)
        self.p = d.up(np.full(self.n + 2 * GUARD, 3.25, np.float32))
        self.at = self.p + 4 * GUARD

    def get(self):
        a = self.d.down(self.p, (self.n + 2 * GUARD,))
        assert (a[:GUARD] == 3.25).all() and (a[GUARD + self.n:] == 3.25).all()
        a = a[GUARD:GUARD + self.n].reshape(self.rows, self.C + self.pad)
        assert (a[:, self.C:] == 3.25).all()
        return a[:, :self.C] if self.rows > 1 or self.pad else a[0]


def close(got, want, what):
    value, bound = want
    off = np.abs(got.reshape(value.shape) - value)
    assert (off <= bound).all(), (what, float((off / bound).max()))


SHAPES = [(1, 1), (5, 2), (3, 3), (300, 31), (9, 32), (17, 33), (1000, 128), (33, 129), (8, 256), (21, 260), (300, 512), (7, 513), (40, 785), (5, 1024), (31, 1279),
          (600, 2048), (3, 2050), (4, 4096), (3, 5001), (2, 8192)]


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("kind", [ref.RMS, ref.LAYER])
def test_norm(D, rows, C, kind):
    Dev, capi = D
    r = np.random.RandomState(rows + C)
    x = (r.standard_normal((rows, C)) * 2 + 1).astype(np.float32)
    gamma, beta = (1 + 0.3 * r.standard_normal(C)).astype(np.float32), r.standard_normal(C).astype(np.float32)
    dy = r.standard_normal((rows, C)).astype(np.float32)
    y, dx, dg, db = ref.norm(x, gamma, beta, dy, kind, EPS)
    with Dev() as d:
        px, pg, pb, pdy = d.up(x), d.up(gamma), d.up(beta), d.up(dy)
        oy, odx, og, ob, st = Out(d, rows, C), Out(d, rows, C), Out(d, 1, C), Out(d, 1, C), d.new(2 * rows)
        capi.check(d.L.seera_norm_fwd(px, pg, pb, oy.at, st, rows, C, kind, EPS))
        close(oy.get(), y, "y")
        capi.check(d.L.seera_norm_bwd(pdy, px, pg, st, odx.at, og.at, ob.at, rows, C, kind))
        first = [o.get().copy() for o in (odx, og, ob)]
        for got, want, what in zip(first, (dx, dg, db), ("dx", "dgamma", "dbeta")):
            close(got, want, what)
        capi.check(d.L.seera_norm_bwd(pdy, px, pg, st, odx.at, og.at, ob.at, rows, C, kind))     # the same bits again
        assert all(np.array_equal(o.get(), f) for o, f in zip((odx, og, ob), first))
        capi.check(d.L.seera_norm_bwd(pdy, px, pg, st, None, og.at, None, rows, C, kind))
        assert np.array_equal(og.get(), first[1])
        want = oy.get().copy()
        capi.check(d.L.seera_norm_fwd(px, pg, pb, px, None, rows, C, kind, EPS))                 # in place, nothing kept
        assert np.array_equal(d.down(px, (rows, C)).ravel(), want.ravel())


def residual_inputs(rows, C, seed):
    r = np.random.RandomState(seed)
    n = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    return {"u": n(rows, C) * 2 + 0.5, "g": n(rows, C) * 2, "res": n(rows, C) * 3, "gamma": 1 + 0.3 * n(C), "scale": 1 + 0.2 * n(C), "gamma2": 1 + 0.3 * n(C),
            "beta2": n(C), "dout": n(rows, C), "dy": n(rows, C)}


def run_residual(D, rows, C, x, kind, act, kind2, pad=0, with_next=True):
    """Both directions through the ABI; the gate and its gradient are columns of wider rows."""
    Dev, capi = D
    have = lambda k: x[k] is not None  # noqa: E731
    with Dev() as d:
        p = {k: (None if a is None else d.up(a)) for k, a in x.items() if k != "g"}
        pg = None
        if have("g"):
            z = np.full((rows, C + pad), np.nan, np.float32)
            z[:, :C] = x["g"]
            pg = d.up(z)
        out, y, st = Out(d, rows, C), Out(d, rows, C), d.new(4 * rows)
        capi.check(d.L.seera_gated_residual_fwd(p["u"], pg, C + pad, p["res"], p["gamma"], p["scale"], out.at, p["gamma2"] if with_next else None,
                                                p["beta2"] if with_next else None, y.at if with_next else None, st, rows, C, kind, act, kind2, EPS, EPS))
        fwd = [out.get()] + ([y.get()] if with_next else [])
        o = {k: Out(d, rows, C, pad if k == "dgate" else 0) for k in ("du", "dgate", "dres")}
        o.update({k: Out(d, 1, C) for k in ("dgamma", "dscale", "dgamma2", "dbeta2")})
        at = lambda k, on: o[k].at if on else None  # noqa: E731
        second = have("dy") and with_next

        def back():
            capi.check(d.L.seera_gated_residual_bwd(p["dout"], p["dy"] if second else None, p["u"], pg, C + pad, p["res"], p["gamma"], p["scale"],
                                                    p["gamma2"] if second else None, st, o["du"].at, at("dgate", have("g")), C + pad, at("dres", have("res")),
                                                    o["dgamma"].at, at("dscale", have("res")), at("dgamma2", second), at("dbeta2", second), rows, C, kind, act,
                                                    kind2))
            return {k: v.get().copy() for k, v in o.items()}
        bwd = back()
        again = back()
        assert all(np.array_equal(bwd[k], again[k]) for k in bwd)
        return fwd, bwd


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("kind,act,kind2", [(ref.RMS, ref.SILU, ref.RMS), (ref.LAYER, ref.SIGMOID, ref.LAYER)])
def test_residual(D, rows, C, kind, act, kind2):
    x = residual_inputs(rows, C, rows * 3 + C)
    fwd, bwd = run_residual(D, rows, C, x, kind, act, kind2, pad=C % 7)
    wf, wb = ref.residual(**x, kind=kind, act=act, kind2=kind2, eps=EPS, eps2=EPS)
    for got, want, what in zip(fwd, wf, ("out", "y")):
        close(got, want, what)
    for k, want in wb.items():
        close(bwd[k], want, k)


@pytest.mark.parametrize("without", [("g",), ("res",), ("g", "res"), ("dout",), ("dy",), ("beta2",), ("next",), ("next", "g", "res")])
@pytest.mark.parametrize("act", [ref.NONE, ref.RELU, ref.TANH])
def test_residual_without_some_of_it(D, without, act):
    rows, C = 37, 132
    x = residual_inputs(rows, C, 11)
    for k in without:
        if k != "next":
            x[k] = None
    nxt = "next" not in without
    fwd, bwd = run_residual(D, rows, C, x, ref.RMS, act, ref.LAYER, with_next=nxt)
    if not nxt:
        x.update(gamma2=None, beta2=None, dy=None)
    wf, wb = ref.residual(**x, kind=ref.RMS, act=act, kind2=ref.LAYER, eps=EPS, eps2=EPS)
    for got, want, what in zip(fwd, wf, ("out", "y")):
        close(got, want, what)
    for k in bwd:
        if k in wb:
            close(bwd[k], wb[k], k)
        else:
            assert (bwd[k] == 3.25).all(), k


def test_residual_gradients_against_differences(D):
    rows, C = 3, 6
    x = residual_inputs(rows, C, 4)
    _, bwd = run_residual(D, rows, C, x, ref.LAYER, ref.SILU, ref.RMS)

    def value(y):
        (out, _), (z, _) = ref.residual(**{**y, "dout": None, "dy": None}, kind=ref.LAYER, act=ref.SILU, kind2=ref.RMS, eps=EPS, eps2=EPS)[0]
        return (out * x["dout"]).sum() + (z * x["dy"]).sum()
    for name, grad in (("u", "du"), ("g", "dgate"), ("res", "dres"), ("gamma", "dgamma"), ("scale", "dscale"), ("gamma2", "dgamma2"), ("beta2", "dbeta2")):
        base = x[name].astype(np.float64)
        for at in list(np.ndindex(base.shape))[::2]:
            step, y = 1e-4, base.copy()
            y[at] += step
            up = value({**x, name: y})
            y[at] -= 2 * step
            diff = (up - value({**x, name: y})) / (2 * step)
            # central differences of a smooth function: step^2 times a third derivative, and the rounding of float32 gradients
            assert abs(diff - bwd[grad][at]) <= 2e-5 + 2e-5 * abs(diff), (name, at)


def test_extreme_rows(D):
    """A row of zeros, one of equal values, a tiny and a large one beside ordinary ones; a NaN and an infinity stay in their rows."""
    Dev, capi = D
    rows, C = 8, 200
    r = np.random.RandomState(0)
    x = r.standard_normal((rows, C)).astype(np.float32)
    x[0], x[1], x[2], x[3] = 0, 4.5, x[2] * 1e-18, x[3] * 1e15
    x[5, 7], x[6, 100] = np.nan, np.inf
    gamma, beta = np.ones(C, np.float32), np.zeros(C, np.float32)
    fine = [0, 1, 2, 3, 4, 7]
    for kind in (ref.RMS, ref.LAYER):
        want, bound = ref.norm(x[fine], gamma, beta, x[fine], kind, EPS)[0]
        with Dev() as d:
            y = d.new(rows * C)
            capi.check(d.L.seera_norm_fwd(d.up(x), d.up(gamma), d.up(beta), y, None, rows, C, kind, EPS))
            got = d.down(y, (rows, C))
        assert (np.abs(got[fine] - want) <= bound).all()
        assert np.isnan(got[5]).all() and np.isnan(got[6, 100])


@pytest.mark.parametrize("act", [ref.NONE, ref.RELU, ref.SIGMOID, ref.TANH, ref.SILU])
def test_gates_far_out(D, act):
    """Gates of +-100 and beyond: nothing overflows on the way to a finite result."""
    rows, C = 4, 64
    x = residual_inputs(rows, C, 1)
    x["g"] = np.tile(np.array([-1e30, -1e4, -100, -88, -20, 0, 20, 88, 100, 1e4, 30, -30, 1e-30, -1e-30, 5, -5], np.float32), (rows, 4))
    if act in (ref.NONE, ref.RELU, ref.SILU):
        x["g"] = np.clip(x["g"], -1e30 if act == ref.SILU else -100, 100)
    fwd, bwd = run_residual(D, rows, C, x, ref.RMS, act, ref.RMS)
    with np.errstate(all="ignore"):
        wf, wb = ref.residual(**x, kind=ref.RMS, act=act, kind2=ref.RMS, eps=EPS, eps2=EPS)
    for got, want in zip(fwd, wf):
        close(got, want, "forward")
    for k in ("du", "dres", "dgate", "dgamma"):
        assert np.isfinite(bwd[k]).all()
    close(bwd["dres"], wb["dres"], "dres")


def test_norms_in_two_recordings(D):
    """Forward and backward recorded twice, replayed in turn with other rows: each recording's sums over the blocks are its own."""
    Dev, capi = D
    rows, C = 700, 516
    with Dev() as d:
        runs = []
        for _ in range(2):
            a = {k: d.new(rows * C) for k in ("u", "g", "res", "dout", "dy", "out", "y", "du", "dgate", "dres")}
            a.update({k: d.new(C) for k in ("gamma", "scale", "gamma2", "beta2", "dgamma", "dscale", "dgamma2", "dbeta2")}, st=d.new(4 * rows))
            capi.check(d.L.seera_graph_begin())
            capi.check(d.L.seera_gated_residual_fwd(a["u"], a["g"], C, a["res"], a["gamma"], a["scale"], a["out"], a["gamma2"], a["beta2"], a["y"], a["st"],
                                                    rows, C, ref.LAYER, ref.SILU, ref.RMS, EPS, EPS))
            capi.check(d.L.seera_gated_residual_bwd(a["dout"], a["dy"], a["u"], a["g"], C, a["res"], a["gamma"], a["scale"], a["gamma2"], a["st"], a["du"],
                                                    a["dgate"], C, a["dres"], a["dgamma"], a["dscale"], a["dgamma2"], a["dbeta2"], rows, C, ref.LAYER, ref.SILU,
                                                    ref.RMS))
            g = d.L.seera_graph_end()
            assert g
            runs.append((a, g))
        for seed in (1, 2):
            data = [residual_inputs(rows, C, 10 * seed + i) for i in range(2)]
            for (a, _), x in zip(runs, data):
                for k, host in x.items():
                    capi.check(d.L.seera_cuda_memcopy_devicetodevice(a[k], d.up(host), host.size))
            for _, g in runs:
                capi.check(d.L.seera_graph_launch(g))
            for (a, _), x in zip(runs, data):
                fwd, bwd = run_residual(D, rows, C, x, ref.LAYER, ref.SILU, ref.RMS)            # the same calls one by one
                for k, want in [("out", fwd[0]), ("y", fwd[1])] + list(bwd.items()):
                    assert np.array_equal(d.down(a[k], want.shape), want), k
        for _, g in runs:
            capi.check(d.L.seera_graph_destroy(g))
