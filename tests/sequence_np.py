"""The gated scan, the norms around a block and AdamW in 64 bits, each with how far a float32 evaluation may be off.

Bounds count roundings: u = 2^-24 is half a step of float32.  They are worked out with the absolute values of what is added, so they hold for every
order of a sum."""
import numpy as np

U = 2.0 ** -24
RMS, LAYER = 0, 1
NONE, RELU, SIGMOID, TANH, SILU = range(5)
f64 = np.float64


def sigmoid(x):
    x = np.asarray(x, f64)
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


# ---- gated scan ------------------------------------------------------------------------------------------------------------------
def scan_fwd(f, v, h0=None, lengths=None):
    """h, h_last and the bounds of both.  A step's roundings: the smaller of a and 1 - a from exp, a sum and a quotient (8 steps of u), their
    product with the difference of h and v, the sum.  Joining pieces of time does each of them up to three times.
    Pieces add a h[before] and what came since apart: |a x + b|, where the two cancel, does not bound the rounding of either, |a x| + |b| does.  `big` is
    the state with the absolute values of everything added."""
    f, v = np.asarray(f, f64), np.asarray(v, f64)
    N, T, C = f.shape
    a, na = sigmoid(f), sigmoid(-f)
    s = np.zeros((N, C)) if h0 is None else np.asarray(h0, f64).copy()
    e, big = np.zeros((N, C)), np.abs(s)
    h, eh = np.zeros((N, T, C)), np.zeros((N, T, C))
    live = np.ones((N, T), bool) if lengths is None else np.arange(T)[None] < np.asarray(lengths)[:, None]
    for t in range(T):
        on = live[:, t]
        old = s[on]
        new = a[on, t] * old + na[on, t] * v[on, t]
        was = big[on]
        big[on] = a[on, t] * was + na[on, t] * np.abs(v[on, t])
        e[on] = a[on, t] * e[on] + U * (big[on] + 10 * np.minimum(a[on, t], na[on, t]) * (was + np.abs(v[on, t])))
        s[on] = new
        h[on, t], eh[on, t] = new, e[on]
    return h, s, 3 * eh + 1e-37, 3 * e + 1e-37


def scan_bwd(f, v, h, dh=None, dlast=None, h0=None, lengths=None):
    """df, dv, dh0 and their bounds, with h as given; `big`: the carried gradient with the absolute values of everything added (see scan_fwd)."""
    f, v, h = (np.asarray(x, f64) for x in (f, v, h))
    N, T, C = f.shape
    a, na = sigmoid(f), sigmoid(-f)
    small = np.minimum(a, na)
    c = np.zeros((N, C)) if dlast is None else np.asarray(dlast, f64).copy()
    dh = np.zeros((N, T, C)) if dh is None else np.asarray(dh, f64)
    e, big = np.zeros((N, C)), np.abs(c)
    df, dv, edf, edv = (np.zeros((N, T, C)) for _ in range(4))
    live = np.ones((N, T), bool) if lengths is None else np.arange(T)[None] < np.asarray(lengths)[:, None]
    before = np.concatenate([np.zeros((N, 1, C)) if h0 is None else np.asarray(h0, f64)[:, None], h[:, :-1]], 1)
    for t in reversed(range(T)):
        on = live[:, t]
        g = dh[on, t] + c[on]
        all_ = np.abs(dh[on, t]) + big[on]
        eg = e[on] + U * all_
        A, NA, S, d = a[on, t], na[on, t], small[on, t], before[on, t] - v[on, t]
        dv[on, t], df[on, t] = NA * g, A * NA * d * g
        edv[on, t] = NA * eg + 12 * U * np.abs(NA * g)
        edf[on, t] = A * NA * (np.abs(d) * eg + np.abs(g) * (U * np.abs(d) + 20 * U * np.abs(d)))
        c[on] = A * g
        big[on] = A * all_
        e[on] = A * eg + U * (A * all_ + 10 * S * all_)
    return df, dv, c, 3 * edf + 1e-37, 3 * edv + 1e-37, 3 * e + 1e-37


# ---- norms -----------------------------------------------------------------------------------------------------------------------
# A mean over the row: at most 16 additions in a thread, 5 in a warp, 16 over warps, the product with 1 / C; a reciprocal root.
_MEAN = 40 * U


def _moments(x, kind, eps, ex):
    """mu, s, N(x) and the bound of N(x), x off by up to ex."""
    mu = x.mean(1, keepdims=True) if kind == LAYER else np.zeros((x.shape[0], 1))
    emu = _MEAN * np.abs(x).mean(1, keepdims=True) + ex.mean(1, keepdims=True) if kind == LAYER else np.zeros_like(mu)
    d = x - mu
    ed = ex + emu + U * np.abs(d)
    var = (d * d).mean(1, keepdims=True) + eps
    es = ((2 * np.abs(d) * ed + ed * ed).mean(1, keepdims=True) + _MEAN * var) / var / 2 + 4 * U         # of s, relative
    s = 1 / np.sqrt(var)
    return mu, s, d * s, ed * s + np.abs(d) * s * (es + 2 * U)


def _norm_grad(b, eb, n, en, s, kind):
    """s (b - [mean b] - n mean(b n)) and its bound, b and n off by up to eb and en."""
    m0 = b.mean(1, keepdims=True) if kind == LAYER else 0.0
    m1 = (b * n).mean(1, keepdims=True)
    em0 = eb.mean(1, keepdims=True) + _MEAN * np.abs(b).mean(1, keepdims=True) if kind == LAYER else 0.0
    em1 = (eb * np.abs(n) + np.abs(b) * en).mean(1, keepdims=True) + _MEAN * np.abs(b * n).mean(1, keepdims=True)
    out = s * (b - m0 - n * m1)
    size = np.abs(b) + np.abs(m0) + np.abs(n * m1)
    return out, s * (eb + em0 + en * np.abs(m1) + np.abs(n) * em1) + 64 * U * s * size       # (64: s has been rounded as well)


def _sum(x, ex):
    """Over the rows: a thread's own, then those side by side, then the blocks': at most 100 additions one after the other for the rows used here."""
    return x.sum(0), ex.sum(0) + 100 * U * np.abs(x).sum(0) + 1e-37


def norm(x, gamma, beta, dy, kind, eps):
    """y, dx, dgamma, dbeta, each with its bound."""
    x, gamma, dy = np.asarray(x, f64), np.asarray(gamma, f64), np.asarray(dy, f64)
    beta = np.zeros(x.shape[1]) if beta is None else np.asarray(beta, f64)
    _, s, n, en = _moments(x, kind, eps, np.zeros_like(x))
    y = n * gamma + beta
    ey = en * np.abs(gamma) + 2 * U * (np.abs(n * gamma) + np.abs(beta))
    b = dy * gamma
    dx = _norm_grad(b, U * np.abs(b), n, en, s, kind)
    return [(y, ey + 1e-37), dx, _sum(dy * n, np.abs(dy) * en), _sum(dy, 0 * dy)]


def gate(g, act):
    """act(g) and its slope; a few roundings each."""
    g = np.asarray(g, f64)
    p = sigmoid(g)
    return {NONE: (g, np.ones_like(g)), RELU: (np.where(g > 0, g, 0), np.where(g > 0, 1.0, 0.0)), SIGMOID: (p, p * (1 - p)),
            TANH: (np.tanh(g), 1 / np.cosh(np.clip(g, -300, 300)) ** 2), SILU: (g * p, p * (1 + g * sigmoid(-g)))}[act]


def residual(u, g, res, gamma, scale, gamma2, beta2, dout, dy, kind, act, kind2, eps, eps2):
    """(out, y) and (du, dgate, dres, dgamma, dscale, dgamma2, dbeta2), each with its bound.  g, res, gamma2 (no second norm), dout and dy may be
    None."""
    to = lambda x: None if x is None else np.asarray(x, f64)  # noqa: E731
    u, g, res, gamma, scale, gamma2, beta2, dout, dy = map(to, (u, g, res, gamma, scale, gamma2, beta2, dout, dy))
    zero = np.zeros_like(u)
    _, s, n, en = _moments(u, kind, eps, zero)
    q, slope = (np.ones_like(u), zero) if g is None else gate(g, act)
    eq, eslope = (zero, zero) if g is None else (8 * U * np.abs(q), 16 * U * (1 + np.abs(g)))
    p = gamma * n
    ep = np.abs(gamma) * en + U * np.abs(p)
    r = zero if res is None else scale * res
    out = r + q * p
    eo = np.abs(q) * ep + eq * np.abs(p) + 3 * U * (np.abs(q * p) + np.abs(r))
    fwd, n2 = [(out, eo + 1e-37)], None
    if gamma2 is not None:
        _, s2, n2, en2 = _moments(out, kind2, eps2, eo)
        b2 = 0.0 if beta2 is None else beta2
        fwd.append((n2 * gamma2 + b2, en2 * np.abs(gamma2) + 2 * U * (np.abs(n2 * gamma2) + np.abs(b2)) + 1e-37))
    if dout is None and dy is None:
        return fwd, None
    d, ed = (zero, zero) if dout is None else (dout, zero)
    if dy is not None:
        a = dy * gamma2
        x, ex = _norm_grad(a, U * np.abs(a), n2, en2, s2, kind2)
        # (s2 itself is off where out is)
        ex = ex + np.abs(x) * ((en2 * np.abs(n2)).mean(1, keepdims=True) + en2.max(1, keepdims=True))
        d, ed = d + x, ed + ex + U * (np.abs(d) + np.abs(x))
    bwd = {}
    b = d * q * gamma
    eb = np.abs(gamma) * (ed * np.abs(q) + np.abs(d) * eq) + 3 * U * np.abs(b)
    bwd["du"] = _norm_grad(b, eb, n, en, s, kind)
    if g is not None:
        t = d * p * slope
        bwd["dgate"] = t, np.abs(p * slope) * ed + np.abs(d * slope) * ep + np.abs(d * p) * eslope + 4 * U * np.abs(t) + 1e-37
    if res is not None:
        bwd["dres"] = scale * d, np.abs(scale) * ed + U * np.abs(scale * d) + 1e-37
        bwd["dscale"] = _sum(d * res, ed * np.abs(res))
    dq = d * q
    bwd["dgamma"] = _sum(dq * n, (ed * np.abs(q) + np.abs(d) * eq) * np.abs(n) + np.abs(dq) * en)
    if dy is not None:
        bwd["dgamma2"], bwd["dbeta2"] = _sum(dy * n2, np.abs(dy) * en2), _sum(dy, zero)
    return fwd, bwd


# ---- AdamW: the averages in float32, bit for bit, each operation rounded by itself -------------------------------------------------------
def f32(*xs):
    return [np.float32(x) for x in xs]


def adamw(w, g, m, v, decay, lr, b1, omb1, b2, omb2, eps, c1, c2, scale):
    """m and v as they come out, w in 64 bits with its bound."""
    lr, b1, omb1, b2, omb2, eps, c1, c2, scale = f32(lr, b1, omb1, b2, omb2, eps, c1, c2, scale)
    with np.errstate(all="ignore"):
        g = g * scale
        m, v = b1 * m + omb1 * g, b2 * v + omb2 * (g * g)
        w, M, V = w.astype(f64), m.astype(f64), v.astype(f64)
        move = lr.astype(f64) * (M / c1) / (np.sqrt(V / c2) + eps)
        keep = w * (1 - f64(lr) * f64(np.float32(decay)))
    return keep - move, m, v, U * (4 * np.abs(keep) + 8 * np.abs(move) + np.abs(w)) + 1e-37


def _hash(place, step):
    low = np.uint64(0xFFFFFFFF)
    place = place.astype(np.uint64)
    x = (place & low) ^ (((place >> np.uint64(32)) * np.uint64(0x632BE5AB)) & low) ^ np.uint64((int(step) * 0x9E3779B1) & 0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0xA3D95F4B)) & low
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x6C8E9D73)) & low
    return x ^ (x >> np.uint64(16))


def _codes(x, inv, unit, top, rnd):
    y = (x * inv * np.float32(unit)).astype(np.float32).view(np.uint32)
    return np.minimum((y + (rnd.astype(np.uint32) << np.uint32(4))) >> np.uint32(20), np.uint32(top))


def pack8(m, v, step, first=0):
    """The state of one tensor, n entries, rounded with the random bits of `step`."""
    n = m.size
    blocks = -(-n // 64)
    M, V = np.zeros(blocks * 64, np.float32), np.zeros(blocks * 64, np.float32)
    M[:n], V[:n] = m, v
    r = _hash(np.arange(first, first + blocks * 64, dtype=np.uint64), step)
    M, V, r = M.reshape(-1, 64), V.reshape(-1, 64), r.reshape(-1, 64)
    tiny = np.finfo(np.float32).tiny
    with np.errstate(all="ignore"):
        am, av = np.abs(M).max(1), np.abs(V).max(1)
        am, av = np.where(am < tiny, np.float32(0), am), np.where(av < tiny, np.float32(0), av)
        im, iv = (np.where(a > 0, np.float32(1) / a, np.float32(0)).astype(np.float32)[:, None] for a in (am, av))
        cm = _codes(np.abs(M), im, 2.0 ** -112, 0x78, r & np.uint64(0xFFFF)) | np.where(M < 0, np.uint32(128), np.uint32(0))
        cv = _codes(V, iv, 2.0 ** -96, 0xF8, r >> np.uint64(16))
    out = np.zeros((blocks, 136), np.uint8)
    body = out[:, :128].reshape(-1, 16, 2, 4)
    body[:, :, 0], body[:, :, 1] = cm.reshape(-1, 16, 4), cv.reshape(-1, 16, 4)
    out[:, :128] = body.reshape(-1, 128)
    out[:, 128:] = np.stack([am, av], 1).astype(np.float32).view(np.uint8)
    return out.reshape(-1)


def unpack8(state, n):
    state = np.asarray(state, np.uint8).reshape(-1, 136)
    codes = state[:, :128].reshape(-1, 16, 2, 4).astype(np.uint32)
    top = np.ascontiguousarray(state[:, 128:]).view(np.float32)
    cm, cv = codes[:, :, 0].reshape(-1, 64), codes[:, :, 1].reshape(-1, 64)
    with np.errstate(all="ignore"):
        m = ((cm & np.uint32(127)) << np.uint32(20)).view(np.float32) * np.float32(2.0 ** 112) * top[:, :1]
        v = (cv << np.uint32(20)).view(np.float32) * np.float32(2.0 ** 96) * top[:, 1:]
    return np.where(cm > 127, -m, m).reshape(-1)[:n], v.reshape(-1)[:n]
