"""Operators of a gated linear recurrent block and of its training: what is measured, and their plain forms.

Three operators, each through the entry points of the binding (`seera_cuda`):
  the gated scan       h[t] = a[t] h[t-1] + (1 - a[t]) v[t] with a = sigmoid(f): `gated_scan_fwd`, `gated_scan_bwd`
  norms and residual   a norm over the features before a block (`norm_fwd`, `norm_bwd`), and what follows a block in one pass: its norm,
                       its gate, the scaled residual and the next block's norm (`gated_residual_fwd`, `gated_residual_bwd`)
  AdamW                one step over many tensors with their states in 32 bits (`adamw_step`) or in 8 (`adamw8_step`, `adamw8_read`)
Everything is float32, as in the rest of the framework, but the states held in 8 bits.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
RMS, LAYER = 0, 1
NONE, RELU, SIGMOID, TANH, SILU = range(5)


def listed():
    return [
        # one new token of eight streams: a recurrent layer's step while answering, all latency
        {"name": "scan_step_8x2048", "kind": "scan_fwd", "N": 8, "T": 1, "C": 2048, "state": True, "ragged": False},
        # one long document read in a single pass: few channels to go by, the time axis has to be split
        {"name": "scan_fwd_1x65536x512", "kind": "scan_fwd", "N": 1, "T": 65536, "C": 512, "state": False, "ragged": False},
        # backward of a training batch, the largest call of the scan
        {"name": "scan_bwd_8x2048x2048", "kind": "scan_bwd", "N": 8, "T": 2048, "C": 2048, "state": False, "ragged": False},
        # backward of a padded batch of odd sizes, sequences of length 0 and 1 among them, with a state carried in and out
        {"name": "scan_bwd_ragged_7x1023x645", "kind": "scan_bwd", "N": 7, "T": 1023, "C": 645, "state": True, "ragged": True},
        # the norm before the first block, forward and backward, of a training batch
        {"name": "norm_16384x1280", "kind": "norm", "rows": 16384, "C": 1280, "norm": LAYER},
        # the same for a small ragged batch of an odd width
        {"name": "norm_333x785", "kind": "norm", "rows": 333, "C": 785, "norm": RMS},
        # the end of a block for one new token of eight streams
        {"name": "residual_step_8x2048", "kind": "residual_fwd", "rows": 8, "C": 2048, "norm": RMS, "next": RMS, "act": SILU},
        # the end of a block in a training batch, with the next block's norm
        {"name": "residual_fwd_16384x2048", "kind": "residual_fwd", "rows": 16384, "C": 2048, "norm": RMS, "next": RMS, "act": SILU},
        # its backward, every gradient
        {"name": "residual_bwd_16384x2048", "kind": "residual_bwd", "rows": 16384, "C": 2048, "norm": RMS, "next": RMS, "act": SILU},
        # an odd width, whose rows do not start on 16 bytes
        {"name": "residual_bwd_2049x1279", "kind": "residual_bwd", "rows": 2049, "C": 1279, "norm": LAYER, "next": LAYER, "act": SIGMOID},
        # the update of a small network: many tensors, little work
        {"name": "adamw_32bit_12x48", "kind": "adamw", "layers": 12, "width": 48, "bits": 32},
        # the update of a large one with its states in 8 bits, read out as a checkpoint does
        {"name": "adamw_8bit_8x1024", "kind": "adamw", "layers": 8, "width": 1024, "bits": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scan_fwd", "scan_bwd", "norm", "residual_fwd", "residual_bwd", "adamw", "adamw"])
    if kind.startswith("scan"):
        most = 1 << 25
        T = 1 if kind == "scan_fwd" and rng.random() < 0.25 else _log(rng, 2, 65536)
        C = min(_log(rng, 1, 4096), max(1, most // T))
        N = _log(rng, 1, max(1, min(64, most // (T * C))))
        return {"kind": kind, "N": N, "T": T, "C": C, "state": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    if kind == "adamw":
        width = _log(rng, 3, 1024)
        return {"kind": kind, "layers": _log(rng, 1, min(64, max(1, 60_000_000 // (8 * width * width)))), "width": width, "bits": rng.choice([8, 32])}
    C = _log(rng, 8, 8192)
    rows = _log(rng, 1, min(65536, max(1, (1 << 25) // C)))
    case = {"kind": kind, "rows": rows, "C": C, "norm": rng.choice([RMS, LAYER])}
    if kind != "norm":
        case.update(next=rng.choice([RMS, LAYER]), act=rng.choice([NONE, RELU, SIGMOID, TANH, SILU]))
    return case


# ---- what a program has in hand ------------------------------------------------------------------------------------------------
def _sizes(case):
    """The tensors of a network of `layers` blocks: two weight matrices and their biases each."""
    D = case["width"]
    return [s for _ in range(case["layers"]) for s in (4 * D * D, 4 * D, 4 * D * D, D)]


def _scan_inputs(case, rand, seed):
    N, T, C = case["N"], case["T"], case["C"]
    # gate logits and candidates side by side in the rows of one projection; gates that remember from a step to a few hundred
    z = torch.cat([rand(N, T, C) * 1.5 + 2.0, rand(N, T, C)], dim=2)
    h0 = rand(N, C) if case["state"] else None
    lengths = None
    if case["ragged"]:
        r = random.Random(seed)
        lengths = [r.randint(0, T) for _ in range(N)]
        for i, v in ((0, T), (1, 0), (2, min(1, T))):
            if i < N:
                lengths[i] = v
        lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    return {"z": z, "h0": h0, "lengths": lengths}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")
    kind = case["kind"]
    st = {"case": case}
    if kind.startswith("scan"):
        N, T, C = case["N"], case["T"], case["C"]
        st.update(_scan_inputs(case, rand, seed))
        st["last"] = torch.empty(N, C, device="cuda")
        if kind == "scan_fwd":
            st["h"] = torch.empty(N, T, C, device="cuda")
        else:
            st["h"] = _scan_fwd(st)[0]
            st["dh"], st["dlast"] = rand(N, T, C), rand(N, C) if case["state"] else None
            st["dz"] = torch.empty(N, T, 2 * C, device="cuda")
            st["dh0"] = torch.empty(N, C, device="cuda") if case["state"] else None
    elif kind == "adamw":
        sizes = _sizes(case)
        starts = np.concatenate([[0], np.cumsum([-(-n // 64) * 64 for n in sizes])]).astype(np.int64)
        total = int(starts[-1])
        # one arena of parameters, each tensor's slot a multiple of 64: what lies between is zero and stays so
        used = torch.zeros(total, device="cuda")
        decay = torch.zeros(total // 64, device="cuda")
        decays = np.array([0.1 if i % 2 == 0 else 0.0 for i in range(len(sizes))], np.float32)         # matrices decay, biases do not
        for o, n, d in zip(starts, sizes, decays):
            used[o:o + n] = 1
            decay[o // 64:(o + n + 63) // 64] = float(d)
        w, g = rand(total) * 0.02 * used, rand(total) * 1e-3 * used
        # averages as they are after ten steps of gradients whose magnitude differs from entry to entry
        size = torch.exp(rand(total) * 1.5) * used
        m, v = rand(total) * 3e-4 * size, (rand(total) ** 2 * 0.5 + 0.1) * 4e-7 * size * size
        g *= size
        st.update(w=w, g=g, decay=decay, t=10)
        st["hp"] = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "scale": 0.5}
        at = lambda x, unit: np.array([x.data_ptr() + int(o) * unit // 64 for o in starts[:-1]], np.uint64)  # noqa: E731
        st["at_w"], st["at_g"], st["n"], st["decays"] = at(w, 256), at(g, 256), np.array(sizes, np.int64), decays
        if case["bits"] == 32:
            st.update(m=m, v=v, at_m=at(m, 256), at_v=at(v, 256))
        else:
            st["state"] = _pack8(m.view(-1, 64), v.view(-1, 64), None)
            st.update(at_state=at(st["state"], 136), m=torch.empty_like(m), v=torch.empty_like(v))
    else:
        rows, C = case["rows"], case["C"]
        st.update(x=rand(rows, C) * 2 + 0.5, gamma=1 + 0.2 * rand(C), beta=0.1 * rand(C))
        st["stats"] = torch.empty(rows, 4 if kind != "norm" else 2, device="cuda")
        new = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        if kind == "norm":
            st.update(dy=rand(rows, C), y=new(rows, C), dx=new(rows, C), dgamma=new(C), dbeta=new(C))
        else:
            st.update(gate=rand(rows, C), res=rand(rows, C) * 3, scale=1 + 0.1 * rand(C), gamma2=1 + 0.2 * rand(C), beta2=0.1 * rand(C))
            if kind == "residual_fwd":
                st.update(out=new(rows, C), y=new(rows, C))
            else:
                st.update(dout=rand(rows, C), dy=rand(rows, C), du=new(rows, C), dgate=new(rows, C), dres=new(rows, C), dparams=[new(C) for _ in range(4)])
                u, out = st["x"], _residual_fwd(st)[0]
                st["stats"] = torch.cat([*_moments(u, case["norm"]), *_moments(out, case["next"])], dim=1).contiguous()
    return st


# ---- plain forms ---------------------------------------------------------------------------------------------------------------
def _shift(x, d, fill):
    """x moved by d steps towards later times, `fill` where nothing comes from."""
    out = torch.full_like(x, fill)
    if d < x.shape[1]:
        out[:, d:] = x[:, :-d]
    return out


def _scan(a, b):
    """All s[t] = a[t] s[t-1] + b[t] along axis 1 from s[-1] = 0, by doubling the distance that is joined."""
    d = 1
    while d < a.shape[1]:
        b = b + a * _shift(b, d, 0.0)
        a = a * _shift(a, d, 1.0)
        d *= 2
    return b


def _gates(st):
    """a, 1 - a and v, and which steps there are."""
    case, z = st["case"], st["z"]
    f, v = z[..., :case["C"]], z[..., case["C"]:]
    live = None
    if st["lengths"] is not None:
        live = (torch.arange(case["T"], device=z.device)[None, :] < st["lengths"][:, None])[..., None]
    return torch.sigmoid(f), torch.sigmoid(-f), v, live


def _scan_fwd(st):
    a, na, v, live = _gates(st)
    b = na * v
    if live is not None:
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    if st["h0"] is not None:
        b = torch.cat([b[:, :1] + a[:, :1] * st["h0"][:, None], b[:, 1:]], dim=1)
    s = _scan(a, b)
    return (s if live is None else torch.where(live, s, 0.0)), s[:, -1].clone()


def _scan_bwd(st):
    a, na, v, live = _gates(st)
    T, dh, h, h0 = a.shape[1], st["dh"], st["h"], st["h0"]
    if live is not None:
        dh, a = torch.where(live, dh, 0.0), torch.where(live, a, 1.0)
    b = a * dh
    if st["dlast"] is not None:
        b = torch.cat([b[:, :-1], b[:, -1:] + a[:, -1:] * st["dlast"][:, None]], dim=1)
    c = _scan(a.flip(1), b.flip(1)).flip(1)                    # c[t] = a[t] (dh[t] + c[t+1])
    after = torch.cat([c[:, 1:], torch.zeros_like(c[:, :1]) if st["dlast"] is None else st["dlast"][:, None]], dim=1)
    before = torch.cat([torch.zeros_like(h[:, :1]) if h0 is None else h0[:, None], h[:, :-1]], dim=1)
    g = dh + after
    df, dv = a * na * (before - v) * g, na * g
    if live is not None:
        df, dv = torch.where(live, df, 0.0), torch.where(live, dv, 0.0)
    dz = torch.cat([df, dv], dim=2)
    return [dz] if h0 is None else [dz, c[:, 0].clone()]


def _moments(x, kind):
    mu = x.mean(dim=1, keepdim=True) if kind == LAYER else torch.zeros_like(x[:, :1])
    return mu, torch.rsqrt((x - mu).square().mean(dim=1, keepdim=True) + EPS)


def _norm(x, kind):
    mu, s = _moments(x, kind)
    return (x - mu) * s, s


def _norm_grad(d, n, s, kind):
    """The gradient of x from that of its normalised values n."""
    m = d.mean(dim=1, keepdim=True) if kind == LAYER else 0.0
    return s * (d - m - n * (d * n).mean(dim=1, keepdim=True))


def _gate(g, act):
    """act(g) and its slope."""
    one = torch.ones_like(g)
    if act == NONE:
        return g, one
    if act == RELU:
        return torch.where(g > 0, g, 0.0), torch.where(g > 0, one, 0.0)
    if act == TANH:
        t = torch.tanh(g)
        return t, 1 - t * t
    p, q = torch.sigmoid(g), torch.sigmoid(-g)
    return (p, p * q) if act == SIGMOID else (g * p, p * (1 + g * q))


def _norm_both(st):
    case = st["case"]
    n, s = _norm(st["x"], case["norm"])
    dx = _norm_grad(st["dy"] * st["gamma"], n, s, case["norm"])
    return [n * st["gamma"] + st["beta"], dx, (st["dy"] * n).sum(dim=0), st["dy"].sum(dim=0)]


def _residual_fwd(st):
    case = st["case"]
    n, _ = _norm(st["x"], case["norm"])
    q, _ = _gate(st["gate"], case["act"])
    out = st["scale"] * st["res"] + q * (st["gamma"] * n)
    n2, _ = _norm(out, case["next"])
    return [out, n2 * st["gamma2"] + st["beta2"]]


def _residual_bwd(st):
    case = st["case"]
    n, s = _norm(st["x"], case["norm"])
    q, slope = _gate(st["gate"], case["act"])
    p = st["gamma"] * n
    n2, s2 = _norm(st["scale"] * st["res"] + q * p, case["next"])
    d = st["dout"] + _norm_grad(st["dy"] * st["gamma2"], n2, s2, case["next"])
    dp = d * q
    du = _norm_grad(dp * st["gamma"], n, s, case["norm"])
    return [du, d * p * slope, st["scale"] * d, (dp * n).sum(dim=0), (d * st["res"]).sum(dim=0), (st["dy"] * n2).sum(dim=0), st["dy"].sum(dim=0)]


# States in 8 bits: 64 neighbouring entries of a tensor are a block of 136 bytes, sixteen times four codes of m and four of v, then the
# largest |m| and the largest v of the block as floats.  A code is the exponent's low bits and three bits of mantissa of the entry over the
# largest one, as a float times a power of two would hold them: m a sign, four exponent bits, v five exponent bits.
_M_UNIT, _V_UNIT = 2.0 ** -112, 2.0 ** -96         # 1.0 times these has the exponent fields 15 and 31
_M_TOP, _V_TOP = 0x78, 0xF8                        # their codes


def _mix(place, step):
    """32 random bits for each place of a step's update, as int64."""
    low = (1 << 32) - 1
    x = (place & low) ^ (((place >> 32) * 0x632BE5AB) & low) ^ ((step * 0x9E3779B1) & low)
    x = ((x ^ (x >> 16)) * 0xA3D95F4B) & low
    x = ((x ^ (x >> 15)) * 0x6C8E9D73) & low
    return x ^ (x >> 16)


def _code(x, unit, top, bits):
    """Codes of x in [0, 1]: the neighbour above with the probability of its nearness; `bits`: 16 random ones, or None for the nearest."""
    y = (x * unit).view(torch.int32)
    y = (y + (0x80000 if bits is None else bits.to(torch.int32) << 4)) >> 20
    return torch.clamp(y, max=top)


def _pack8(m, v, rnd):
    am, av = m.abs().amax(dim=1), v.amax(dim=1)
    tiny = torch.finfo(torch.float32).tiny
    am, av = torch.where(am < tiny, 0.0, am), torch.where(av < tiny, 0.0, av)
    im, iv = (torch.where(a > 0, a.reciprocal(), 0.0)[:, None] for a in (am, av))
    cm = _code(m.abs() * im, _M_UNIT, _M_TOP, None if rnd is None else rnd & 0xFFFF) | torch.where(m < 0, 128, 0)
    cv = _code(v * iv, _V_UNIT, _V_TOP, None if rnd is None else rnd >> 16)
    out = torch.empty(m.shape[0], 136, dtype=torch.uint8, device=m.device)
    out[:, :128].view(-1, 16, 2, 4)[:, :, 0] = cm.view(-1, 16, 4).to(torch.uint8)
    out[:, :128].view(-1, 16, 2, 4)[:, :, 1] = cv.view(-1, 16, 4).to(torch.uint8)
    out[:, 128:] = torch.stack([am, av], dim=1).view(torch.uint8)
    return out


def _unpack8(state):
    codes = state[:, :128].view(-1, 16, 2, 4).to(torch.int32)
    scales = state[:, 128:].contiguous().view(torch.float32)
    cm, cv = codes[:, :, 0].reshape(-1, 64), codes[:, :, 1].reshape(-1, 64)
    m = ((cm & 127) << 20).view(torch.float32) * (1 / _M_UNIT) * scales[:, :1]
    v = (cv << 20).view(torch.float32) * (1 / _V_UNIT) * scales[:, 1:]
    return torch.where(cm > 127, -m, m), v


def _scalars(st):
    """What a step's scalars are, rounded to 32 bits: lr, beta1, 1 - beta1, beta2, 1 - beta2, eps, the corrections, the gradient's factor."""
    h, t = st["hp"], st["t"]
    return [float(np.float32(x)) for x in (h["lr"], h["beta1"], 1 - h["beta1"], h["beta2"], 1 - h["beta2"], h["eps"],
                                           1 - h["beta1"] ** t, 1 - h["beta2"] ** t, h["scale"])]


def _adamw(st):
    lr, b1, omb1, b2, omb2, eps, c1, c2, scale = _scalars(st)
    eight = st["case"]["bits"] == 8
    w, g = st["w"].view(-1, 64), st["g"].view(-1, 64) * scale
    m, v = _unpack8(st["state"]) if eight else (st["m"].view(-1, 64), st["v"].view(-1, 64))
    m, v = b1 * m + omb1 * g, b2 * v + omb2 * (g * g)
    keep = 1 - lr * st["decay"][:, None]
    w.copy_(w * keep - lr * (m / c1) / (torch.sqrt(v / c2) + eps))
    if eight:
        place = torch.arange(w.numel(), device=w.device).view(-1, 64)
        st["state"].copy_(_pack8(m, v, _mix(place, st["t"])))
        m, v = _unpack8(st["state"])
    st["m"].view(-1, 64).copy_(m)
    st["v"].view(-1, 64).copy_(v)
    st["t"] += 1
    return [st["w"], st["m"], st["v"]]


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def _at(x):
    return 0 if x is None else x.data_ptr()


def _run_own(st):
    from ml_framework_b200 import seera_cuda as sc
    case = st["case"]
    kind = case["kind"]
    if kind.startswith("scan"):
        N, T, C = case["N"], case["T"], case["C"]
        f = st["z"].data_ptr()
        if kind == "scan_fwd":
            sc.gated_scan_fwd(f, f + 4 * C, 2 * C, _at(st["h0"]), _at(st["lengths"]), _at(st["h"]), _at(st["last"]), N, T, C)
            return [st["h"], st["last"]]
        df = st["dz"].data_ptr()
        sc.gated_scan_bwd(f, f + 4 * C, 2 * C, _at(st["h0"]), _at(st["lengths"]), _at(st["h"]), _at(st["dh"]), _at(st["dlast"]),
                          df, df + 4 * C, 2 * C, _at(st["dh0"]), N, T, C)
        return [st["dz"]] if st["h0"] is None else [st["dz"], st["dh0"]]
    if kind == "adamw":
        s = _scalars(st)
        if case["bits"] == 32:
            sc.adamw_step(st["at_w"], st["at_g"], st["at_m"], st["at_v"], st["n"], st["decays"], *s)
        else:
            sc.adamw8_step(st["at_w"], st["at_g"], st["at_state"], st["n"], st["decays"], *s, float(st["t"]))
            sc.adamw8_read(_at(st["state"]), _at(st["m"]), _at(st["v"]), st["m"].numel())
        st["t"] += 1
        return [st["w"], st["m"], st["v"]]
    rows, C = case["rows"], case["C"]
    if kind == "norm":
        sc.norm_fwd(_at(st["x"]), _at(st["gamma"]), _at(st["beta"]), _at(st["y"]), _at(st["stats"]), rows, C, case["norm"], EPS)
        sc.norm_bwd(_at(st["dy"]), _at(st["x"]), _at(st["gamma"]), _at(st["stats"]), _at(st["dx"]), _at(st["dgamma"]), _at(st["dbeta"]), rows, C,
                    case["norm"])
        return [st["y"], st["dx"], st["dgamma"], st["dbeta"]]
    if kind == "residual_fwd":
        sc.gated_residual_fwd(_at(st["x"]), _at(st["gate"]), C, _at(st["res"]), _at(st["gamma"]), _at(st["scale"]), _at(st["out"]),
                              _at(st["gamma2"]), _at(st["beta2"]), _at(st["y"]), _at(st["stats"]), rows, C, case["norm"], case["act"], case["next"],
                              EPS, EPS)
        return [st["out"], st["y"]]
    dg, ds, dg2, db2 = st["dparams"]
    sc.gated_residual_bwd(_at(st["dout"]), _at(st["dy"]), _at(st["x"]), _at(st["gate"]), C, _at(st["res"]), _at(st["gamma"]), _at(st["scale"]),
                          _at(st["gamma2"]), _at(st["stats"]), _at(st["du"]), _at(st["dgate"]), C, _at(st["dres"]), _at(dg), _at(ds), _at(dg2),
                          _at(db2), rows, C, case["norm"], case["act"], case["next"])
    return [st["du"], st["dgate"], st["dres"], dg, ds, dg2, db2]


def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "scan_fwd":
        return list(_scan_fwd(state))
    if kind == "scan_bwd":
        return _scan_bwd(state)
    if kind == "adamw":
        return _adamw(state)
    return {"norm": _norm_both, "residual_fwd": _residual_fwd, "residual_bwd": _residual_bwd}[kind](state)


def work(case):
    """Each input read once, each output written once."""
    kind = case["kind"]
    if kind.startswith("scan"):
        n, c = case["N"] * case["T"] * case["C"], case["N"] * case["C"]
        state = 4 * c * (1 if case["state"] else 0)
        if kind == "scan_fwd":
            return {"bytes": 12 * n + 4 * c + state, "flops": 12 * n}
        return {"bytes": 24 * n + 3 * state, "flops": 20 * n}
    if kind == "adamw":
        n = sum(_sizes(case))
        return {"bytes": n * (28 if case["bits"] == 32 else 12 + 2 * 136 / 64 + 8), "flops": 16 * n}
    n = case["rows"] * case["C"]
    return {"norm": {"bytes": 20 * n, "flops": 22 * n}, "residual_fwd": {"bytes": 20 * n, "flops": 24 * n},
            "residual_bwd": {"bytes": 32 * n, "flops": 60 * n}}[kind]


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------------
def _exact_scan(case, st):
    """Step by step in time."""
    C, T, N = case["C"], case["T"], case["N"]
    f, v = st["z"][..., :C].double(), st["z"][..., C:].double()
    a = 1 / (1 + torch.exp(-f))
    na = 1 / (1 + torch.exp(f))
    length = torch.full((N,), T, device=f.device) if st["lengths"] is None else st["lengths"]
    alive = torch.arange(T, device=f.device)[:, None] < length[None, :]
    zero = torch.zeros(N, C, dtype=torch.float64, device=f.device)
    if case["kind"] == "scan_fwd":
        s = zero if st["h0"] is None else st["h0"].double()
        h = torch.zeros(N, T, C, dtype=torch.float64, device=f.device)
        u = na * v
        for t in range(T):
            new = torch.addcmul(u[:, t], a[:, t], s)
            s = new if st["lengths"] is None else torch.where(alive[t][:, None], new, s)
            h[:, t] = s if st["lengths"] is None else torch.where(alive[t][:, None], new, zero)
        return [h, s]
    dh, h = st["dh"].double(), st["h"].double()
    c = zero if st["dlast"] is None else st["dlast"].double()
    g = torch.zeros(N, T, C, dtype=torch.float64, device=f.device)
    for t in reversed(range(T)):
        on = alive[t][:, None]
        now = dh[:, t] + c
        g[:, t] = torch.where(on, now, zero)
        c = torch.where(on, a[:, t] * now, c)
    h[:, 1:] = h[:, :-1].clone()
    h[:, 0] = 0 if st["h0"] is None else st["h0"].double()
    dz = torch.cat([a * na * (h - v) * g, na * g], dim=2)
    return [dz] if st["h0"] is None else [dz, c]


def _exact_norm(x, kind):
    x = x - x.mean(1, keepdim=True) if kind == LAYER else x
    return x / torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind.startswith("scan"):
        return _exact_scan(case, st)
    if kind == "adamw":
        lr, b1, omb1, b2, omb2, eps, c1, c2, scale = _scalars(st)
        g = st["g"].double() * scale
        if case["bits"] == 32:
            m, v = st["m"].double(), st["v"].double()
        else:
            m, v = (x.reshape(-1).double() for x in _unpack8(st["state"]))
        m, v = b1 * m + omb1 * g, b2 * v + omb2 * g ** 2
        w = st["w"].double()
        w = w - lr * st["decay"].double().repeat_interleave(64) * w - lr * (m / c1) / ((v / c2) ** 0.5 + eps)
        return [w, m, v] if case["bits"] == 32 else [w, None, None]          # which neighbour a state is rounded to has no value in 64 bits
    # norms: the gradients come from the formula of the forward pass alone
    names = {"norm": ("x", "gamma", "beta"), "residual_fwd": ("x", "gate", "res", "gamma", "scale", "gamma2", "beta2")}
    leaf = {k: st[k].double().requires_grad_(kind != "residual_fwd") for k in names["norm" if kind == "norm" else "residual_fwd"]}
    n = _exact_norm(leaf["x"], case["norm"])
    if kind == "norm":
        y = n * leaf["gamma"] + leaf["beta"]
        return [y.detach(), *torch.autograd.grad(y, [leaf["x"], leaf["gamma"], leaf["beta"]], st["dy"].double())]
    g = leaf["gate"]
    q = {NONE: lambda: g, RELU: lambda: g.clamp(min=0), SIGMOID: lambda: 1 / (1 + torch.exp(-g)),
         TANH: lambda: torch.tanh(g), SILU: lambda: g / (1 + torch.exp(-g))}[case["act"]]()
    out = leaf["scale"] * leaf["res"] + q * n * leaf["gamma"]
    y = _exact_norm(out, case["next"]) * leaf["gamma2"] + leaf["beta2"]
    if kind == "residual_fwd":
        return [out, y]
    return list(torch.autograd.grad([out, y], [leaf[k] for k in ("x", "gate", "res", "gamma", "scale", "gamma2", "beta2")],
                                    [st["dout"].double(), st["dy"].double()]))
