"""A small network of gated recurrent blocks, as layers of the front end and as a function in 64 bits (torch autograd), for the tests on the CPU stand-in and
on the device."""
import numpy as np
import torch

N, T, IN, U, CLASSES = 5, 21, 6, 12, 4


def build(S, head="softmax", seed=0, norm="rms", gate="silu"):
    """Two blocks over (N, T, IN): projection to U by a plain recurrence, then [norm, gated recurrence, residual end] twice, then the head."""
    np.random.seed(seed)
    layers = [S.Input((T, IN)), S.GatedRecurrence(IN, U)]
    Norm = S.RMSNorm if norm == "rms" else S.LayerNorm
    for _ in range(2):
        trunk = layers[-1]
        layers += [Norm(U), S.GatedRecurrence(U, U, output_gate=True), S.GatedResidual(U, residual=trunk, activation=gate, norm=norm)]
    layers.append(Norm(U))
    if head == "softmax":
        layers += [S.GatedRecurrence(U, U, return_sequences=False), S.Dense(U, CLASSES, activation="softmax")]
    model = S.Sequential(layers)
    r = np.random.RandomState(seed + 1)
    for l in model.param_layers:                     # norms and scales away from ones and zeros
        w, b = (p.to_numpy() for p in l.get_weights())
        l.set_weights((w + 0.2 * r.standard_normal(w.shape)).astype(np.float32), (b + 0.2 * r.standard_normal(b.shape)).astype(np.float32))
    return model


def data(seed=0, classes=True):
    r = np.random.RandomState(seed)
    X = r.standard_normal((N, T, IN)).astype(np.float32)
    if classes:
        Y = np.eye(CLASSES, dtype=np.float32)[r.randint(0, CLASSES, N)]
    else:
        Y = r.standard_normal((N, T, U)).astype(np.float32)
    return X, Y


def params64(model):
    return [[torch.tensor(p.to_numpy().astype(np.float64), requires_grad=True) for p in l.get_weights()] for l in model.param_layers]


def _norm(x, p, kind):
    mu = x.mean(-1, keepdim=True) if kind == "layer" else 0.0
    eps = 1e-5 if kind == "layer" else 1e-6
    return (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps) * p[0] + p[1]


def _scan(z, units, lengths):
    f, v = z[..., :units], z[..., units:2 * units]
    a = torch.sigmoid(f)
    s, out = torch.zeros(z.shape[0], units, dtype=z.dtype), []
    for t in range(z.shape[1]):
        new = a[:, t] * s + (1 - a[:, t]) * v[:, t]
        on = torch.ones(z.shape[0], 1, dtype=torch.bool) if lengths is None else (torch.as_tensor(np.asarray(lengths)) > t)[:, None]
        s = torch.where(on, new, s)
        out.append(torch.where(on, new, torch.zeros_like(new)))
    return torch.stack(out, 1), s


def forward64(P, X, head="softmax", norm="rms", gate="silu", lengths=None):
    """The network's output (probabilities of the softmax head, or the last norm's output)."""
    it = iter(P)
    x = torch.tensor(X, dtype=torch.float64)
    p = next(it)
    x, _ = _scan(x @ p[0] + p[1], U, lengths)
    act = {"silu": torch.nn.functional.silu, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "relu": torch.relu, None: lambda g: g}[gate]
    for _ in range(2):
        y = _norm(x, next(it), norm)
        p = next(it)
        z = y @ p[0] + p[1]
        h, _ = _scan(z, U, lengths)
        p = next(it)
        mu = h.mean(-1, keepdim=True) if norm == "layer" else 0.0
        n = (h - mu) / torch.sqrt(((h - mu) ** 2).mean(-1, keepdim=True) + 1e-6)
        x = p[1] * x + act(z[..., 2 * U:]) * p[0] * n
    x = _norm(x, next(it), norm)
    if head != "softmax":
        return x
    p = next(it)
    _, last = _scan(x @ p[0] + p[1], U, lengths)
    p = next(it)
    return torch.softmax(last @ p[0] + p[1], -1)


def loss64(out, Y, head="softmax"):
    Y = torch.tensor(Y, dtype=torch.float64)
    if head == "softmax":
        return -(Y * torch.log(out.clamp(1e-7, 1 - 1e-7))).sum(-1).mean()
    return ((out - Y) ** 2).mean()


def check_step(S, tol, head="softmax", norm="rms", gate="silu", lengths=None, seed=0, passes=1):
    """Output, loss and every gradient of one pass against 64 bits; the last of `passes`."""
    model = build(S, head, seed, norm, gate)
    X, Y = data(seed, head == "softmax")
    P = params64(model)
    want = forward64(P, X, head, norm, gate, lengths)
    total = loss64(want, Y, head)
    total.backward()
    L = S.Loss()
    for _ in range(passes):
        out = model.forward(S.Tensor(X, is_leaf=True), lengths=lengths)
        loss = (L.categorical_cross_entropy if head == "softmax" else L.mse)(out, S.Tensor(Y, is_leaf=True))
        model.zero_grad()
        S.autograd4nn(loss)
    rel = lambda a, b: np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30)  # noqa: E731
    assert rel(out.to_numpy(), want.detach().numpy()) < tol
    assert abs(loss.item() - total.item()) < tol * max(1.0, abs(total.item()))
    for l, p in zip(model.param_layers, P):
        for t, q, name in zip((l.weights, l.bais), p, ("weights", "bais")):
            assert rel(t.grad.to_host_f32().reshape(q.shape), q.grad.numpy()) < tol, (l, name)
    return model
