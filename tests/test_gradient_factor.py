"""The factor of the fp16 modes' gradient copies on residual trunks of Dense layers, where the gradient past a block may be larger or smaller than the one
through its norm by any factor."""
import numpy as np
import pytest

from test_host_logic_cpu import host  # noqa: F401  (fixture)

ROWS, IN, U, OUT = 24, 10, 32, 20


def build(S, size, norm="rms", gamma=1.0):
    """Two blocks on a trunk whose rows are of the given size: Dense -> [norm -> Dense -> residual end -> Dense] twice -> norm -> Dense."""
    np.random.seed(0)
    Norm = S.RMSNorm if norm == "rms" else S.LayerNorm
    layers = [S.Input((IN,)), S.Dense(IN, U, "relu")]
    for _ in range(2):
        trunk = layers[-1]
        layers += [Norm(U), S.Dense(U, U, activation="tanh"), S.GatedResidual(U, residual=trunk, norm=norm), S.Dense(U, U, "relu")]
    model = S.Sequential(layers + [Norm(U), S.Dense(U, OUT, "sigmoid")])
    first = model.param_layers[0]
    w, b = (p.to_numpy() for p in first.get_weights())
    first.set_weights(w * np.float32(size / np.clip(size, 1, 8)), b)
    for l in model.param_layers:                     # a small gamma makes a block's part small beside the trunk too
        if isinstance(l, (Norm, S.GatedResidual)):
            g, b = (p.to_numpy() for p in l.get_weights())
            l.set_weights(g * np.float32(gamma if isinstance(l, Norm) else min(gamma, 1)), b)
    return model


def data(size=1.0):
    r = np.random.RandomState(1)
    return (r.standard_normal((ROWS, IN)) * np.clip(size, 1, 8)).astype(np.float32), r.standard_normal((ROWS, OUT)).astype(np.float32)


CASES = [(1.0, "rms", 1.0), (3e4, "rms", 1.0), (3e4, "layer", 1.0), (1e-4, "rms", 1.0), (1.0, "rms", 1e-5), (100.0, "layer", 1e3),
         (300.0, "rms", 1.0), (300.0, "layer", 1.0), (100.0, "layer", 100.0), (1500.0, "rms", 1.0), (1500.0, "layer", 0.01)]
# Against 64 bits: tanh's and the sigmoid's slopes are formed from their outputs, 1 - y^2 and y (1 - y), with an absolute error of 2^-24, which is all there is of them where
# gamma n passes 17 (e^-17 = 4e-8): no gammas above 1.
COMPARED = [c for c in CASES if c[2] <= 1]
# Mode 4 holds weights up to 65504 / 256 = 255.9 and activations up to 65504 / 16 = 4094 (its documented ranges): rows of 3e4 are outside.
IN_RANGE = [c for c in COMPARED if c[0] < 2000]


@pytest.mark.parametrize("size,norm,gamma", CASES)
def test_factor_is_that_of_the_gradient_that_is_copied(host, monkeypatch, size, norm, gamma):
    """Mode 4: 256 times the entry that the factor was taken from is fp16's end; two copies hold entries down to some 2^-20 of it."""
    S, fake = host.seera, host.fake
    largest = lambda p, n: float(np.abs(fake.to_host_f32(p, (n,))).max())  # noqa: E731
    seen, now = [], [None]
    product = fake.matmul_act_bwd

    def take(p, n):
        now[0] = largest(p, n)

    def matmul_act_bwd(A, B, y, g, dA, dB, db, M, N, K, *more):
        seen.append(largest(g, M * N) / now[0])
        return product(A, B, y, g, dA, dB, db, M, N, K, *more)
    monkeypatch.setattr(fake, "get_precision", lambda: 4)
    monkeypatch.setattr(fake, "grad_scale_update", take)
    monkeypatch.setattr(fake, "grad_scale_of_loss", take)
    monkeypatch.setattr(fake, "matmul_act_bwd", matmul_act_bwd)
    X, Y = data(size)
    S.autograd4nn(S.Loss().mse(build(S, size, norm, gamma).forward(X), S.Tensor(Y, is_leaf=True)))
    assert len(seen) == 6
    assert max(seen) < 250 and min(seen) > 2.0 ** -8, seen


def test_a_pass_without_such_layers_sets_it_once(host, monkeypatch):
    S, fake = host.seera, host.fake
    calls = []
    monkeypatch.setattr(fake, "get_precision", lambda: 4)
    for name in ("grad_scale_update", "grad_scale_of_loss"):
        monkeypatch.setattr(fake, name, lambda p, n, name=name: calls.append(name))
    X, Y = data()
    np.random.seed(0)
    model = S.Sequential([S.Input((IN,)), S.Dense(IN, U, "tanh"), S.Dense(U, U, "relu"), S.Dense(U, OUT, "sigmoid")])
    S.autograd4nn(S.Loss().mse(model.forward(X), S.Tensor(Y, is_leaf=True)))
    assert calls == ["grad_scale_of_loss"]


@pytest.mark.gpu
@pytest.mark.parametrize("mode,tol,size,norm,gamma", [(3, 2e-5, *c) for c in COMPARED] + [(4, 2e-3, *c) for c in IN_RANGE])
def test_gradients_against_64_bits(mode, tol, size, norm, gamma):
    """Products of at most 32 terms, six of them one after the other: fp32-class in mode 3; mode 4 forms weight gradients from one fp16 copy each, 2^-12 of an entry."""
    import torch
    from ml_framework_b200 import seera as S, seera_cuda as sc
    sc.init(0)
    sc.set_precision(mode)
    try:
        model = build(S, size, norm, gamma)
        X, Y = data(size)
        for _ in range(2):
            loss = S.Loss().mse(model.forward(X), S.Tensor(Y, is_leaf=True))
            model.zero_grad()
            S.autograd4nn(loss)
        P = [[torch.tensor(p.to_numpy().astype(np.float64), requires_grad=True) for p in l.get_weights()] for l in model.param_layers]
        it = iter(P)
        values = []

        def dense(x, act):
            p = next(it)
            values.append(act(x @ p[0] + p[1]))
            return values[-1]

        def n(x, eps):
            mu = x.mean(-1, keepdim=True) if norm == "layer" else 0.0
            return (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + eps)
        eps = 1e-6 if norm == "rms" else 1e-5
        x = dense(torch.tensor(X, dtype=torch.float64), torch.relu)
        for _ in range(2):
            p = next(it)
            h = dense(n(x, eps) * p[0] + p[1], torch.tanh)
            p = next(it)
            x = dense(p[1] * x + p[0] * n(h, 1e-6), torch.relu)
        p = next(it)
        ((dense(n(x, eps) * p[0] + p[1], torch.sigmoid) - torch.tensor(Y, dtype=torch.float64)) ** 2).mean().backward()
        assert mode != 4 or max(float(v.detach().abs().max()) for v in values) < 4094
        for l, p in zip(model.param_layers, P):
            for t, q in zip((l.weights, l.bais), p):
                want = q.grad.numpy()
                off = np.linalg.norm(t.grad.to_host_f32().reshape(want.shape) - want) / np.linalg.norm(want)
                assert off < tol, (l, off)
    finally:
        sc.set_precision(3)
