"""Norms over many rows a block, which are loaded while the row before is worked on, against the same rows a few at a time: what belongs to a row is the same
bits, and the sums over the rows are those of 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
# every width of a block, whole vectors and single words; enough rows for more than four a block of any of them (at most 16 blocks of 8 rows or 32 of one an SM)
WIDTHS = [(64, 80000), (255, 80000), (500, 20000), (513, 20000), (767, 20000), (768, 20000), (1000, 20000), (1279, 10000), (1280, 10000), (1536, 10000), (2047, 8000), (2048, 8000), (2559, 6000), (2560, 6000), (3300, 6000), (4095, 6000),
          (4096, 6000)]


@pytest.mark.parametrize("C,rows", WIDTHS)
@pytest.mark.parametrize("kind", [0, 1])
def test_rows_of_many_are_those_of_a_few(C, rows, kind):
    import torch
    from ml_framework_b200 import seera_cuda as sc
    sc.init(0)
    gen = torch.Generator(device="cuda").manual_seed(C + kind)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    u, gate, res, dout, dy = (new(rows, C) for _ in range(5))
    gamma, scale, gamma2, beta2 = (1 + 0.2 * new(C) for _ in range(4))
    torch.cuda.synchronize()

    def run(a, b, sums):
        """Rows a .. b - 1: y, dx of the norm; out, y, du, dgate, dres of the residual end; the sums over the rows."""
        n = b - a
        at = lambda t: t.data_ptr() + 4 * a * C  # noqa: E731
        o = [torch.empty(n, C, device="cuda") for _ in range(7)]
        st, st4 = torch.empty(n, 2, device="cuda"), torch.empty(n, 4, device="cuda")
        p = [t.data_ptr() for t in o]
        s = [t.data_ptr() for t in sums]
        torch.cuda.synchronize()
        sc.norm_fwd(at(u), gamma.data_ptr(), beta2.data_ptr(), p[0], st.data_ptr(), n, C, kind, 1e-5)
        sc.norm_bwd(at(dy), at(u), gamma.data_ptr(), st.data_ptr(), p[1], s[0], s[1], n, C, kind)
        sc.gated_residual_fwd(at(u), at(gate), C, at(res), gamma.data_ptr(), scale.data_ptr(), p[2], gamma2.data_ptr(), beta2.data_ptr(), p[3], st4.data_ptr(), n, C,
                              kind, 4, 1 - kind, 1e-5, 1e-5)
        sc.gated_residual_bwd(at(dout), at(dy), at(u), at(gate), C, at(res), gamma.data_ptr(), scale.data_ptr(), gamma2.data_ptr(), st4.data_ptr(), p[4], p[5], C, p[6],
                              s[2], s[3], s[4], s[5], n, C, kind, 4, 1 - kind)
        sc.stream_synchronize()
        return o
    sums, again, few = ([torch.empty(C, device="cuda") for _ in range(6)] for _ in range(3))
    whole = run(0, rows, sums)
    twice = run(0, rows, again)
    assert all(torch.equal(a, b) for a, b in zip(whole + sums, twice + again))
    step = 148
    for a in range(0, rows, 40 * step):                     # a part in 40: a block has one row of it, or a warp
        b = min(a + step, rows)
        for x, y in zip(whole, run(a, b, few)):
            assert torch.equal(x[a:b], y)
    # the sums over the rows: of the terms in 64 bits, to which a few roundings of each and of at most 100 + rows / 148 additions come
    x, g, r, d, e = (t.double() for t in (u, gate, res, dout, dy))

    def moments(x, kind, eps=1e-5):
        mu = x.mean(1, keepdim=True) if kind else 0.0
        s = 1 / torch.sqrt(((x - mu) ** 2).mean(1, keepdim=True) + eps)
        return (x - mu) * s, s
    n, _ = moments(x, kind)
    q = g * torch.sigmoid(g)
    out = scale.double() * r + q * gamma.double() * n
    n2, s2 = moments(out, 1 - kind)
    a = e * gamma2.double()
    d = d + s2 * (a - (a.mean(1, keepdim=True) if 1 - kind else 0.0) - n2 * (a * n2).mean(1, keepdim=True))
    for got, term in zip(sums, (e * n, e, d * q * n, d * r, e * n2, e)):
        assert ((got.double() - term.sum(0)).abs() <= (160 + rows / 148) * U * term.abs().sum(0)).all()
