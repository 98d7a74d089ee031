"""The gated scan against 64 bits on both sides of where its forms change: steps by a thread a state or split, a block or a cluster a tile."""
import numpy as np
import pytest

import test_gpu_gated_scan as base

pytestmark = pytest.mark.gpu
D = base.D
# one sequence: few steps; about a round of blocks, and more than one, around 4 and 9 steps a round; tiles just below and at the places of a round
SHAPES = [(1, 2, 512), (1, 3, 512), (1, 4, 512), (1, 5, 512), (1, 9, 512), (16, 8, 333), (300, 7, 33), (300, 8, 33), (300, 18, 33), (300, 19, 33), (64, 13, 1024), (64, 14, 1024),
          (64, 28, 1024), (64, 62, 1024), (64, 63, 1024), (295, 200, 32), (296, 200, 32), (297, 200, 31), (148, 130, 64)]


@pytest.mark.parametrize("N,T,C", SHAPES)
@pytest.mark.parametrize("state,ragged", [(False, False), (True, True)])
def test_forward(D, N, T, C, state, ragged):
    base.test_forward(D, N, T, C, state, ragged)


@pytest.mark.parametrize("N,T,C", SHAPES)
@pytest.mark.parametrize("state,ragged,given", [(True, True, "both"), (False, False, "dlast")])
def test_backward(D, N, T, C, state, ragged, given):
    base.test_backward(D, N, T, C, state, ragged, given)


def test_parts_of_a_sequence_are_the_whole(D):
    """Parts of lengths that take different forms, each from the state of the one before, within a few roundings of the whole."""
    Dev, capi = D
    N, T, C = 2, 900, 96
    r = np.random.RandomState(0)
    f, v = (r.standard_normal((N, T, C)).astype(np.float32) for _ in range(2))
    with Dev() as d:
        h, last = d.new(N * T * C), d.new(N * C)
        capi.check(d.L.seera_gated_scan_fwd(d.up(f), d.up(v), C, None, None, h, last, N, T, C))
        whole = d.down(h, (N, T, C))
        s, t, parts = d.up(np.zeros((N, C), np.float32)), 0, []
        for k in (1, 2, 3, 4, 5, 8, 17, 60, 100, 700):
            part = d.new(N * k * C)
            capi.check(d.L.seera_gated_scan_fwd(d.up(f[:, t:t + k]), d.up(v[:, t:t + k]), C, s, None, part, s, N, k, C))
            parts.append(d.down(part, (N, k, C)))
            t += k
        assert t == T
        got = np.concatenate(parts, 1)
        assert np.abs(got - whole).max() <= 2.0 ** -19 * np.abs(whole).max()          # gates near 1/2: a state is off by few roundings, which fade
        # (the state comes from runs of steps, the outputs from steps: the same sums in another order)
        assert np.abs(d.down(s, (N, C)) - parts[-1][:, -1]).max() <= 2.0 ** -19 * np.abs(whole).max()
