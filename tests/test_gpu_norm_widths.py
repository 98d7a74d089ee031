"""Norms and residual ends against 64 bits at the widths where a row's threads change."""
import pytest

import sequence_np as ref
import test_gpu_norms as base

pytestmark = pytest.mark.gpu
D = base.D
THREADS = (32, 64, 96, 128, 160, 192, 256, 320, 416, 512)
SHAPES = [(rows, 8 * t + more) for t in THREADS for rows, more in ((7, -1), (450, 0), (4, 1), (11, 4))]


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("kind", [ref.RMS, ref.LAYER])
def test_norm(D, rows, C, kind):
    base.test_norm(D, rows, C, kind)


@pytest.mark.parametrize("rows,C", SHAPES)
@pytest.mark.parametrize("kind,act,kind2", [(ref.RMS, ref.SILU, ref.LAYER), (ref.LAYER, ref.TANH, ref.RMS)])
def test_residual(D, rows, C, kind, act, kind2):
    base.test_residual(D, rows, C, kind, act, kind2)
