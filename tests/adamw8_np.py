"""The rounding of 8-bit averages whose steps are bounded, as a model for the tests: sequence_np.pack8 with a v above zero held at the smallest code at least."""
import numpy as np

import sequence_np as ref


def pack8_bounded(m, v, step, first=0):
    """The state of one tensor, n entries, rounded with the random bits of `step`."""
    state = ref.pack8(m, v, step, first).reshape(-1, 136)
    codes = state[:, :128].reshape(-1, 16, 2, 4).copy()
    top = np.ascontiguousarray(state[:, 132:]).view(np.float32)
    V = np.zeros(state.shape[0] * 64, np.float32)
    V[:v.size] = v
    least = (V.reshape(-1, 64) > 0) & (top > 0) & np.isfinite(top)
    codes[:, :, 1] = np.maximum(codes[:, :, 1], least.reshape(-1, 16, 4))
    state = state.copy()
    state[:, :128] = codes.reshape(-1, 128)
    return state.reshape(-1)
