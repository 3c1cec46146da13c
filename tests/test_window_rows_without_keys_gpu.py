"""Rows that see no key, as a padded batch's next layer has them: their result was NaN, and so is what was computed from it."""
import numpy as np
import pytest

import window_oracle
from conftest import seeded
from test_window_gpu import gradients

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("Hkv", [1, 2])
@pytest.mark.parametrize("lens, window, align, sinks", [
    ([200, 700], 64, "start", 0),                # behind the last key's window, from the middle of a tile on
    ([1, 129], 1, "start", 0),                   # all rows but one; the diagonal
    ([300, 0], 64, "end", 0),                    # in front of the first key; a sequence without keys
    ([300, 699], 64, "end", 2),                  # ... with a few sinks
    ([690, 128], 64, "end", 20),                 # ... and with many
    ([350, 40], 500, "end", 3),                  # a window longer than the sequence
])
def test_their_queries_are_not_read(lens, window, align, sinks, Hkv, d):
    """NaN and infinities in the rows' queries and in the gradient of their result: the others' gradients are the same bits."""
    B, H, S = 2, 2, 700
    q, k, v = (seeded(i, B, (H, Hkv, Hkv)[i], S, d).astype(np.float16) for i in range(3))
    g = seeded(5, B, H, S, d)
    _, clean = gradients(q, k, v, g, window, sinks, lens, align)
    dead = np.stack([~window_oracle.seen(S, S, n, window, sinks, align).any(1) for n in lens])
    assert dead.any() and not dead.all()
    for b in range(B):
        q[b][:, dead[b]] = np.nan
        q[b][:, np.flatnonzero(dead[b])[::3]] = np.inf
        g[b][:, dead[b]] = np.nan
    for grad_dtype in ("float32", "float16"):
        out, got = gradients(q, k, v, g, window, sinks, lens, align, grad_dtype)
        assert all(np.isnan(out[b][:, dead[b]]).all() and np.isfinite(out[b][:, ~dead[b]]).all() for b in range(B))
        for name, a, b in zip("qkv", got, clean):
            assert np.isfinite(a).all(), name
            assert np.array_equal(a, b.astype(a.dtype)), name
