"""Gradients of rows that see one key or few, where dS is what is left of a difference."""
import numpy as np
import pytest

import window_oracle
from conftest import seeded
from test_window_gpu import gradients

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("Hkv", [1, 2])
def test_rows_of_one_key(Hkv, d):
    """A window of one key: the weight is 1, O = V, and dS = dO V - dO O = 0 with the dO that both are formed of.

    O in fp16 is V exactly (the weight's exponential and the sum are the same to 2^-12.5, less than half a step of fp16 however
    they are rounded).  What is left of dS is the sums': d products in a matrix unit, 2^-23 of the sum of their sizes each, and d in
    fp32, 2^-24 each; two factors of 1 + 2^-12.5 and its rounding to fp16, of which 2^-25 is left near zero.  dQ is one such
    product, dK one for each query head."""
    B, H, S = 1, 2, 700
    q, k, v = (seeded(i, B, (H, Hkv, Hkv)[i], S, d).astype(np.float16) for i in range(3))
    g = seeded(5, B, H, S, d)
    _, (dq, dk, dv) = gradients(q, k, v, g, 1, 0, None, "start", "float32", "float16")
    q, k, v, g = (x.astype(np.float64) for x in (q, k, v, g.astype(np.float16)))
    kk, vv = (np.repeat(x, H // Hkv, 1) for x in (k, v))
    left = ((np.abs(g) * np.abs(vv)).sum(-1) * d * 1.5 * 2.0 ** -23 / np.sqrt(d) * 1.01 + 2.0 ** -25)[..., None]
    assert (np.abs(dq) <= left * np.abs(kk)).all(), (np.abs(dq) / (left * np.abs(kk))).max()
    bound = (left * np.abs(q)).reshape(B, Hkv, H // Hkv, S, d).sum(2)
    assert (np.abs(dk) <= bound * (1 + 2.0 ** -20)).all()
    want = g.reshape(B, Hkv, H // Hkv, S, d).sum(2)
    assert (np.abs(dv - want) <= 2.0 ** -11 * np.abs(g).reshape(B, Hkv, H // Hkv, S, d).sum(2)).all()      # weights in fp16


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("S, window, sinks, lens", [(921, 100, 1, [921, 600]), (700, 40, 0, [300, 650]), (400, 3, 2, [400, 17])])
def test_padded_batches(S, window, sinks, lens, d):
    """The rows behind the last key see fewer and fewer.  P, dS and dO are rounded to fp16 once each, at random: a gradient is a sum of
    products of two of them, off by (2^-11)^2 / 3 per factor in the mean of squares over a binade's rounding errors at most; that is
    2^-11 sqrt(2 / 3) of the root of the sum of their squares, and for dQ and dK dS is a difference whose parts are at most twice the norm
    of what is left here: 2^-10 of the norm."""
    B, H = 2, 4
    q, k, v = (seeded(i, B, (H, 2, 2)[i], S, d).astype(np.float16) for i in range(3))
    g = seeded(5, B, H, S, d)
    want = window_oracle.backward(q, k, v, g, lens, window, sinks, "start")
    _, got = gradients(q, k, v, g, window, sinks, lens, "start")
    for name, a, b in zip("qkv", got, want):
        assert np.linalg.norm(a - b) <= 2.0 ** -10 * np.linalg.norm(b), (name, np.linalg.norm(a - b) / np.linalg.norm(b))
