"""CPU suite of attention with a sliding window: refusals before any launch, the layers' checks, the oracle's gradients against
differences of its forward pass."""
import ctypes

import numpy as np
import pytest

import tensorax_b200 as ts
import tensorax_b200.functional as F
import window_oracle
from tensorax_b200 import _C, _lib
from tensorax_b200.nn import GroupedQueryAttention


def forward_desc(**more):
    return _lib.SdpaDesc(**{**dict(q=16, k=16, v=16, out=16, batch=1, q_heads=4, kv_heads=2, seq_q=8, seq_k=8, d_k=64, d_v=64,
                                   dtype=_lib.TX_DTYPE_F16, causal=1), **more})


def backward_desc(**more):
    return _lib.SdpaBwdDesc(**{**dict(q=16, k=16, v=16, out=16, dout=16, lse=16, dq=16, dk=16, dv=16, batch=1, q_heads=4,
                                      kv_heads=2, seq_q=8, seq_k=8, d=64, causal=1), **more})


@pytest.mark.skipif(_lib.cuda_is_available(), reason="descriptors hold no real pointers")
def test_refusals():
    lib = _lib.load()

    def forward(desc, **window):
        rc = lib.tx_sdpa_window_forward(ctypes.byref(desc), ctypes.byref(_lib.WindowDesc(**{"window": 4, **window})))
        return rc, lib.tx_last_error()

    def backward(desc, **window):
        rc = lib.tx_sdpa_window_backward(ctypes.byref(desc), ctypes.byref(_lib.WindowDesc(**{"window": 4, **window})))
        return rc, lib.tx_last_error()

    for call, desc in ((forward, forward_desc()), (backward, backward_desc())):
        assert call(desc)[0] == 2                                    # taken, but for the missing device
        assert call(desc, window=2 ** 50, sinks=2 ** 50, align_end=1)[0] == 2
        for bad in (dict(window=0), dict(window=-1), dict(sinks=-1)):
            assert call(desc, **bad)[0] == 1 and b"window" in call(desc, **bad)[1]
        assert call(desc, align_end=2)[0] == 1
    assert forward(forward_desc(causal=0))[0] == 1 and forward(forward_desc(mask=16))[0] == 1
    assert forward(forward_desc(flags=_lib.TX_SDPA_F32_VIA_F16))[0] == 1 and forward(forward_desc(flags=_lib.TX_SDPA_P_IN_SMEM))[0] == 1
    assert forward(forward_desc(kv_heads=3))[0] == 1
    assert backward(backward_desc(causal=0))[0] == 1 and backward(backward_desc(flags=_lib.TX_SDPA_FORCE_SIMT))[0] == 1
    assert backward(backward_desc(d=32))[0] == 5
    assert lib.tx_sdpa_window_forward(ctypes.byref(forward_desc()), None) == 1
    assert lib.tx_sdpa_window_backward(ctypes.byref(backward_desc()), None) == 1
    assert lib.tx_sdpa_window_forward(None, ctypes.byref(_lib.WindowDesc(window=1))) == 1


def test_descriptor_layout():
    assert ctypes.sizeof(_lib.WindowDesc) == 24


def test_python_layer_refuses():
    q = ts.Tensor.randn((1, 2, 4, 64))
    with pytest.raises(ValueError, match="4D"):
        F.scaled_dot_product_attention_window(ts.Tensor.randn((2, 4, 64)), q, q, 3)
    with pytest.raises(ValueError, match="grad_dtype"):
        F.scaled_dot_product_attention_window(q, q, q, 3, grad_dtype="int8")
    for bad in (dict(window=0), dict(window=3, sinks=-1), dict(window=3, align="middle")):
        with pytest.raises(RuntimeError, match="SDPA window"):
            _C.window_desc(**bad)
    with pytest.raises(RuntimeError, match="CUDA path only"):
        F.scaled_dot_product_attention_window(q, q, q, 3)
    layer = GroupedQueryAttention(2, 1)
    with pytest.raises(ValueError, match="head counts"):
        layer.forward_bhsd(q, q, q, window=3)
    with pytest.raises(ValueError, match="no dense mask"):
        layer.forward_bhsd(q, ts.Tensor.randn((1, 1, 4, 64)), ts.Tensor.randn((1, 1, 4, 64)), mask=q, window=3)


@pytest.mark.parametrize("align,window,sinks,n", [("start", 3, 1, 7), ("end", 4, 0, 6), ("start", 2, 0, 4)])
def test_oracle_gradients_against_differences(align, window, sinks, n):
    """Central differences of the oracle's forward pass; rows that see nothing (the last case has some) are left out."""
    rng = np.random.default_rng(0)
    x = [rng.standard_normal(s) for s in ((1, 2, 7, 4), (1, 1, 7, 4), (1, 1, 7, 4))]
    g = rng.standard_normal((1, 2, 7, 4))

    def loss():
        return np.nansum(window_oracle.forward(*x, [n], window, sinks, align) * g)

    for t, grad in zip(x, window_oracle.backward(*x, g, [n], window, sinks, align)):
        for i in np.ndindex(t.shape):
            old, h = t[i], 1e-5
            t[i] = old + h
            up = loss()
            t[i] = old - h
            down = loss()
            t[i] = old
            # differences are off by h^2 times a third derivative (of order 1) and 1e-16 / h
            assert abs((up - down) / (2 * h) - grad[i]) < 1e-8
