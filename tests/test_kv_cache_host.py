"""CPU suite of the quantised K/V cache: refusals before any launch, descriptor layouts, the oracle's own rounding."""
import ctypes

import numpy as np
import pytest

import kv_oracle
from tensorax_b200 import _C, _lib

CACHE = dict(k=4096, v=8192, k_scale=64, v_scale=128, pages=8, kv_heads=2, page_size=16, d=64, format=_lib.TX_KV_E4M3)


def write_desc(cache=None, **more):
    return _lib.KvWriteDesc(**{**dict(cache=_lib.KvCache(**{**CACHE, **(cache or {})}), k=16, v=16, page_table=16, batch=2,
                                      tokens=3, table_len=4, dtype=_lib.TX_DTYPE_F16), **more})


def read_desc(cache=None, **more):
    return _lib.KvReadDesc(**{**dict(cache=_lib.KvCache(**{**CACHE, **(cache or {})}), k=16, v=16, page_table=16, batch=2,
                                     tokens=3, table_len=4, dtype=_lib.TX_DTYPE_F32), **more})


def attention_desc(cache=None, **more):
    return _lib.KvAttentionDesc(**{**dict(cache=_lib.KvCache(**{**CACHE, **(cache or {})}), q=16, out=16, page_table=16,
                                          kv_lens=16, batch=2, q_heads=4, tokens=3, table_len=4, dtype=_lib.TX_DTYPE_F16), **more})


CALLS = {"write": ("tx_kv_cache_write", write_desc), "read": ("tx_kv_cache_read", read_desc),
         "attention": ("tx_kv_cache_attention", attention_desc)}
INVALID, UNSUPPORTED = 1, 5
BAD_CACHE = [
    (dict(k=None), INVALID, b"null"), (dict(v_scale=None), INVALID, b"null"), (dict(k=4097), INVALID, b"aligned"),
    (dict(k_scale=66), INVALID, b"aligned"), (dict(pages=0), INVALID, b"positive"), (dict(kv_heads=0), INVALID, b"positive"),
    (dict(d=96), UNSUPPORTED, b"head dim"), (dict(page_size=8), INVALID, b"power of two"), (dict(page_size=48), INVALID, b"power of two"),
    (dict(format=2), INVALID, b"format"), (dict(pages=2 ** 31), UNSUPPORTED, b"too large"),
    (dict(page_size=65536), None, b""),
]
BAD = {
    "write": [(dict(k=None), INVALID, b"null"), (dict(page_table=None), INVALID, b"null"), (dict(v=24), INVALID, b"aligned"),
              (dict(batch=0), INVALID, b"positive"), (dict(tokens=0), INVALID, b"positive"), (dict(dtype=7), INVALID, b"dtype"),
              (dict(flags=1), INVALID, b"flags"), (dict(src_tokens=2), INVALID, b"fewer rows"),
              (dict(table_len=2 ** 28), UNSUPPORTED, b"too large"), (dict(src_tokens=2, rows=16), None, b"")],
    "read": [(dict(v=None), INVALID, b"null"), (dict(k=20), INVALID, b"aligned"), (dict(tokens=-1), INVALID, b"positive"),
             (dict(table_len=0), INVALID, b"positive"), (dict(flags=4), INVALID, b"flags")],
    "attention": [(dict(q=None), INVALID, b"null"), (dict(kv_lens=None), INVALID, b"null"), (dict(out=8), INVALID, b"aligned"),
                  (dict(tokens=65), UNSUPPORTED, b"64"), (dict(tokens=0), UNSUPPORTED, b"64"), (dict(q_heads=5), INVALID, b"multiple"),
                  (dict(window=-1), INVALID, b"negative"), (dict(sinks=-1), INVALID, b"negative"), (dict(window=2), INVALID, b"hold"),
                  (dict(flags=1), INVALID, b"flags"), (dict(tree=12), INVALID, b"aligned"), (dict(window=2 ** 40), None, b"")],
}


def refusal(name, desc):
    lib = _lib.load()
    return getattr(lib, CALLS[name][0])(ctypes.byref(desc)), lib.tx_last_error()


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.skipif(_lib.cuda_is_available(), reason="descriptors hold no real pointers")
def test_refusals(name):
    make = CALLS[name][1]
    assert getattr(_lib.load(), CALLS[name][0])(None) == INVALID
    for cases, build in ((BAD_CACHE, lambda more: make(cache=more)), (BAD[name], lambda more: make(**more))):
        for more, want, words in cases:
            rc, message = refusal(name, build(more))
            if want is None:
                assert rc == 2 and b"no CUDA device" in message, more        # taken, but for the missing device
            else:
                assert rc == want and words in message, (more, rc, message)


def test_descriptor_layouts():
    cache = 4 * 8 + 4 * 8 + 2 * 4
    assert ctypes.sizeof(_lib.KvCache) == cache
    assert ctypes.sizeof(_lib.KvWriteDesc) == cache + 6 * 8 + 4 * 8 + 2 * 4 + 8
    assert ctypes.sizeof(_lib.KvReadDesc) == cache + 5 * 8 + 3 * 8 + 2 * 4 + 8
    assert ctypes.sizeof(_lib.KvAttentionDesc) == cache + 6 * 8 + 6 * 8 + 2 * 4 + 8


def test_python_layer_refuses():
    for bad in (dict(format="fp8"), dict(page_size=24), dict(page_size=8), dict(d=80), dict(pages=0)):
        with pytest.raises(RuntimeError, match="K/V cache"):
            _C.KvCacheImpl(**{**dict(pages=4, kv_heads=2, page_size=16, d=64, format="int8"), **bad})
    for bad in ([2 ** 31], [0.5], np.array([-1.0])):
        with pytest.raises(RuntimeError, match="index array"):
            _C.IndexImpl(bad)
    with pytest.raises(RuntimeError, match=r"start must have shape \[3\]"):
        _C.index_array([1, 2], (3,), "K/V cache write", "start")


def test_oracle_rounds_to_the_nearest_code():
    """The table of values against the format's definition, and against every code's neighbours."""
    assert kv_oracle.E4M3[1] == 2.0 ** -9 and kv_oracle.E4M3[8] == 2.0 ** -6 and kv_oracle.E4M3[126] == 448.0
    assert (np.diff(kv_oracle.E4M3) > 0).all()
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 64)) * np.exp(rng.standard_normal((50, 1)) * 8)).astype(np.float32)
    x[0], x[1, 3], x[2, 5] = 0, np.nan, np.inf
    for fmt in ("e4m3", "int8"):
        codes, scales = kv_oracle.quantise(x, fmt)
        back = kv_oracle.values(codes, scales, fmt)
        assert np.isnan(back[1:3]).all() and (back[0] == 0).all()
        fine = np.r_[0, 3:50]
        amax = np.abs(x[fine]).max(-1, keepdims=True)
        # half a step: 1/254 of the row's largest, or 2^-4 of the value (2^-10 of the scale where codes are subnormal)
        half = amax / 254 * 1.0000002 if fmt == "int8" else np.maximum(np.abs(x[fine]) * 2.0 ** -4, scales[fine, None] * 2.0 ** -10)
        assert (np.abs(back[fine] - x[fine]) <= half).all()
        if fmt == "e4m3":
            assert (scales[fine[1:]] * 448 >= amax[1:, 0]).all() and (scales[fine[1:]] * 224 < amax[1:, 0]).all()
