"""Attention over the cache at the number of rows a K/V head from which the fifth-generation tensor cores take the call: more than
32 with e4m3 codes, more than 64 with int8."""
import numpy as np
import pytest

from conftest import seeded
from test_kv_cache_gpu import check_attention, filled, tensor, words_of

pytestmark = pytest.mark.gpu

CASES = [
    # B, Hq, Hkv, T, S, page, q_lens, window, sinks, shape
    (1, 4, 1, 8, 2000, 16, None, None, 0, "tree"),               # 32
    (1, 32, 1, 1, 1500, 64, None, None, 0, "chain"),             # 32: one token of many heads
    (2, 3, 1, 11, 1300, 32, [11, 4], None, 0, "chain"),          # 33
    (1, 33, 1, 1, 3000, 128, None, 700, 3, "chain"),             # 33
    (2, 12, 2, 7, 2500, 64, [7, 2], 900, 5, "tree"),             # 42, two K/V heads
    (1, 3, 1, 16, 1100, 16, None, 200, 150, "tree"),             # 48, more than a tile of sinks
    (2, 2, 1, 32, 4000, 64, [32, 17], None, 0, "tree"),          # 64
    (1, 16, 1, 4, 2500, 16, None, 1000, 4, "tree"),              # 64
    (2, 13, 1, 5, 2222, 32, [5, 0], 600, 17, "chain"),           # 65
    (1, 5, 1, 13, 1025, 16, None, None, 0, "chain"),             # 65, one key in the last share
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_rows_about_the_switch(case, d, fmt):
    B, Hq, Hkv, T, S, page, q_lens, window, sinks, shape = CASES[case]
    cache, table, kv = filled(300 + case, B, Hkv, S, d, page, fmt)
    q = seeded(case, B, Hq, T, d).astype(np.float16)
    nodes = q_lens or [T] * B
    kv_lens = [S - 37 * b for b in range(B)]
    tree, words = words_of(shape, case, B, T)
    many = Hq // Hkv * T > (32 if fmt == "e4m3" else 64)
    for out_dtype in ("float32", "float16"):
        got = cache.attend(tensor(q), table, kv_lens, q_lens=q_lens, tree=tree, window=window, sinks=sinks, out_dtype=out_dtype).numpy()
        check_attention(got, q, kv, kv_lens, nodes, words, window, sinks, False, out_dtype == "float16", fp16_cache=many)
        for b in range(B):
            assert (got[b, :, nodes[b]:] == 0).all()
