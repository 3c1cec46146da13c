"""Page tables that name pages which do not exist: what is reported, whose rows are NaN, and whose are not."""
import numpy as np
import pytest

import tensorax_b200 as ts
from conftest import seeded
from tensorax_b200 import _C, _lib
from tensorax_b200.nn import QuantizedKVCache

pytestmark = pytest.mark.gpu


def tensor(x):
    return ts.Tensor._wrap(_C.from_numpy(np.ascontiguousarray(x)))


def filled(B, S, d, page, fmt):
    """A cache of B sequences of S keys, one K/V head, and its page table."""
    table_len = S // page
    table = np.random.default_rng(1).permutation(B * table_len).reshape(B, table_len).astype(np.int32)
    cache = QuantizedKVCache(B * table_len, 1, d, page, fmt)
    cache.write(tensor(seeded(2, B, 1, S, d)), tensor(seeded(3, B, 1, S, d)), table)
    return cache, table


def finish_reports():
    with pytest.raises(RuntimeError, match="does not exist"):
        _lib.check(_lib.load().tx_sdpa_finish(None))
    _lib.check(_lib.load().tx_sdpa_finish(None))                  # once


@pytest.mark.parametrize("entry", [-1, -2, -3, -2 ** 31, "pages", 2 ** 31 - 1])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads", [1, 30, 40])                    # 2, 60 and 80 rows a K/V head
def test_every_entry_outside_the_cache_is_reported(heads, fmt, entry):
    """In the first, a middle and the last page of a sequence."""
    B, S, d, page = 1, 320, 64, 16
    cache, table = filled(B, S, d, page, fmt)
    q = tensor(seeded(4, B, heads, 2, d).astype(np.float16))
    good = cache.attend(q, table, [S]).numpy()
    for place in (0, 9, 19):
        bad = table.copy()
        bad[0, place] = cache.num_pages if entry == "pages" else entry
        out = cache.attend(q, bad, [S], sync=False)
        finish_reports()
        assert np.isnan(out.numpy()).all(), place
        with pytest.raises(RuntimeError, match="does not exist"):
            cache.read(bad, S)
        kv = tensor(seeded(2, B, 1, S, d)), tensor(seeded(3, B, 1, S, d))
        with pytest.raises(RuntimeError, match="does not exist"):
            cache.write(*kv, bad)
    assert np.array_equal(cache.attend(q, table, [S]).numpy(), good)
