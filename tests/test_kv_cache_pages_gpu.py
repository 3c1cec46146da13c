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


@pytest.mark.parametrize("what", ["page", "length"])
@pytest.mark.parametrize("fmt, dtype, d, heads", [("e4m3", np.float16, 64, 1), ("int8", np.float16, 128, 1), ("e4m3", np.float16, 128, 40),
                                                  ("int8", np.float16, 64, 40), ("e4m3", np.float16, 256, 6), ("int8", np.float32, 64, 2)])
def test_other_sequences_have_their_rows(fmt, dtype, d, heads, what):
    """A call of several waves of CTAs in which every seventh sequence names a page that does not exist, or more keys than its table
    has: the others' rows are the same bits as ever, and so are those of calls queued behind it before anyone asks."""
    B, S, page, T = 700, 64, 16, 2
    cache, table = filled(B, S, d, page, fmt)
    q = tensor(seeded(4, B, heads, T, d).astype(dtype))
    want = cache.attend(q, table, [S] * B).numpy()
    assert np.isfinite(want).all()
    wrong = np.arange(B) % 7 == 0
    bad, lens = table.copy(), np.full(B, S)
    if what == "page":
        bad[wrong, 2] = -1
    else:
        lens[wrong] = S + 1
    for _ in range(3):
        got = cache.attend(q, bad, lens, sync=False)
        behind = cache.attend(q, table, [S] * B, sync=False)
        finish_reports()
        got = got.numpy()
        assert np.isnan(got[wrong]).all() and np.array_equal(got[~wrong], want[~wrong])
        assert np.array_equal(behind.numpy(), want)


def test_a_report_of_a_write_or_read_stops_nothing():
    """What was queued behind a write and a read that leave tokens out -- attention over the cache, prompts with and without a
    window, a layer's gradients -- is what it is without them."""
    import tensorax_b200.functional as F
    B, S, d, page = 2, 64, 64, 16
    cache, table = filled(B, S, d, page, "e4m3")
    q = tensor(seeded(4, B, 3, 2, d).astype(np.float16))
    prompt = [_C.from_numpy(seeded(5 + i, 1, 2, 600, d).astype(np.float16)) for i in range(3)]
    grad = tensor(seeded(9, 1, 2, 600, d))

    def behind():
        out = [cache.attend(q, table, [S] * B, sync=False).numpy(),
               _C.to_numpy(_C.scaled_dot_product_attention_ex(*prompt, causal=True, sync=False)),
               _C.to_numpy(_C.scaled_dot_product_attention_window(*prompt, 100, 3, sync=False))]
        leaves = [ts.Tensor._wrap(x, True) for x in prompt]
        result = F.scaled_dot_product_attention_window(*leaves, 100, 3)
        try:
            result.backward(grad)
        except RuntimeError as e:                          # backward waits, and tells what was reported before it
            assert "does not exist" in str(e)
            _lib.check(_lib.load().tx_sdpa_finish(None))
            result = F.scaled_dot_product_attention_window(*leaves, 100, 3)
            result.backward(grad)
        return out + [result.numpy()] + [t.grad.numpy() for t in leaves]

    want = behind()
    kv = tensor(seeded(2, B, 1, S, d)), tensor(seeded(3, B, 1, S, d))
    bad = table.copy()
    bad[1, 3] = 10 ** 6
    for call in (lambda: cache.write(*kv, bad, sync=False), lambda: cache.read(bad, S, sync=False)):
        call()
        got = behind()
        assert all(np.isfinite(x).all() and np.array_equal(x, y) for x, y in zip(got, want))
