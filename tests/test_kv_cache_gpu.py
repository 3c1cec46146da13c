"""The quantised K/V cache on the device against its definition in 64 bits: codes and scales to the bit, values read back, and
attention of one token, chains and trees over it."""
import ctypes

import numpy as np
import pytest

import kv_oracle
import tensorax_b200 as ts
import tensorax_b200.functional as F
from conftest import seeded
from tensorax_b200 import _C, _lib
from tensorax_b200.nn import QuantizedKVCache

pytestmark = pytest.mark.gpu

FORMATS = ["e4m3", "int8"]


def tensor(x):
    return ts.Tensor._wrap(_C.from_numpy(np.ascontiguousarray(x)))


def page_table(seed, pages, B, table_len):
    return np.random.default_rng(seed).permutation(pages)[: B * table_len].reshape(B, table_len).astype(np.int32)


def strong(seed, *shape):
    """Rows of different strength."""
    return seeded(seed, *shape) * np.exp(seeded(seed + 1, *shape[:-1], 1))


# ------------------------------------------------------------------ write, read
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("B,H,T,d,page", [(1, 1, 1, 64, 16), (3, 2, 37, 128, 16), (2, 3, 130, 256, 64)])
def test_write_then_read(B, H, T, d, page, dtype, fmt):
    """Codes and scales are the definition's, everything else stays as it was, and reading gives codes times scales."""
    start = [(7 * b) % 40 for b in range(B)]
    counts = [max(T - 5 * b, 0) for b in range(B)]
    table_len = (40 + T) // page + 1
    pages = B * table_len + 2
    table = page_table(5, pages, B, table_len)
    cache = QuantizedKVCache(pages, H, d, page, fmt)
    for buf in cache._impl._bufs:
        buf.upload(np.full(buf.nbytes, 0x2a, np.uint8))
    kv = [strong(1 + 2 * i, B, H, T, d).astype(dtype) for i in range(2)]
    kv[0][0, 0, 0] = 0
    if T > 6:
        kv[0][0, 0, 1, 3], kv[1][0, 0, 2, 0], kv[1][0, 0, 3, 7] = np.inf, np.nan, -np.inf
        kv[1][0, 0, 4] *= dtype(2e-4 if dtype == np.float16 else 1e-38)          # subnormal numbers among them
        kv[0][0, 0, 5, :2] = 448, -448
    before = cache._impl.to_numpy()
    cache.write(tensor(kv[0]), tensor(kv[1]), table, start, counts)
    codes, scales = cache._impl.to_numpy()
    read = cache.read(table, T, start, counts, dtype=np.dtype(dtype).name)
    for i in range(2):
        want_codes, want_scales = before[0][i].copy(), before[1][i].copy()
        c, f = kv_oracle.quantise(kv[i], fmt)
        for b in range(B):
            pos = start[b] + np.arange(counts[b])
            want_codes[table[b][pos // page], :, pos % page] = c[b, :, : counts[b]].swapaxes(0, 1)
            want_scales[table[b][pos // page], :, pos % page] = f[b, :, : counts[b]].T
        assert np.array_equal(scales[i].view(np.uint32), want_scales.view(np.uint32)) or np.array_equal(scales[i], want_scales, equal_nan=True)
        assert np.array_equal(codes[i], want_codes)
        got = read[i].numpy()
        for b in range(B):
            # the fp32 product, then the type read: |have - want| <= ((1 + 2^-24)(1 + u) - 1) |want|, u half an eps, or half a
            # subnormal step more (in Python's floats: numpy's fp16 ones round u + 2^-24 back to u, and 2^-25 to nothing)
            want = kv_oracle.values(c[b, :, : counts[b]], f[b, :, : counts[b]], fmt)
            have = got[b, :, : counts[b]].astype(np.float64)
            fine = np.isfinite(want)
            assert np.array_equal(np.isnan(have), ~fine)
            half, least = float(np.finfo(dtype).eps) / 2, float(np.finfo(dtype).smallest_subnormal) / 2
            assert (np.abs(have - want)[fine] <= np.abs(want[fine]) * ((1 + 2.0 ** -24) * (1 + half) - 1) + least).all()
            assert (got[b, :, counts[b]:] == 0).all()


def test_rows_pick_the_accepted_nodes():
    """`rows`: the accepted nodes of a tree are written in line, the same node twice if so asked."""
    B, H, T, d, page = 2, 2, 9, 64, 16
    table = page_table(3, 8, B, 2)
    k, v = strong(1, B, H, T, d), strong(5, B, H, T, d)
    rows = np.array([[0, 3, 8], [2, 2, 7]])
    cache = QuantizedKVCache(8, H, d, page, "int8")
    cache.write(tensor(k), tensor(v), cache.indices(table), start=[14, 3], counts=[3, 2], rows=rows)
    got = cache.read(table, 3, start=[14, 3], counts=[3, 2], dtype="float32")
    for x, y in zip((k, v), got):
        for b, n in ((0, 3), (1, 2)):
            picked = x[b][:, rows[b, :n]]
            assert np.array_equal(y.numpy()[b, :, :n], kv_oracle.values(*kv_oracle.quantise(picked, "int8"), "int8").astype(np.float32))


@pytest.mark.parametrize("what", ["page", "negative page", "position", "row"])
def test_what_does_not_exist_is_reported_and_left_out(what):
    B, H, T, d, page = 1, 2, 20, 64, 16
    cache = QuantizedKVCache(4, H, d, page, "e4m3")
    for buf in cache._impl._bufs:
        buf.upload(np.zeros(buf.nbytes, np.uint8))
    table, start, rows = np.array([[1, 2]]), [0], np.arange(T)[None]
    if what == "page":
        table = np.array([[1, 4]])
    elif what == "negative page":
        table = np.array([[1, -1]])
    elif what == "position":
        start = [16]
    else:
        rows = np.where(rows < 16, rows, T)
    k = strong(1, B, H, T, d)
    with pytest.raises(RuntimeError, match="does not exist"):
        cache.write(tensor(k), tensor(k), table, start=start, rows=rows)
    codes, _ = cache._impl.to_numpy()
    there = table[0][start[0] // page]
    assert codes[0][there].any() and not codes[0][[p for p in range(4) if p != there]].any()
    cache.write(tensor(k), tensor(k), [[1, 2]])              # the failure was one call's
    if what in ("page", "negative page"):
        with pytest.raises(RuntimeError, match="does not exist"):
            cache.read(table, T)
        for heads in (1, 40):
            with pytest.raises(RuntimeError, match="does not exist"):
                cache.attend(tensor(seeded(3, B, H * heads, 2, d).astype(np.float16)), table, [T])
    _lib.check(_lib.load().tx_sdpa_finish(None))


@pytest.mark.parametrize("length", [41, 2 ** 31 - 1])
@pytest.mark.parametrize("heads", [1, 40])
def test_more_keys_than_the_page_table_holds(heads, length):
    """Reported, the sequence's rows NaN (the failure is the whole call's: another sequence may or may not have its rows)."""
    B, H, d, page = 2, 1, 64, 16
    cache, table, _ = filled(3, B, H, 32, d, page, "int8")
    q = tensor(seeded(4, B, H * heads, 2, d).astype(np.float16))
    out = cache.attend(q, table, [length, 32], sync=False)
    with pytest.raises(RuntimeError, match="does not exist"):
        _lib.check(_lib.load().tx_sdpa_finish(None))
    assert np.isnan(out.numpy()[0]).all()
    assert np.isfinite(cache.attend(q, table, [32, 32]).numpy()).all()


# ------------------------------------------------------------------ attention
def filled(seed, B, H, S, d, page, fmt, spread=0.5):
    """A cache of S tokens per sequence, its page table, and the values it holds [2][B, H, S, d]."""
    table_len = (S + page - 1) // page
    pages = B * table_len + 1
    table = page_table(seed, pages, B, table_len)
    cache = QuantizedKVCache(pages, H, d, page, fmt)
    kv = [(seeded(seed + 1 + i, B, H, S, d) * np.exp(spread * seeded(seed + 3 + i, B, H, S, 1))).astype(np.float32) for i in range(2)]
    cache.write(tensor(kv[0]), tensor(kv[1]), table)
    return cache, table, [kv_oracle.values(*kv_oracle.quantise(x, fmt), fmt) for x in kv]


def words_of(shape, seed, B, T):
    if shape == "chain":
        return None, np.array([[(2 << t) - 1 for t in range(T)]] * B, dtype=np.uint64)
    rng = np.random.default_rng(seed)
    words = np.zeros((B, T), dtype=object)
    for b in range(B):
        for t in range(T):
            parent = int(rng.integers(max(-1, t - 4), t)) if t else -1
            words[b, t] = (int(words[b, parent]) if parent >= 0 else 0) | 1 << t
    words = words.astype(np.uint64)
    return words, words


def check_attention(got, q, kv, kv_lens, q_lens, words, window, sinks, fp32, out16, fp16_cache=False):
    """Every element within what the roundings of the products can make of it.

    fp16 queries: a weight is rounded to fp16 (2^-11 of it); the score's sum of d products in fp32 may lose 2^-23 of the
    sum of their sizes per addition (matrix units cut off), `e` in all; both the weight and the sum of the weights carry e.
    fp32: a weight is two fp16 numbers (2^-22), so is a query (2^-22 per product).  2^-19: the exponential (2^-22), the
    scales' products and the partial sums.  fp16 results are rounded once more.
    fp16_cache: many rows a head; keys and values times their scales are rounded to fp16 (2^-11 of a product, of a value; an
    element below 2^-14 of 224 in the tile's largest row, to 2^-25 of that: 2^-30 of the largest value), and the exponential may be the
    polynomial one (2^-12.5 in weight and sum).  Weights more than 2^24 (and 2^8 for a maximum not yet raised) below the
    row's largest are lost: with up to 2^10 keys in a tile's row, 2^-7 of that at most here, 2^-17 of the largest value."""
    B, Hq, T, d = q.shape
    G = Hq // kv[0].shape[1]
    for b in range(B):
        n, ctx = q_lens[b], kv_lens[b] - q_lens[b]
        see = kv_oracle.visible(ctx, n, words[b], window, sinks)
        for h in range(Hq):
            want, weight, size = kv_oracle.attention(q[b, h, :n], kv[0][b, h // G, : kv_lens[b]], kv[1][b, h // G, : kv_lens[b]], see)
            have = got[b, h, :n].astype(np.float64)
            assert np.array_equal(np.isnan(have), np.isnan(want)), (b, h)
            e = size * (d * 2.0 ** -23 * (2 if fp32 else 1) + 2.0 ** -22)
            bound = weight * ((2.0 ** -21 if fp32 else 2.0 ** -11) + 2 * e[:, None] + 2.0 ** -19) + 1e-30
            if fp16_cache:
                top = np.abs(kv[1][b, h // G, : kv_lens[b]]).max(initial=0.0)
                bound = bound + weight * (2.0 ** -11 + 2.0 ** -11.5 + 2 * 2.0 ** -11 * size[:, None]) + 2.0 ** -17 * top
            if out16:
                bound = bound + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
            assert (np.abs(have - want) <= bound)[~np.isnan(want)].all(), (b, h, np.nanmax(np.abs(have - want) / bound))


MANY = [
    # as CASES below; more than 64 rows a head: the tcgen05 kernel
    (1, 8, 1, 64, 64, 16, None, None, 0, "tree"),               # two query tiles, no context
    (2, 5, 1, 13, 1, 16, [1, 0], None, 0, "tree"),              # one key; one sequence without nodes
    (2, 3, 1, 23, 300, 32, [23, 7], None, 0, "chain"),          # one query tile, three tiles of keys
    (1, 6, 2, 64, 513, 64, None, 130, 70, "tree"),              # sinks and window apart, nodes over two tiles
    (2, 16, 2, 33, 2000, 128, [33, 12], 700, 5, "tree"),        # two parts of 256 rows
    (1, 4, 1, 64, 4100, 256, None, 3000, 200, "chain"),
    (1, 4, 1, 50, 1030, 16, None, 64, 0, "tree"),
]

CASES = [
    # B, Hq, Hkv, T, S (keys of the longest sequence), page, q_lens, window, sinks, shape
    (1, 1, 1, 1, 1, 16, None, None, 0, "chain"),
    (3, 4, 2, 1, 300, 16, None, None, 0, "chain"),
    (2, 8, 1, 2, 129, 32, None, None, 0, "chain"),
    (2, 4, 2, 5, 700, 64, [5, 2], None, 0, "tree"),
    (2, 6, 2, 9, 1000, 128, [9, 0], 150, 4, "tree"),
    (1, 4, 1, 17, 513, 16, None, 64, 0, "chain"),
    (2, 16, 2, 64, 333, 64, [64, 33], 100, 70, "tree"),
    (1, 2, 2, 64, 64, 16, None, None, 0, "tree"),               # no context at all
    (2, 4, 4, 3, 2050, 256, None, 2000, 1, "tree"),
]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(case, d, dtype, fmt):
    B, Hq, Hkv, T, S, page, q_lens, window, sinks, shape = CASES[case]
    cache, table, kv = filled(100 + case, B, Hkv, S, d, page, fmt)
    q = seeded(case, B, Hq, T, d).astype(dtype)
    nodes = q_lens or [T] * B
    kv_lens = [S - 37 * b if S - 37 * b >= max(nodes[b], 1) else S for b in range(B)]
    tree, words = words_of(shape, case, B, T)
    for out_dtype in ("float32", "float16"):
        out = cache.attend(tensor(q), table, kv_lens, q_lens=q_lens, tree=tree, window=window, sinks=sinks, out_dtype=out_dtype)
        assert out.dtype == out_dtype
        got = out.numpy()
        check_attention(got, q, kv, kv_lens, nodes, words, window, sinks, dtype == np.float32, out_dtype == "float16",
                        fp16_cache=dtype == np.float16 and d <= 128 and Hq // Hkv * T > 64)
        for b in range(B):
            assert (got[b, :, nodes[b]:] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("case", range(len(MANY)))
def test_attention_of_many_rows(case, d, fmt):
    B, Hq, Hkv, T, S, page, q_lens, window, sinks, shape = MANY[case]
    cache, table, kv = filled(200 + case, B, Hkv, S, d, page, fmt)
    q = seeded(case, B, Hq, T, d).astype(np.float16)
    nodes = [min(n, S) for n in (q_lens or [T] * B)]
    kv_lens = [S - 37 * b if S - 37 * b >= max(nodes[b], 1) else S for b in range(B)]
    tree, words = words_of(shape, case, B, T)
    for out_dtype in ("float32", "float16"):
        got = cache.attend(tensor(q), table, kv_lens, q_lens=q_lens, tree=tree, window=window, sinks=sinks, out_dtype=out_dtype).numpy()
        check_attention(got, q, kv, kv_lens, nodes, words, window, sinks, False, out_dtype == "float16", fp16_cache=True)
        for b in range(B):
            assert (got[b, :, nodes[b]:] == 0).all()
    again = cache.attend(tensor(q), table, kv_lens, q_lens=q_lens, tree=tree, window=window, sinks=sinks, out_dtype="float16").numpy()
    assert np.array_equal(got, again, equal_nan=True)


def test_fp32_queries_keep_fp32_accuracy():
    """Long sums at the fp32 path's tolerance: 1e-5 on unit-variance data."""
    cache, table, kv = filled(7, 1, 1, 20000, 128, 64, "int8", spread=0.0)
    q = seeded(3, 1, 2, 1, 128)
    got = cache.attend(tensor(q), table, [20000]).numpy()
    for h in range(2):
        want, _, _ = kv_oracle.attention(q[0, h], kv[0][0, 0], kv[1][0, 0], np.ones((1, 20000), bool))
        assert np.abs(got[0, h] - want).max() <= 1e-5


def test_a_node_that_sees_nothing_and_words_of_all_bits():
    cache, table, kv = filled(9, 1, 1, 64, 64, 16, "e4m3")
    words = np.zeros((1, 64), np.uint64)
    words[0, 1], words[0, 63] = 1 << 1, 2 ** 64 - 1
    q = seeded(4, 1, 1, 64, 64).astype(np.float16)
    got = cache.attend(tensor(q), table, [64], tree=words).numpy()
    assert np.isnan(got[0, 0, 0]).all() and np.isnan(got[0, 0, 2:63]).all()
    check_attention(got, q, kv, [64], [64], words, None, 0, False, False)
    q = seeded(4, 1, 2, 64, 64).astype(np.float16)                # 128 rows
    got = cache.attend(tensor(q), table, [64], tree=words).numpy()
    assert np.isnan(got[0, :, 0]).all() and np.isnan(got[0, :, 2:63]).all()
    check_attention(got, q, kv, [64], [64], words, None, 0, False, False, fp16_cache=True)


def test_values_of_any_magnitude():
    """Scales from 2^-60 to 2^60 beside one another: each row's share is what its scale says."""
    B, H, S, d = 1, 1, 200, 64
    table = page_table(1, 13, 1, 13)
    for fmt in FORMATS:
        k, v = seeded(1, B, H, S, d), seeded(2, B, H, S, d)
        for power in (-60.0, 60.0):
            mixed = v * np.where(np.arange(S) % 3 == 0, 1.0, 2.0 ** power)[:, None].astype(np.float32)
            cache = QuantizedKVCache(13, H, d, 16, fmt)
            cache.write(tensor(k), tensor(mixed), table)
            kv = [kv_oracle.values(*kv_oracle.quantise(x, fmt), fmt) for x in (k, mixed)]
            q = seeded(3, B, 4, 1, d).astype(np.float16)
            check_attention(cache.attend(tensor(q), table, [S]).numpy(), q, kv, [S], [1], [[1]], None, 0, False, False)
            q = seeded(3, B, 16, 6, d).astype(np.float16)
            got = cache.attend(tensor(q), table, [S]).numpy()
            words = [[(2 << t) - 1 for t in range(6)]]
            check_attention(got, q, kv, [S], [6], words, None, 0, False, False, fp16_cache=True)


@pytest.mark.parametrize("fmt", FORMATS)
def test_what_is_not_finite_stays_where_it_is_seen(fmt):
    """A NaN key or value makes NaN of the nodes that see it; keys past the end and outside the window are never used."""
    B, H, S, T, d, page, window = 1, 1, 150, 3, 64, 16, 40
    table = page_table(1, 10, 1, 10)
    k, v = seeded(1, B, H, 160, d), seeded(2, B, H, 160, d)
    k[0, 0, 149, 5] = np.nan                     # node 2: only it sees that
    v[0, 0, 148, 1] = np.inf                     # node 1, which node 2 does not see
    k[0, 0, 20], v[0, 0, 30] = np.nan, np.inf    # outside every window
    k[0, 0, 150:], v[0, 0, 150:] = np.nan, np.nan
    cache = QuantizedKVCache(10, H, d, page, fmt)
    cache.write(tensor(k), tensor(v), table)
    tree = np.array([[0b001, 0b011, 0b101]], np.uint64)
    for heads in (2, 40):                        # 6 rows, and 120
        q = seeded(3, B, heads, T, d).astype(np.float16)
        got = cache.attend(tensor(q), table, [S], tree=tree, window=window).numpy()
        assert np.isfinite(got[0, :, 0]).all() and np.isnan(got[0, :, 1]).all() and np.isnan(got[0, :, 2]).all()
        kv = [np.nan_to_num(kv_oracle.values(*kv_oracle.quantise(x, fmt), fmt)) for x in (k, v)]
        check_attention(got[:, :, :1], q[:, :, :1], kv, [148], [1], [[1]], window, 0, False, False, fp16_cache=heads > 2)


def test_queries_that_are_not_finite():
    cache, table, kv = filled(9, 1, 1, 50, 64, 16, "int8")
    for dtype in (np.float16, np.float32):
        q = seeded(4, 1, 2, 1, 64).astype(dtype)
        q[0, 0, 0, 3] = np.nan
        got = cache.attend(tensor(q), table, [50]).numpy()
        assert np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1]).all()


def test_fp32_queries_of_any_magnitude():
    cache, table, kv = filled(11, 1, 1, 300, 128, 16, "int8", spread=0.0)
    for power in (2.0 ** -100, 2.0 ** -30, 2.0 ** 3):
        q = (seeded(4, 1, 2, 1, 128) * power).astype(np.float32)
        q[0, 1, 0, :64] *= np.float32(2.0 ** -9)
        got = cache.attend(tensor(q), table, [300]).numpy()
        check_attention(got, q, kv, [300], [1], [[1]], None, 0, True, False)


def test_rows_of_nodes_that_do_not_exist_stay(lib=None):
    """The library writes rows t < q_lens[b] and no others."""
    cache, table, _ = filled(13, 2, 1, 100, 64, 16, "e4m3")
    q = seeded(4, 2, 2, 7, 64).astype(np.float16)
    dq, table_dev = tensor(q), cache.indices(table)
    out = _lib.to_device(np.full((2, 2, 7, 64), -3.0, np.float32))
    lens, nodes = cache.indices([100, 60]), cache.indices([4, 0])
    desc = _lib.KvAttentionDesc(cache=cache._impl.desc, q=dq._c_tensor.data_ptr, out=out.ptr, page_table=table_dev.data_ptr,
                                kv_lens=lens.data_ptr, q_lens=nodes.data_ptr, batch=2, q_heads=2, tokens=7,
                                table_len=table.shape[1], dtype=_lib.TX_DTYPE_F16)
    _lib.check(_lib.load().tx_kv_cache_attention(ctypes.byref(desc)))
    _lib.check(_lib.load().tx_sdpa_finish(None))
    got = out.download((2, 2, 7, 64), np.float32)
    assert (got[0, :, 4:] == -3).all() and (got[1] == -3).all() and (got[0, :, :4] != -3).all()


@pytest.mark.parametrize("heads", [2, 60])
def test_sequences_of_fewer_keys_than_nodes(heads):
    """An idle place of a batch (no key), and a sequence that is shorter than the call: no key, no result."""
    cache, table, kv = filled(17, 3, 1, 40, 64, 16, "int8")
    q = seeded(4, 3, heads, 3, 64).astype(np.float16)
    for dtype in (np.float16, np.float32) if heads == 2 else (np.float16,):
        got = cache.attend(tensor(q.astype(dtype)), table, [0, 2, 40]).numpy()
        assert np.isnan(got[0]).all() and np.isnan(got[1, :, 2]).all()
        assert np.isfinite(got[1, :, :2]).all() and np.isfinite(got[2]).all()


def test_the_same_bits_every_time():
    cache, table, _ = filled(15, 2, 2, 3000, 128, 64, "e4m3")
    q = tensor(seeded(4, 2, 8, 6, 128).astype(np.float16))
    first = cache.attend(q, table, [3000, 1711]).numpy()
    for _ in range(3):
        assert np.array_equal(first, cache.attend(q, table, [3000, 1711]).numpy())


def test_a_cache_beyond_32_bits():
    """Pages whose bytes and rows lie past 2^32: the offsets are 64-bit."""
    H, d, page, fmt = 8, 256, 256, "int8"
    pages = (2 ** 32 + 2 ** 29) // (H * d * page)                 # 4.5 GiB of codes each
    cache = QuantizedKVCache(pages, H, d, page, fmt)
    table = np.array([[pages - 1, 0, pages - 2]])
    k, v = seeded(1, 1, H, 600, d).astype(np.float16), seeded(2, 1, H, 600, d).astype(np.float16)
    cache.write(tensor(k), tensor(v), table)
    kv = [kv_oracle.values(*kv_oracle.quantise(x, fmt), fmt) for x in (k, v)]
    back = cache.read(table, 600, dtype="float32")
    for x, y in zip(kv, back):
        assert np.array_equal(x.astype(np.float32), y.numpy())
    q = seeded(3, 1, H, 1, d).astype(np.float16)
    check_attention(cache.attend(tensor(q), table, [600]).numpy(), q, kv, [600], [1], [[1]], None, 0, False, False)


# ------------------------------------------------------------------ as they are used
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_serving_loop(fmt):
    """A prompt is written, then trees of drafts are written, attended and cut down to the accepted path, step by step; each
    step's attention is that over the tokens kept so far."""
    B, Hq, Hkv, d, page, window, sinks = 2, 4, 2, 64, 16, 90, 2
    rng = np.random.default_rng(0)
    lens = np.array([70, 33])
    table = page_table(2, 40, B, 16)
    cache = QuantizedKVCache(40, Hkv, d, page, fmt)
    table_dev = cache.indices(table)
    held = [[seeded(10 * b + i, Hkv, lens[b], d).astype(np.float16) for i in range(2)] for b in range(B)]
    prompt = [np.zeros((B, Hkv, 70, d), np.float16) for _ in range(2)]
    for b in range(B):
        for i in range(2):
            prompt[i][b, :, : lens[b]] = held[b][i]
    cache.write(tensor(prompt[0]), tensor(prompt[1]), table_dev, counts=lens, sync=False)
    T = 7
    for step in range(4):
        k, v, q = (seeded(100 + 3 * step + i, B, (Hkv, Hkv, Hq)[i], T, d).astype(np.float16) for i in range(3))
        cache.write(tensor(k), tensor(v), table_dev, start=lens, sync=False)
        tree, words = words_of("tree", step, B, T)
        got = cache.attend(tensor(q), table_dev, lens + T, tree=tree, window=window, sinks=sinks).numpy()
        full = [np.zeros((B, Hkv, lens.max() + T, d)) for _ in range(2)]
        for b in range(B):
            for i, new in enumerate((k, v)):
                x = np.concatenate([held[b][i], new[b]], 1)
                full[i][b, :, : lens[b] + T] = kv_oracle.values(*kv_oracle.quantise(x, fmt), fmt)
        check_attention(got, q, full, lens + T, [T] * B, words, window, sinks, False, False)
        # the path to a node is accepted
        paths = [[u for u in range(T) if int(words[b, int(rng.integers(T))]) >> u & 1] for b in range(B)]
        n = max(map(len, paths))
        rows = np.array([p + [0] * (n - len(p)) for p in paths])
        cache.write(tensor(k), tensor(v), table_dev, start=lens, counts=[len(p) for p in paths], rows=rows, sync=False)
        for b in range(B):
            held[b] = [np.concatenate([held[b][i], x[b][:, paths[b]]], 1) for i, x in enumerate((k, v))]
        lens = lens + [len(p) for p in paths]
    kb, _ = cache.read(table_dev, int(lens.max()), counts=lens, dtype="float32")
    for b in range(B):
        assert np.array_equal(kb.numpy()[b, :, : lens[b]], kv_oracle.values(*kv_oracle.quantise(held[b][0], fmt), fmt).astype(np.float32))


def test_calls_in_two_graphs_and_on_two_streams():
    """Write and attention recorded in graphs of two streams and replayed on other inputs, both at once."""
    torch = pytest.importorskip("torch")
    lib = _lib.load()
    B, Hq, Hkv, T, S, d, page = 2, 8, 2, 4, 500, 128, 64
    jobs = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        st = ctypes.c_void_p(stream.cuda_stream)
        codes = [torch.zeros(20, Hkv, page, d, dtype=torch.uint8, device="cuda") for _ in range(2)]
        scales = [torch.zeros(20, Hkv, page, device="cuda") for _ in range(2)]
        table = torch.randperm(20)[:16].view(B, 8).int().cuda()
        k, v = (torch.empty(B, Hkv, S, d, dtype=torch.float16, device="cuda").normal_() for _ in range(2))
        q, out = torch.empty(B, Hq, T, d, dtype=torch.float16, device="cuda").normal_(), torch.zeros(B, Hq, T, d, device="cuda")
        lens = torch.tensor([S, S - 100], dtype=torch.int32, device="cuda")
        cache = _lib.KvCache(k=codes[0].data_ptr(), v=codes[1].data_ptr(), k_scale=scales[0].data_ptr(), v_scale=scales[1].data_ptr(),
                             pages=20, kv_heads=Hkv, page_size=page, d=d, format=_lib.TX_KV_E4M3)
        write = _lib.KvWriteDesc(cache=cache, k=k.data_ptr(), v=v.data_ptr(), page_table=table.data_ptr(), batch=B, tokens=S,
                                 table_len=8, dtype=_lib.TX_DTYPE_F16, stream=st)
        attend = _lib.KvAttentionDesc(cache=cache, q=q.data_ptr(), out=out.data_ptr(), page_table=table.data_ptr(),
                                      kv_lens=lens.data_ptr(), batch=B, q_heads=Hq, tokens=T, table_len=8, dtype=_lib.TX_DTYPE_F16,
                                      stream=st)

        def call(write=write, attend=attend):
            _lib.check(lib.tx_kv_cache_write(ctypes.byref(write)))
            _lib.check(lib.tx_kv_cache_attention(ctypes.byref(attend)))

        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
            call()
        jobs.append((graph, call, (k, v, q), out, (codes, scales, table, lens)))
    for _ in range(3):
        want = []
        for _, call, inputs, out, _ in jobs:
            for t in inputs:
                t.normal_()
            torch.cuda.synchronize()
            call()
            torch.cuda.synchronize()
            want.append(out.clone())
            out.zero_()
        torch.cuda.synchronize()
        for graph, *_ in jobs:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(job[3], w) for job, w in zip(jobs, want))


@pytest.mark.parametrize("T", [1, 24])
def test_calls_that_follow_each_other_without_a_wait(T):
    """Queries, keys, lengths and pages are written on the stream right in front of the calls that read them, and overwritten
    right behind: the same bits as with a wait after every step."""
    torch = pytest.importorskip("torch")
    lib, stream = _lib.load(), torch.cuda.Stream()
    st = ctypes.c_void_p(stream.cuda_stream)
    B, Hq, Hkv, d, page, table_len, steps = 2, 8, 2, 128, 16, 40, 12
    generator = torch.Generator(device="cuda").manual_seed(1)
    new = [torch.randn(steps, B, Hkv, T, d, generator=generator, device="cuda").half() for _ in range(2)]
    qs = torch.randn(steps, B, Hq, T, d, generator=generator, device="cuda").half()
    plain = [torch.randn(B, Hkv, 640, d, generator=generator, device="cuda").half() for _ in range(2)]
    tables = torch.stack([torch.randperm(B * table_len).view(B, table_len) for _ in range(steps)]).int().cuda()

    def run(wait):
        codes, scales = [torch.zeros(B * table_len, Hkv, page, d, dtype=torch.uint8, device="cuda") for _ in range(2)], \
                        [torch.zeros(B * table_len, Hkv, page, device="cuda") for _ in range(2)]
        k, v, q = torch.zeros_like(new[0][0]), torch.zeros_like(new[1][0]), torch.zeros_like(qs[0])
        table, start, lens = torch.zeros_like(tables[0]), torch.zeros(B, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.int32, device="cuda")
        out, step_out = torch.zeros(B, Hq, T, d, device="cuda"), torch.zeros(B, Hq, 1, d, device="cuda")
        q1 = torch.zeros(B, Hq, 1, d, dtype=torch.float16, device="cuda")
        cache = _lib.KvCache(k=codes[0].data_ptr(), v=codes[1].data_ptr(), k_scale=scales[0].data_ptr(), v_scale=scales[1].data_ptr(),
                             pages=B * table_len, kv_heads=Hkv, page_size=page, d=d, format=_lib.TX_KV_E4M3)
        write = _lib.KvWriteDesc(cache=cache, k=k.data_ptr(), v=v.data_ptr(), page_table=table.data_ptr(), start=start.data_ptr(),
                                 batch=B, tokens=T, table_len=table_len, dtype=_lib.TX_DTYPE_F16, stream=st)
        attend = _lib.KvAttentionDesc(cache=cache, q=q.data_ptr(), out=out.data_ptr(), page_table=table.data_ptr(), kv_lens=lens.data_ptr(),
                                      batch=B, q_heads=Hq, tokens=T, table_len=table_len, dtype=_lib.TX_DTYPE_F16, stream=st)
        window = _lib.SdpaDesc(q=q1.data_ptr(), k=plain[0].data_ptr(), v=plain[1].data_ptr(), kv_lens=lens.data_ptr(), out=step_out.data_ptr(),
                               batch=B, q_heads=Hq, kv_heads=Hkv, seq_q=1, seq_k=640, d_k=d, d_v=d, dtype=_lib.TX_DTYPE_F16, causal=1, stream=st)
        rule, got = _lib.WindowDesc(window=50, sinks=2, align_end=1), []
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for i in range(steps):
                for to, x in ((k, new[0][i]), (v, new[1][i]), (q, qs[i]), (table, tables[i]), (q1, qs[i][:, :, :1])):
                    to.copy_(x)
                start.fill_(16 * i)
                _lib.check(lib.tx_kv_cache_write(ctypes.byref(write)))
                lens.fill_(16 * i + T)
                _lib.check(lib.tx_kv_cache_attention(ctypes.byref(attend)))
                _lib.check(lib.tx_sdpa_window_forward(ctypes.byref(window), ctypes.byref(rule)))
                for x in (q, q1, k, v):
                    x.fill_(float("nan"))
                got += [out.clone(), step_out.clone()]
                if wait:
                    torch.cuda.synchronize()
        torch.cuda.synchronize()
        _lib.check(lib.tx_sdpa_finish(st))
        return got

    want = run(True)
    assert all(torch.isfinite(x).all() for x in want[1::2])
    for _ in range(3):
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(run(False), want))


def test_functional_refusals():
    cache = QuantizedKVCache(4, 2, 64, 16)
    x = tensor(seeded(1, 1, 2, 3, 64))
    with pytest.raises(ValueError, match="4D"):
        F.kv_cache_write(cache, tensor(seeded(1, 2, 3, 64)), x, [[0]])
    with pytest.raises(ValueError, match="CUDA"):
        F.kv_cache_write(cache, x.cpu(), x.cpu(), [[0]])
    with pytest.raises(RuntimeError, match="of the cache"):
        cache.write(tensor(seeded(1, 1, 3, 3, 64)), tensor(seeded(1, 1, 3, 3, 64)), [[0]])
    with pytest.raises(RuntimeError, match="page_table"):
        cache.write(x, x, [0])
    with pytest.raises(RuntimeError, match="kv_lens"):
        cache.attend(x, [[0]], [3, 3])
    with pytest.raises(RuntimeError, match="hold the call"):
        cache.attend(x, [[0]], [3], window=2)
    x.requires_grad = True
    with pytest.raises(ValueError, match="no backward"):
        cache.attend(x, [[0]], [3])
