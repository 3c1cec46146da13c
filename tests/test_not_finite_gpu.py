"""Infinities and NaN among keys and values that some rows see: those rows are what the definition makes of them, wherever in a
tile the key lies, and rows that do not see it have their own result."""
import numpy as np
import pytest

import kv_oracle
import tensorax_b200 as ts
import window_oracle
from conftest import seeded
from tensorax_b200 import _C
from tensorax_b200.nn import QuantizedKVCache

pytestmark = pytest.mark.gpu


def tensor(x):
    return ts.Tensor._wrap(_C.from_numpy(np.ascontiguousarray(x)))


# ------------------------------------------------------------------ attention over the cache
def check_cache_rows(got, q, codes, kv_lens, words, window, sinks, many):
    """Rows that see a key whose scale is not finite are NaN; the others are within what the roundings can make of them.

    A weight is rounded to fp16 (2^-11 of it); the score's sum of d products in fp32 may lose 2^-23 of the sum of their sizes per
    addition, e in all, carried by the weight and by the sum of the weights; 2^-19 for exponentials, scales and partial sums.
    many (rows a head, tcgen05): keys and values times their scales are rounded to fp16 too (2^-11 of a product, of a value), the
    exponential may be the polynomial one (1.6e-4 < 2^-12.5 in weight and sum), and weights more than 2^24 (and 2^8 for a
    maximum not yet raised) below the row's largest are lost: with 2^10 keys a row at most, 2^-17 of the largest value."""
    B, Hq, T, d = q.shape
    kv = [kv_oracle.values(*c) for c in codes]
    bad = ~(np.isfinite(kv[0]).all(-1) & np.isfinite(kv[1]).all(-1))
    kv = [np.where(bad[..., None], 0.0, x) for x in kv]
    G, seen_bad, fine = Hq // kv[0].shape[1], 0, 0
    for b in range(B):
        ctx = kv_lens[b] - T
        see = kv_oracle.visible(ctx, T, words[b], window, sinks)
        for h in range(Hq):
            k, v, broken = (x[b, h // G, : kv_lens[b]] for x in (kv[0], kv[1], bad))
            nan = (see & broken).any(1)
            assert np.isnan(got[b, h, nan]).all(), (b, h)
            want, weight, size = kv_oracle.attention(q[b, h], k, v, see)
            e = size * (d * 2.0 ** -23 + 2.0 ** -22)
            bound = weight * (2.0 ** -11 + 2 * e[:, None] + 2.0 ** -19) + 1e-30
            if many:
                bound = bound + weight * (2.0 ** -11 + 2.0 ** -11.5 + 2 * 2.0 ** -11 * size[:, None]) + 2.0 ** -17 * np.abs(v).max()
            assert (np.abs(got[b, h].astype(np.float64) - want) <= bound)[~nan].all(), (b, h)
            seen_bad, fine = seen_bad + int(nan.sum()), fine + int((~nan).sum())
    assert seen_bad and fine


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads, T", [(2, 3), (8, 5), (16, 4), (40, 3)])          # 6, 40, 64 and 120 rows a K/V head
@pytest.mark.parametrize("where", ["node", "context"])
def test_a_key_at_every_place_of_a_tile(where, heads, T, d, fmt):
    """Sixteen sequences, the key one place further in each.  "node": the last node, which only it sees.  "context": the first
    key of the window of the last node, a root; the others stand below it and see from one key further on."""
    B, window = 16, 90
    kv_lens = [177 + b + T for b in range(B)]
    page, table_len = 16, 13
    table = np.random.default_rng(3).permutation(B * table_len).reshape(B, table_len).astype(np.int32)
    kv = [seeded(1 + i, B, 1, page * table_len, d) for i in range(2)]
    for b in range(B):
        ctx = kv_lens[b] - T
        at = kv_lens[b] - 1 if where == "node" else ctx - window + 1
        kv[b % 2][b, 0, at, (5 * b) % d] = (np.nan, np.inf, -np.inf)[b % 3]
    cache = QuantizedKVCache(B * table_len, 1, d, page, fmt)
    cache.write(tensor(kv[0]), tensor(kv[1]), table)
    codes = [(*kv_oracle.quantise(x, fmt), fmt) for x in kv]
    if where == "node":
        words, limit = np.array([[1 << t | 1 for t in range(T)]] * B, np.uint64), None
    else:
        words, limit = np.array([[1 << t | 1 << (T - 1) for t in range(T)]] * B, np.uint64), window
    q = seeded(7, B, heads, T, d).astype(np.float16)
    got = cache.attend(tensor(q), table, kv_lens, tree=words, window=limit).numpy()
    check_cache_rows(got, q, codes, kv_lens, words, limit, 0, heads * T > (32 if fmt == "e4m3" else 64))


# ------------------------------------------------------------------ prompts and steps over plain keys
def check_head(got, q, k, v, see, near, f16):
    """One head with one bad element of K or V.  Rows that see a NaN or +inf score are NaN, a score of -inf has no weight, a value
    that is not finite shows in its column of the rows that see it.  Of the other rows those `near` the key may show it; what they
    show of anything else is within the bounds of the windowed attention's tests (roundings of weights, 2^-11 and 2^-12.5 for the
    polynomial exponential; e for the scores' sums; 2^-17 of |v| for weights that are lost)."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    d = q.shape[1]
    with np.errstate(invalid="ignore"):
        s = np.where(see, q @ k.T / np.sqrt(d), -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p = p / p.sum(1, keepdims=True)
    nan = np.isnan(p).any(1)
    assert np.isnan(got[nan]).all()
    vv, kk, pp = (np.where(np.isfinite(x), x, 0.0) for x in (v, k, p))
    want, weight = pp @ vv, pp @ np.abs(vv)
    size = np.where(see & (np.isfinite(k).all(1) | ~np.isneginf(s)), np.abs(q) @ np.abs(kk).T, 0).max(1) / np.sqrt(d)
    e = size * (3 * d * 2.0 ** -23 + 2.0 ** -21)
    bound = weight * ((2.0 ** -11 + 2.0 ** -11.5 if f16 else 2.0 ** -21) + 2 * e[:, None] + 2.0 ** -19) + 1e-30
    if f16:
        bound = bound + 2.0 ** -17 * np.abs(vv).max()
    with np.errstate(invalid="ignore"):
        fine = np.abs(got.astype(np.float64) - want) <= bound
    shows = (see[:, :, None] & ~np.isfinite(v)[None]).any(1)          # a row sees that value
    assert not np.isfinite(got[shows]).any()
    fine |= nan[:, None] | shows | (near[:, None] & ~np.isfinite(got))
    assert fine.all(), np.argwhere(~fine)[:4]
    return int(nan.sum() + shows.any(1).sum())


def spoil(q, k, v, head, at, d):
    """NaN or an infinity in key `at` of a head: in K (+inf times positive elements: a score of +inf; and of -inf), or in V."""
    c = 7 * head % d
    q[..., c] = np.abs(q[..., c]) + q.dtype.type(0.1)
    (k if head % 5 < 3 else v)[at, c] = (np.nan, np.inf, -np.inf, np.nan, np.inf)[head % 5]


@pytest.mark.parametrize("dtype, d", [(np.float16, 64), (np.float16, 128), (np.float16, 256), (np.float16, 512), (np.float32, 64),
                                      (np.float32, 128), (np.float32, 160)])
@pytest.mark.parametrize("window, sinks", [(100, 3), (None, 0)])
def test_prompts(window, sinks, dtype, d):
    """Twenty heads, the key one place further in each; `window` None: causal."""
    H, S = 20, 700
    q, k, v = (seeded(i, 1, H, S, d).astype(dtype) for i in range(3))
    for h in range(H):
        spoil(q[0, h], k[0, h], v[0, h], h, 400 + h, d)
    impls = [_C.from_numpy(x) for x in (q, k, v)]
    if window is None:
        got = _C.to_numpy(_C.scaled_dot_product_attention_ex(*impls, causal=True))
    else:
        got = _C.to_numpy(_C.scaled_dot_product_attention_window(*impls, window, sinks))
    see = window_oracle.seen(S, S, S, window or S, sinks, "start")
    met = 0
    for h in range(H):
        near = np.zeros(S, bool)
        for a in range(0, S, 128):                       # a tile of rows sees keys within 128 of it
            used = np.flatnonzero(see[a: a + 128].any(0))
            near[a: a + 128] = np.abs(used - (400 + h)).min() <= 128
        assert not near.all()
        met += check_head(got[0, h], q[0, h], k[0, h], v[0, h], see, near, dtype == np.float16)
    assert met


@pytest.mark.parametrize("dtype, d", [(np.float16, 64), (np.float16, 128), (np.float16, 256), (np.float32, 64), (np.float32, 128)])
@pytest.mark.parametrize("G, Sq", [(1, 1), (4, 1), (5, 3), (4, 6)])
def test_steps(G, Sq, dtype, d):
    """The last rows of twenty sequences; 24 rows a K/V head are beyond the decoding steps' kernels in fp16."""
    B, S, window, sinks = 20, 400, 100, 3
    lens = [330 + b for b in range(B)]
    q, k, v = (seeded(i, B, (G, 1, 1)[i], (Sq, S, S)[i], d).astype(dtype) for i in range(3))
    for b in range(B):
        spoil(q[b], k[b, 0], v[b, 0], b, 300 + b, d)
    got = _C.to_numpy(_C.scaled_dot_product_attention_window(*(_C.from_numpy(x) for x in (q, k, v)), window, sinks, "end", kv_lens=lens))
    met = 0
    for b in range(B):
        see = window_oracle.seen(Sq, S, lens[b], window, sinks, "end")
        for h in range(G):
            met += check_head(got[b, h], q[b, h], k[b, 0], v[b, 0], see, np.ones(Sq, bool), dtype == np.float16)
    assert met


def test_a_longer_prompt_of_shared_heads():
    """The key in the first of several tiles that a row walks, and in the last."""
    H, S, d, window = 16, 1500, 128, 600
    for first in (0, 640, 1484):
        q, k, v = seeded(1, 1, H, S, d), seeded(2, 1, 4, S, d), seeded(3, 1, 4, S, d)
        q, k, v = (x.astype(np.float16) for x in (q, k, v))
        for h in range(4):
            k[0, h, first + 5 * h, 3] = np.nan
        got = _C.to_numpy(_C.scaled_dot_product_attention_window(*(_C.from_numpy(x) for x in (q, k, v)), window, 0))
        see = window_oracle.seen(S, S, S, window, 0, "start")
        for h in range(H):
            at = first + 5 * (h // 4)
            assert check_head(got[0, h], q[0, h], k[0, h // 4], v[0, h // 4], see, np.abs(np.arange(S) - at) < window + 256, True)
