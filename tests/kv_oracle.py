"""The quantised cache and the attention over it in numpy, 64 bits, from their definitions."""
import numpy as np

# the values of the 127 codes without a sign that are numbers: exponent field, three bits behind the point
E4M3 = np.array([(c & 7) * 2.0 ** -9 if c < 8 else (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10) for c in range(127)])


def quantise(x, fmt):
    """x [..., d] -> (codes, scales [...]); codes as the cache keeps them."""
    x = np.asarray(x, np.float32)
    fine = np.isfinite(x).all(-1)
    x = np.where(fine[..., None], x, np.float32(0))
    amax = np.abs(x).max(-1)
    if fmt == "int8":
        scale = np.maximum(amax * (np.float32(1) / np.float32(127)), np.float32(2.0 ** -126)).astype(np.float32)
        codes = np.clip(np.rint(x / scale[..., None]), -127, 127).astype(np.int8)
    else:
        m, e = np.frexp(amax.astype(np.float64))
        scale = np.exp2(np.maximum(np.where(amax > 0, np.where(m <= 0.875, e - 9, e - 8), -126), -126).astype(np.float64))
        y = np.abs(x.astype(np.float64)) / scale[..., None]
        hi = np.clip(np.searchsorted(E4M3, y), 1, 126)
        lo = hi - 1
        below, above = y - E4M3[lo], E4M3[hi] - y
        code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
        codes = (code + 128 * np.signbit(x)).astype(np.uint8)
        scale = scale.astype(np.float32)
    codes[~fine] = 0
    return codes, np.where(fine, scale, np.float32(np.nan)).astype(np.float32)


def values(codes, scales, fmt):
    c = codes.astype(np.float64) if fmt == "int8" else E4M3[np.minimum(codes & 127, 126)] * np.where(codes & 128, -1.0, 1.0)
    return c * np.asarray(scales, np.float64)[..., None]


def rows_of(cache, table, h, positions, page):
    """Rows of one sequence and head from pages [pages, H, page, ...]."""
    positions = np.asarray(positions)
    return cache[np.asarray(table)[positions // page], h, positions % page]


def visible(ctx, nodes, words, window, sinks):
    """[nodes, ctx + nodes]: what each node sees."""
    see = np.zeros((nodes, ctx + nodes), bool)
    for t in range(nodes):
        word = int(words[t])
        depth = max(bin(word).count("1"), 1) - 1
        j = np.arange(ctx)
        see[t, :ctx] = True if not window else (j > ctx + depth - window) | (j < sinks)
        for u in range(nodes):
            see[t, ctx + u] = word >> u & 1
    return see


def attention(q, k, v, see):
    """q [T, d], k, v [n, d], see [T, n] -> (O, sum_j p_j |v_j|, the largest sum of |q||k| in a visible score), 64 bits."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, weight = (np.full((len(q), v.shape[1]), np.nan) for _ in range(2))
    size = np.full(len(q), np.nan)
    for t in range(len(q)):
        if not see[t].any():
            continue
        kk, vv = k[see[t]], v[see[t]]
        s = kk @ q[t] / np.sqrt(q.shape[1])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[t], weight[t] = p @ vv, p @ np.abs(vv)
        size[t] = (np.abs(kk) @ np.abs(q[t])).max() / np.sqrt(q.shape[1])
    return out, weight, size
