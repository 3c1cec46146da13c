"""Attention with a sliding window and sinks, and its gradients, in numpy and 64 bits, from the definition."""
import numpy as np


def seen(Sq, Sk, n, window, sinks, align):
    """[Sq, Sk]: row i of a sequence of n keys sees key j."""
    pos = np.arange(Sq)[:, None] + (n - Sq if align == "end" else 0)
    key = np.arange(Sk)[None, :]
    return (key < n) & (key <= pos) & ((key > pos - window) | (key < sinks))


def _softmax(q, k, see):
    with np.errstate(invalid="ignore"):
        s = np.where(see, q @ np.where(see.any(0)[:, None], k, 0).T / np.sqrt(q.shape[-1]), -np.inf)
        alive = see.any(1)
        p = np.exp(s - np.where(alive, s.max(1, initial=-np.inf, where=see), 0)[:, None])
    return np.where(alive[:, None], p / np.where(alive, p.sum(1), 1)[:, None], 0.0), alive


def forward(q, k, v, lens, window, sinks, align="start", with_size=False):
    """q [B,Hq,Sq,d], k, v [B,Hkv,Sk,*] -> O (and sum_j p_j |v_j|, and the largest sum of |q||k| in a row's visible score)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    B, H, Sq, d = q.shape
    G, Sk = H // k.shape[1], k.shape[2]
    out, weight = (np.full((B, H, Sq, v.shape[3]), np.nan) for _ in range(2))
    size = np.zeros((B, H, Sq))
    for b in range(B):
        see = seen(Sq, Sk, lens[b], window, sinks, align)
        used = see.any(0)
        for h in range(H):
            p, alive = _softmax(q[b, h], k[b, h // G], see)
            vv = np.where(used[:, None], v[b, h // G], 0)
            out[b, h][alive], weight[b, h][alive] = (p @ vv)[alive], (p @ np.abs(vv))[alive]
            if with_size:
                kk = np.where(used[:, None], k[b, h // G], 0)
                size[b, h] = np.where(see, np.abs(q[b, h]) @ np.abs(kk).T, 0).max(1) / np.sqrt(d)
    return (out, weight, size) if with_size else out


def backward(q, k, v, grad, lens, window, sinks, align="start"):
    """(dq, dk, dv); a row that sees nothing has no part."""
    q, k, v, grad = (np.asarray(x, np.float64) for x in (q, k, v, grad))
    B, H, Sq, d = q.shape
    G, Sk, scale = H // k.shape[1], k.shape[2], 1 / np.sqrt(d)
    dq, dk, dv = np.zeros_like(q), np.zeros_like(k), np.zeros_like(v)
    for b in range(B):
        see = seen(Sq, Sk, lens[b], window, sinks, align)
        used = see.any(0)[:, None]
        for h in range(H):
            kk, vv, g = np.where(used, k[b, h // G], 0), np.where(used, v[b, h // G], 0), grad[b, h]
            p, _ = _softmax(q[b, h], kk, see)
            dp = g @ vv.T
            ds = p * (dp - (p * dp).sum(1, keepdims=True)) * scale
            dq[b, h] = ds @ kk
            dk[b, h // G] += ds.T @ q[b, h]
            dv[b, h // G] += p.T @ g
    return dq, dk, dv
