"""Attention of windowed models and their quantised K/V cache: the operators' measured cases.

Every case is a dict of plain values; ``listed()``, ``draw(rng)``, ``prepare(case, seed)``, ``run(state)`` and
``work(case)`` are as in ``cases.py`` beside this file.  ``run`` computes the operators in elementary torch operations,
or, where ``own`` is true, through the package's entry points; ``exact(case, seed)`` gives the results in 64 bits.

Kinds of work ("kind"):
  window  attention in which a row sees the last ``window`` keys up to its own position and the first ``sinks`` ones.
          "align" says where row i stands: "start": at position i; "end": the rows are the last ones of their sequence
          (a single token against the cache the serving loop keeps, or a chunk of a long prompt)
  train   the same, forward and the three gradients
  cache   a call's keys and values quantised into pages as they are written, and the last ``back`` tokens of each
          sequence read back as values
  tree    attention of ``T`` drafted tokens over the pages: a tree ("tree"), a chain, or with T = 1 a plain decoding step
"""
import ctypes
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16}
_SIZES = {"float32": 4, "float16": 2}


def _window(kind, B, Hq, Hkv, Sq, Sk, d, window, sinks, dtype="float16", lens="full", align="start", name=None):
    c = {"kind": kind, "B": B, "Hq": Hq, "Hkv": Hkv, "Sq": Sq, "Sk": Sk, "d": d, "window": window, "sinks": sinks,
         "dtype": dtype, "lens": lens, "align": align}
    return c if name is None else {"name": name, **c}


def _cache(B, Hkv, T, S, back, d, page, fmt, dtype="float16", name=None):
    c = {"kind": "cache", "B": B, "Hkv": Hkv, "T": T, "S": S, "back": back, "d": d, "page": page, "format": fmt,
         "dtype": dtype}
    return c if name is None else {"name": name, **c}


def _tree(B, Hq, Hkv, T, S, d, page, fmt, window=0, sinks=0, dtype="float16", shape="tree", ragged=False, name=None):
    c = {"kind": "tree", "B": B, "Hq": Hq, "Hkv": Hkv, "T": T, "S": S, "d": d, "page": page, "format": fmt,
         "window": window, "sinks": sinks, "dtype": dtype, "shape": shape, "ragged": ragged}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # One small prompt of a small model: launch and host time only.
        _window("window", 1, 4, 4, 250, 250, 64, 64, 4, name="window_small_d64"),
        # A padded batch of long prompts with four query heads per K/V head.
        _window("window", 2, 16, 4, 8192, 8192, 128, 1024, 4, lens="half", name="window_prefill_d128"),
        # float32 attention at a head width and a length that are no tile multiples.
        _window("window", 2, 8, 8, 1000, 1000, 80, 200, 3, "float32", name="window_fp32_d80"),
        # One decoding step: single tokens against plain caches of which the window and the sinks are read.
        _window("window", 8, 32, 8, 1, 8192, 128, 2048, 4, lens="half", align="end", name="window_decode_d128"),
        # A training step's attention: forward and the three gradients.
        _window("train", 4, 16, 16, 2048, 2048, 128, 512, 4, name="window_train_d128"),
        # The same at an odd length with padding, narrow heads and shared K/V heads.
        _window("train", 2, 12, 4, 921, 921, 64, 100, 1, lens="half", name="window_train_ragged_d64"),
        # A step's new tokens appended to their sequences, and the last of them read back.
        _cache(32, 8, 1, 2048, 64, 128, 16, "int8", name="cache_append_int8"),
        # A batch of prompts written as they leave the projections, and read back for the next chunk.
        _cache(8, 8, 4096, 4096, 4096, 128, 64, "e4m3", name="cache_prompt_e4m3"),
        # One decoding step of a batch of long sequences: the cache is read once, nothing else is large.
        _tree(16, 32, 8, 1, 8192, 128, 64, "e4m3", name="decode_e4m3_d128"),
        # A small batch's drafts of different sizes, over pages that are no multiple of a tile.
        _tree(4, 12, 4, 13, 1500, 64, 16, "int8", ragged=True, name="tree_int8_d64"),
        # Full trees over long contexts with a window: the largest drafts.
        _tree(8, 32, 8, 64, 16384, 128, 64, "e4m3", window=8192, sinks=4, name="tree_window_e4m3_d128"),
        # float32 queries over an eight-bit cache.
        _tree(2, 8, 2, 7, 1000, 128, 32, "int8", dtype="float32", shape="chain", name="chain_fp32_int8_d128"),
    ]


# ------------------------------------------------------------------ more cases of the same ranges
def _log_int(rng, lo, hi):
    """Uniform in the logarithm; every value between the bounds, odd ones too."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(["window", "window", "window32", "step", "train", "train", "cache", "cache", "tree", "tree", "tree"])
    sinks = rng.choice([0, 1, 4, 4, 16, 130])
    if kind == "window":
        S, hkv = _log_int(rng, 64, 8192), rng.choice([1, 2, 4, 8])
        return _window("window", rng.randint(1, 4), hkv * rng.choice([1, 1, 2, 4]), hkv, S, S, rng.choice([64, 64, 128, 128, 256]),
                       _log_int(rng, 16, 4096), sinks, lens=rng.choice(["full", "half"]))
    if kind == "window32":
        S, h = _log_int(rng, 16, 2048), rng.randint(1, 12)
        return _window("window", rng.randint(1, 3), h, h, S, S, rng.choice([32, 64, 80, 128]), _log_int(rng, 8, 1024), sinks,
                       "float32", lens=rng.choice(["full", "half"]))
    if kind == "step":
        hkv, dtype = rng.choice([1, 2, 4, 8]), rng.choice(["float16", "float16", "float32"])
        return _window("window", _log_int(rng, 1, 32), hkv * rng.choice([1, 2, 4, 8]), hkv, rng.choice([1, 1, 1, 2, 5, 128, 500]),
                       _log_int(rng, 512, 16384), rng.choice([64, 128]), _log_int(rng, 64, 4096), sinks, dtype,
                       lens=rng.choice(["full", "half"]), align="end")
    if kind == "train":
        S, hkv = _log_int(rng, 64, 4096), rng.choice([2, 4, 8])
        return _window("train", rng.randint(1, 4), hkv * rng.choice([1, 1, 4]), hkv, S, S, rng.choice([64, 128, 128, 256]),
                       _log_int(rng, 16, 2048), sinks, lens=rng.choice(["full", "half"]))
    page, fmt, d = rng.choice([16, 32, 64, 128]), rng.choice(["e4m3", "int8"]), rng.choice([64, 128, 128, 256])
    if kind == "cache":
        T = rng.choice([1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 4096)])
        S = max(T, _log_int(rng, 64, 4096))
        return _cache(_log_int(rng, 1, 64 if T <= 64 else 8), rng.choice([1, 2, 4, 8]), T, S, _log_int(rng, 1, S), d, page, fmt,
                      rng.choice(["float16", "float16", "float32"]))
    T = rng.choice([1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 4, 64), _log_int(rng, 16, 64)])
    hkv, window = rng.choice([1, 2, 4, 8]), rng.choice([0, 0, _log_int(rng, 64, 8192)])
    return _tree(_log_int(rng, 1, 16), hkv * rng.choice([1, 2, 4, 8]), hkv, T, _log_int(rng, 64, 32768), d, page, fmt, window,
                 sinks if window else 0, rng.choice(["float16", "float16", "float16", "float32"]),
                 rng.choice(["tree", "tree", "chain"]), ragged=rng.random() < 0.4)


def draw(rng):
    most = max(_dense_cost(c) for c in listed())
    while True:
        c = _draw_once(rng)
        if _dense_cost(c) <= most:
            return c


def _dense_cost(c):
    """What the case costs in its plain form: all scores of its tensors, without a window."""
    if c["kind"] == "cache":
        return 64.0 * c["B"] * c["Hkv"] * (c["T"] + c["back"]) * c["d"]
    Sq, Sk = (c["T"], c["S"] + 64) if c["kind"] == "tree" else (c["Sq"], c["Sk"])
    return c["B"] * c["Hq"] * Sq * Sk * (c["d"] + 64.0) * (3.5 if c["kind"] == "train" else 1.0) + 64.0 * c["B"] * c["Hkv"] * Sk * c["d"]


# ------------------------------------------------------------------ what the program has in hand
def _lengths(case, seed):
    """Valid keys of each sequence: all of them, or uniform in [Sk/2, Sk] as a padded batch has them."""
    if case["lens"] == "full":
        return [case["Sk"]] * case["B"]
    g = torch.Generator().manual_seed(seed * 7919 + 17)
    lo = max(case["Sk"] // 2, min(case["Sq"], case["Sk"]) if case["align"] == "end" else 1)
    return torch.randint(lo, case["Sk"] + 1, (case["B"],), generator=g).tolist()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed * 6007 + 5)
    dtype, B, d, Hkv = _DTYPES[case["dtype"]], case["B"], case["d"], case["Hkv"]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    s = {"case": case}
    if case["kind"] in ("window", "train"):
        Hq, Sq, Sk = case["Hq"], case["Sq"], case["Sk"]
        s["lens"] = _lengths(case, seed)
        s["dev_lens"] = torch.tensor(s["lens"], dtype=torch.int32, device="cuda")
        s["q"], s["k"], s["v"] = normal(B, Hq, Sq, d), normal(B, Hkv, Sk, d), normal(B, Hkv, Sk, d)
        if case["kind"] == "train":
            s["grad"] = normal(B, Hq, Sq, d, dtype=torch.float32)
        else:
            s["out"] = torch.empty((B, Hq, Sq, d), dtype=dtype, device="cuda")
        return s
    # pages in no order, as a server that has run for a while hands them out; a few of them belong to nobody
    T, S, page = case["T"], case["S"], case["page"]
    table_len = (S + T + page - 1) // page
    pages = B * table_len + 3
    s["table"] = torch.randperm(pages, generator=host)[: B * table_len].view(B, table_len).to(torch.int32).cuda()
    codes = [torch.zeros((pages, Hkv, page, d), dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros((pages, Hkv, page), dtype=torch.float32, device="cuda") for _ in range(2)]
    if case["kind"] == "cache":
        # tokens of different strength, as keys have them; a few rows carry an outlier
        strength = torch.exp(torch.randn((B, Hkv, T, 1), generator=gen, device="cuda") * 0.5)
        s["k"], s["v"] = (normal(B, Hkv, T, d, dtype=torch.float32) * strength).to(dtype), normal(B, Hkv, T, d, scale=0.7)
        most = S - T
        ctx = [most] * B if most == 0 else torch.randint(0, most + 1, (B,), generator=host).tolist()
        total = [c + T for c in ctx]
        counts = [min(t, case["back"]) for t in total]
        s["start"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
        s["back_count"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        s["back_start"] = torch.tensor([t - c for t, c in zip(total, counts)], dtype=torch.int32, device="cuda")
        s["out_k"], s["out_v"] = (torch.zeros((B, Hkv, case["back"], d), dtype=dtype, device="cuda") for _ in range(2))
        known, known_strength = normal(pages, Hkv, page, d, dtype=torch.float32), 1.0
    else:
        Hq = case["Hq"]
        s["q"] = normal(B, Hq, T, d)
        nodes = torch.randint(max(1, T // 2), T + 1, (B,), generator=host).tolist() if case["ragged"] else [T] * B
        ctx = torch.randint(S // 2, S + 1, (B,), generator=host).tolist()
        words = []
        for b in range(B):
            row = []
            for t in range(T):
                parent = t - 1 if case["shape"] == "chain" else int(torch.randint(max(-1, t - 9), t, (1,), generator=host))
                row.append((row[parent] if parent >= 0 else 0) | (1 << t))
            words.append([w - (1 << 64) if w >= 1 << 63 else w for w in row])
        s["words"] = torch.tensor(words, dtype=torch.int64, device="cuda")
        s["q_lens"] = torch.tensor(nodes, dtype=torch.int32, device="cuda")
        s["kv_lens"] = torch.tensor([c + n for c, n in zip(ctx, nodes)], dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros((B, Hq, T, d), dtype=dtype, device="cuda")
        known, known_strength = normal(pages, Hkv, page, d, dtype=torch.float32), 0.7
    for i in range(2):
        x = known if i == 0 else normal(pages, Hkv, page, d, dtype=torch.float32) * known_strength
        codes[i][:], scales[i][:] = _quantise(x, case["format"])
    s["codes"], s["scales"] = codes, scales
    return s


# ------------------------------------------------------------------ the plain forms
def _quantise(x, fmt):
    """Codes (as bytes) and scales of the rows of x: a row's last dimension shares a scale."""
    x = x.float()
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine.unsqueeze(-1), x, torch.zeros_like(x))
    amax = x.abs().amax(-1)
    if fmt == "int8":
        scale = (amax / 127.0).clamp_min(2.0 ** -126)
        codes = torch.round(x / scale.unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
    else:
        m, e = torch.frexp(amax)
        e = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)
        scale = torch.ldexp(torch.ones_like(amax), e)
        codes = (x / scale.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.view(torch.uint8), torch.where(fine, scale, torch.full_like(scale, math.nan))


def _values(codes, scales, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float() * scales.unsqueeze(-1)


def _slots(table, page, position):
    """Page and place in it of the tokens at position [B, n] of their sequences."""
    return torch.gather(table.long(), 1, position // page), position % page


def _seen(case, row_pos, key_pos):
    """Whether a key at key_pos lies in the window of a row at row_pos or among the sinks."""
    if not case["window"]:
        return key_pos <= row_pos
    return (key_pos <= row_pos) & ((key_pos > row_pos - case["window"]) | (key_pos < case["sinks"]))


def _positions(case, lens):
    pos = torch.arange(case["Sq"], device="cuda").view(1, -1)
    return pos + (lens.view(-1, 1) - case["Sq"] if case["align"] == "end" else 0)


def _softmax(scores, seen):
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_window(s):
    case = s["case"]
    G, scale, lens = case["Hq"] // case["Hkv"], case["d"] ** -0.5, s["dev_lens"].long()
    q, k, v = s["q"].float().unflatten(1, (-1, G)), s["k"].float().unsqueeze(2), s["v"].float().unsqueeze(2)
    key = torch.arange(case["Sk"], device="cuda").view(1, 1, -1)
    seen = _seen(case, _positions(case, lens).unsqueeze(-1), key) & (key < lens.view(-1, 1, 1))
    p = _softmax(torch.matmul(q, k.transpose(-1, -2)) * scale, seen[:, None, None])
    out = torch.matmul(p, v)
    if case["kind"] == "window":
        return out.flatten(1, 2).to(s["q"].dtype)
    g = s["grad"].unflatten(1, (-1, G))
    # a row that sees no key is 0/0 in the result and has no part in the gradients
    dead = ~seen.any(-1)[:, None, None, :, None]
    p, alive = p.masked_fill_(dead, 0.0), out.masked_fill(dead, 0.0)
    dv = torch.matmul(p.transpose(-1, -2), g).sum(2)
    ds = torch.matmul(g, v.transpose(-1, -2)).sub_((g * alive).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q).sum(2)
    dtype = s["q"].dtype
    return [out.flatten(1, 2).to(dtype), dq.flatten(1, 2).to(dtype), dk.to(dtype), dv.to(dtype)]


def _plain_cache(s):
    case = s["case"]
    at, place = _slots(s["table"], case["page"], s["start"].long().view(-1, 1) + torch.arange(case["T"], device="cuda"))
    row = torch.arange(case["back"], device="cuda").view(1, -1)
    valid = row < s["back_count"].view(-1, 1)
    from_, from_place = _slots(s["table"], case["page"], torch.where(valid, s["back_start"].long().view(-1, 1) + row, 0))
    return [_plain_cache_one(case, s[n], s["codes"][i], s["scales"][i], at, place, from_, from_place, valid, s["out_" + n])
            for i, n in enumerate(("k", "v"))]


def _plain_cache_one(case, new, codes, scales, at, place, from_, from_place, valid, out):
    c, f = _quantise(new.transpose(1, 2), case["format"])
    codes[at, :, place] = c
    scales[at, :, place] = f
    back = _values(codes[from_, :, from_place], scales[from_, :, from_place], case["format"])
    return torch.where(valid[:, None, :, None], back.transpose(1, 2).to(out.dtype), out)


def _plain_tree(s):
    case = s["case"]
    T, B, G, fmt = case["T"], case["B"], case["Hq"] // case["Hkv"], case["format"]
    n = s["table"].shape[1] * case["page"]
    key = torch.arange(n, device="cuda").view(1, -1).expand(B, -1)
    at, place = _slots(s["table"], case["page"], key)
    k, v = (_values(s["codes"][i][at, :, place], s["scales"][i][at, :, place], fmt).transpose(1, 2).unsqueeze(2) for i in range(2))
    bits = (s["words"].unsqueeze(-1) >> torch.arange(T, device="cuda")) & 1                       # [B, T, node]
    ctx = (s["kv_lens"] - s["q_lens"]).long().view(B, 1, 1)
    depth = bits.sum(-1, keepdim=True) - 1
    node = (key.unsqueeze(1) - ctx).expand(B, T, n)
    in_tree = (node >= 0) & (node < s["q_lens"].view(B, 1, 1))
    seen = torch.where(in_tree, torch.gather(bits, 2, node.clamp(0, T - 1)) > 0,
                       (node < 0) & _seen(case, ctx + depth, key.unsqueeze(1)))
    q = s["q"].float().unflatten(1, (-1, G))
    p = _softmax(torch.matmul(q, k.transpose(-1, -2)) * case["d"] ** -0.5, seen[:, None, None])
    out = torch.matmul(p, v).flatten(1, 2).to(s["out"].dtype)
    alive = torch.arange(T, device="cuda").view(1, -1) < s["q_lens"].view(-1, 1)
    return torch.where(alive[:, None, :, None], out, s["out"])


# ------------------------------------------------------------------ the package's entry points
class _Shared:
    """A tensor of the package as an object torch can look at without a copy; keeps the tensor alive."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.__cuda_array_interface__ = {"shape": tensor.shape, "typestr": "<f2" if tensor.dtype == "float16" else "<f4",
                                         "data": (tensor._c_tensor.data_ptr, False), "version": 2}


def _view(tensor):
    return torch.as_tensor(_Shared(tensor), device="cuda")


class _Lent:
    """A torch tensor's memory as a buffer of the package; keeps the tensor alive."""

    def __init__(self, tensor):
        self.tensor, self.ptr = tensor, tensor.data_ptr()


def _lend(t, requires_grad=False):
    from tensorax_b200 import _C
    from tensorax_b200.tensor import Tensor
    dtype = "float16" if t.dtype == torch.float16 else "float32"
    return Tensor._wrap(_C.TensorImpl(list(t.shape), dtype, "cuda", buf=_Lent(t)), requires_grad)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dtype_code(_lib, case):
    return _lib.TX_DTYPE_F16 if case["dtype"] == "float16" else _lib.TX_DTYPE_F32


def _own_window(s):
    from tensorax_b200 import _lib
    case, f16 = s["case"], s["case"]["dtype"] == "float16"
    desc = _lib.SdpaDesc(q=s["q"].data_ptr(), k=s["k"].data_ptr(), v=s["v"].data_ptr(), mask=None,
                         kv_lens=s["dev_lens"].data_ptr(), out=s["out"].data_ptr(), batch=case["B"], q_heads=case["Hq"],
                         kv_heads=case["Hkv"], seq_q=case["Sq"], seq_k=case["Sk"], d_k=case["d"], d_v=case["d"],
                         dtype=_dtype_code(_lib, case), causal=1, flags=_lib.TX_SDPA_OUT_F16 if f16 else 0, stream=_stream(),
                         lse=None)
    win = _lib.WindowDesc(window=case["window"], sinks=case["sinks"], align_end=int(case["align"] == "end"))
    _lib.check(_lib.load().tx_sdpa_window_forward(ctypes.byref(desc), ctypes.byref(win)))
    return s["out"]


def _own_train(s):
    import tensorax_b200.functional as F
    case = s["case"]
    q, k, v = (_lend(s[n], True) for n in ("q", "k", "v"))
    out = F.scaled_dot_product_attention_window(q, k, v, case["window"], case["sinks"], kv_lens=s["lens"], align=case["align"],
                                                out_dtype="float16", grad_dtype="float16")
    out.backward(_lend(s["grad"]))
    return [_view(out), _view(q.grad), _view(k.grad), _view(v.grad)]


def _pages(_lib, s):
    case = s["case"]
    (k, v), (ks, vs) = s["codes"], s["scales"]
    return _lib.KvCache(k=k.data_ptr(), v=v.data_ptr(), k_scale=ks.data_ptr(), v_scale=vs.data_ptr(), pages=k.shape[0],
                        kv_heads=case["Hkv"], page_size=case["page"], d=case["d"],
                        format=_lib.TX_KV_INT8 if case["format"] == "int8" else _lib.TX_KV_E4M3)


def _own_cache(s):
    from tensorax_b200 import _lib
    case, lib, table = s["case"], _lib.load(), s["table"]
    common = dict(cache=_pages(_lib, s), page_table=table.data_ptr(), batch=case["B"], table_len=table.shape[1],
                  dtype=_dtype_code(_lib, case), stream=_stream())
    write = _lib.KvWriteDesc(k=s["k"].data_ptr(), v=s["v"].data_ptr(), start=s["start"].data_ptr(), tokens=case["T"], **common)
    _lib.check(lib.tx_kv_cache_write(ctypes.byref(write)))
    read = _lib.KvReadDesc(k=s["out_k"].data_ptr(), v=s["out_v"].data_ptr(), start=s["back_start"].data_ptr(),
                           counts=s["back_count"].data_ptr(), tokens=case["back"], **common)
    _lib.check(lib.tx_kv_cache_read(ctypes.byref(read)))
    return [s["out_k"], s["out_v"]]


def _own_tree(s):
    from tensorax_b200 import _lib
    case, table = s["case"], s["table"]
    desc = _lib.KvAttentionDesc(cache=_pages(_lib, s), q=s["q"].data_ptr(), out=s["out"].data_ptr(),
                                page_table=table.data_ptr(), kv_lens=s["kv_lens"].data_ptr(),
                                q_lens=s["q_lens"].data_ptr() if case["ragged"] else None,
                                tree=s["words"].data_ptr() if case["shape"] == "tree" else None, batch=case["B"],
                                q_heads=case["Hq"], tokens=case["T"], table_len=table.shape[1],
                                window=case["window"], sinks=case["sinks"],
                                dtype=_dtype_code(_lib, case),
                                flags=_lib.TX_SDPA_OUT_F16 if case["dtype"] == "float16" else 0, stream=_stream())
    _lib.check(_lib.load().tx_kv_cache_attention(ctypes.byref(desc)))
    return s["out"]


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"window": _own_window, "train": _own_train, "cache": _own_cache, "tree": _own_tree}[kind](s)
    return {"window": _plain_window, "train": _plain_window, "cache": _plain_cache, "tree": _plain_tree}[kind](s)


# ------------------------------------------------------------------ what a pass cannot do without
def _visible(rows, keys, window, sinks, first):
    """Pairs of a row and a key it sees: `rows` rows, the first at position `first`, `keys` keys."""
    pos = torch.arange(rows, dtype=torch.float64) + first
    upto = (pos + 1).clamp(0, keys)
    lo = (pos + 1 - window).clamp(min=0).minimum(upto) if window else torch.zeros_like(pos)
    return float((upto - lo + lo.clamp(max=sinks)).sum())


def work(case):
    B, Hkv, d, size = case["B"], case["Hkv"], case["d"], _SIZES[case["dtype"]]
    if case["kind"] == "cache":
        rows, back = B * Hkv * case["T"], B * Hkv * min(case["back"], (case["S"] + case["T"] + 1) // 2)
        return {"bytes": 2.0 * (rows + back) * (d * (size + 1) + 4), "flops": 4.0 * (rows + back) * d}
    Hq, window, sinks = case["Hq"], case["window"], case["sinks"]
    if case["kind"] == "tree":
        T, ctx = case["T"], 0.75 * case["S"]
        nodes = 0.75 * T if case["ragged"] else T
        keys = (min(ctx, window + sinks) if window else ctx) + nodes
        # a node sees the context and its ancestors, of which a tree has few
        pairs = B * Hq * nodes * (keys - nodes + (nodes / 2 if case["shape"] == "chain" else min(nodes, 6)))
        return {"bytes": B * Hkv * keys * (2.0 * d + 8) + 2.0 * B * Hq * nodes * d * size, "flops": 4.0 * pairs * d}
    # lengths uniform in [Sk/2, Sk] average three quarters of the keys
    Sq, Sk = case["Sq"], case["Sk"]
    keys = Sk if case["lens"] == "full" else 0.75 * Sk
    first = max(keys - Sq, 0) if case["align"] == "end" else 0
    attention = 4.0 * B * Hq * d * _visible(Sq, keys, window, sinks, first)
    read = keys if case["align"] == "start" else min(keys, Sq + window + sinks)
    rows_q, rows_k = B * Hq * Sq * d, B * Hkv * read * d
    if case["kind"] == "train":
        # out, dQ, dK, dV written in 16 bits, dO read in 32
        return {"bytes": size * (3 * rows_q + 2 * rows_k + 2 * B * Hkv * Sk * d) + 4.0 * rows_q, "flops": 3.5 * attention}
    return {"bytes": float(size * (2 * rows_q + 2 * rows_k)), "flops": attention}


# ------------------------------------------------------------------ the definitions, in 64 bits
def _exact_quantised(x, fmt):
    """The values that the codes of x stand for, row by row of the last dimension (inputs are finite)."""
    x = x.double()
    top = x.abs().max(dim=-1, keepdim=True).values
    if fmt == "int8":
        step = (top.float() / 127.0).clamp(min=2.0 ** -126).double()               # the scale is kept in 32 bits
        return torch.round(x / step) * step
    step = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(min=-126))
    y = x / step
    # four significant bits, and multiples of 2^-9 below 2^-6
    unit = torch.exp2((torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3).clamp(min=-9))
    return torch.round(y / unit) * unit * step


def _exact_stored(codes, scales, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).double() * scales.double().unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    B, d, Hkv, page = case["B"], case["d"], case["Hkv"], case["page"] if "page" in case else 0
    if case["kind"] == "cache":
        outs = [s["out_k"].double(), s["out_v"].double()]
        for i, new in enumerate((s["k"], s["v"])):
            fresh = _exact_quantised(new, case["format"])
            for b in range(B):
                first, count, start = int(s["back_start"][b]), int(s["back_count"][b]), int(s["start"][b])
                where = torch.arange(first, first + count, device="cuda")
                held = s["table"][b].long()[where // page]
                old = _exact_stored(s["codes"][i][held, :, where % page], s["scales"][i][held, :, where % page], case["format"])
                rows = old.permute(1, 0, 2).clone()
                written = where >= start
                rows[:, written] = fresh[b][:, where[written] - start]
                outs[i][b, :, :count] = rows
        return outs
    Hq, window, sinks = case["Hq"], case["window"], case["sinks"]
    G = Hq // Hkv
    if case["kind"] == "tree":
        out = s["out"].double()
        for b in range(B):
            total, nodes = int(s["kv_lens"][b]), int(s["q_lens"][b])
            ctx = total - nodes
            where = torch.arange(total, device="cuda")
            held = s["table"][b].long()[where // page]
            k, v = (_exact_stored(s["codes"][i][held, :, where % page], s["scales"][i][held, :, where % page],
                                  case["format"]).permute(1, 0, 2).repeat_interleave(G, 0) for i in range(2))
            hidden = torch.zeros((nodes, total), dtype=torch.bool, device="cuda")
            for t in range(nodes):
                word = int(s["words"][b, t]) % (1 << 64)
                depth = bin(word).count("1") - 1
                if window:
                    hidden[t, min(sinks, ctx): max(0, min(ctx, ctx + depth - window + 1))] = True
                for u in range(nodes):
                    hidden[t, ctx + u] = not word >> u & 1
            w = (torch.einsum("htd,hjd->htj", s["q"][b, :, :nodes].double(), k) / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[b, :, :nodes] = torch.einsum("htj,hjd->htd", torch.softmax(w, -1), v)
        return out
    train = case["kind"] == "train"
    outs = [s["q"].new_zeros((B, Hq, case["Sq"], d), dtype=torch.float64)]
    if train:
        outs += [torch.zeros_like(s[n], dtype=torch.float64) for n in ("q", "k", "v")]
    for b in range(B):
        n = s["lens"][b]
        i = torch.arange(case["Sq"], device="cuda").unsqueeze(1) + (n - case["Sq"] if case["align"] == "end" else 0)
        j = torch.arange(n, device="cuda").unsqueeze(0)
        hidden = (j > i) | ((j <= i - window) & (j >= sinks))
        dead = hidden.all(1, keepdim=True)                   # rows without a key: no value, no part in the gradients
        for h in range(Hkv):
            mine = slice(h * G, (h + 1) * G)
            q, k, v = (t.double().requires_grad_(train) for t in (s["q"][b, mine], s["k"][b, h, :n], s["v"][b, h, :n]))
            w = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden & ~dead, -math.inf), -1)
            o = w.masked_fill(dead, 0.0) @ v
            outs[0][b, mine] = o.detach().masked_fill(dead, math.nan)
            if train:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["grad"][b, mine].double())
                outs[1][b, mine], outs[2][b, h, :n], outs[3][b, h, :n] = gq, gk, gv
    return outs if train else outs[0]
