"""Attention with a sliding window and sinks on the device against its definition in 64 bits: every kernel that takes it, at the
sizes and masks where its tile lists begin and end."""
import ctypes

import numpy as np
import pytest

import tensorax_b200 as ts
import tensorax_b200.functional as F
import window_oracle
from conftest import seeded
from tensorax_b200 import _C, _lib
from tensorax_b200.nn import GroupedQueryAttention, QuantizedKVCache

pytestmark = pytest.mark.gpu


def tensor(x, requires_grad=False):
    return ts.Tensor._wrap(_C.from_numpy(np.ascontiguousarray(x)), requires_grad)


def run(q, k, v, window, sinks, lens, align, out_dtype="float32", flags=0):
    return _C.to_numpy(_C.scaled_dot_product_attention_window(
        *(_C.from_numpy(x) for x in (q, k, v)), window, sinks, align, kv_lens=lens, out_dtype=out_dtype, flags=flags))


def check(got, q, k, v, lens, window, sinks, align, tensor_cores, out16=False):
    """Every element within what the roundings can make of it.  Scores are sums of d products in fp32 (a matrix unit may
    lose 2^-23 of the sum of their sizes per addition): e in all, carried by a weight and by the sum of the weights.
    fp16: a weight is rounded to fp16, 2^-11 of it, the sum of unrounded weights divides; the polynomial exponential is off by
    1.6e-4 < 2^-12.5 in weight and sum alike.  fp32: pairs of fp16 numbers, 2^-21 in all.  2^-19 for exponents and sums.
    Weights more than 2^24 below the row's largest (and 2^8 for a maximum not yet raised) are lost: 2^-14 of |v| at most."""
    want, weight, size = window_oracle.forward(q, k, v, lens, window, sinks, align, with_size=True)
    f16 = q.dtype == np.float16
    assert (np.isnan(got) == np.isnan(want)).all(), np.argwhere(np.isnan(got) != np.isnan(want))[:4]
    e = size * (q.shape[-1] * 2.0 ** -23 * (1 if f16 or not tensor_cores else 3) + 2.0 ** -21)
    bound = weight * ((2.0 ** -11 + 2.0 ** -11.5 if f16 and tensor_cores else 2.0 ** -21) + 2 * e[..., None] + 2.0 ** -19) + 1e-30
    if f16 and tensor_cores:
        bound = bound + 2.0 ** -17 * np.abs(np.nan_to_num(v.astype(np.float64), posinf=0, neginf=0)).max()
    if out16:
        bound = bound + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    ok = np.abs(got.astype(np.float64) - want) <= bound
    assert ok[~np.isnan(want)].all(), np.nanmax(np.abs(got.astype(np.float64) - want) / bound)


CASES = [
    # B, Hq, Hkv, Sq, Sk, window, sinks, lens, align
    (1, 2, 2, 1, 1, 1, 0, None, "start"),
    (1, 2, 1, 300, 300, 1, 0, None, "start"),
    (2, 4, 2, 513, 513, 130, 3, [513, 260], "start"),        # one row behind two query tiles; padding
    (1, 2, 1, 700, 700, 64, 0, [200], "start"),              # rows behind the last key's window see nothing
    (1, 2, 1, 700, 700, 64, 1, [200], "start"),              # ... but the sink
    (1, 2, 2, 1000, 1000, 200, 300, None, "start"),          # sinks longer than the window, over several tiles
    (1, 1, 1, 385, 385, 100000, 5, None, "start"),           # a window longer than everything: causal
    (2, 2, 1, 200, 900, 150, 4, [900, 431], "end"),          # a chunk of a long prompt
    (1, 2, 1, 300, 300, 50, 2, [100], "end"),                # more rows than keys: the first stand before the sequence
    (2, 2, 2, 256, 1100, 256, 0, [1100, 0], "end"),          # a sequence without keys
    (1, 2, 1, 640, 256, 128, 7, None, "start"),              # more rows than keys
]


@pytest.mark.parametrize("d", [64, 128, 256, 512])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_fp16(case, d):
    B, Hq, Hkv, Sq, Sk, window, sinks, lens, align = CASES[case]
    q, k, v = seeded(case, B, Hq, Sq, d), seeded(50 + case, B, Hkv, Sk, d), seeded(90 + case, B, Hkv, Sk, d)
    q, k, v = (x.astype(np.float16) for x in (q, k, v))
    full = lens or [Sk] * B
    check(run(q, k, v, window, sinks, lens, align), q, k, v, full, window, sinks, align, True)
    check(run(q, k, v, window, sinks, lens, align, "float16"), q, k, v, full, window, sinks, align, True, True)
    if case in (2, 5, 7):
        check(run(q, k, v, window, sinks, lens, align, flags=_lib.TX_SDPA_FORCE_SIMT), q, k, v, full, window, sinks, align, False)


@pytest.mark.parametrize("d", [32, 64, 80, 128, 160])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_fp32(case, d):
    """Pairs of fp16 numbers up to d = 128, CUDA cores beyond; 1e-5, the fp32 path's tolerance on unit-variance data."""
    B, Hq, Hkv, Sq, Sk, window, sinks, lens, align = CASES[case]
    q, k, v = seeded(case, B, Hq, Sq, d), seeded(50 + case, B, Hkv, Sk, d), seeded(90 + case, B, Hkv, Sk, d)
    got = run(q, k, v, window, sinks, lens, align)
    check(got, q, k, v, lens or [Sk] * B, window, sinks, align, True)
    want = window_oracle.forward(q, k, v, lens or [Sk] * B, window, sinks, align)
    assert np.nanmax(np.abs(got - want), initial=0.0) <= 1e-5


STEPS = [
    # B, Hq, Hkv, Sq, Sk, window, sinks, lens
    (1, 1, 1, 1, 1, 1, 0, None),
    (3, 4, 1, 1, 1000, 100, 4, [1000, 0, 37]),
    (2, 8, 4, 1, 3000, 2000, 1, [2999, 1024]),
    (1, 2, 2, 1, 777, 5, 300, None),
    (2, 9, 3, 3, 500, 130, 2, [500, 2]),                      # a step of three tokens; a sequence of fewer keys than rows
    (40, 4, 2, 1, 600, 64, 4, "ramp"),                        # lengths brought to the device first
]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_decoding_step(case, d, dtype):
    """Few rows per K/V head, the last ones of their sequences: of a cache only the window and the sinks are read."""
    B, Hq, Hkv, Sq, Sk, window, sinks, lens = STEPS[case]
    if lens == "ramp":
        lens = [1 + (17 * i) % Sk for i in range(B)]
    q, k, v = (x.astype(dtype) for x in (seeded(case, B, Hq, Sq, d), seeded(50 + case, B, Hkv, Sk, d), seeded(90 + case, B, Hkv, Sk, d)))
    full = lens or [Sk] * B
    for b in range(B):                                       # what no row sees may be anything
        hidden = ~window_oracle.seen(Sq, Sk, full[b], window, sinks, "end").any(0)
        k[b][:, hidden], v[b][:, hidden] = np.nan, np.inf
    check(run(q, k, v, window, sinks, lens, "end"), q, k, v, full, window, sinks, "end", dtype == np.float16 and Sk < 128)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("align", ["start", "end"])
def test_few_rows_with_and_without_the_row_statistic(d, align):
    """The two kernels for few fp16 rows: the one that leaves the statistic for the backward, and the one that does not."""
    B, Hq, Hkv, Sq, Sk, window, sinks, lens = 2, 6, 2, 5, 300, 40, 3, [300, 123]
    q, k, v = (seeded(i, B, h, s, d).astype(np.float16) for i, (h, s) in enumerate(((Hq, Sq), (Hkv, Sk), (Hkv, Sk))))
    g = seeded(9, B, Hq, Sq, d)
    check(run(q, k, v, window, sinks, lens, align), q, k, v, lens, window, sinks, align, False)
    out, got = gradients(q, k, v, g, window, sinks, lens, align)
    check(out, q, k, v, lens, window, sinks, align, False)
    for name, a, b in zip("qkv", got, window_oracle.backward(q, k, v, g, lens, window, sinks, align)):
        assert np.linalg.norm(a - b) <= 2.0 ** -8 * np.linalg.norm(b), name
    half, _ = gradients(q, k, v, g, window, sinks, lens, align, "float16", "float16")
    assert np.abs(half.astype(np.float32) - out).max() <= 2.0 ** -11 * np.abs(out).max()


def test_what_lies_behind_the_last_key_may_be_anything():
    for d, dtype in ((64, np.float16), (128, np.float16), (256, np.float16), (64, np.float32), (160, np.float32)):
        q, k, v = (seeded(i, 2, 2, 400, d).astype(dtype) for i in range(3))
        lens = [333, 150]
        clean = run(q, k, v, 100, 4, lens, "start")
        for b in range(2):
            k[b, :, lens[b]:], v[b, :, lens[b]:] = np.nan, np.inf
        got = run(q, k, v, 100, 4, lens, "start")
        assert np.isfinite(got).all()
        if dtype == np.float16:
            assert np.array_equal(got, clean)
        check(got, q, k, v, lens, 100, 4, "start", dtype == np.float16 or d <= 128)


def test_a_window_of_everything_is_the_causal_mask():
    """Bit for bit, where the tiles are the same."""
    for d in (64, 128, 256):
        q, k, v = (_C.from_numpy(seeded(i, 2, 4, 700, d).astype(np.float16)) for i in range(3))
        a = _C.to_numpy(_C.scaled_dot_product_attention_ex(q, k, v, causal=True, kv_lens=[700, 300]))
        b = _C.to_numpy(_C.scaled_dot_product_attention_window(q, k, v, 2 ** 40, 2 ** 40, kv_lens=[700, 300]))
        assert np.array_equal(a, b)


# ------------------------------------------------------------------ gradients
TRAIN = [
    # B, Hq, Hkv, S, window, sinks, lens, align
    (1, 1, 1, 1, 1, 0, None, "start"),
    (2, 4, 2, 300, 64, 0, None, "start"),
    (2, 4, 1, 921, 100, 1, [921, 400], "start"),              # padding; sink tiles in a launch of their own
    (1, 2, 2, 700, 64, 0, [200], "start"),                    # rows that see nothing
    (1, 2, 1, 1500, 128, 200, None, "start"),                 # two tiles of sinks
    (1, 2, 2, 513, 100000, 0, None, "start"),
    (2, 2, 2, 260, 90, 3, [260, 0], "start"),
    (1, 2, 1, 400, 120, 2, [300], "end"),
]


def gradients(q, k, v, g, window, sinks, lens, align, grad_dtype="float32", out_dtype="float32"):
    tq, tk, tv = (tensor(x, True) for x in (q, k, v))
    out = F.scaled_dot_product_attention_window(tq, tk, tv, window, sinks, kv_lens=lens, align=align, out_dtype=out_dtype,
                                                grad_dtype=grad_dtype)
    out.backward(tensor(g))
    assert tq.grad.dtype == tk.grad.dtype == tv.grad.dtype == grad_dtype
    return out.numpy(), [t.grad.numpy() for t in (tq, tk, tv)]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(TRAIN)))
def test_gradients(case, d):
    """Operands (P, dO, dS) are rounded to fp16: 2^-11 each, so a product of two of them is off by 2^-10 of the sum of its
    terms' sizes; a gradient's norm is held to 2^-8 of the whole (their sum, the statistics', and what cancels in dP - D)."""
    B, Hq, Hkv, S, window, sinks, lens, align = TRAIN[case]
    q, k, v = (x.astype(np.float16) for x in (seeded(case, B, Hq, S, d), seeded(50 + case, B, Hkv, S, d), seeded(90 + case, B, Hkv, S, d)))
    g = seeded(7, B, Hq, S, d)
    full = lens or [S] * B
    want = window_oracle.backward(q, k, v, g, full, window, sinks, align)
    for grad_dtype, out_dtype in (("float32", "float32"), ("float16", "float16")):
        _, got = gradients(q, k, v, g, window, sinks, lens, align, grad_dtype, out_dtype)
        for name, a, b in zip("qkv", got, want):
            assert np.isfinite(a).all(), name
            norm = np.linalg.norm(b)
            # (a single key has the gradient zero in q and k: what is left there is the cancellation's rounding)
            assert np.linalg.norm(a - b) <= 2.0 ** -8 * max(norm, np.linalg.norm(g) * 2.0 ** -3), (name, np.linalg.norm(a - b) / max(norm, 1e-30))
            for n in range(B):                           # no part in anything: nothing, exactly
                see = window_oracle.seen(S, S, full[n], window, sinks, align)
                assert not a[n][:, ~see.any(1 if name == "q" else 0)].any(), name


SINKS = [
    # B, Hq, Hkv, Sq, Sk, window, sinks, lens, align: the sinks' tiles are seen by many more rows than the others
    (1, 4, 2, 1200, 1200, 64, 17, None, "start"),
    (2, 3, 1, 700, 700, 50, 64, [700, 9], "start"),           # fewer keys than sinks
    (1, 2, 1, 1200, 1200, 64, 65, None, "start"),
    (1, 6, 2, 601, 30, 8, 20, None, "start"),                 # rows far behind the last key
    (2, 2, 1, 900, 10, 4, 16, [10, 3], "start"),              # all keys are sinks
    (3, 2, 2, 640, 640, 32, 16, [640, 1, 0], "start"),
    (1, 2, 2, 500, 900, 40, 5, [800], "end"),
    (2, 2, 2, 500, 700, 40, 5, [700, 300], "end"),            # rows in front of the first key
]


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", range(len(SINKS)))
def test_gradients_of_sinks(case, d):
    """As test_gradients, the norm taken over the sinks' rows alone, then over the others."""
    B, Hq, Hkv, Sq, Sk, window, sinks, lens, align = SINKS[case]
    q, k, v = (x.astype(np.float16) for x in (seeded(case, B, Hq, Sq, d), seeded(50 + case, B, Hkv, Sk, d), seeded(90 + case, B, Hkv, Sk, d)))
    g, full = seeded(7, B, Hq, Sq, d), lens or [Sk] * B
    want = window_oracle.backward(q, k, v, g, full, window, sinks, align)
    _, got = gradients(q, k, v, g, window, sinks, lens, align)
    for name, a, b in zip("qkv", got, want):
        assert np.isfinite(a).all(), name
        for part in ((a, b),) if name == "q" else ((a[:, :, :sinks], b[:, :, :sinks]), (a[:, :, sinks:], b[:, :, sinks:])):
            norm = np.linalg.norm(part[1])
            if not norm:                                         # no such rows, or no part in anything
                assert not part[0].any(), name
                continue
            assert np.linalg.norm(part[0] - part[1]) <= 2.0 ** -8 * norm, (name, np.linalg.norm(part[0] - part[1]) / max(norm, 1e-30))


def test_what_lies_behind_the_last_key_has_no_part_in_gradients():
    for d in (64, 128, 256):
        q, k, v = (seeded(i, 2, 2, 400, d).astype(np.float16) for i in range(3))
        g, lens = seeded(5, 2, 2, 400, d), [333, 150]
        _, clean = gradients(q, k, v, g, 100, 4, lens, "start")
        for b in range(2):
            k[b, :, lens[b]:], v[b, :, lens[b]:] = np.nan, np.inf
        _, got = gradients(q, k, v, g, 100, 4, lens, "start")
        assert all(np.array_equal(a, b) for a, b in zip(got, clean))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens, align, sinks", [([200, 700], "start", 0), ([300, 0], "end", 2), ([690, 128], "end", 20)])
def test_gradients_of_rows_that_see_nothing_are_not_read(d, lens, align, sinks):
    """A loss over all rows hands the NaN of rows without keys back as their gradient: it goes nowhere."""
    B, H, S, window = 2, 2, 700, 64
    q, k, v = (seeded(i, B, H, S, d).astype(np.float16) for i in range(3))
    g = seeded(5, B, H, S, d)
    _, clean = gradients(q, k, v, g, window, sinks, lens, align)
    dead = np.stack([~window_oracle.seen(S, S, n, window, sinks, align).any(1) for n in lens])
    assert dead.any()
    for b in range(B):
        g[b][:, dead[b]] = np.nan
    _, got = gradients(q, k, v, g, window, sinks, lens, align)
    assert all(np.isfinite(a).all() and np.array_equal(a, b) for a, b in zip(got, clean))


def test_gradients_against_differences():
    """Central differences of the kernel's own forward pass, along random directions.  fp32 results of fp16 products: a loss
    of n terms is off by about 2^-11 sqrt(n) |g||o| / sqrt(n); the step is large enough for that to be a few per cent."""
    B, H, S, d, window, sinks = 1, 2, 200, 64, 40, 2
    q, k, v = (seeded(i, B, H, S, d).astype(np.float16) for i in range(3))
    g = seeded(5, B, H, S, d)
    _, grads = gradients(q, k, v, g, window, sinks, None, "start")
    rng = np.random.default_rng(0)
    for i, x in enumerate((q, k, v)):
        step = (rng.integers(0, 2, x.shape) * 2 - 1) * 2.0 ** -5
        pair = []
        for sign in (1, -1):
            moved = [q, k, v]
            moved[i] = (x.astype(np.float64) + sign * step).astype(np.float16)
            pair.append((moved[i].astype(np.float64), (run(*moved, window, sinks, None, "start").astype(np.float64) * g).sum()))
        along = (grads[i].astype(np.float64) * (pair[0][0] - pair[1][0])).sum()
        size = np.linalg.norm(grads[i]) * np.linalg.norm(pair[0][0] - pair[1][0]) / np.sqrt(x.size)
        assert abs((pair[0][1] - pair[1][1]) - along) <= 0.1 * abs(along) + 3 * size, (i, pair[0][1] - pair[1][1], along)


def test_the_same_bits_every_time():
    q, k, v = (seeded(i, 2, 4, 1000, 128).astype(np.float16) for i in range(3))
    g = seeded(5, 2, 4, 1000, 128)
    first = gradients(q, k, v, g, 200, 4, [1000, 600], "start")
    for _ in range(2):
        again = gradients(q, k, v, g, 200, 4, [1000, 600], "start")
        assert np.array_equal(first[0], again[0]) and all(np.array_equal(a, b) for a, b in zip(first[1], again[1]))


@pytest.mark.parametrize("d", [64, 128])
def test_forward_and_backward_in_a_graph_beside_an_eager_step(d):
    """A training step recorded in a graph and replayed on other inputs while the eager step's buffers live."""
    torch = pytest.importorskip("torch")
    lib, stream = _lib.load(), torch.cuda.Stream()
    B, H, S = 2, 4, 1100
    q, k, v = (torch.empty(B, H, S, d, device="cuda", dtype=torch.float16).normal_() for _ in range(3))
    g, out, lse = torch.randn(B, H, S, d, device="cuda"), torch.zeros(B, H, S, d, device="cuda"), torch.zeros(B, H, S, device="cuda")
    grads = [torch.zeros(B, H, S, d, device="cuda", dtype=torch.float16) for _ in range(3)]
    st = ctypes.c_void_p(stream.cuda_stream)
    fwd = _lib.SdpaDesc(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), batch=B, q_heads=H, kv_heads=H, seq_q=S,
                        seq_k=S, d_k=d, d_v=d, dtype=_lib.TX_DTYPE_F16, causal=1, stream=st, lse=lse.data_ptr())
    bwd = _lib.SdpaBwdDesc(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), dout=g.data_ptr(), lse=lse.data_ptr(),
                           dq=grads[0].data_ptr(), dk=grads[1].data_ptr(), dv=grads[2].data_ptr(), batch=B, q_heads=H, kv_heads=H,
                           seq_q=S, seq_k=S, d=d, causal=1, flags=_lib.TX_BWD_GRADS_F16, stream=st)
    win = _lib.WindowDesc(window=100, sinks=3)

    def call():
        _lib.check(lib.tx_sdpa_window_forward(ctypes.byref(fwd), ctypes.byref(win)))
        _lib.check(lib.tx_sdpa_window_backward(ctypes.byref(bwd), ctypes.byref(win)))

    torch.cuda.synchronize()
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        call()
    for _ in range(3):
        for t in (q, k, v, g):
            t.normal_()
        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        want = [t.clone() for t in (out, *grads)]
        for t in (out, *grads):
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, *grads), want))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_decoding_step_in_a_graph(d):
    """Recorded once, replayed as the sequences grow: lengths and queries are read when it runs."""
    torch = pytest.importorskip("torch")
    lib, stream = _lib.load(), torch.cuda.Stream()
    B, Hq, Hkv, S = 3, 8, 2, 500
    q = torch.empty(B, Hq, 1, d, device="cuda", dtype=torch.float16).normal_()
    k, v = (torch.empty(B, Hkv, S, d, device="cuda", dtype=torch.float16).normal_() for _ in range(2))
    out, lens = torch.zeros(B, Hq, 1, d, device="cuda"), torch.tensor([100, 1, 499], dtype=torch.int32, device="cuda")
    desc = _lib.SdpaDesc(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), kv_lens=lens.data_ptr(), out=out.data_ptr(), batch=B, q_heads=Hq,
                         kv_heads=Hkv, seq_q=1, seq_k=S, d_k=d, d_v=d, dtype=_lib.TX_DTYPE_F16, causal=1, stream=ctypes.c_void_p(stream.cuda_stream))
    win = _lib.WindowDesc(window=70, sinks=3, align_end=1)
    torch.cuda.synchronize()
    _lib.check(lib.tx_sdpa_window_forward(ctypes.byref(desc), ctypes.byref(win)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream, capture_error_mode="relaxed"):
        _lib.check(lib.tx_sdpa_window_forward(ctypes.byref(desc), ctypes.byref(win)))
    for step in range(4):
        q.normal_()
        lens.copy_(torch.tensor([100 + 100 * step, 1 + step, 499], dtype=torch.int32))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(out.cpu().numpy(), *(x.cpu().numpy() for x in (q, k, v)), lens.tolist(), 70, 3, "end", False)


# ------------------------------------------------------------------ as they are used
def test_prompt_in_chunks_then_steps():
    """A layer with a window: the whole prompt at once, the same in chunks against what has been kept, single tokens against
    plain buffers and against the quantised cache.  The quantised steps are off by the codes' rounding: int8 rows are within
    1/254 of their largest element (4 sigma here at most: 1/60), so scores and values move by a few per cent."""
    H, Hkv, S, d, window, sinks = 4, 2, 300, 64, 80, 4
    layer = GroupedQueryAttention(H, Hkv)
    q, k, v = (seeded(i, 1, (H, Hkv, Hkv)[i], S, d).astype(np.float16) for i in range(3))
    whole = layer.forward_bhsd(tensor(q), tensor(k), tensor(v), window=window, sinks=sinks).numpy()
    check(whole, q, k, v, [S], window, sinks, "start", True)
    for first, last in ((0, 128), (128, 290), (290, 299), (299, 300)):
        part = layer.forward_bhsd(tensor(q[:, :, first:last]), tensor(k), tensor(v), kv_lens=[last], window=window, sinks=sinks,
                                  align="end").numpy()
        assert np.abs(part - whole[:, :, first:last]).max() <= 2e-3
    cache = QuantizedKVCache(10, Hkv, d, 32, "int8")
    table = [list(range(10))]
    cache.write(tensor(k), tensor(v), table)
    step = layer.forward_cached(tensor(q[:, :, 299:]), cache, table, [300], window=window, sinks=sinks).numpy()
    assert np.abs(step - whole[:, :, 299:]).max() <= 0.05
    with pytest.raises(ValueError, match="head counts"):
        GroupedQueryAttention(4, 4).forward_cached(tensor(q[:, :, 299:]), cache, table, [300])
