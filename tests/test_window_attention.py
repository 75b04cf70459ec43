"""window.attention (kea_window_attention) against a dense softmax in 64 bits.

Bounds, u = 2^-24: a score is a dot product of d terms in FP32 scaled once, off by at most es = (d + 3) u scale sum |q k| + 3 u |s|;
a weight exp(s - max) by 2 es + 8 u of itself; the sums over n keys take n + 16 additions and rescalings of u each; for the
16-bit types the weights are rounded to the type (half a step h of themselves, and 2^-25 where FP16 has no smaller number, the
largest weight of a row being 1 or more before the division), in the sum as well as in the product at most; the output takes half
a step of its type. All of it applies to sum_j p_j |v_j|."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from kea_kernels import _hip, window

DEV = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def expected(q, k, v, left, right, sinks, lengths=None, starts=None, scale=None):
    """(the output in 64 bits, how far the kernel's may be from it), on the CPU; unseen keys are left out altogether."""
    dtype = q.dtype
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    b, tq, h, d = q.shape
    tk, hk = k.shape[1:3]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, err = torch.zeros(b, tq, h, d, dtype=torch.float64), torch.zeros(b, tq, h, d, dtype=torch.float64)
    hs = HALF_STEP[dtype]
    rounded = 0.0 if dtype == F32 else hs
    for i in range(b):
        n = tk if lengths is None else min(max(int(lengths[i]), 0), tk)
        at = n - tq if starts is None else int(starts[i])
        p = torch.arange(tq)[:, None] + at
        j = torch.arange(n)
        seen = torch.ones(tq, n, dtype=torch.bool)
        if right is not None:
            seen &= j <= p + right
        if left is not None:
            seen &= (j >= p - left) | (j < sinks)
        seen &= (p >= 0) & (p < n)
        used = seen.any(0)
        kk, vv, seen = k[i, :n][used], v[i, :n][used], seen[:, used]
        if not seen.any():
            continue
        for x in range(h):
            kx, vx = kk[:, x * hk // h], vv[:, x * hk // h]
            s = (q[i, :, x] @ kx.t()) * scale
            mag = (q[i, :, x].abs() @ kx.abs().t()) * abs(scale)
            w = torch.where(seen, s, torch.tensor(-math.inf, dtype=torch.float64))
            w = torch.nan_to_num(torch.softmax(w, 1))  # (rows that see nothing)
            es = torch.where(seen, (d + 3) * U * mag + 3 * U * s.abs(), torch.zeros(1, dtype=torch.float64)).amax(1, keepdim=True)
            o, a = w @ vx, w @ vx.abs()
            e = a * (2 * es + (len(kx) + 24) * U + 2 * rounded) * 1.05
            if dtype == F16:
                e = e + 2.0**-25 * (seen.double() @ vx.abs())
            out[i, :, x], err[i, :, x] = o, e + (o.abs() + e) * hs + (2.0**-25 if dtype == F16 else 1e-37) * seen.any(1, keepdim=True)
    return out, err


def check(got, want, err):
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off[err == 0] == 0).all()
    worst = (off / err.clamp_min(1e-300))[err > 0].max().item() if (err > 0).any() else 0.0
    assert worst <= 1, f"{worst:.3g} times the bound"


def heads(b, t, h, d, dtype, g, size=1.0):
    return (size * torch.randn(b, t, h, d, generator=g)).to(dtype).to(DEV)


WINDOWS = [(None, 0, 0), (None, None, 0), (0, 0, 0), (5, 0, 2), (16, 16, 1), (63, 0, 4), (64, 7, 70), (100, None, 3), (200, 3, 0), (0, 0, 1), (31, 40, 33)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t", [1, 2, 31, 33, 64, 65, 130, 300])
def test_whole_sequences(t, dtype):
    g = torch.Generator().manual_seed(t)
    for i, (left, right, sinks) in enumerate(WINDOWS):
        h, hk, d = [(2, 2, 64), (4, 1, 128), (6, 2, 80), (1, 1, 8), (3, 3, 256), (2, 1, 40)][(i + t) % 6]
        q, k, v = heads(2, t, h, d, dtype, g), heads(2, t, hk, d, dtype, g), heads(2, t, hk, d, dtype, g)
        got = window.attention(q, k, v, left=left, right=right, sinks=sinks)
        assert got.shape == q.shape and got.dtype == dtype
        check(got, *expected(q, k, v, left, right, sinks))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tq,tk,h,hk,d", [(1, 1, 4, 4, 64), (1, 77, 8, 2, 128), (1, 1000, 8, 1, 128), (3, 600, 4, 2, 64), (4, 4100, 4, 4, 128), (1, 5000, 2, 1, 256),
                                          (7, 333, 6, 3, 96), (20, 900, 16, 2, 64), (2, 3000, 33, 1, 32), (150, 1200, 4, 2, 128)])
def test_tokens_against_a_cache(tq, tk, h, hk, d, dtype):
    """Sequences of their own lengths (none, one, some, all), queries the last tokens; what the cache holds behind them is NaN."""
    g = torch.Generator().manual_seed(tq + tk)
    lengths = torch.tensor([0, 1, tk // 2 + 1, tk, max(1, tk - 3)], dtype=torch.int32)
    q, k, v = heads(5, tq, h, d, dtype, g), heads(5, tk, hk, d, dtype, g), heads(5, tk, hk, d, dtype, g)
    for i, n in enumerate(lengths.tolist()):
        k[i, n:] = float("nan")
        v[i, n:] = float("nan")
    for left, right, sinks in ((None, 0, 0), (255, 0, 4), (9, 0, 0), (2000, 0, 65), (0, 0, 1), (None, None, 0)):
        got = window.attention(q, k, v, left=left, right=right, sinks=sinks, kv_lengths=lengths.to(DEV))
        check(got, *expected(q, k, v, left, right, sinks, lengths))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_padded_clips_and_positions(dtype):
    """Padded clips (starts of zero), pieces in the middle of a sequence, queries partly or wholly outside it, lengths past the
    tensor: rows outside are zeros."""
    g = torch.Generator().manual_seed(1)
    q, k, v = heads(4, 90, 4, 64, dtype, g), heads(4, 150, 2, 64, dtype, g), heads(4, 150, 2, 64, dtype, g)
    for lengths, starts in (([90, 1, 0, 37], [0, 0, 0, 0]), ([150, 100, 120, 60], [10, 60, -40, 200]), ([1000, -5, 150, 150], [60, 0, -89, 149]),
                            ([150, 150, 150, 150], [2**31 - 1, -(2**31), -90, 150])):
        ln, st = torch.tensor(lengths, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32)
        for left, right, sinks in ((40, 0, 2), (16, 16, 0), (None, None, 0)):
            got = window.attention(q, k, v, left=left, right=right, sinks=sinks, kv_lengths=ln.to(DEV), q_starts=st.to(DEV))
            check(got, *expected(q, k, v, left, right, sinks, lengths, starts))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,tq", [(200, 200), (700, 1), (300, 5)])
def test_unseen_keys_have_no_part(t, tq, dtype):
    """NaN and infinities in keys and values reach the queries that see them and no others; the type's lowest and highest
    values among the seen ones are numbers like others."""
    g = torch.Generator().manual_seed(2)
    clean = [heads(1, n, 2, 64, dtype, g) for n in (tq, t, t)]
    q, k, v = (x.clone() for x in clean)
    bad = t - 60  # seen by positions bad .. bad + 20
    k[0, bad], v[0, bad] = float("nan"), float("inf")
    v[0, bad - 1, 0] = float("-inf")
    got = window.attention(q, k, v, left=20, right=0, sinks=1)[0].cpu()
    want, err = expected(*clean, 20, 0, 1)
    want, err = want[0], err[0]
    p = torch.arange(tq) + t - tq
    sees = ((p >= bad - 1) & (p <= bad + 20))
    assert got[~sees].isfinite().all() and ((got[~sees].double() - want[~sees]).abs() <= err[~sees]).all()
    if tq == t:
        assert got[(p >= bad) & (p <= bad + 20)].isnan().all() and (got[bad - 1, 0] == float("-inf")).all()
        assert got[bad - 1, 1].isfinite().all()
    v = clean[2].clone()
    v[0, bad] = torch.finfo(dtype).max
    v[0, bad + 1] = torch.finfo(dtype).min
    got = window.attention(q, clean[1], v, left=20, right=0, sinks=1)
    want, err = expected(clean[0], clean[1], v, 20, 0, 1)
    inside = want[0].abs().amax((1, 2)) < torch.finfo(dtype).max / 2
    assert ((got[0].cpu().double() - want[0]).abs() <= err[0])[inside].all()


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,tq", [(90, 90), (3000, 1)])
def test_seen_nan_scores_show(t, tq, dtype):
    """Keys of NaN alone (in one of several parts of the keys, too) make the rows that see one NaN, and only those."""
    g = torch.Generator().manual_seed(8)
    q, k, v = heads(3, tq, 2, 64, dtype, g), heads(3, t, 2, 64, dtype, g), heads(3, t, 2, 64, dtype, g)
    k[0, t - 70:t - 1] = float("nan")
    k[1, :] = float("nan")
    got = window.attention(q, k, v)
    assert got[:2, -1].isnan().all() and got[2].isfinite().all()
    clean = k.clone()
    clean[:2] = 0
    want, err = expected(q, clean, v, None, 0, 0)
    check(got[2:], want[2:], err[2:])
    if tq > 1:
        assert got[1].isnan().all()
        first = t - 70
        assert got[0, :first].isfinite().all() and got[0, first:].isnan().all()


MANY = [(60, 150, 4, 2, 64), (140, 150, 4, 2, 128), (260, 150, 2, 2, 80), (60, 150, 6, 2, 40), (130, 150, 4, 2, 256), (1, 2600, 8, 4, 64)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,h,hk,d", MANY)
def test_many_rows(b, t, h, hk, d, dtype):
    """Enough rows for the tiles of 128, which end in the middle of one: whole sequences, padded clips with NaN behind them,
    the last tokens of ragged ones."""
    g = torch.Generator().manual_seed(b + d)
    q, k, v = heads(b, t, h, d, dtype, g), heads(b, t, hk, d, dtype, g), heads(b, t, hk, d, dtype, g)
    check(window.attention(q, k, v, left=70, sinks=5), *expected(q, k, v, 70, 0, 5))
    lengths = torch.randint(0, t + 1, (b,), generator=g, dtype=torch.int32)
    lengths[:3] = torch.tensor([t, 0, 1], dtype=torch.int32)[:b]
    for i, n in enumerate(lengths.tolist()):
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    zeros = torch.zeros(b, dtype=torch.int32)
    for left, right, sinks, starts in ((20, 16, 1, zeros), (None, None, 0, zeros), (31, 0, 2, None)):
        got = window.attention(q, k, v, left=left, right=right, sinks=sinks, kv_lengths=lengths.to(DEV),
                               q_starts=None if starts is None else starts.to(DEV))
        check(got, *expected(q, k, v, left, right, sinks, lengths, starts))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_and_bad_values(dtype):
    """Tiles of 128 rows: infinities and NaN of keys and values reach the queries that see them and no others."""
    g = torch.Generator().manual_seed(12)
    b, t = 60, 150
    q, k, v = heads(b, t, 4, 64, dtype, g), heads(b, t, 2, 64, dtype, g), heads(b, t, 2, 64, dtype, g)
    want, err = expected(q, k, v, 20, 0, 1)
    bad = 90  # seen by positions 90 .. 110
    k[::2, bad], v[::2, bad], v[::2, bad - 1, 0] = float("nan"), float("inf"), float("-inf")
    got = window.attention(q, k, v, left=20, sinks=1).cpu()
    p = torch.arange(t)
    sees = (p >= bad - 1) & (p <= bad + 20)
    check(got[1::2], want[1::2], err[1::2])
    check(got[::2, ~sees], want[::2, ~sees], err[::2, ~sees])
    assert got[::2, bad:bad + 21].isnan().all() and (got[::2, bad - 1, :2] == float("-inf")).all()
    check(got[::2, bad - 1, 2:], want[::2, bad - 1, 2:], err[::2, bad - 1, 2:])


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(dtype):
    """Scores in the thousands (one key takes all), equal scores, a negative and a zero scale."""
    g = torch.Generator().manual_seed(3)
    q, k, v = heads(1, 140, 2, 64, dtype, g, 20), heads(1, 140, 2, 64, dtype, g, 20), heads(1, 140, 2, 64, dtype, g)
    for scale in (None, 0.0, -0.01, 3.0):
        for left, right, sinks in ((None, None, 0), (30, 0, 2)):
            check(window.attention(q, k, v, left=left, right=right, sinks=sinks, scale=scale),
                  *expected(q, k, v, left, right, sinks, scale=scale))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Slices of a fused projection, heads in front of tokens, keys shared by the batch (stride 0), an out of its own strides."""
    g = torch.Generator().manual_seed(4)
    b, t, h, d = 3, 70, 2, 64
    fused = torch.randn(b, t, 3 * h * d + 16, generator=g).to(dtype).to(DEV)
    q, k, v = (fused[..., i * h * d:(i + 1) * h * d].view(b, t, h, d) for i in range(3))
    check(window.attention(q, k, v, left=10, right=3, sinks=1), *expected(q, k, v, 10, 3, 1))
    q, k, v = (torch.randn(b, h, t, d, generator=g).to(dtype).to(DEV).transpose(1, 2) for _ in range(3))
    check(window.attention(q, k, v, left=10, sinks=1), *expected(q, k, v, 10, 0, 1))
    k, v = (x[:1].expand(b, t, h, d) for x in (k, v))
    base = torch.full((b, t + 1, h, d + 8), 3.0, dtype=dtype, device=DEV)
    out = base[:, :t, :, :d]
    got = window.attention(q, k, v, left=10, sinks=1, out=out)
    assert got.data_ptr() == out.data_ptr()
    check(out, *expected(q, k, v, 10, 0, 1))
    assert (base[:, t] == 3).all() and (base[..., d:] == 3).all()


@pytest.mark.gpu
@torch.inference_mode()
def test_offsets_past_32_bits():
    """Keys and values further apart than 2^31 bytes within a sequence, sequences more than 2^32 bytes apart."""
    g = torch.Generator().manual_seed(5)
    step, tk, d = 1 << 24, 150, 64  # 150 tokens 32 MiB apart: 4.9 GB
    base = torch.zeros(2 * tk * step + 64, dtype=F16, device=DEV)
    k, v = (base[o:].as_strided((2, tk, 1, d), (tk * step, step, d, 1)) for o in (0, 128))
    k.copy_(torch.randn(2, tk, 1, d, generator=g))
    v.copy_(torch.randn(2, tk, 1, d, generator=g))
    for tq in (1, 150):
        q = heads(2, tq, 2, d, F16, g)
        check(window.attention(q, k, v, left=70, sinks=3), *expected(q, k, v, 70, 0, 3))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("tq,tk", [(1, 2000), (130, 130)])
def test_captured_calls_replay(tq, tk):
    """Graphs on two streams at once with eager calls between them (each has a workspace of its own), lengths that move on
    between replays; the same bits every time."""
    g = torch.Generator().manual_seed(6)
    k, v = heads(2, tk, 2, 64, BF16, g), heads(2, tk, 2, 64, BF16, g)
    qs = [heads(2, tq, 8, 64, BF16, g) for _ in range(2)]
    lengths = torch.tensor([tk - 20, tk // 2], dtype=torch.int32, device=DEV)
    call = lambda q: window.attention(q, k, v, left=700, sinks=4, kv_lengths=lengths)  # noqa: E731
    call(qs[0])
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for q, stream in zip(qs, streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            outs.append(call(q))
        graphs.append(graph)
    for _ in range(4):
        want = [call(q).clone() for q in qs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        again = call(qs[0])
        torch.cuda.synchronize()
        assert torch.equal(again, want[0]) and torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        check(again, *expected(qs[0], k, v, 700, 0, 4, lengths.tolist()))
        lengths += 5


@pytest.mark.gpu
@torch.inference_mode()
def test_empty():
    q, k = torch.empty(0, 3, 2, 64, device=DEV), torch.empty(0, 3, 2, 64, device=DEV)
    assert window.attention(q, k, k).shape == (0, 3, 2, 64)
    q, k = torch.ones(2, 0, 2, 64, device=DEV), torch.ones(2, 3, 2, 64, device=DEV)
    assert window.attention(q, k, k).shape == (2, 0, 2, 64)
    q, k = torch.ones(2, 3, 2, 64, device=DEV), torch.ones(2, 0, 2, 64, device=DEV)
    assert not window.attention(q, k, k, left=4).any()


# ---- without a GPU -----------------------------------------------------------------------------------------------------------

def test_refusals():
    q, k = torch.zeros(2, 5, 4, 64), torch.zeros(2, 9, 2, 64)
    lengths = torch.zeros(2, dtype=torch.int32)
    for args, kw, message in [
        ((q[0], k, k), {}, "q must be"), ((q.double(), k, k), {}, "q must be"), ((q, k.half(), k), {}, "k must be"), ((q, k, k[:, :8]), {}, "v"),
        ((q, k[:1], k[:1]), {}, "k must be"), ((q, k[..., :32], k[..., :32]), {}, "k must be"), ((q[:, :, :3], k, k), {}, "multiple"),
        ((q[..., :60], k[..., :60], k[..., :60]), {}, "head size"), ((torch.zeros(1, 1, 1, 264),) * 3, {}, "head size"),
        ((torch.zeros(2, 5, 4, 66)[..., :64], k, k), {}, "16 bytes"), ((torch.zeros(2, 5, 64, 4).transpose(2, 3), k, k), {}, "16 bytes"),
        ((torch.zeros(2, 64, 4, 5).transpose(1, 3), k, k), {}, "16 bytes"), ((q, k, k), dict(left=-1), "left"), ((q, k, k), dict(right=1.5), "right"),
        ((q, k, k), dict(sinks=-2), "sinks"), ((q, k, k), dict(kv_lengths=lengths.long()), "kv_lengths"),
        ((q, k, k), dict(q_starts=lengths[:1]), "q_starts"), ((q, k, k), dict(out=torch.zeros(2, 5, 4, 64).half()), "out must be"),
        ((q, k, k), dict(out=torch.zeros(2, 1, 4, 64).expand(2, 5, 4, 64)), "share memory"), ((q, k, k), dict(out=q), "overlaps"),
        ((q, k, k), {}, "GPU"),
    ]:
        with pytest.raises(ValueError, match=message):
            window.attention(*args, **kw)
    with pytest.raises(RuntimeError, match="inference only"):
        window.attention(q.requires_grad_(), k, k)


def test_library_refusals():
    L = _hip.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    t = _hip.Heads(p, 64, 64, 64)
    good = dict(q=t, k=t, v=t, o=t, dt=0, b=1, tq=1, tk=1, h=2, hk=1, d=64, left=0, right=0, sinks=0, scale=1.0, ln=None, st=None, ws=None, wb=0,
                stream=None)
    for change, rc in [(dict(dt=3), -1), (dict(b=-1), -1), (dict(tk=(1 << 30) + 1), -1), (dict(h=3, hk=2), -1), (dict(hk=0), -1), (dict(d=12), -1),
                       (dict(d=264), -1), (dict(left=-1), -1), (dict(sinks=-1), -1), (dict(k=_hip.Heads(p + 4, 64, 64, 64)), -2),
                       (dict(o=_hip.Heads(p, 64, 66, 64)), -2), (dict(ln=p + 2), -2), (dict(q=_hip.Heads(None, 64, 64, 64)), -1), (dict(b=0), 0)]:
        assert L.kea_window_attention(*(good | change).values()) == rc, change
    assert L.kea_window_attention_workspace(0, 1, 1, 1, 3, 2, 64, 0, 0, 0) < 0


def test_a_scale_that_is_no_number_is_refused():
    q = torch.zeros(1, 0, 2, 64)
    for scale in (float("nan"), float("inf"), -float("inf"), 1e300):
        with pytest.raises(ValueError, match="scale"):
            window.attention(q, q, q, scale=scale)
    t, L = _hip.Heads(16, 64, 64, 64), _hip.lib()
    for scale in (float("nan"), float("inf")):
        assert L.kea_window_attention(t, t, t, t, 0, 0, 1, 1, 2, 1, 64, 0, 0, 0, scale, None, None, None, 0, None) == -1


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("tq", [1, 60])
def test_scales_at_the_end_of_the_range(tq):
    """A scale of zero weighs all keys alike whatever their products, one of 2^-126 and below is taken as it is. (Its product with
    log2(e) is off by at most 2^-150, 1.5 u of 2^-127, where a bound of u is counted: the sum of d products has 4 u to spare.)"""
    g = torch.Generator().manual_seed(21)
    q, k, v = heads(2, tq, 2, 64, F32, g, 2.0**60), heads(2, 70, 2, 64, F32, g, 2.0**60), heads(2, 70, 2, 64, F32, g)
    for scale in (0.0, 1.25 * 2.0**-126, -2.0**-127):
        want, err = expected(q, k, v, 30, 0, 1, scale=scale)
        check(window.attention(q, k, v, left=30, sinks=1, scale=scale), want, err)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_a_scale_of_zero(dtype):
    """The mean of what is seen, and NaN for a query that is no number."""
    g = torch.Generator().manual_seed(22)
    q, k, v = heads(2, 40, 2, 64, dtype, g, 100), heads(2, 40, 2, 64, dtype, g, 100), heads(2, 40, 2, 64, dtype, g)
    want, err = expected(q, k, v, 9, 0, 1, scale=0.0)
    q[0, 5, 1, 7], q[1, 9, 0, 3] = float("nan"), float("inf")
    got = window.attention(q, k, v, left=9, sinks=1, scale=0.0)
    bad = torch.zeros(2, 40, 2, dtype=torch.bool)
    bad[0, 5, 1] = bad[1, 9, 0] = True
    assert got[bad].isnan().all()
    check(got[~bad], want[~bad], err[~bad])


def test_any_number_of_first_tokens():
    """As many first tokens as an int64 says: the parts of the keys are those of all keys seen."""
    L = _hip.lib()
    want = L.kea_window_attention_workspace(2, 1, 1, 5000, 2, 2, 64, 10, 0, 5000)
    for sinks in (1 << 30, (1 << 63) - 1):
        assert L.kea_window_attention_workspace(2, 1, 1, 5000, 2, 2, 64, 10, 0, sinks) == want > 0


def test_an_out_over_the_lengths_is_refused():
    q, words = torch.zeros(2, 5, 4, 8), torch.zeros(400, dtype=torch.int32)
    out = words[:320].view(torch.float32).view(2, 5, 4, 8)
    for kw in (dict(kv_lengths=words[318:320]), dict(q_starts=words[:2])):
        with pytest.raises(ValueError, match="overlaps"):
            window.attention(q, q, q, out=out, **kw)
    with pytest.raises(ValueError, match="GPU"):
        window.attention(q, q, q, out=out, kv_lengths=words[320:322])


LN2 = 0.693147182464599609375  # in FP32; its FP32 product with log2(e) is 1, so that weights are 2^(s - max)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("tk,a,b", [(128, 3, 40), (128, 33, 100), (5000, 7, 4000), (5000, 2500, 33), (50000, 100, 49000)])
def test_parts_join_without_loss(tk, a, b, d):
    """Two keys count, in the parts of two waves or workgroups, the rest weigh 2^-200. Key a's score is 0 and key b's -x, so that the
    output is 1 for v = (1 at a, 0 at b) over 1 + 2^-x, and 2^-x over that for the reverse. x is a multiple of 2^-21 below 4: in FP32
    every difference of scores is exact, weights and the factor of a part are one exp2 of 2 u each, their products and sums u each:
    2^-x is off by 5 u, 1 + 2^-x by a third of that and u at most (x >= 1), then come three products or quotients of u, and u for
    2.7e-9 x in the exponent: 11 u. (Exponents rounded behind 2^4 or 2^5 would add 11 or 22.)"""
    g = torch.Generator().manual_seed(tk + a)
    h = d  # head i reads element i of the keys
    x = 1 + torch.randint(0, 3 * 2**21, (d,), generator=g) / 2**21
    q = torch.eye(h).view(1, 1, h, d).to(DEV)
    k = torch.full((1, tk, 1, d), -200.0)
    k[0, a], k[0, b] = 0, -x
    v = torch.zeros(1, tk, 1, d)
    v[0, a, 0, ::2], v[0, b, 0, 1::2] = 1, 1
    got = window.attention(q, k.to(DEV), v.to(DEV), scale=LN2)[0, 0].cpu().double()
    w = torch.exp2(-x.double())[:, None]
    want = torch.cat([1 / (1 + w), w / (1 + w)], 1).repeat(1, d // 2)
    worst = ((got - want).abs() / want).max().item() / U
    assert worst <= 11, f"{worst:.3g} u"


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 40, 128, 256])
@pytest.mark.parametrize("tq,tk", [(1, 100), (1, 6000), (30, 700), (300, 300)])
def test_small_values_keep_their_digits(tq, tk, d, dtype):
    """Values 2^100 smaller give an output 2^100 smaller to the bit: the scores are small, so that no weight is below 2^-10, and
    every product and sum stays a normal number."""
    g = torch.Generator().manual_seed(tk + d)
    q, k, v = heads(1, tq, 2, d, dtype, g, 0.25), heads(1, tk, 1, d, dtype, g), heads(1, tk, 1, d, dtype, g)
    want = window.attention(q, k, v)
    assert torch.equal(window.attention(q, k, v * 2.0**-100), want * 2.0**-100)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 40, 80, 128, 200, 256])
@pytest.mark.parametrize("b,t,tq", [(1, 300, 300), (1, 3000, 4), (2, 130, 130), (1, 100, 3), (40, 150, 150)])
def test_unseen_keys_leave_the_bits(b, t, tq, d, dtype):
    """NaN, infinities and the type's largest values in keys and values: who does not see them has the same bits as without them,
    in every form (tiles of 32 rows whose keys are shared out or split, of 128 rows, ragged heads); who does has their sum."""
    g = torch.Generator().manual_seed(t + d)
    q, k, v = heads(b, tq, 4, d, dtype, g), heads(b, t, 2, d, dtype, g), heads(b, t, 2, d, dtype, g)
    lengths = torch.full((b,), t - 10, dtype=torch.int32, device=DEV)
    starts = torch.full((b,), t - 10 - tq, dtype=torch.int32, device=DEV) if tq < t else torch.zeros(b, dtype=torch.int32, device=DEV)
    call = lambda k, v: window.attention(q, k, v, left=20, right=0, sinks=1, kv_lengths=lengths, q_starts=starts)  # noqa: E731
    want = call(k, v)
    p = torch.arange(tq) + int(starts[0])
    real = p < t - 10
    bad = t - 42 if tq == t else t - 33  # seen by positions bad .. bad + 20 (tq < t: the middle of the queries is the first)
    for at_k, at_v in ((float("nan"), float("inf")), (0.0, torch.finfo(dtype).max), (float("inf"), float("nan")), (0.0, -float("inf"))):
        k1, v1 = k.clone(), v.clone()
        k1[:, bad], v1[:, bad], v1[:, bad + 1] = at_k, at_v, at_v
        k1[:, t - 10:], v1[:, t - 10:] = float("nan"), float("inf")
        got = call(k1, v1)
        sees = (p >= bad) & (p <= bad + 21) & real
        assert torch.equal(got[:, ~sees], want[:, ~sees]), (at_k, at_v)
        if at_k == 0 and at_v > 0:  # two of the largest value: finite sums, within the bounds but for the last binade
            x, e = expected(q, k1[:, :t - 10], v1[:, :t - 10], 20, 0, 1, starts=starts.tolist())
            off = (got[:, sees].cpu().double() - x[:, sees]).abs() <= e[:, sees]
            assert (off | (x[:, sees].abs() > torch.finfo(dtype).max / 2)).all()
        elif at_k == 0:
            assert (got[:, sees] == at_v).all()
        else:
            first = sees & (p <= bad + 20)
            assert got[:, first].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 120, 256])
def test_unseen_keys_leave_the_bits_of_many_fp32_rows(d):
    """As above, with enough FP32 rows for the tiles of 128 (2560 of 32 rows, for heads over 64)."""
    test_unseen_keys_leave_the_bits(140, 150, 150, d, F32)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,tq,h,hk,d", [(2, 33, 1, 2, 1, 64), (2, 200, 200, 2, 2, 128), (2, 3000, 2, 2, 1, 64), (2, 2600, 2600, 8, 4, 80), (2, 90, 90, 2, 1, 256)])
def test_weights_add_up_to_one(b, t, tq, h, hk, d, dtype):
    """Values that are all c give c: the weights that the product takes are the ones that are summed. Every sixteenth key weighs 1,
    the others just less than halfway from 1/2 to the 16-bit type's next number: rounded to 1/2, all sums are exact (fewer than 2^12
    keys, c of 11 bits at most), and the quotient is off by 2 u. (The weights as they were would add up to 2^-8.2 more in BF16, and
    c is just below 2.) In FP32 either sum is off by t + 16 roundings of u at most."""
    x = {BF16: 0.50194, F16: 0.50024, F32: 0.3}[dtype]
    q, k = torch.zeros(b, tq, h, d), torch.zeros(b, t, hk, d)
    q[..., 0], k[..., 0] = 1, -1
    k[:, ::16, :, 0] = 0
    for c in (2 - torch.finfo(dtype).eps, 1.0, -3.96875):
        v = torch.full((b, t, hk, d), c)
        got = window.attention(q.to(dtype).to(DEV), k.to(dtype).to(DEV), v.to(dtype).to(DEV), scale=-math.log(x), right=None)
        if dtype == F32:
            assert ((got - c).abs() <= abs(c) * 2 * (t + 20) * U).all()
        else:
            assert (got == c).all()
