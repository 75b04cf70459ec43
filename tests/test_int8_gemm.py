"""int8.gemm and Int8Linear (kea_int8_gemm): int8 rows x int8 weights with scales for each token and channel, against exact
integer sums and the epilogue in 64 bits.

Bounds: u = 2^-24 is half a step of FP32. The sum is exact; r = f(acc) * s * a + b takes a conversion, a product and a fused
multiply-add, so it is within u * (3 |v| + |v + b|) of the exact value (v = acc s a); SiLU on the hardware's exp2 and
reciprocal (a step of 2^-23 each, the exponent's argument two more times |r|) adds |silu| (|r| + 4) 2^-23 and passes r's own
error on with a slope of at most 1.1; the residual adds two roundings; the output half a step of its type (and half the
smallest subnormal of FP16, 2^-25)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from kea_kernels import _hip, int8, lowbit

DEV = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def make(m, n, k, seed, scales=torch.float32, extreme=False):
    """q int8 [1, M, ldq], qs, w int8 [N, K] view of padded rows, ws; the bytes behind K hold garbage."""
    g = torch.Generator().manual_seed(seed)
    ldq, ldw = lowbit.round_up(k, 16), lowbit.round_up(k, 16) + 16 * (seed % 2)
    q = torch.randint(-128, 128, (1, m, ldq), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, ldw), generator=g, dtype=torch.int8)
    if extreme:
        q[:, ::2, :k], w[:, :k] = -128, -128
    qs = (torch.rand(1, m, generator=g) * 0.02 + 1e-3).to(scales)
    ws = (torch.rand(n, generator=g) * 0.02 + 1e-3).to(scales)
    return q.to(DEV), qs.to(DEV), w.to(DEV)[:, :k], ws.to(DEV)


def sums(q, w):
    k = w.shape[1]
    a, b = q.reshape(-1, q.shape[-1])[:, :k].cpu().numpy().astype(np.int32), w.cpu().numpy().astype(np.int32)
    return torch.from_numpy(a.astype(np.float64) @ b.astype(np.float64).T)  # exact: below 2^53


def expected(q, qs, w, ws, bias, silu, residual, factor, dtype):
    """The value in 64 bits and how far the kernel's may be from it."""
    v = sums(q, w) * qs.cpu().double().reshape(-1, 1) * ws.cpu().double()
    b = torch.zeros(1, dtype=torch.float64) if bias is None else bias.cpu().double()
    r = v + b
    err = U * (3 * v.abs() + r.abs())
    if silu:
        s = r / (1 + torch.exp(-r))
        err = 1.1 * err + s.abs() * (r.abs() + 4) * 2 * U
        r = s
    if residual is not None:
        y = residual.cpu().double() + factor * r
        err = factor * err + U * ((factor * r).abs() + y.abs())
        r = y
    err = err + (r.abs() + err) * HALF_STEP[dtype] + (2.0**-25 if dtype == torch.float16 else 2.0**-149)
    return r, err


def check(out, want, err):
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    worst = ((out - want).abs() / err).max().item()
    assert worst <= 1, f"{worst:.3g} times the bound"


# every path of the kernel: single rows, ragged tiles on both sides, k below, at and past a step of 64 / 128, long k
SIZES = [(1, 1, 1), (1, 17, 16), (1, 640, 2560), (1, 2560, 640), (2, 130, 63), (3, 1030, 641), (5, 64, 65), (15, 256, 129), (16, 1024, 4096),
         (17, 33, 127), (31, 48, 1000), (33, 1030, 640), (64, 64, 128), (65, 129, 257), (100, 300, 4100), (125, 1024, 1024),
         (128, 128, 64), (129, 255, 192), (200, 512, 2048), (257, 513, 1025), (300, 4096, 320), (375, 1030, 641), (1000, 256, 512),
         (1000, 1024, 1024), (2049, 130, 96), (4100, 1025, 160), (2000, 4096, 1024)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sums_are_exact(m, n, k):
    q, _, w, _ = make(m, n, k, m + n + k)
    got = int8.gemm(q, None, w, None, out_dtype=torch.int32)
    assert torch.equal(got.cpu().double(), sums(q, w))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(2, 3, 131071), (70, 130, 131071), (300, 300, 60000)])
def test_the_largest_sums_are_exact(m, n, k):
    q, _, w, _ = make(m, n, k, 7, extreme=True)
    got = int8.gemm(q, None, w, None, out_dtype=torch.int32)
    assert torch.equal(got.cpu().double(), sums(q, w))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(6000, 2050, 641), (1500, 10243, 641), (2500, 5121, 1000), (1000, 2050, 1500), (8001, 257, 1500), (500, 5121, 1500)])
def test_the_widest_tiles(m, n, k):
    """Sizes that take tiles of 256 x 256, or four stages ahead, with ragged edges: the sums, and the epilogue's types."""
    q, qs, w, ws = make(m, n, k, m)
    want = sums(q, w)
    assert torch.equal(int8.gemm(q, None, w, None, out_dtype=torch.int32).cpu().double(), want)
    bias, residual = torch.linspace(-3, 3, n, device=DEV), torch.linspace(-2, 2, m * n, device=DEV).view(m, n)
    for b, silu, res, dtype in ((bias, True, None, torch.bfloat16), (None, False, residual, torch.float32), (bias, False, None, torch.float16)):
        rows = slice(m - 300, m)  # (the first and last rows: all have the sums of above)
        got = int8.gemm(q, qs, w, ws, b, out_dtype=dtype, silu=silu, residual=res, residual_factor=0.5)
        check(got[rows], *expected(q[:, rows], qs[:, rows], w, ws, b, silu, None if res is None else res[rows], 0.5, dtype))
        check(got[:300], *expected(q[:, :300], qs[:, :300], w, ws, b, silu, None if res is None else res[:300], 0.5, dtype))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("scales", [torch.float32, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 2560, 640), (16, 1024, 4096), (33, 1030, 641), (257, 513, 1025), (1000, 1024, 1024)])
def test_epilogue(m, n, k, dtype, scales):
    q, qs, w, ws = make(m, n, k, m + k, scales)
    g = torch.Generator().manual_seed(n)
    bias = torch.randn(n, generator=g).to(scales).to(DEV)
    residual = torch.randn(m, n, generator=g).to(DEV)
    for b, silu, res in ((None, False, None), (bias, False, None), (bias, True, None), (None, True, residual), (bias, False, residual)):
        got = int8.gemm(q, qs, w, ws, b, out_dtype=dtype, silu=silu, residual=res, residual_factor=0.5)
        assert got.dtype == dtype and tuple(got.shape) == (m, n)
        check(got, *expected(q, qs, w, ws, b, silu, res, 0.5, dtype))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(3, 70, 90), (40, 130, 260), (300, 260, 1000)])
def test_views_stay_inside_their_rows(m, n, k):
    """q with spare rows and columns, strided out and residual: what lies between the rows is left as it was."""
    q, qs, w, ws = make(m, n, k, 3)
    wide = torch.zeros(m + 2, q.shape[2] + 48, dtype=torch.int8, device=DEV)
    wide[:m, :q.shape[2]] = q[0]
    base = torch.full((m + 1, n + 5), 7.0, device=DEV)
    out, res = base[:m, 2:n + 2], torch.randn(m, n + 3, device=DEV)[:, :n]
    want, err = expected(q, qs, w, ws, None, False, res, 1.0, torch.float32)
    got = int8.gemm(wide[:m], qs, w, ws, out=out, residual=res)
    assert got.data_ptr() == out.data_ptr()
    check(out, want, err)
    assert (base[m] == 7).all() and (base[:, :2] == 7).all() and (base[:, n + 2:] == 7).all()
    res = res.contiguous()
    int8.gemm(q, qs, w, ws, out=res, residual=res)  # in place
    check(res, want, err)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(3, 70, 90), (40, 131, 260), (300, 267, 1000), (600, 1031, 128)])
def test_outputs_at_any_alignment(m, n, k, dtype):
    """Rows of out and of the residual that start at odd elements and lie an odd number of elements apart."""
    q, qs, w, ws = make(m, n, k, 5)
    base = torch.full((m + 1, n + 4), 7.0, device=DEV).to(dtype)[:, :n + 3]
    base = base.contiguous() if n % 2 == 0 else torch.full((m + 1, n + 2), 7.0, device=DEV).to(dtype)
    out, res = base[:m, 1:n + 1], torch.randn(m, n + 3, device=DEV)[:, 3:]
    int8.gemm(q, qs, w, ws, out=out, residual=res, residual_factor=-2.0)
    want, err = expected(q, qs, w, ws, None, False, res, -2.0, dtype)
    check(out, want, err.abs() + 4 * U * (want - res.cpu().double()).abs())
    assert (base[m] == 7).all() and (base[:, 0] == 7).all() and (base[:, n + 1:] == 7).all()


@pytest.mark.gpu
@torch.inference_mode()
def test_rows_far_apart():
    """Leading dimensions that 32-bit offsets within a tile do not reach."""
    far = 1 << 24
    base = torch.zeros(130 * far, dtype=torch.int8, device=DEV)
    q = base.as_strided((130, 200), (far, 1))
    q.copy_(torch.randint(-128, 128, (130, 200), dtype=torch.int8))
    w = torch.randint(-128, 128, (140, 208), dtype=torch.int8).to(DEV)[:, :200]
    assert torch.equal(int8.gemm(q, None, w, None, out_dtype=torch.int32).cpu().double(), sums(q, w))


@pytest.mark.gpu
@torch.inference_mode()
def test_offsets_past_32_bits():
    """Rows of q and out beyond 2^31 bytes."""
    k, n, m = 4096, 32, 600000
    q = torch.zeros(m, k, dtype=torch.int8, device=DEV)
    q[-3:] = torch.randint(-128, 128, (3, k), dtype=torch.int8, device=DEV)
    w = torch.randint(-128, 128, (n, k), dtype=torch.int8, device=DEV)
    got = int8.gemm(q, None, w, None, out_dtype=torch.int32)
    assert torch.equal(got[-3:].cpu().double(), sums(q[-3:], w)) and not got[:-3].any()
    base = torch.zeros(3, 1 << 30, dtype=torch.float32, device=DEV)  # rows of out 2^32 bytes apart
    one = torch.ones(3, device=DEV)
    int8.gemm(q[-3:].contiguous(), one, w, torch.ones(n, device=DEV), out=base[:, 5:5 + n])
    assert torch.equal(base[:, 5:5 + n].cpu().double(), sums(q[-3:], w))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(1, 2560, 640), (16, 1024, 4096), (300, 512, 2048)])
def test_captured_calls_replay(m, n, k):
    """Two graphs of the same shape on two streams, replayed at once and with eager calls between, give the eager bits."""
    q, qs, w, ws = make(m, n, k, 11)
    other = make(m, n, k, 12)[0]
    want = [int8.gemm(x, qs, w, ws).clone() for x in (q, other)]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, stream in zip((q, other), streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                outs.append(int8.gemm(x, qs, w, ws))
            graphs.append(graph)
    for _ in range(5):
        for out in outs:
            out.fill_(-1)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = int8.gemm(q, qs, w, ws)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0])
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.gpu
@torch.inference_mode()
def test_linear_layer():
    """Int8Linear.linear is the quantizer and the product: the sums of its own int8 rows, within the epilogue's bound."""
    g = torch.Generator().manual_seed(0)
    dense = torch.randn(130, 271, generator=g)
    layer = int8.Int8Linear.from_dense(dense, torch.randn(130, generator=g), DEV)
    back = layer.weight.cpu().double() * layer.scale.cpu().double()[:, None]
    assert ((back - dense.double()).abs() <= layer.scale.cpu().double()[:, None] * (0.5 + 1e-4)).all()
    for x in (torch.randn(271, generator=g), torch.randn(7, 271, generator=g), torch.randn(2, 5, 271, generator=g)):
        x = x.to(DEV)
        rows = x.reshape(-1, 271)
        q, qs, _ = lowbit.quantize(rows[None], (0, 271, 1, rows.shape[0]), rows.shape[0], 271, 1)
        for dtype in (torch.float32, torch.bfloat16):
            y = layer.linear(x, activation="silu", out_dtype=dtype)
            assert y.shape == (*x.shape[:-1], 130)
            check(y.reshape(-1, 130), *expected(q, qs, layer.weight, layer.scale, layer.bias, True, None, 1.0, dtype))
    for empty in ((0, 271), (2, 0, 271), (0, 3, 271)):
        assert layer.linear(torch.empty(empty, device=DEV)).shape == (*empty[:-1], 130)
    norm = torch.nn.LayerNorm(271, device=DEV)
    x = torch.randn(4, 271, generator=g).to(DEV)
    q, qs, _ = lowbit.quantize(x[None], (0, 271, 1, 4), 4, 271, 1, norm=norm, input_activation="silu")
    assert torch.equal(layer.linear(x, norm=norm, input_activation="silu"), int8.gemm(q, qs, layer.weight, layer.scale, layer.bias))


@pytest.mark.gpu
@torch.inference_mode()
def test_empty_rows_and_unaligned_views_on_the_gpu():
    q, qs, w, ws = make(4, 8, 32, 1)
    assert int8.gemm(q[:, :0], qs[:, :0], w, ws).shape == (0, 8)
    flat = torch.zeros(4 * 48 + 1, dtype=torch.int8, device=DEV)
    with pytest.raises(ValueError, match="16 bytes"):
        int8.gemm(flat[1:].view(4, 48), qs, w, ws)


@pytest.mark.gpu
@torch.inference_mode()
def test_a_layer_owns_its_weight():
    w = torch.randint(-128, 128, (40, 64), dtype=torch.int8).to(DEV)
    scale, bias, x = torch.ones(40, device=DEV), torch.zeros(40, device=DEV), torch.randn(3, 64, device=DEV)
    layer = int8.Int8Linear.prepare(w, scale, bias, DEV)
    want = layer.linear(x)
    w.zero_(), scale.zero_(), bias.fill_(1)
    assert torch.equal(layer.linear(x), want)


@pytest.mark.gpu
@torch.inference_mode()
def test_one_row_of_any_stride_and_out_beside_the_residual():
    q, qs, w, ws = make(4, 70, 200, 9)
    want = int8.gemm(q, qs, w, ws)
    one = torch.as_strided(q, (1, q.shape[2]), (100, 1), 0)
    assert torch.equal(int8.gemm(one, qs[:, :1], w, ws), want[:1])
    both = torch.zeros(4, 140, device=DEV)
    both[:, :70] = 1
    int8.gemm(q, qs, w, ws, out=both[:, 70:], residual=both[:, :70])
    assert torch.equal(both[:, 70:], int8.gemm(q, qs, w, ws, residual=torch.ones(4, 70, device=DEV))) and (both[:, :70] == 1).all()


# ---- without a GPU -----------------------------------------------------------------------------------------------------------

def test_an_output_that_overlaps_is_refused():
    q, qs, w, ws = _cpu()
    far = torch.zeros(64, 8)
    for out, kw in ((far[:4], dict(residual=far[1:5])), (far.view(32, 16)[:4, :8], dict(residual=far.view(32, 16)[:4, 4:12])),
                    (far[:1], dict(residual=far.view(-1)[4:12].view(1, 8)))):
        with pytest.raises(ValueError, match="shares memory"):
            int8.gemm(q[:, :out.shape[0]], qs[:, :out.shape[0]], w, ws, out=out, **kw)
    words = torch.zeros(64, dtype=torch.int32)
    with pytest.raises(ValueError, match="shares memory"):
        int8.gemm(words.view(torch.int8)[:128].view(4, 32), None, w, None, out=words[16:48].view(4, 8))
    with pytest.raises(ValueError, match="GPU"):
        int8.gemm(q, qs, w, ws, out=far[:4], residual=far[:4])
    with pytest.raises(ValueError, match="8192"):
        int8.Int8Linear.prepare(torch.zeros(4, 8193, dtype=torch.int8), torch.ones(4), None, "cuda:0")


def _cpu(m=4, n=8, k=32):
    return (torch.zeros(1, m, k, dtype=torch.int8), torch.ones(1, m), torch.zeros(n, k, dtype=torch.int8), torch.ones(n))


def test_refusals():
    q, qs, w, ws = _cpu()
    bad = [
        (dict(q=q.expand(2, 4, 32)), "one activation part"), (dict(q=q.float()), "int8"), (dict(w=w.short()), "int8"),
        (dict(w=torch.zeros(8, 48, dtype=torch.int8)), "elements"), (dict(qs=torch.ones(1, 5)), "qs"),
        (dict(qs=torch.ones(1, 4, dtype=torch.bfloat16)), "qs"), (dict(qs=None), "qs"), (dict(ws=torch.ones(9)), "wscale"),
        (dict(ws=torch.ones(16)[::2]), "wscale"), (dict(bias=torch.ones(7)), "bias"),
        (dict(w=torch.zeros(8, 33, dtype=torch.int8)[:, :32]), "16 bytes"), (dict(w=torch.zeros(32, 16, dtype=torch.int8).t()), "column"),
        (dict(residual=torch.zeros(4, 8, dtype=torch.float16)), "residual"), (dict(residual=torch.zeros(4, 9)), "residual"),
        (dict(out=torch.zeros(4, 9)), "out"), (dict(out=torch.zeros(8, 4).t()), "out"), (dict(out=torch.zeros(1, 8).expand(4, 8)), "out"),
        (dict(out_dtype=torch.float64), "dtype"), (dict(out_dtype=torch.int32, silu=True), "int32"),
        (dict(w=torch.zeros(8, 0, dtype=torch.int8)), "K"), (dict(w=torch.zeros(0, 32, dtype=torch.int8)), "N >= 1"),
        (dict(), "run on the GPU"),
    ]
    for change, message in bad:
        a = dict(q=q, qs=qs, w=w, ws=ws, bias=None) | change
        with pytest.raises(ValueError, match=message):
            int8.gemm(a.pop("q"), a.pop("qs"), a.pop("w"), a.pop("ws"), a.pop("bias"), **a)
    with pytest.raises(RuntimeError, match="inference only"):
        int8.gemm(q, qs.requires_grad_(), w, ws)


def test_a_last_row_that_ends_inside_16_bytes_is_refused():
    q, qs, _, ws = _cpu(k=20)
    rows = torch.zeros(8 * 32 - 12, dtype=torch.int8)
    with pytest.raises(ValueError, match="16 bytes"):
        int8.gemm(q.new_zeros(1, 4, 32), qs, rows.as_strided((8, 20), (32, 1)), ws)
    w = int8.pad_rows(torch.arange(160).to(torch.int8).view(8, 20))
    assert w.stride(0) == 32 and torch.equal(w.reshape(-1), torch.arange(160).to(torch.int8))
    assert int8.pad_rows(w).data_ptr() == w.data_ptr()
    one = torch.zeros(20, dtype=torch.int8).view(1, 20)
    assert int8.pad_rows(one).untyped_storage().nbytes() == 32


def test_library_refusals():
    """kea_int8_gemm checks sizes, types and alignment before anything is launched."""
    L = _hip.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    good = dict(q=p, ldq=32, qs=p, qd=0, w=p, ldw=32, ws=p, wd=0, b=None, bd=0, y=p, yd=0, ldy=8, r=None, ldr=0, f=1.0, m=4, n=8,
                k=32, flags=0, stream=None)
    for change, rc in [(dict(k=0), -1), (dict(k=131072), -1), (dict(n=0), -1), (dict(m=-1), -1), (dict(ldq=16), -1), (dict(ldy=7), -1),
                       (dict(yd=4), -1), (dict(yd=3, flags=1), -1), (dict(yd=3, r=p, ldr=8), -1), (dict(flags=2), -1), (dict(qd=2), -1),
                       (dict(b=p, bd=2), -1), (dict(q=None), -1), (dict(qs=None), -1), (dict(q=p + 4), -2), (dict(ldw=40), -2),
                       (dict(y=p + 2), -2), (dict(r=p, ldr=4), -1), (dict(m=0), 0), (dict(n=1 << 31), -1)]:
        assert L.kea_int8_gemm(*(good | change).values()) == rc, change


def test_linear_refusals():
    for args in ((torch.zeros(4, 8), torch.ones(4), None), (torch.zeros(4, 8, dtype=torch.int8), torch.ones(5), None),
                 (torch.zeros(4, 8, dtype=torch.int8), torch.full((4,), float("nan")), None)):
        with pytest.raises(ValueError):
            int8.Int8Linear.prepare(*args, "cuda:0")
    with pytest.raises(ValueError, match="GPU devices only"):
        int8.Int8Linear.prepare(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4), None, "cpu")
    with pytest.raises(ValueError, match="finite"):
        int8.Int8Linear.from_dense(torch.full((2, 2), float("inf")))


class _Gpu1:
    type, index = "cuda", 1


def test_launches_are_made_from_the_tensors_device(monkeypatch):
    """on_device switches to a GPU that is not the current one, whose default stream the handle 0 would otherwise name."""
    entered = []

    class Guard:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            entered.append(self.d.index)

        def __exit__(self, *_):
            pass

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    with _hip.on_device(_Gpu1()):
        assert entered == [1]
    with _hip.on_device(torch.device("cuda", 0)):
        assert entered == [1]


def test_a_norm_that_requires_grad_is_refused():
    layer = int8.Int8Linear(torch.zeros(4, 16, dtype=torch.int8), torch.ones(4), None)
    with pytest.raises(RuntimeError, match="inference only"):
        layer.linear(torch.zeros(2, 16), norm=torch.nn.LayerNorm(16))
    with pytest.raises(RuntimeError, match="inference only"):
        layer.linear(torch.zeros(0, 16), norm=torch.nn.LayerNorm(16))
    assert layer.linear(torch.zeros(0, 16), norm=torch.nn.LayerNorm(16).requires_grad_(False)).shape == (0, 4)


@pytest.mark.parametrize("n,k,ld,offset", [(2, 10, 16, 0), (5, 20, 32, 0), (3, 1, 16, 0), (2, 16, 32, 16), (1, 10, 16, 0), (4, 31, 48, 32)])
def test_pad_rows_gives_what_gemm_takes(n, k, ld, offset):
    """Rows whose storage ends with the last one's elements, short of 16 bytes, are copied; with the bytes there they are not."""
    for tail, kept in ((0, k % 16 == 0), (lowbit.round_up(k, 16) - k, True)):
        flat = torch.arange(offset + (n - 1) * ld + k + tail).to(torch.int8)
        w = flat.as_strided((n, k), (ld, 1), offset)
        rows = int8.pad_rows(w)
        assert torch.equal(rows, w) and (rows.data_ptr() == w.data_ptr()) == kept
        q, qs, _, ws = _cpu(k=lowbit.round_up(k, 16), n=n)
        with pytest.raises(ValueError, match="GPU"):  # all that is left to refuse
            int8.gemm(q, qs, rows, ws)
