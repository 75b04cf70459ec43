"""int4.gemm, int4.pack and Int4Linear (kea_int4_gemm): int8 rows x 4-bit weights with scales for each token and each group of a
row's weights, against the definition in 64 bits.

Bounds: u = 2^-24 is half a step of FP32. A sum over a group, or over 128 k of a longer one, is exact; the scaled sums are joined
by one fused multiply-add each and, between waves, one addition each, at most 8 of them: (steps + 8) u sum |s_g S_g| over the
steps. The row's scale and the bias take one fused multiply-add, u |r|; SiLU on the hardware's exp2 and reciprocal adds
|silu| (|r| + 4) 2^-23 and passes r's own error on with a slope of at most 1.1; the residual adds two roundings; the output half a
step of its type (and half the smallest subnormal of FP16, 2^-25)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kea_kernels import _hip, int4, lowbit

DEV = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def make(m, n, k, group, seed, scales=torch.float32):
    """q int8 [1, M, ldq] with garbage behind K, qs, weight int8 [N, K], scales [N, groups], on the CPU."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (1, m, lowbit.round_up(k, 16)), generator=g, dtype=torch.int8)
    w = torch.randint(-8, 8, (n, k), generator=g, dtype=torch.int8)
    qs = (torch.rand(1, m, generator=g) * 0.02 + 1e-3).to(scales)
    ws = ((torch.rand(n, -(-k // group), generator=g) + 0.05) * 0.02 * torch.where(torch.rand(n, 1, generator=g) < 0.2, -1.0, 1.0)).to(scales)
    return q, qs, w, ws


def expected(q, qs, w, ws, group, bias, silu, residual, factor, dtype):
    """The value in 64 bits and how far the kernel's may be from it."""
    n, k = w.shape
    step = min(group, 128)
    steps = -(-k // step)
    qd, wd = torch.zeros(q.shape[1], steps * step, dtype=torch.float64), torch.zeros(n, steps * step, dtype=torch.float64)
    qd[:, :k], wd[:, :k] = q[0, :, :k].double(), w.double()
    s = ws.double().repeat_interleave(max(1, group // step), 1)[:, :steps]
    acc = torch.zeros(len(qd), n, dtype=torch.float64)
    size = torch.zeros_like(acc)
    for i in range(steps):
        part = (qd[:, i * step:(i + 1) * step] @ wd[:, i * step:(i + 1) * step].t()) * s[:, i]
        acc += part
        size += part.abs()
    v, b = acc * qs.double().reshape(-1, 1), torch.zeros(1, dtype=torch.float64) if bias is None else bias.cpu().double()
    r = v + b
    err = U * ((steps + 8) * size * qs.double().reshape(-1, 1).abs() + r.abs())
    if silu:
        t = r / (1 + torch.exp(-r))
        err = 1.1 * err + t.abs() * (r.abs() + 4) * 2 * U
        r = t
    if residual is not None:
        y = residual.cpu().double() + factor * r
        err = abs(factor) * err + U * ((factor * r).abs() + y.abs())
        r = y
    err = err + (r.abs() + err) * HALF_STEP[dtype] + (2.0**-25 if dtype == torch.float16 else 2.0**-126)
    return r, err


def check(out, want, err):
    out = out.cpu().double()
    assert torch.isfinite(out).all()
    worst = ((out - want).abs() / err).max().item()
    assert worst <= 1, f"{worst:.3g} times the bound"


def on_gpu(q, qs, w, ws, group):
    return q.to(DEV), qs.to(DEV), int4.pack(w.to(DEV), ws.to(DEV), group)


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (16, 128, 128), (17, 129, 64), (33, 640, 32), (5, 300, 512), (40, 1000, 256)])
def test_packing_keeps_every_weight(n, k, group):
    _, _, w, ws = make(1, n, k, group, n + k)
    p = int4.pack(w, ws, group)
    assert torch.equal(p.dense(), w.float() * ws.repeat_interleave(group, 1)[:, :k])
    assert p.words.numel() == -(-n // 16) * -(-k // 128) * 256 and p.scales.shape == (-(-n // 16), -(-k // group), 16)
    # the layout that the header states, a weight at a time
    b = p.words.view(torch.uint8).view(-1, 16)
    for row, at in ((0, 0), (n - 1, k - 1), (n // 2, k // 2), (n // 3, 2 * k // 3)):
        tile, i, block, kk = row // 16, row % 16, at // 128, at % 128
        h, j, u, low = kk // 64, kk % 64 // 16, kk % 16 // 8, kk % 8
        byte = int(b[(tile * -(-k // 128) + block) * 64 + 16 * j + i, 8 * h + 4 * u + low % 4])
        nibble = byte >> 4 if low >= 4 else byte & 15
        assert (nibble if nibble < 8 else nibble - 16) == int(w[row, at])


def test_pack_refusals():
    w, s = torch.zeros(4, 100, dtype=torch.int8), torch.ones(4, 2)
    for bad in (lambda: int4.pack(w, s, 48), lambda: int4.pack(w, s, 16), lambda: int4.pack(w, s, 64.0), lambda: int4.pack(w, s, 128),
                lambda: int4.pack(w.float(), s, 64), lambda: int4.pack(w[0], s, 64), lambda: int4.pack(w, s.double(), 64),
                lambda: int4.pack(w + 8, s, 64), lambda: int4.pack(w - 9, s, 64), lambda: int4.pack(w, s * float("nan"), 64),
                lambda: int4.pack(w, s * float("inf"), 64), lambda: int4.pack(w, s * 1e38, 64), lambda: int4.pack(w[:0], s[:0], 64),
                lambda: int4.pack(w[:, :0], s, 64)):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(int4.pack(w + 7, s, 64).dense(), torch.full((4, 100), 7.0))
    assert torch.equal(int4.pack(w - 8, s.half(), 64).dense(), torch.full((4, 100), -8.0))


# single rows, ragged tiles on both sides, k below, at and past a step of 16 / 32 / 64 / 128, shares of the waves of none and many
SIZES = [(1, 1, 1), (1, 17, 16), (1, 640, 2560), (1, 2560, 640), (2, 130, 63), (3, 1030, 641), (5, 64, 65), (13, 1024, 4096), (15, 256, 129),
         (16, 48, 1000), (17, 33, 127), (31, 96, 384), (33, 1030, 640), (64, 64, 128), (65, 129, 257), (100, 300, 4100), (125, 1024, 1024),
         (128, 128, 64), (129, 255, 192), (200, 512, 2048), (257, 513, 1025), (300, 4096, 320), (375, 1030, 641), (1000, 256, 512),
         (2049, 130, 96), (1500, 1025, 160)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("group", [32, 64, 128, 512])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(m, n, k, group):
    for i, (scales, dtype) in enumerate(((torch.float32, torch.float32), (torch.float16, torch.bfloat16))):
        q, qs, w, ws = make(m, n, k, group, m + n + k + i, scales)
        qg, qsg, wg = on_gpu(q, qs, w, ws, group)
        check(int4.gemm(qg, qsg, wg, out_dtype=dtype), *expected(q, qs, w, ws, group, None, False, None, 1.0, dtype))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,group", [(1, 130, 200, 32), (7, 1030, 640, 64), (40, 61, 1024, 128), (150, 257, 300, 64), (700, 300, 520, 32)])
def test_epilogue(m, n, k, group, dtype):
    q, qs, w, ws = make(m, n, k, group, 3)
    qg, qsg, wg = on_gpu(q, qs, w, ws, group)
    bias, residual = torch.linspace(-3, 3, n), torch.linspace(-2, 2, m * n).view(m, n)
    for b, silu, res, factor in ((bias, False, None, 1.0), (bias.half(), True, None, 1.0), (None, True, residual, 0.5), (bias, False, residual, -2.0)):
        got = int4.gemm(qg, qsg, wg, None if b is None else b.to(DEV), silu=silu, residual=None if res is None else res.to(DEV),
                        residual_factor=factor, out_dtype=dtype)
        check(got, *expected(q, qs, w, ws, group, b, silu, res, factor, dtype))
    y = residual.to(DEV)
    if dtype == torch.float32:  # in place
        assert int4.gemm(qg, qsg, wg, out=y, residual=y, residual_factor=0.5) is y
        check(y, *expected(q, qs, w, ws, group, None, False, residual, 0.5, dtype))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m,n,k", [(2000, 2050, 900), (3000, 700, 130), (500, 1050, 4097), (260, 4001, 4000), (300, 700, 1111), (1300, 130, 6000), (800, 1550, 506)])
def test_tiles_of_many_rows(m, n, k, group):
    """Sizes that take tiles of 32 x 64 to 128 x 128, by one, two or four groups of waves, stages past the end among them."""
    q, qs, w, ws = make(m, n, k, group, m + n + k, torch.float32 if group > 64 else torch.float16)
    qg, qsg, wg = on_gpu(q, qs, w, ws, group)
    bias = torch.linspace(-3, 3, n)
    got = int4.gemm(qg, qsg, wg, bias.to(DEV), silu=True, out_dtype=torch.float16)
    for rows in (slice(0, 150), slice(m - 150, m)):
        check(got[rows], *expected(q[:, rows], qs[:, rows], w, ws, group, bias, True, None, 1.0, torch.float16))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("group", [32, 64, 128, 256])
@pytest.mark.parametrize("m,n,k", [(1, 30, 2048), (1, 30, 2049), (13, 50, 2177), (16, 1024, 4096), (2, 8193, 2100), (1, 8192, 2200)])
def test_tokens_of_wide_layers(m, n, k, group):
    """Four and eight waves to a workgroup, with and without a block of k for each of them."""
    q, qs, w, ws = make(m, n, k, group, m + n + k, torch.float32 if group > 64 else torch.float16)
    qg, qsg, wg = on_gpu(q, qs, w, ws, group)
    bias = torch.linspace(-3, 3, n)
    got = int4.gemm(qg, qsg, wg, bias.to(DEV), silu=True, out_dtype=torch.float16)
    check(got, *expected(q, qs, w, ws, group, bias, True, None, 1.0, torch.float16))


@pytest.mark.gpu
@torch.inference_mode()
def test_rows_far_apart():
    """Rows of q 2^23 bytes and more apart, past 32 bits in all."""
    q, qs, w, ws = make(300, 40, 200, 64, 17)
    _, qsg, wg = on_gpu(q, qs, w, ws, 64)
    store = torch.empty(299 * (1 << 24) + 256, dtype=torch.int8, device=DEV)
    far = store.as_strided((300, 208), (1 << 24, 1))
    far.copy_(q[0])
    check(int4.gemm(far, qsg, wg), *expected(q, qs, w, ws, 64, None, False, None, 1.0, torch.float32))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 17, 40), (5, 130, 200), (33, 100, 640), (300, 131, 150)])
def test_outputs_inside_larger_ones(m, n, k, dtype):
    """Any alignment and row stride of out, and nothing is written around it; q a view of wider rows."""
    q, qs, w, ws = make(m, n, k, 64, 5)
    _, qsg, wg = on_gpu(q, qs, w, ws, 64)
    ldq = q.shape[2]
    wide = torch.full((m, ldq + 48), 77, dtype=torch.int8, device=DEV)
    wide[:, 16:16 + ldq] = q[0].to(DEV)
    for left in (0, 1, 3):
        big = torch.full((m + 2, n + 7), 5.0, dtype=dtype, device=DEV)
        out = big[1:m + 1, left:left + n]
        assert int4.gemm(wide[:, 16:16 + ldq], qsg, wg, out=out) is out
        check(out, *expected(q, qs, w, ws, 64, None, False, None, 1.0, dtype))
        big[1:m + 1, left:left + n] = 5.0
        assert bool((big == 5.0).all())


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k,group", [(3, 40, 5000, 128), (130, 200, 9000, 32), (1, 16, 1 << 20, 64)])
def test_largest_values_and_long_rows(m, n, k, group):
    """Extreme integers in long rows: a step's sum is the largest there is."""
    q, qs, w, ws = make(m, n, k, group, 9)
    q[:, ::2], w[::2] = -128, -8
    qg, qsg, wg = on_gpu(q, qs, w, ws, group)
    check(int4.gemm(qg, qsg, wg), *expected(q, qs, w, ws, group, None, False, None, 1.0, torch.float32))


@pytest.mark.gpu
@torch.inference_mode()
def test_calls_are_the_same_to_the_bit_and_rows_stand_alone():
    q, qs, w, ws = make(200, 520, 1100, 64, 11)
    qg, qsg, wg = on_gpu(q, qs, w, ws, 64)
    one = int4.gemm(qg, qsg, wg)
    assert torch.equal(one, int4.gemm(qg, qsg, wg))
    qsg2 = qsg.clone()
    qsg2[0, 7] = float("nan")
    two = int4.gemm(qg, qsg2, wg)
    assert torch.isnan(two[7]).all() and torch.equal(torch.cat((one[:7], one[8:])), torch.cat((two[:7], two[8:])))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(1, 1030, 640), (40, 256, 512), (500, 512, 640)])
def test_captured_calls_replay(m, n, k):
    q, qs, w, ws = make(m, n, k, 64, 13)
    qg, qsg, wg = on_gpu(q, qs, w, ws, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        int4.gemm(qg, qsg, wg)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = int4.gemm(qg, qsg, wg, silu=True)
    g = torch.Generator().manual_seed(1)
    for _ in range(4):
        qg.copy_(torch.randint(-128, 128, q.shape, generator=g, dtype=torch.int8))
        want = int4.gemm(qg, qsg, wg, silu=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.gpu
@torch.inference_mode()
def test_linear_layer():
    g = torch.Generator().manual_seed(2)
    weight, bias = torch.randn(70, 300, generator=g) / 17, torch.randn(70, generator=g)
    layer = int4.Int4Linear.from_dense(weight, bias, 64, "cuda:0")
    x = torch.randn(3, 5, 300, generator=g).to(DEV)
    q, qs, _ = lowbit.quantize(x, (x.stride(0), x.stride(1), 1, 5), 15, 300, 1)
    want = int4.gemm(q, qs, layer.weight, layer.bias, silu=True).view(3, 5, 70)
    assert torch.equal(layer.linear(x, activation="silu"), want)
    assert torch.equal(layer.linear(x[1, 2], activation="silu"), want[1, 2])
    assert layer.linear(x[:0]).shape == (0, 5, 70) and layer.linear(x, out_dtype=torch.float16).dtype == torch.float16
    # rounding to int8 rows and 4-bit weights: half a step of each, as far as 300 products can add up
    dense, w4 = x.cpu().double() @ weight.double().t() + bias.double(), layer.weight.dense().cpu().double()
    step_w, step_x = (weight.double() - w4).abs(), x.cpu().double().abs().amax(2, keepdim=True) / 254
    bound = x.cpu().double().abs() @ step_w.t() + step_x * w4.abs().sum(1) + 1e-4
    assert bool(((layer.linear(x).cpu().double() - dense).abs() <= bound).all())
    half_group = weight.view(70, -1)[:, :64].abs().amax(1) / 7 / 2
    assert bool((step_w[:, :64].amax(1) <= half_group.double() * 1.001).all())
    layer2 = int4.Int4Linear.prepare(torch.randint(-8, 8, (20, 100), generator=g, dtype=torch.int8), torch.ones(20, 1, dtype=torch.float64), None, 128, "cuda")
    assert layer2.weight.scales.dtype == torch.float32 and layer2.linear(torch.ones(100, device=DEV)).shape == (20,)


@pytest.mark.gpu
@torch.inference_mode()
def test_empty_rows():
    _, _, w, ws = make(1, 20, 100, 64, 1)
    p = int4.pack(w.to(DEV), ws.to(DEV), 64)
    out = int4.gemm(torch.empty(1, 0, 112, dtype=torch.int8, device=DEV), torch.empty(1, 0, device=DEV), p)
    assert out.shape == (0, 20)


@torch.inference_mode()
def test_refusals():
    q, qs, w, ws = make(4, 20, 100, 64, 1)
    p = int4.pack(w, ws, 64)
    for bad in (lambda: int4.gemm(q.float(), qs, p), lambda: int4.gemm(q.expand(2, -1, -1), qs, p), lambda: int4.gemm(q[:, :, :96], qs, p),
                lambda: int4.gemm(q, qs[:, :3], p), lambda: int4.gemm(q, qs.double(), p), lambda: int4.gemm(q, qs, p, torch.zeros(19)),
                lambda: int4.gemm(q, qs, p, out_dtype=torch.int32), lambda: int4.gemm(q, qs, p, out=torch.empty(4, 21)),
                lambda: int4.gemm(q, qs, p, out=torch.empty(20, 4).t()), lambda: int4.gemm(q, qs, p, residual=torch.empty(4, 20).half()),
                lambda: int4.gemm(q, qs, p, residual=torch.empty(4, 19)), lambda: int4.gemm(q[0, :, 1:], qs, p),
                lambda: int4.gemm(q, qs, int4.Weight(p.words[:-1], p.scales, 20, 100, 64)),
                lambda: int4.gemm(q, qs, int4.Weight(p.words, p.scales, 33, 100, 64)),
                lambda: int4.gemm(q, qs, int4.Weight(p.words, p.scales, 20, 100, 32)),
                lambda: int4.gemm(q, qs, int4.Weight(p.words, p.scales.half(), 20, 300, 64)),
                lambda: int4.gemm(q, qs, p)):  # (the last: tensors on the CPU)
        with pytest.raises(ValueError):
            bad()
    buffer = torch.empty(4, 112)
    with pytest.raises(ValueError, match="shares memory"):
        int4.gemm(buffer.view(torch.int8)[:, :112].view(1, 4, 112), qs, p, out=buffer[:, 2:22])
    y = torch.empty(5, 20)
    with pytest.raises(ValueError, match="shares memory"):
        int4.gemm(q, qs, p, out=y[1:], residual=y[:4])


def test_derivatives_are_refused():
    q, qs, w, ws = make(4, 20, 100, 64, 1)
    p = int4.pack(w, ws, 64)
    with pytest.raises(RuntimeError, match="inference only"):
        int4.gemm(q, qs.requires_grad_(), p)
    with pytest.raises(RuntimeError, match="inference only"):
        int4.gemm(q, qs.detach(), p, residual=torch.zeros(4, 20, requires_grad=True))


def test_library_refusals():
    fn, one, odd = _hip.lib().kea_int4_gemm, ctypes.c_void_p(16), ctypes.c_void_p(8)
    good = dict(q=one, ldq=112, qs=one, qd=0, w=one, ws=one, wd=0, group=64, b=None, bd=0, y=one, yd=0, ldy=20, r=None, ldr=0, f=1.0, m=4, n=20, k=100,
                flags=0)
    call = lambda **kw: fn(*{**good, **kw}.values(), None)  # noqa: E731
    for bad in (dict(m=-1), dict(n=0), dict(k=0), dict(k=(1 << 20) + 1, ldq=1 << 21), dict(group=0), dict(group=48), dict(group=16), dict(ldq=96), dict(ldy=19),
                dict(r=one, ldr=19), dict(yd=3), dict(flags=2), dict(qd=2), dict(wd=2), dict(b=one, bd=2), dict(q=None), dict(w=None), dict(y=None),
                dict(qs=None), dict(ws=None), dict(m=1 << 30, n=1 << 20)):
        if "n" in bad and bad.get("n") == 1 << 20:
            bad = {**bad, "ldy": 1 << 20}
        assert call(**bad) == -1, bad
    for bad in (dict(q=odd), dict(w=odd), dict(ws=odd), dict(ldq=104), dict(y=ctypes.c_void_p(18)), dict(qs=ctypes.c_void_p(18))):
        assert call(**bad) == -2, bad
    assert call(m=0) == 0


def test_linear_refusals():
    w = torch.zeros(4, 100)
    with pytest.raises(ValueError, match="GPU"):
        int4.Int4Linear.from_dense(w, device="cpu")
    with pytest.raises(ValueError, match="finite"):
        int4.Int4Linear.from_dense(w * float("nan"))
    with pytest.raises(ValueError, match="power of two"):
        int4.Int4Linear.from_dense(w, group=100)
