"""norms.block_norm (kea_block_norm): y = x + factor * act(gate) * post(block), z = pre(y), against the formulas in 64 bits.

Bounds follow the FP32 steps (u = 2^-24, half a step): a sum of d elements in chains of at most d / 64 + 16 additions is off by
that many u times the mean of the magnitudes; differences, products and sums take one u each; square root, reciprocal and the
added eps four together; a sigmoid (|g| + 4) 2^-23 of itself, a tanh 4 * 2^-23; every output half a step of its type (and 2^-25,
half of FP16's smallest number). Errors of a norm's input pass through it: into the mean, the centred values and the variance."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch
import torch.nn.utils.parametrize
import torch.nn.utils.prune

from kea_kernels import _hip, lowbit, norms

DEV = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def module(kind, d, g, dtype=F32, eps=1e-5):
    if not kind:
        return None
    m = torch.nn.LayerNorm(d, eps=eps) if kind == "layer" else torch.nn.RMSNorm(d, eps=eps)
    with torch.no_grad():
        m.weight.copy_(1 + 0.3 * torch.randn(d, generator=g))
        if kind == "layer":
            m.bias.copy_(0.3 * torch.randn(d, generator=g))
    return m.to(DEV, dtype)


def normed(v, ev, m):
    """(norm of v, bound on the kernel's error) from v in 64 bits and a bound on its input's error."""
    if m is None:
        return v, ev
    d = v.shape[1]
    depth = d // 64 + 16
    layer = hasattr(m, "bias")
    mean = v.mean(1, keepdim=True) if layer else torch.zeros(1, dtype=torch.float64)
    emean = ev.mean(1, keepdim=True) + depth * U * v.abs().mean(1, keepdim=True) if layer else 0.0
    c = v - mean
    ec = ev + emean + (U * c.abs() if layer else 0.0)
    var = (c * c).mean(1, keepdim=True)
    evar = 2 * (c.abs() * ec).mean(1, keepdim=True) + (ec * ec).mean(1, keepdim=True) + (depth + 2) * U * var
    rstd = 1 / torch.sqrt(var + m.eps)
    rel = 0.5 * evar / (var + m.eps) * 1.01 + 4 * U
    z, ez = c * rstd, ec * rstd + (c * rstd).abs() * (rel + 2 * U)
    if m.weight is not None:
        w = m.weight.detach().cpu().double()
        z, ez = z * w, ez * w.abs() + U * (z * w).abs()
    if layer and m.bias is not None:
        z = z + m.bias.detach().cpu().double()
        ez = ez + U * z.abs()
    return z, ez * 1.01


def expected(x, block, post, gate, act, factor, pre):
    x, o = x.cpu().double(), block.cpu().double()
    d = x.shape[-1]
    x, o = x.reshape(-1, d), o.reshape(-1, d)
    p, ep = normed(o, torch.zeros_like(o), post)
    if gate is not None:
        g = gate.cpu().double().reshape(-1, d)
        g = g.repeat_interleave(o.shape[0] // g.shape[0], 0)
        eg = torch.zeros_like(g)
        if act == "sigmoid":
            s = 1 / (1 + torch.exp(-g))
            g, eg = s, s * (g.abs() + 4) * 2 * U
        if act == "tanh":
            g, eg = torch.tanh(g), torch.full_like(g, 8 * U)
        p, ep = p * g, ep * g.abs() + p.abs() * eg + U * (p * g).abs()
    y = x + factor * p
    ey = abs(factor) * ep + U * ((factor * p).abs() + y.abs())
    return (y, ey), normed(y, ey, pre)


def check(out, want, err):
    out = out.reshape(want.shape)
    bound = err + (want.abs() + err) * HALF_STEP[out.dtype] + TINY[out.dtype]
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.3g} times the bound"


def check_rows8(q, qs, z, ez):
    """The int8 rows of z: the scale of the largest, every code the nearest to within z's own error, zeros behind d."""
    d = z.shape[1]
    assert q.dtype == torch.int8 and qs.dtype == F32 and q.shape == (1, z.shape[0], lowbit.round_up(d, 16))
    top, s = z.abs().amax(1), qs[0].cpu().double()
    assert ((s - (top / 127).clamp_min(1e-30)).abs() <= ez.amax(1) / 127 + 2 * U * top / 127 + 1e-36).all()
    code = q[0, :, :d].cpu().double()
    assert ((code * s[:, None] - z).abs() <= s[:, None] * (0.5 + 1e-5) + ez).all() and (q[0, :, :d] >= -127).all()
    assert not q[0, :, d:].any()


def tensors(rows, d, stream, block, g, gates=0):
    x = (2 * torch.randn(rows, d, generator=g)).to(stream).to(DEV)
    o = (torch.randn(rows, d, generator=g) * (0.2 + torch.rand(rows, 1, generator=g)) + 0.3).to(block).to(DEV)
    gate = torch.randn(gates, d, generator=g).to(block).to(DEV) if gates else None
    return x, o, gate


SIZES = [(1, 1), (1, 8), (3, 2), (5, 7), (4, 63), (1, 64), (7, 65), (2, 255), (3, 256), (9, 511), (6, 512), (2, 520), (1, 640), (5, 1000),
         (33, 1024), (4, 1031), (3, 2040), (2, 2048), (5, 2049), (2, 2056), (3, 4096), (2, 4097), (2, 5120), (1, 8192), (2, 8200), (3, 10001),
         (2, 16384), (1, 32767), (2, 32768)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("rows,d", SIZES)
def test_row_lengths(rows, d):
    g = torch.Generator().manual_seed(rows * 40000 + d)
    for stream, block, post, pre in ((F32, F16, "layer", "rms"), (BF16, BF16, "rms", "layer"), (F16, F32, "", "layer"), (F32, BF16, "layer", "")):
        x, o, gate = tensors(rows, d, stream, block, g, 1)
        post, pre = module(post, d, g), module(pre, d, g)
        (y, ey), (z, ez) = expected(x, o, post, gate, "sigmoid", 0.5, pre)
        got = norms.block_norm(x, o, post=post, gate=gate, gate_activation="sigmoid", factor=0.5, pre=pre)
        assert got[0].dtype == stream and got[0].shape == x.shape
        check(got[0], y, ey)
        if pre is None:
            assert got[1] is None
        else:
            assert got[1].dtype == block
            check(got[1], z, ez)
        got = norms.block_norm(x, o, post=post, gate=gate, gate_activation="sigmoid", factor=0.5, pre=pre, quantize=True)
        check(got[0], y, ey)
        check_rows8(got[1], got[2], z, ez)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("act", ["", "sigmoid", "tanh"])
@pytest.mark.parametrize("stream", [F32, F16, BF16])
@pytest.mark.parametrize("block", [F32, F16, BF16])
def test_types_gates_and_norms(stream, block, act):
    g = torch.Generator().manual_seed(3)
    for d in (72, 77):
        for gates in (0, 1, 3, 12):
            for post in ("", "rms", "layer"):
                x, o, gate = tensors(12, d, stream, block, g, gates)
                x, o = x.view(3, 4, d), o.view(3, 4, d)
                post_m, pre_m = module(post, d, g, block), module("rms" if post == "layer" else "layer", d, g, F16)
                shaped = gate if gates < 3 else gate.view(3, -1, d)
                (y, ey), (z, ez) = expected(x, o, post_m, gate, act if gates else "", -1.5, pre_m)
                got = norms.block_norm(x, o, post=post_m, gate=shaped, gate_activation=act, factor=-1.5, pre=pre_m)
                assert got[0].shape == got[1].shape == x.shape
                check(got[0], y, ey)
                check(got[1], z, ez)


@pytest.mark.gpu
@torch.inference_mode()
def test_many_rows():
    g = torch.Generator().manual_seed(4)
    x, o, gate = tensors(70001, 24, BF16, BF16, g, 70001)
    pre = module("rms", 24, g)
    got = norms.block_norm(x, o, gate=gate, gate_activation="tanh", pre=pre)
    (y, ey), (z, ez) = expected(x, o, None, gate, "tanh", 1.0, pre)
    check(got[0], y, ey)
    check(got[1], z, ez)


@pytest.mark.gpu
@torch.inference_mode()
def test_millions_of_rows():
    """More rows than 2^32 / 1024: rows of 8, each normalised to the same values."""
    x = torch.arange(8, dtype=F32, device=DEV).repeat(5_000_003, 1)
    pre = module("layer", 8, torch.Generator().manual_seed(1))
    _, z = norms.block_norm(x, x.half(), factor=0.0, pre=pre)
    (_, _), (want, err) = expected(x[:1], x[:1].half(), None, None, "", 0.0, pre)
    check(z[:1], want, err)
    assert (z == z[0]).all()


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("d", [64, 1024, 1031])
def test_norm_alone_and_rows_of_the_stream(d):
    """Without a block: the norm of x, as values or int8 rows; without a norm: the rows that lowbit.quantize makes, to the bit."""
    g = torch.Generator().manual_seed(5)
    for dtype in (F32, F16, BF16):
        x = torch.randn(6, d, generator=g).to(dtype).to(DEV)
        for kind in ("rms", "layer"):
            m = module(kind, d, g, dtype)
            z, ez = normed(x.cpu().double(), torch.zeros(6, d, dtype=torch.float64), m)
            y, got = norms.block_norm(x, None, pre=m)
            assert y is x and got.dtype == dtype
            check(got, z, ez)
            y, q, qs = norms.block_norm(x, None, pre=m, quantize=True)
            check_rows8(q, qs, z, ez)
        _, q, qs = norms.block_norm(x, None, quantize=True)
        want = lowbit.quantize((x.float() if dtype == BF16 else x)[None], (0, d, 1, 6), 6, d, 1)
        assert torch.equal(q, want[0]) and torch.equal(qs, want[1])
    x, o, _ = tensors(6, d, F32, F16, g)
    y, q, qs = norms.block_norm(x, o, factor=0.5, quantize=True)
    want = lowbit.quantize(y[None], (0, d, 1, 6), 6, d, 1)
    assert torch.equal(q, want[0]) and torch.equal(qs, want[1])


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("d", [96, 1024, 99, 4096])
def test_views_in_place_and_parameters(d):
    """Strided rows on every side, out in place, norms without weight or bias, eps None: what lies between rows stays."""
    g = torch.Generator().manual_seed(6)
    base = torch.full((9, d + 24), 5.0, device=DEV)
    base[:8, 8:8 + d] = 2 * torch.randn(8, d, generator=g).to(DEV)
    x = base[:8, 8:8 + d]
    o = torch.randn(8, 2 * d, generator=g).to(BF16).to(DEV)[:, d:]
    gate = torch.randn(4, d + 8, generator=g).to(BF16).to(DEV)[:, :d]
    post, pre = SimpleNamespace(weight=None, bias=None, eps=1e-6), SimpleNamespace(weight=None, eps=2.0**-23)
    (y, ey), (z, ez) = expected(x, o, post, gate, "", 0.7, pre)
    pre.eps = None
    got = norms.block_norm(x, o, post=post, gate=gate, factor=0.7, pre=pre, out=x)
    assert got[0].data_ptr() == x.data_ptr()
    check(x, y, ey)
    check(got[1], z, ez)
    assert (base[8] == 5).all() and (base[:, :8] == 5).all() and (base[:, 8 + d:] == 5).all()


@pytest.mark.gpu
@torch.inference_mode()
def test_one_bad_row_stays_one():
    """Infinities and NaN of one row, and rows of zeros, leave the others alone."""
    g = torch.Generator().manual_seed(7)
    x, o, gate = tensors(9, 200, F32, F32, g, 1)
    pre, post = module("layer", 200, g), module("rms", 200, g)
    clean = norms.block_norm(x, o, post=post, gate=gate, pre=pre)
    x2, o2 = x.clone(), o.clone()
    o2[3, 5], x2[5, 7] = float("nan"), float("inf")
    x2[7], o2[7] = 0, 0
    bad = norms.block_norm(x2, o2, post=post, gate=gate, pre=pre)
    for a, b in zip(clean, bad):
        for r in (0, 1, 2, 4, 6, 8):
            assert torch.equal(a[r], b[r])
        assert b[3].isnan().all()
    assert bad[1][5].isnan().all() and bad[0][5, 7] == float("inf") and bad[0][5, :7].isfinite().all()
    assert (bad[0][7] == 0).all() and torch.allclose(bad[1][7], pre.bias)


@pytest.mark.gpu
@torch.inference_mode()
def test_offsets_past_32_bits():
    d, far = 1024, 1 << 30
    g = torch.Generator().manual_seed(8)
    base = torch.zeros(5 * far // 4 + 5 * d, dtype=BF16, device=DEV)
    x = base.as_strided((5, d), (far // 4 * 1, 1))  # rows 2^28 elements apart: the last past 2^31 bytes
    x.copy_(torch.randn(5, d, generator=g).to(BF16))
    o = torch.randn(5, d, generator=g).to(BF16).to(DEV)
    pre = module("rms", d, g)
    (y, ey), (z, ez) = expected(x, o, None, None, "", 1.0, pre)
    got = norms.block_norm(x, o, pre=pre, out=x)
    check(x, y, ey)
    check(got[1], z, ez)


@pytest.mark.gpu
@torch.inference_mode()
def test_captured_calls_replay_on_their_stream():
    g = torch.Generator().manual_seed(9)
    x, o, gate = tensors(50, 1024, F32, F16, g, 10)
    post, pre = module("layer", 1024, g), module("rms", 1024, g)
    call = lambda: norms.block_norm(x, o, post=post, gate=gate, gate_activation="sigmoid", factor=0.5, pre=pre, quantize=True)  # noqa: E731
    want = [t.clone() for t in call()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        out = call()
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        again = call()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(again, want))


@pytest.mark.gpu
@torch.inference_mode()
def test_no_rows():
    x = torch.empty(0, 16, device=DEV)
    y, z = norms.block_norm(x, x.half(), pre=torch.nn.RMSNorm(16, device=DEV))
    assert y.shape == (0, 16) and z.shape == (0, 16) and z.dtype == F16
    assert norms.block_norm(x, x, quantize=True)[1].shape == (1, 0, 16)


@pytest.mark.gpu
@torch.inference_mode()
def test_small_gates_keep_their_digits():
    """tanh of gates down to 2^-60, without a stream that hides them. Below 1/4 a series, whose next term is 2^-26 of its value,
    in three roundings that count; above, at most 8 u from 1 - 2 / (1 + e^(2 g)); two roundings more to the output."""
    gate = torch.cat([s * 2.0 ** torch.linspace(-60, 4, 1300) for s in (1, -1)] + [torch.tensor([0.0, 0.25, -0.25])]).to(DEV)[None]
    o = torch.linspace(-3, 3, gate.shape[1], device=DEV)[None]
    y, _ = norms.block_norm(torch.zeros_like(o), o, gate=gate, gate_activation="tanh")
    g = gate.cpu().double()
    want = torch.tanh(g) * o.cpu().double()
    assert ((y.cpu().double() - want).abs() <= want.abs() * U * torch.where(g.abs() < 0.25, 6.0, 8 / torch.tanh(g).abs() + 2)).all()


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("d", [99, 1024, 4100])
def test_out_as_the_block_and_beside_the_stream(d):
    g = torch.Generator().manual_seed(11)
    x, o, gate = tensors(8, d, BF16, BF16, g, 8)
    want, _ = norms.block_norm(x, o, gate=gate, factor=0.5)
    both = torch.empty(8, 2 * d, dtype=BF16, device=DEV)
    both[:, :d] = x
    norms.block_norm(both[:, :d], o, gate=gate, factor=0.5, out=both[:, d:])
    assert torch.equal(both[:, d:], want) and torch.equal(both[:, :d], x)
    norms.block_norm(x, o, gate=gate, factor=0.5, out=o)
    assert torch.equal(o, want)


# ---- without a GPU -----------------------------------------------------------------------------------------------------------

def test_an_output_that_overlaps_is_refused():
    x, o, gate = torch.zeros(64, 32), torch.zeros(6, 32), torch.zeros(6, 32)
    for args in ((x[:6], o, gate, x[1:7]), (x[:6], x[6:12], gate, x[3:9]), (x[:6], o, x[20:26], x[20:26]), (x[:1], o[:1], x[:1], x[:1]),
                 (x[:6], o, gate, x.view(-1)[16:208].view(6, 32))):
        with pytest.raises(ValueError, match="shares memory"):
            norms.block_norm(*args[:2], gate=args[2], out=args[3])
    with pytest.raises(ValueError, match="GPU"):
        norms.block_norm(x.view(32, 64)[:, :32], x.view(32, 64)[:, :32], out=x.view(32, 64)[:, 32:])


def test_refusals():
    x, o = torch.zeros(6, 32), torch.zeros(6, 32, dtype=F16)
    ln, rms = torch.nn.LayerNorm(32), torch.nn.RMSNorm(32)
    call = norms.block_norm
    for args, kw, message in [
        ((x, o[:5]), {}, "block is"), ((x.double(), o), {}, "x must be"), ((x, o.int()), {}, "block must be"),
        ((x, o), dict(gate=torch.zeros(4, 32, dtype=F16)), "gate"), ((x, o), dict(gate=torch.zeros(1, 32)), "gate"),
        ((x, o), dict(gate=torch.zeros(1, 16, dtype=F16)), "gate"), ((x, o), dict(gate=torch.zeros(0, 32, dtype=F16)), "gate"),
        ((x, o), dict(gate=o, gate_activation="relu"), "activation"), ((x, o), dict(pre=torch.nn.LayerNorm(16)), "normalizes"),
        ((x, o), dict(post=torch.nn.LayerNorm((6, 32))), "normalizes"),
        ((x, o), dict(pre=SimpleNamespace(weight=torch.ones(16), eps=1.0)), "elements"),
        ((x, o), dict(pre=SimpleNamespace(weight=torch.ones(32), bias=torch.zeros(32, dtype=F16), eps=1.0)), "weight is"),
        ((x, o), dict(out=torch.zeros(6, 32, dtype=F16)), "out must have"), ((x, o), dict(out=torch.zeros(1, 32).expand(6, 32)), "overlap"),
        ((x, None), {}, "without a block"), ((x, None), dict(pre=ln, gate=x[:1]), "without a block"), ((x, None), dict(pre=ln, out=x), "without a block"),
        ((torch.zeros(32, 6).t(), o), {}, "contiguous elements"), ((torch.zeros(3, 4, 32)[:, :2], o.view(3, 2, 32)), {}, "one stride"),
        ((torch.zeros(1, 40000), torch.zeros(1, 40000)), {}, "32768"), ((x, o), dict(pre=rms), "GPU"),
    ]:
        with pytest.raises(ValueError, match=message):
            call(*args, **kw)
    with pytest.raises(RuntimeError, match="inference only"):
        call(x.clone().requires_grad_(), o, pre=ln)


def test_library_refusals():
    L = _hip.lib()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    none, layer = _hip.Norm(0, 0, None, None, 0.0), _hip.Norm(1, 0, p, p, 1e-5)
    good = dict(x=p, xd=0, ldx=32, b=p, bd=1, ldb=32, m=4, d=32, post=none, g=None, ldg=0, gr=1, ga=0, f=1.0, y=p, ldy=32, pre=layer, z=p,
                ldz=32, q=None, ldq=0, qs=None, stream=None)
    for change, rc in [(dict(d=0), -1), (dict(d=32769), -1), (dict(m=-1), -1), (dict(xd=3), -1), (dict(ldx=31), -1), (dict(ldy=31), -1),
                       (dict(g=p, ldg=31), -1), (dict(gr=0), -1), (dict(ga=3), -1), (dict(pre=none), -1), (dict(q=p, ldq=32, qs=p), -1),
                       (dict(z=None, q=p, ldq=32), -1), (dict(b=None), -1), (dict(x=p + 2), -2), (dict(z=p + 1), -2), (dict(x=None), -1),
                       (dict(pre=_hip.Norm(3, 0, None, None, 0.0)), -1), (dict(pre=_hip.Norm(1, 0, p + 2, None, 0.0)), -1), (dict(m=0), 0)]:
        assert L.kea_block_norm(*(good | change).values()) == rc, change


def test_a_bias_that_is_no_parameter_makes_a_layer_norm():
    """The native call takes a module's own parameters; a bias that a LayerNorm keeps elsewhere (pruned, parametrized, as a
    buffer, an attribute) is not taken for the bias that an RMSNorm lacks."""
    class Shifted(torch.nn.Module):
        def forward(self, b):
            return b + 1

    pruned, parametrized, buffered, plain = (torch.nn.LayerNorm(8) for _ in range(4))
    torch.nn.utils.prune.identity(pruned, "bias")
    torch.nn.utils.parametrize.register_parametrization(parametrized, "bias", Shifted())
    del buffered.bias, plain.bias
    buffered.register_buffer("bias", torch.ones(8))
    plain.bias = torch.ones(8)
    odd = torch.nn.RMSNorm(8)
    odd.bias = torch.ones(8)
    for m in (pruned, parametrized, buffered, plain, odd):
        with pytest.raises(LookupError):
            norms._parameters(m, 8)
        assert norms._norm("pre", m, 8, torch.device("cpu"))[0].kind == 1
    assert [norms._parameters(m, 8)[0] for m in (None, torch.nn.LayerNorm(8), torch.nn.LayerNorm(8, bias=False), torch.nn.RMSNorm(8))] == [0, 1, 1, 2]
    assert norms._parameters(type("Own", (torch.nn.RMSNorm,), {})(8), 8)[0] == 2


def test_parameters_that_require_grad_are_refused():
    """Without rows, so that the refusal is all that can happen."""
    x = torch.zeros(0, 8)
    fresh, frozen = torch.nn.LayerNorm(8), torch.nn.RMSNorm(8).requires_grad_(False)
    half = torch.nn.LayerNorm(8).requires_grad_(False)
    half.bias.requires_grad_()
    for kw in (dict(pre=fresh), dict(post=fresh, pre=frozen), dict(pre=half)):
        with pytest.raises(RuntimeError, match="inference only"):
            norms.block_norm(x, x, **kw)
        with torch.no_grad():
            norms.block_norm(x, x, **kw)
    with pytest.raises(RuntimeError, match="inference only"):
        norms.block_norm(x, None, pre=fresh)
    norms.block_norm(x, x, post=frozen, pre=frozen)


@pytest.mark.gpu
def test_parameters_that_require_grad_are_refused_on_the_gpu():
    x = torch.randn(4, 64, device=DEV)
    fresh = torch.nn.LayerNorm(64, device=DEV)
    frozen = torch.nn.LayerNorm(64, device=DEV).requires_grad_(False)
    want = norms.block_norm(x, x, pre=frozen)
    for kw in (dict(pre=fresh), dict(post=fresh, pre=frozen), dict(pre=fresh, quantize=True)):
        with pytest.raises(RuntimeError, match="inference only"):
            norms.block_norm(x, x, **kw)
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(norms.block_norm(x, x, pre=fresh), want))


def test_an_out_over_a_norms_parameters_is_refused():
    x, norm, flat = torch.zeros(2, 8), torch.nn.LayerNorm(8).requires_grad_(False), torch.zeros(40)
    for name in ("weight", "bias"):
        for which in ("post", "pre"):
            setattr(norm, name, torch.nn.Parameter(flat[12:20], requires_grad=False))
            with pytest.raises(ValueError, match="shares memory"):
                norms.block_norm(x, x, out=flat[:16].view(2, 8), **{which: norm})
            with pytest.raises(ValueError, match="GPU"):
                norms.block_norm(x, x, out=flat[20:36].view(2, 8), **{which: norm})
            setattr(norm, name, torch.nn.Parameter(torch.ones(8), requires_grad=False))


@pytest.mark.gpu
@torch.inference_mode()
def test_an_out_over_a_norms_parameters_is_refused_on_the_gpu():
    x, norm = torch.randn(1, 64, device=DEV), torch.nn.LayerNorm(64, device=DEV)
    for out in (norm.weight.view(1, 64), norm.bias.view(1, 64)):
        for kw in (dict(post=norm), dict(pre=norm)):
            with pytest.raises(ValueError, match="shares memory"):
                norms.block_norm(x, x, out=out, **kw)
