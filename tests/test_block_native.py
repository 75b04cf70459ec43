"""The native call path of int8.gemm, norms.block_norm and window.attention (kea_native): it takes the ordinary calls, gives
the Python path's bits, shapes and strides, and leaves everything else to that path; and a layer made of the three, run as
a model would, against the same layer in 64 bits."""
from __future__ import annotations

import math
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad

from kea_kernels import _hip, int8, lowbit, norms, window

DEV = "cuda"


def _same(a, b):
    for x, y in zip(a, b, strict=True):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and torch.equal(x, y)


@pytest.mark.gpu
@torch.inference_mode()
def test_gemm(monkeypatch):
    g = torch.Generator().manual_seed(0)
    q = torch.randint(-128, 128, (1, 40, 112), generator=g, dtype=torch.int8).to(DEV)
    w = int8.pad_rows(torch.randint(-128, 128, (50, 100), generator=g, dtype=torch.int8).to(DEV))
    qs, ws, bias = (torch.rand(n, generator=g).to(DEV) for n in (40, 50, 50))
    res = torch.randn(40, 50, generator=g).to(DEV)
    calls = [(q, qs, w, ws), (q[0], qs.half(), w, ws.half(), bias.half()), (q[:, :1], qs[:1], w, ws), (q, qs[None], w, ws, bias),
             (q[:, :3], qs[:3], w[:1], ws[:1])]
    options = [dict(), dict(out_dtype=torch.float16, silu=True), dict(out_dtype=torch.bfloat16)]
    for args in calls:
        for kw in options + ([dict(residual=res, residual_factor=0.5)] if args[0].shape[-2] == 40 else []):
            native = int8._native_gemm(*args, *[None] * (5 - len(args)), kw.get("out"), kw.get("out_dtype", torch.float32), kw.get("silu", False),
                                       kw.get("residual"), kw.get("residual_factor", 1.0))
            assert native is not None
            with monkeypatch.context() as mp:
                mp.setattr(int8, "_native_gemm", lambda *a: None)
                _same([native], [int8.gemm(*args, **kw)])
    out = torch.empty(40, 64, device=DEV)[:, :50]
    assert int8.gemm(q, qs, w, ws, out=out) is out or torch.equal(out, int8.gemm(q, qs, w, ws))
    for bad in (dict(out=out[:, :49]), dict(residual=res.half()), dict(out_dtype=torch.float64)):
        with pytest.raises(ValueError):
            int8.gemm(q, qs, w, ws, **bad)
    with torch.inference_mode(False), pytest.raises(RuntimeError, match="inference only"):
        int8.gemm(q, qs.clone().requires_grad_(), w, ws)


@pytest.mark.gpu
@torch.inference_mode()
def test_block_norm(monkeypatch):
    g = torch.Generator().manual_seed(1)
    ln, rms = torch.nn.LayerNorm(96, device=DEV), torch.nn.RMSNorm(96, device=DEV, dtype=torch.bfloat16)
    bare = torch.nn.LayerNorm(96, elementwise_affine=False, device=DEV)
    x = torch.randn(2, 6, 96, generator=g).to(DEV)
    wide = torch.randn(2, 6, 200, generator=g).half().to(DEV)[..., 8:104]
    gate = torch.randn(2, 1, 96, generator=g).half().to(DEV)
    for kw in (dict(pre=ln), dict(post=rms, pre=bare, gate=gate, gate_activation="tanh", factor=0.5), dict(post=ln, quantize=True),
               dict(pre=rms, quantize=True), dict(post=bare), dict(gate=gate[0, 0], pre=ln)):
        args = (kw.get("post"), kw.get("gate"), kw.get("gate_activation", ""), kw.get("factor", 1.0), kw.get("pre"), kw.get("quantize", False), None)
        for a, b in ((x, wide), (x[:, :1], wide[:, :1]), (x.bfloat16(), wide), (x[0], wide[1])):
            if kw.get("gate") is not None and a.dim() == 2:
                continue
            native = norms._native(a, b, *args)
            assert native is not None
            with monkeypatch.context() as mp:
                mp.setattr(norms, "_native", lambda *_: None)
                _same(native, norms.block_norm(a, b, **kw))
    class Odd(torch.nn.LayerNorm):  # a weight that is no parameter of the module's own
        @property
        def weight(self):
            return torch.full((96,), 2.0, device=DEV)
    odd = Odd.__new__(Odd)
    torch.nn.Module.__init__(odd)
    odd.normalized_shape, odd.eps, odd.bias = (96,), 1e-5, None
    assert norms._native(x, wide, None, None, "", 1.0, odd, False, None) is None
    assert torch.allclose(norms.block_norm(x, wide, pre=odd)[1].float(), 2 * norms.block_norm(x, wide, pre=bare)[1].float(), atol=1e-2)
    for bad in (dict(pre=torch.nn.LayerNorm(95, device=DEV)), dict(pre=ln.cpu() if False else torch.nn.LayerNorm(96)), dict(gate=gate.float())):
        with pytest.raises(ValueError):
            norms.block_norm(x, wide, **bad)


@pytest.mark.gpu
@torch.inference_mode()
def test_window(monkeypatch):
    g = torch.Generator().manual_seed(2)
    fused = torch.randn(2, 50, 3, 4, 64, generator=g).half().to(DEV)
    q, k, v = fused.unbind(2)
    lengths = torch.tensor([50, 20], dtype=torch.int32, device=DEV)
    for kw in (dict(), dict(left=5, right=2, sinks=1, kv_lengths=lengths, q_starts=torch.zeros_like(lengths)), dict(left=1 << 40, right=None, scale=0.3)):
        args = (kw.get("left"), kw.get("right", 0), kw.get("sinks", 0), kw.get("scale"), kw.get("kv_lengths"), kw.get("q_starts"))
        for a in (q, q[:, -1:]):
            native = window._native(a, k, v, *args)
            assert native is not None
            with monkeypatch.context() as mp:
                mp.setattr(window, "_native", lambda *_: None)
                _same([native], [window.attention(a, k, v, **kw)])
    for bad in (dict(left=-1), dict(sinks=-1), dict(kv_lengths=lengths.long())):
        with pytest.raises(ValueError):
            window.attention(q, k, v, **bad)


class Layer:
    """x -> x + 0.5 gate post(W_out attention(W_qkv pre(x))), then x + W_down silu(W_up pre2(x)): the three operators as a
    streaming layer with 8-bit weights chains them, int8 rows between norms and products."""

    def __init__(self, d, heads, kv_heads, ff, g):
        self.d, self.heads, self.kv_heads, self.dk = d, heads, kv_heads, d // heads
        dense = lambda n, k: torch.randn(n, k, generator=g) / math.sqrt(k)  # noqa: E731
        n = (heads + 2 * kv_heads) * self.dk
        self.qkv, self.out = int8.Int8Linear.from_dense(dense(n, d)), int8.Int8Linear.from_dense(dense(d, d), torch.randn(d, generator=g))
        self.up, self.down = int8.Int8Linear.from_dense(dense(ff, d)), int8.Int8Linear.from_dense(dense(d, ff))
        self.norms = [torch.nn.RMSNorm(d, eps=1e-5, device=DEV) for _ in range(2)] + [torch.nn.LayerNorm(d, device=DEV)]
        self.gate = torch.randn(d, generator=g).half().to(DEV)

    def __call__(self, x, cache, seen, window_size=20, sinks=2):
        """x [B, T, d], tokens behind the `seen` ones of each sequence whose keys and values lie in cache [2, B, Tmax, Hkv, dk]."""
        b, t, d = x.shape
        pre, post, pre2 = self.norms
        _, q, qs = norms.block_norm(x, None, pre=pre, quantize=True)
        y = int8.gemm(q, qs, self.qkv.weight, self.qkv.scale, out_dtype=torch.float16).view(b, t, -1, self.dk)
        at = seen[:, None] + torch.arange(t, device=DEV)
        for i, part in enumerate((y[:, :, self.heads:self.heads + self.kv_heads], y[:, :, self.heads + self.kv_heads:])):
            cache[i][torch.arange(b, device=DEV)[:, None], at.long()] = part
        a = window.attention(y[:, :, :self.heads], cache[0], cache[1], left=window_size, sinks=sinks, kv_lengths=(seen + t).int())
        o = self.out.linear(a.view(b, t, d), out_dtype=torch.float16)
        x, q, qs = norms.block_norm(x, o, post=post, gate=self.gate, gate_activation="sigmoid", factor=0.5, pre=pre2, quantize=True)
        h = int8.gemm(q, qs, self.up.weight, self.up.scale, silu=True)
        q, qs, _ = lowbit.quantize(h[None], (0, h.stride(0), 1, b * t), b * t, h.shape[1], 1)
        flat = x.view(b * t, d)
        return int8.gemm(q, qs, self.down.weight, self.down.scale, residual=flat, out=flat).view(b, t, d)

    def plain(self, x, window_size=20, sinks=2):
        """The whole sequences at once in 64 bits, activations unrounded."""
        pre, post, pre2 = self.norms
        weight = lambda w: w.weight.cpu().double() * w.scale.cpu().double()[:, None]  # noqa: E731

        def norm(v, m):
            c = v - v.mean(-1, keepdim=True) if hasattr(m, "bias") else v
            z = c / torch.sqrt((c * c).mean(-1, keepdim=True) + m.eps) * m.weight.detach().cpu().double()
            return z + m.bias.detach().cpu().double() if hasattr(m, "bias") else z

        b, t, d = x.shape
        x = x.cpu().double()
        y = (norm(x, pre) @ weight(self.qkv).t()).view(b, t, -1, self.dk).transpose(1, 2)
        group = self.heads // self.kv_heads
        q, k, v = y[:, :self.heads], *(y[:, s:s + self.kv_heads].repeat_interleave(group, 1) for s in (self.heads, self.heads + self.kv_heads))
        i, j = torch.arange(t)[:, None], torch.arange(t)
        mask = (j <= i) & ((j >= i - window_size) | (j < sinks))
        s = (q @ k.transpose(2, 3) / math.sqrt(self.dk)).masked_fill(~mask, float("-inf"))
        a = (s.softmax(-1) @ v).transpose(1, 2).reshape(b, t, d)
        o = a @ weight(self.out).t() + self.out.bias.cpu().double()
        x = x + 0.5 * torch.sigmoid(self.gate.cpu().double()) * norm(o, post)
        h = norm(x, pre2) @ weight(self.up).t()
        return x + (h / (1 + torch.exp(-h))) @ weight(self.down).t()


@pytest.mark.gpu
@torch.inference_mode()
def test_a_layer_over_whole_sequences_and_token_by_token():
    """The prompt in one call, then one token at a time: each token's output is the whole sequence's in 64 bits up to the int8
    rounding of four activations (steps of 1/127 of a row's largest value, a third of a step in the mean, four times; 0.02 of
    the layer's output in norm), and the same tokens in one call or one by one differ by as little."""
    g = torch.Generator().manual_seed(5)
    layer = Layer(256, 4, 2, 512, g)
    b, t, more = 2, 45, 5
    x = torch.randn(b, t + more, 256, generator=g).to(DEV)
    want = layer.plain(x)
    cache = torch.full((2, b, 64, 2, 64), float("nan"), dtype=torch.float16, device=DEV)
    outs = [layer(x[:, :t].contiguous(), cache, torch.zeros(b, dtype=torch.int64, device=DEV))]
    for i in range(more):
        outs.append(layer(x[:, t + i:t + i + 1].contiguous(), cache, torch.full((b,), t + i, dtype=torch.int64, device=DEV)))
    got = torch.cat(outs, 1).cpu().double()
    assert torch.isfinite(got).all()
    off = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    assert off < 0.02, off


def test_a_missing_native_library_is_an_error(monkeypatch):
    def missing():
        raise RuntimeError("missing")
    monkeypatch.setattr(_hip, "native", missing)
    with pytest.raises(RuntimeError, match="missing"):
        window.attention(*(torch.zeros(1, 1, 1, 64),) * 3)


def test_forward_mode_tangents_are_refused():
    """A dual tensor requires no grad, but its tangent would be lost all the same."""
    x, q, qs = torch.zeros(0, 16), torch.zeros(0, 16, dtype=torch.int8), torch.ones(0)
    w, ws, bias, heads = torch.zeros(4, 16, dtype=torch.int8), torch.ones(4), torch.zeros(4), torch.zeros(1, 0, 1, 8)
    norm = torch.nn.RMSNorm(16).requires_grad_(False)
    layer = int8.Int8Linear(w, ws, None)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        moving = SimpleNamespace(weight=dual(torch.ones(16)), eps=1e-5)
        calls = [lambda: norms.block_norm(dual(x), x), lambda: norms.block_norm(x, dual(x), pre=norm), lambda: norms.block_norm(x, x, pre=moving),
                 lambda: int8.gemm(q, qs, w, ws, dual(bias)), lambda: int8.gemm(q, dual(qs), w, ws), lambda: layer.linear(dual(x)),
                 lambda: window.attention(dual(heads), heads, heads), lambda: window.attention(heads, heads, dual(heads))]
        for call in calls:
            with pytest.raises(RuntimeError, match="inference only"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="inference only"):  # (which leaves forward mode on)
                call()
            with torch.inference_mode():
                call()
        norms.block_norm(x, x, pre=norm)
        window.attention(heads, heads, heads)


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused_on_the_gpu():
    x, norm, moving = torch.randn(3, 64, device=DEV), *(torch.nn.RMSNorm(64, device=DEV).requires_grad_(False) for _ in range(2))
    q, qs, w, ws = torch.zeros(3, 64, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV), torch.zeros(4, 64, dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    heads = torch.randn(1, 5, 2, 64, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        moving._parameters["weight"] = dual(moving.weight)  # (as torch.func.functional_call leaves it)
        for call in (lambda: norms.block_norm(x, dual(x), pre=norm), lambda: norms.block_norm(x, x, pre=moving), lambda: int8.gemm(q, dual(qs), w, ws), lambda: window.attention(heads, dual(heads), heads)):
            with pytest.raises(RuntimeError, match="inference only"):
                call()
        norms.block_norm(x, x, pre=norm), int8.gemm(q, qs, w, ws), window.attention(heads, heads, heads)
