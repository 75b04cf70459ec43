"""The native call path of int4.gemm and the paged cache's operators (kea_native): it takes the ordinary calls, gives the Python path's
bits, and leaves everything else to that path; and a decoder's layers made of them, run as a model would: a prompt in pieces, then
token by token in a captured graph, against the same layers in 64 bits on the values that the cache and the weights stand for."""
from __future__ import annotations

import math

import pytest
import torch
import torch.autograd.forward_ad

from kea_kernels import _hip, int4, lowbit, norms, paged

DEV = "cuda"


@pytest.mark.gpu
@torch.inference_mode()
def test_gemm(monkeypatch):
    g = torch.Generator().manual_seed(0)
    q = torch.randint(-128, 128, (1, 40, 112), generator=g, dtype=torch.int8).to(DEV)
    w = int4.pack(torch.randint(-8, 8, (50, 100), generator=g, dtype=torch.int8).to(DEV), torch.rand(50, 2, generator=g).to(DEV), 64)
    h = int4.pack(torch.randint(-8, 8, (50, 100), generator=g, dtype=torch.int8).to(DEV), torch.rand(50, 4, generator=g).half().to(DEV), 32)
    qs, bias = (torch.rand(n, generator=g).to(DEV) for n in (40, 50))
    res = torch.randn(40, 50, generator=g).to(DEV)
    for args in ((q, qs, w), (q[0], qs.half(), h, bias.half()), (q[:, :1], qs[:1], w), (q, qs[None], h, bias)):
        for kw in [dict(), dict(out_dtype=torch.float16, silu=True), dict(out_dtype=torch.bfloat16)] + (
                [dict(residual=res, residual_factor=0.5)] if args[0].shape[-2] == 40 else []):
            p = args[2]
            native = int4._native_gemm(args[0], args[1], p.words, p.scales, 50, 100, p.group, args[3] if len(args) > 3 else None, None,
                                       kw.get("out_dtype", torch.float32), kw.get("silu", False), kw.get("residual"), kw.get("residual_factor", 1.0))
            assert native is not None
            with monkeypatch.context() as mp:
                mp.setattr(int4, "_native_gemm", lambda *a: None)
                other = int4.gemm(*args, **kw)
            assert native.dtype == other.dtype and torch.equal(native, other)
    out = torch.empty(40, 64, device=DEV)[:, :50]
    assert torch.equal(int4.gemm(q, qs, w, out=out), int4.gemm(q, qs, w))
    for bad in (dict(out=out[:, :49]), dict(residual=res.half()), dict(out_dtype=torch.float64), dict(bias=bias[:49])):
        with pytest.raises(ValueError):
            int4.gemm(q, qs, w, **bad)
    with pytest.raises(ValueError):
        int4.gemm(q, qs, int4.Weight(w.words, w.scales, 70, 100, 64))
    with torch.inference_mode(False), pytest.raises(RuntimeError, match="inference only"):
        int4.gemm(q, qs.clone().requires_grad_(), w)


@pytest.mark.gpu
@torch.inference_mode()
def test_paged(monkeypatch):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(9, h, 64, generator=g).half().to(DEV) for h in (4, 2, 2))
    table = torch.randperm(20, generator=g).int().view(2, 10).to(DEV)
    lengths, offsets = torch.tensor([100, 150], dtype=torch.int32, device=DEV), torch.tensor([0, 5, 8], dtype=torch.int32, device=DEV)

    def run(native):
        torch.manual_seed(3)
        cache = paged.Cache.empty(20, 16, 2, 64, DEV)
        for t in (cache.k, cache.v):
            t.random_(-100, 100)
        for t in (cache.k_scale, cache.v_scale):
            t.uniform_(0.01, 0.02)
        four = (cache.k, cache.v, cache.k_scale, cache.v_scale)
        with monkeypatch.context() as mp:
            if not native:
                mp.setattr(paged, "_native", lambda *a: None)
            else:
                n = _hip.native()
                assert n.paged_write(*four, k, v, table, lengths, offsets) is True
                assert n.paged_read(*four, table, lengths, 7, None, torch.float16) is not None
                assert n.paged_attention(*four, q, table, lengths, offsets, None, None) is not None
                assert n.paged_attention(*four, q[:8], table, lengths, None, 5, 0.3) is not None
            paged.write(cache, k, v, table, lengths, offsets)
            outs = [paged.attention(q, cache, table, lengths, offsets), paged.attention(q[:8], cache, table, lengths, left=5, scale=0.3),
                    paged.attention(q[:, :2].float(), cache, table, lengths, offsets, left=2**40)]
            for dtype in (torch.float32, torch.float16, torch.bfloat16):
                outs += [*paged.read(cache, table, lengths, 7, out_dtype=dtype), *paged.read(cache, table, lengths, 50, starts=offsets[:2], out_dtype=dtype)]
        return [*outs, *four]

    for x, y in zip(run(True), run(False), strict=True):
        assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and torch.equal(x, y)
    cache = paged.Cache.empty(20, 16, 2, 64, DEV)
    for bad in (dict(q=q[:7], q_offsets=None), dict(q=q[..., :48]), dict(q=q[:, :3]), dict(table=table.long()), dict(kv_lengths=lengths[:1]), dict(left=-1),
                dict(q_offsets=lengths), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            paged.attention(**{**dict(q=q, cache=cache, table=table, kv_lengths=lengths, q_offsets=offsets), **bad})
    with torch.inference_mode(False), pytest.raises(RuntimeError, match="inference only"):
        paged.write(cache, k.clone().requires_grad_(), v, table, lengths, offsets)


def test_forward_mode_tangents_are_refused():
    w = int4.pack(torch.zeros(4, 32, dtype=torch.int8), torch.ones(4, 1), 32)
    cache, x = paged.Cache.empty(1, 16, 1, 16, "cpu"), torch.zeros(1, 1, 16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: int4.gemm(torch.zeros(1, 2, 32, dtype=torch.int8), dual(torch.ones(1, 2)), w), lambda: paged.write(cache, dual(x), x, table, lengths),
                     lambda: paged.attention(dual(x), cache, table, lengths)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()


# ---- two layers of a decoder --------------------------------------------------------------------------------------------------

D, HEADS, KV, HD, FF = 256, 8, 2, 64, 640


class Layer:
    """Norm, attention and feed-forward with 4-bit weights over a paged cache; a residual stream in FP32."""

    def __init__(self, g, dev):
        def linear(n, k):
            return int4.Int4Linear.from_dense(torch.randn(n, k, generator=g) / math.sqrt(k), group=64, device=dev)

        self.qkv, self.out, self.up, self.down = linear((HEADS + 2 * KV) * HD, D), linear(D, HEADS * HD), linear(FF, D), linear(D, FF)
        self.norms = [torch.nn.RMSNorm(D, eps=1e-5, device=dev).requires_grad_(False) for _ in range(2)]
        for n in self.norms:
            n.weight.copy_(1 + 0.1 * torch.randn(D, generator=g))
        self.cache = paged.Cache.empty(24, 16, KV, HD, dev)

    def __call__(self, x, table, lengths, offsets):
        q, qs = norms.block_norm(x, None, pre=self.norms[0], quantize=True)[1:]
        h = int4.gemm(q, qs, self.qkv.weight, out_dtype=torch.float16).view(-1, HEADS + 2 * KV, HD)
        paged.write(self.cache, h[:, HEADS:HEADS + KV], h[:, HEADS + KV:], table, lengths, offsets)
        o = paged.attention(h[:, :HEADS], self.cache, table, lengths, offsets)
        oq, os, _ = lowbit.quantize(o.view(1, -1, HEADS * HD), (0, HEADS * HD, 1, len(o)), len(o), HEADS * HD, 1)
        x = int4.gemm(oq, os, self.out.weight, residual=x)
        q, qs = norms.block_norm(x, None, pre=self.norms[1], quantize=True)[1:]
        u = int4.gemm(q, qs, self.up.weight, silu=True)
        uq, us, _ = lowbit.quantize(u[None], (0, FF, 1, len(u)), len(u), FF, 1)
        return int4.gemm(uq, us, self.down.weight, residual=x)


def dense_layer(layer, x, lengths):
    """The same in 64 bits over whole sequences, without rounding rows, keys or values."""
    w = {n: getattr(layer, n).weight.dense().cpu().double() for n in ("qkv", "out", "up", "down")}
    norm = lambda v, m: v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * m.weight.cpu().double()  # noqa: E731
    outs = []
    for n, v in zip(lengths, x.split(lengths)):
        h = (norm(v, layer.norms[0]) @ w["qkv"].t()).view(n, -1, HD)
        o = torch.empty(n, HEADS, HD, dtype=torch.float64)
        for i in range(HEADS):
            kv = HEADS + i * KV // HEADS
            s = (h[:, i] @ h[:, kv].t() / math.sqrt(HD)).masked_fill(torch.triu(torch.ones(n, n, dtype=torch.bool), 1), -math.inf)
            o[:, i] = torch.softmax(s, 1) @ h[:, kv + KV]
        v = v + o.view(n, -1) @ w["out"].t()
        u = norm(v, layer.norms[1]) @ w["up"].t()
        outs.append(v + u / (1 + torch.exp(-u)) @ w["down"].t())
    return torch.cat(outs)


@pytest.mark.gpu
@torch.inference_mode()
def test_layers_over_a_prompt_in_pieces_and_token_by_token():
    g = torch.Generator().manual_seed(5)
    layers, lengths = [Layer(g, DEV) for _ in range(2)], [130, 61, 90]
    x = torch.randn(sum(lengths), D, generator=g).to(DEV)
    parts = x.split(lengths)
    table = torch.randperm(24, generator=g).int()[:21].view(3, 7)
    table = torch.cat([table, torch.full((3, 2), -1, dtype=torch.int32)], 1)
    for i, n in enumerate(lengths):
        table[i, -(-n // 16):] = -1
    spare = iter(sorted(set(range(24)) - set(table.flatten().tolist())))
    for i, n in enumerate(lengths):
        for j in range(-(-n // 16)):
            if table[i, j] < 0:
                table[i, j] = next(spare)
    table = table.to(DEV)
    done, outs = [0, 0, 0], [[], [], []]

    def step(news):
        nonlocal done
        rows = torch.cat([parts[b][done[b]:done[b] + n] for b, n in enumerate(news)])
        done = [a + n for a, n in zip(done, news)]
        at = torch.tensor([sum(news[:b]) for b in range(4)], dtype=torch.int32, device=DEV)
        ln = torch.tensor(done, dtype=torch.int32, device=DEV)
        for layer in layers:
            rows = layer(rows, table, ln, at)
        for b in range(3):
            outs[b].append(rows[at[b]:at[b + 1]])

    for news in ((100, 40, 0), (5, 1, 70), (20, 1, 0)):
        step(news)
    # what is left one token at a time, in a captured graph that follows the lengths
    left = [a - b for a, b in zip(lengths, done)]
    rows, ln, at = torch.zeros(3, D, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = rows
        for layer in layers:
            y = layer(y, table, ln, at)
    while any(left):
        live = [b for b in range(3) if left[b]]
        for i, b in enumerate(live):
            rows[i] = parts[b][done[b]]
        rows[len(live):] = float("nan")  # (rows of no sequence)
        done = [a + (b in live) for b, a in enumerate(done)]
        left = [a - (b in live) for b, a in enumerate(left)]
        at.copy_(torch.tensor([len([b for b in live if b < i]) for i in range(4)]))
        ln.copy_(torch.tensor(done))
        graph.replay()
        torch.cuda.synchronize()
        for i, b in enumerate(live):
            outs[b].append(y[i:i + 1].clone())
    got = torch.cat([torch.cat(o) for o in outs]).cpu().double()
    want = x.cpu().double()
    for layer in layers:
        want = dense_layer(layer, want, lengths)
    # rows, keys and values in 8 bits: each rounding is off by 1/254 of a row's largest element at most, about 1/254/sqrt(3) * 3 of its
    # root mean square; ten of them in line, and weights of 64 products apart, stay within 8 %
    error = (got - want).square().mean().sqrt() / want.square().mean().sqrt()
    assert torch.isfinite(got).all() and error < 0.08, error
    # the pieces do not matter beyond the rounding of sums: all at once gives the same within a few steps of 8 bits
    cold = [Layer.__new__(Layer) for _ in layers]
    for a, b in zip(cold, layers):
        a.__dict__.update(b.__dict__)
        a.cache = paged.Cache.empty(24, 16, KV, HD, DEV)
    y, at = x, torch.tensor([0, 130, 191, 281], dtype=torch.int32, device=DEV)
    for layer in cold:
        y = layer(y, table, torch.tensor(lengths, dtype=torch.int32, device=DEV), at)
    error = (got - y.cpu().double()).square().mean().sqrt() / want.square().mean().sqrt()
    assert error < 0.02, error
