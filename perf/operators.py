"""The operators of a transformer layer with 8-bit weights, as a program built on kea_kernels calls them.

  gemm    int8.gemm: the int8 rows that lowbit.quantize makes times int8 weights, with a scale for each row (token) and each
          weight row (channel): the layers that do not stand 1 or 2 bits
  norm    norms.block_norm: a block's output normalised, gated, scaled and added to the residual stream, and the next block's
          input normalised, as values or as the int8 rows that the product reads, in one pass
  attend  window.attention: attention within a sliding window and to the first few tokens, over clips, long recordings, and one
          token at a time against a cache

Row counts are tokens: one at a time, frames of a clip (125 for 10 s), of a batch, of a long recording. Matrix shapes are the
encoder's (1024 <-> 4096) and the decoder's (640 -> 2560, 640 -> 1030), and odd ones.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PACKAGE = str(Path(__file__).resolve().parents[1] / "kea-kernels_amd")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(4096, 1024), (1024, 4096), (1024, 1024), (2048, 1024), (4096, 4096), (2560, 640), (1030, 640)]  # (n, k)
EPS = 1e-5


def listed() -> list:
    def gemm(name, m, n, k, **more):
        return {"name": name, "op": "gemm", "m": m, "n": n, "k": k, "scales": "f32", "bias": False, "silu": False,
                "residual": False, "out": "f16", **more}

    def norm(name, rows, d, **more):
        return {"name": name, "op": "norm", "rows": rows, "d": d, "stream": "f32", "block": "f16", "post": "", "pre": "layer",
                "gate": "", "act": "", "factor": 0.5, "quantize": False, **more}

    def attend(name, batch, tq, tk, **more):
        return {"name": name, "op": "attend", "batch": batch, "tq": tq, "tk": tk, "heads": 8, "kv_heads": 8, "d": 128,
                "left": 1023, "right": 0, "sinks": 4, "dtype": "bf16", "ragged": False, "packed": False, **more}

    return [
        # one step of a decoder: a token's row through its input projection
        gemm("gemm_token", 1, 2560, 640, scales="f16", bias=True),
        # a few streams' tokens through a down projection, added to the residual stream
        gemm("gemm_16_down", 16, 1024, 4096, residual=True, out="f32"),
        # a joint network's logits over the frames of a 30-s clip: odd sizes, rows that are no multiple of 16 long
        gemm("gemm_375_odd", 375, 1030, 641, bias=True, out="f32"),
        # the up projection of eight 10-s clips with its activation
        gemm("gemm_1000_up", 1000, 4096, 1024, silu=True),
        # a long recording in one call
        gemm("gemm_16000", 16000, 4096, 4096, bias=True, out="bf16"),
        # one token between two blocks
        norm("norm_token", 1, 1024, stream="f16", post="rms", pre="rms", factor=1.0),
        # eight clips between two feed-forwards, the next block's input as int8 rows
        norm("norm_1000_rows8", 1000, 1024, post="layer", gate="clip", quantize=True),
        # a gate of its own for each token, a width that no vector load fits
        norm("norm_999_odd", 999, 1031, stream="bf16", block="bf16", post="rms", pre="layer", gate="token", act="sigmoid"),
        # a long recording, wide rows
        norm("norm_16000", 16000, 4096, stream="bf16", block="bf16", post="rms", pre="rms", gate="channel", act="tanh"),
        # one token of 16 streams of different ages, each against its own long cache
        attend("attend_token", 16, 1, 16000, kv_heads=2, ragged=True),
        # two padded 60-s clips with limited context to both sides, on the encoder's fused projection
        attend("attend_clips", 2, 750, 750, left=128, right=128, sinks=1, dtype="f32", ragged=True, packed=True),
        # a recording of 13 minutes, causal
        attend("attend_long", 1, 10000, 10000, kv_heads=4),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number in lo .. hi, even over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("gemm", "norm", "attend"))
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "gemm":
        n, k = rng.choice(SHAPES) if rng.random() < 0.6 else (_spread(rng, 1, 4100), _spread(rng, 1, 4100))
        out = rng.choice(("f32", "f16", "bf16"))
        return {"op": op, "m": _spread(rng, 1, 16000), "n": n, "k": k, "scales": rng.choice(("f32", "f16")), "bias": yes(),
                "silu": yes(), "residual": yes(), "out": out}
    if op == "norm":
        d = rng.choice((640, 1024, 2048, 4096)) if yes() else _spread(rng, 2, 4100)
        stream, post, pre = rng.choice(("f32", "f16", "bf16")), rng.choice(("", "rms", "layer")), rng.choice(("", "rms", "layer"))
        block = rng.choice(("f32", "f16", "bf16"))
        return {"op": op, "rows": _spread(rng, 1, 16000), "d": d, "stream": stream, "block": block, "post": post, "pre": pre,
                "gate": rng.choice(("", "channel", "clip", "token")), "act": rng.choice(("", "sigmoid", "tanh")),
                "factor": rng.choice((0.5, 1.0, 0.1)), "quantize": pre != "" and block != "f32" and yes()}
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"op": op, "heads": kv_heads * rng.choice((1, 2, 4) if kv_heads < 8 else (1,)), "kv_heads": kv_heads,
            "d": rng.choice((64, 128, 80)), "sinks": rng.choice((0, 1, 4, 17)), "dtype": rng.choice(("f32", "f16", "bf16")),
            "ragged": yes(), "packed": False}
    if yes():  # tokens against a cache
        tk = _spread(rng, 1, 20000)
        return {**case, "batch": _spread(rng, 1, 32), "tq": min(tk, rng.choice((1, 1, 1, 4))), "tk": tk, "left": _spread(rng, 1, 4096),
                "right": 0}
    t = _spread(rng, 1, 6000)
    return {**case, "batch": max(1, min(8, 6000 // t)), "tq": t, "tk": t, "left": _spread(rng, 1, 2048),
            "right": rng.choice((0, 0, 5, 128)), "packed": kv_heads == case["heads"]}


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _rows8(x):
    """Float rows as int8 with a scale each, rows padded to whole 16 bytes as lowbit.quantize leaves them."""
    s = (x.abs().amax(1) / 127).clamp_min(1e-30)
    q = torch.zeros(x.shape[0], -(-x.shape[1] // 16) * 16, dtype=torch.int8, device=x.device)
    q[:, :x.shape[1]] = torch.round(x / s[:, None]).to(torch.int8)
    return q, s


def _norm_module(kind, d, randn):
    """The norm that a model holds in front of or behind a block."""
    if not kind:
        return None
    m = torch.nn.LayerNorm(d, eps=EPS) if kind == "layer" else torch.nn.RMSNorm(d, eps=EPS)
    m = m.to("cuda").requires_grad_(False)
    m.weight.copy_(1 + 0.1 * randn(d))
    if kind == "layer":
        m.bias.copy_(0.1 * randn(d))
    return m


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "gemm":
        m, n, k, st = case["m"], case["n"], case["k"], DTYPES[case["scales"]]
        q, qs = _rows8(randn(m, k) * (0.5 + torch.rand(m, 1, generator=g, device="cuda")))
        w, ws = _rows8(randn(n, k) / math.sqrt(k))
        return {"case": case, "q": q[None], "qs": qs.to(st)[None], "w": w[:, :k], "ws": ws.to(st),
                "bias": 0.1 * randn(n) if case["bias"] else None, "residual": randn(m, n) if case["residual"] else None}
    if case["op"] == "norm":
        rows, d, st, bt = case["rows"], case["d"], DTYPES[case["stream"]], DTYPES[case["block"]]
        gates = {"": 0, "channel": 1, "clip": 1 if rows % 8 else 8, "token": rows}[case["gate"]]
        return {"case": case, "x": (2 * randn(rows, d)).to(st), "block": (randn(rows, d) * (0.2 + randn(rows, 1).abs())).to(bt),
                "post": _norm_module(case["post"], d, randn), "pre": _norm_module(case["pre"], d, randn),
                "gate": randn(gates, d).to(bt) if gates else None}
    b, tq, tk, h, hk, d, dt = (case[x] for x in ("batch", "tq", "tk", "heads", "kv_heads", "d", "dtype"))
    if case["packed"]:  # slices of a fused projection
        q, k, v = randn(b, tk, 3 * h * d).to(DTYPES[dt]).view(b, tk, 3, h, d).unbind(2)
    else:
        q, k, v = (randn(b, t, heads, d).to(DTYPES[dt]) for t, heads in ((tq, h), (tk, hk), (tk, hk)))
    lengths = starts = None
    if case["ragged"]:
        low = max(tq if tq < tk else 1, tk // 4)
        lengths = torch.randint(low, tk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        starts = torch.zeros_like(lengths) if tq == tk else lengths - tq
    return {"case": case, "q": q, "k": k, "v": v, "lengths": lengths, "starts": starts}


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state: dict):
    case = state["case"]
    if own:
        return _own(case, state)
    return {"gemm": _gemm, "norm": _norm, "attend": _attend}[case["op"]](case, state)


def _own(case, s):
    from kea_kernels import int8, norms, window
    if case["op"] == "gemm":
        return int8.gemm(s["q"], s["qs"], s["w"], s["ws"], s["bias"], silu=case["silu"], residual=s["residual"],
                         residual_factor=0.5, out_dtype=DTYPES[case["out"]])
    if case["op"] == "norm":
        out = norms.block_norm(s["x"], s["block"], post=s["post"], gate=s["gate"], gate_activation=case["act"],
                               factor=case["factor"], pre=s["pre"], quantize=case["quantize"])
        if case["quantize"]:  # the values that the int8 rows stand for, in the block's type
            y, q, qs = out
            return y, (q[0, :, :case["d"]].float() * qs[0, :, None]).to(s["block"].dtype)
        return out
    return window.attention(s["q"], s["k"], s["v"], left=case["left"], right=case["right"], sinks=case["sinks"],
                            kv_lengths=s["lengths"], q_starts=s["starts"])


def _gemm(case, s):
    k = case["k"]
    r = (s["q"][0, :, :k].float() @ s["w"].float().t()) * s["qs"][0].float()[:, None] * s["ws"].float()
    if s["bias"] is not None:
        r = r + s["bias"]
    if case["silu"]:
        r = r * torch.sigmoid(r)
    if s["residual"] is not None:
        r = s["residual"] + 0.5 * r
    return r.to(DTYPES[case["out"]])


def _normed(v, m):
    if m is None:
        return v
    if isinstance(m, torch.nn.LayerNorm):
        c = v - v.mean(1, keepdim=True)
        return c * torch.rsqrt((c * c).mean(1, keepdim=True) + m.eps) * m.weight + m.bias
    return v * torch.rsqrt((v * v).mean(1, keepdim=True) + m.eps) * m.weight


def _norm(case, s):
    p = _normed(s["block"].float(), s["post"])
    if s["gate"] is not None:
        g = s["gate"].float()
        g = torch.sigmoid(g) if case["act"] == "sigmoid" else torch.tanh(g) if case["act"] == "tanh" else g
        p = (p.view(g.shape[0], -1, p.shape[1]) * g[:, None]).view_as(p)
    y = s["x"].float() + case["factor"] * p
    if s["pre"] is None:
        return y.to(s["x"].dtype), None
    z = _normed(y, s["pre"])
    if case["quantize"]:
        scale = (z.abs().amax(1, keepdim=True) / 127).clamp_min(1e-30)
        z = torch.round(z / scale) * scale
    return y.to(s["x"].dtype), z.to(s["block"].dtype)


def _attend(case, s):
    q = s["q"].float().transpose(1, 2)                                          # [B, H, T, D]
    b, h, tq, d = q.shape
    tk, hk = s["k"].shape[1:3]
    dev = q.device
    lengths = torch.full((b,), tk, device=dev) if s["lengths"] is None else s["lengths"].long()
    starts = lengths - tq if s["starts"] is None else s["starts"].long()
    pos = starts[:, None] + torch.arange(tq, device=dev)                        # [B, Tq]
    if tq == 1 and case["sinks"] + case["left"] + 1 < tk:  # the keys that a single token can see, taken out of the cache
        near = torch.arange(-case["left"], 1, device=dev) + pos                 # [B, left + 1]
        first = torch.arange(case["sinks"], device=dev).expand(b, -1)
        keys = torch.cat([first, near], 1)
        seen = torch.cat([first < pos - case["left"], near >= 0], 1)[:, None]   # (a sink inside the window counts once)
        at = keys.clamp(0, tk - 1)[:, None, :, None].expand(-1, hk, -1, d)
        k, v = (s[x].gather(1, at.transpose(1, 2)).float().transpose(1, 2) for x in ("k", "v"))
        visible = seen & ((keys < lengths[:, None]) & (keys <= pos))[:, None]
    else:
        k, v = (s[x].float().transpose(1, 2) for x in ("k", "v"))
        j = torch.arange(tk, device=dev)
        p = pos[:, :, None]
        visible = (j <= p + case["right"]) & ((j >= p - case["left"]) | (j < case["sinks"])) & (j < lengths[:, None, None])
    visible = (visible & ((pos >= 0) & (pos < lengths[:, None]))[:, :, None])[:, None, None]
    q = q.reshape(b, hk, h // hk, tq, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()[:, :, None]) * (1 / math.sqrt(d))   # [B, Hkv, G, Tq, Tk]
    scores = scores.masked_fill(~visible, float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    out = torch.matmul(e / e.sum(-1, keepdim=True).clamp_min(1e-30), v.contiguous()[:, :, None])
    return out.view(b, h, tq, d).transpose(1, 2).to(s["q"].dtype).contiguous()


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        b = m * k + n * k + (m + n) * size[case["scales"]] + m * n * size[case["out"]]
        return {"bytes": b + 4 * n * case["bias"] + 4 * m * n * case["residual"], "flops": 2 * m * n * k}
    if case["op"] == "norm":
        rows, d, x, o = case["rows"], case["d"], size[case["stream"]], size[case["block"]]
        z = 0 if not case["pre"] else rows * d + 4 * rows if case["quantize"] else rows * d * o
        gates = {"": 0, "channel": 1, "clip": 1 if rows % 8 else 8, "token": rows}[case["gate"]]
        vectors = {"": 0, "rms": 4, "layer": 8}
        return {"bytes": rows * d * (2 * x + o) + z + gates * d * o + d * (vectors[case["post"]] + vectors[case["pre"]]),
                "flops": 16 * rows * d}
    b, tq, tk, h, hk, d = (case[x] for x in ("batch", "tq", "tk", "heads", "kv_heads", "d"))
    length = 5 * tk // 8 if case["ragged"] else tk   # (the mean of the drawn lengths)
    start = 0 if tq == tk else max(0, length - tq)
    pairs, keys = 0, min(length, case["sinks"])
    for p in range(start, min(start + tq, length)):
        low, high = max(0, p - case["left"]), min(length - 1, p + case["right"])
        pairs += high - low + 1 + min(low, case["sinks"])
    low, high = max(0, start - case["left"]), min(length - 1, start + tq - 1 + case["right"])
    keys = high - low + 1 + min(low, case["sinks"])
    return {"bytes": size[case["dtype"]] * b * d * (h * tq * 2 + 2 * hk * keys), "flops": 4 * d * h * b * pairs}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        acc = s["q"][0].double()[:, :case["k"]].mm(s["w"].double().t().contiguous())
        r = torch.einsum("mn,m,n->mn", acc, s["qs"][0].double(), s["ws"].double())
        if case["bias"]:
            r += s["bias"].double()
        if case["silu"]:
            r /= 1 + torch.exp(-r)
        return s["residual"].double() + r / 2 if case["residual"] else r
    if case["op"] == "norm":
        def moments(v, m):
            if isinstance(m, torch.nn.LayerNorm):
                var, mean = torch.var_mean(v, 1, unbiased=False, keepdim=True)
                return (v - mean) / torch.sqrt(var + m.eps) * m.weight.double() + m.bias.double()
            return v / torch.sqrt(v.square().mean(1, keepdim=True) + m.eps) * m.weight.double()

        p = s["block"].double()
        if s["post"] is not None:
            p = moments(p, s["post"])
        if s["gate"] is not None:
            g = s["gate"].double().repeat_interleave(case["rows"] // s["gate"].shape[0], 0)
            p = p * {"": lambda v: v, "sigmoid": lambda v: 1 / (1 + torch.exp(-v)), "tanh": torch.tanh}[case["act"]](g)
        y = s["x"].double() + case["factor"] * p
        if s["pre"] is None:
            return y, None
        z = moments(y, s["pre"])
        if case["quantize"]:
            unit = (z.abs().amax(1) / 127).clamp_min(1e-30)[:, None]
            z = torch.round(z / unit) * unit
        return y, z
    b, tq, tk, h, hk = (case[x] for x in ("batch", "tq", "tk", "heads", "kv_heads"))
    out = torch.zeros(b, tq, h, case["d"], dtype=torch.float64, device="cuda")
    for i in range(b):
        n = tk if s["lengths"] is None else int(s["lengths"][i])
        at = n - tq if s["starts"] is None else int(s["starts"][i])
        for first in range(0, tq, 256):  # a block of queries, and the keys that one of them can see
            p = torch.arange(first, min(first + 256, tq), device="cuda") + at
            p = p[(p >= 0) & (p < n)]
            if not p.numel():
                continue
            low, high = max(0, int(p[0]) - case["left"]), min(n - 1, int(p[-1]) + case["right"])
            j = torch.cat([torch.arange(min(case["sinks"], low), device="cuda"), torch.arange(low, high + 1, device="cuda")])
            unseen = (j > p[:, None] + case["right"]) | ((j < p[:, None] - case["left"]) & (j >= case["sinks"]))
            for head in range(h):
                kv = head * hk // h
                w = s["q"][i, p - at, head].double().mm(s["k"][i, j, kv].double().t().contiguous()) / math.sqrt(case["d"])
                out[i, p - at, head] = w.masked_fill(unseen, -math.inf).softmax(1).mm(s["v"][i, j, kv].double())
    return out
