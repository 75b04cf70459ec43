"""The operators of a decoder's layer with 4-bit weights and an 8-bit cache in pages, as a program built on kea_kernels calls them.

  gemm    int4.gemm: the int8 rows that lowbit.quantize makes times 4-bit weights with a scale for each group of a row's weights
  write   paged.write and paged.read of the same places: the new tokens' keys and values, quantised to int8 in the cache's pages
          with a scale for each token and head, and what the cache holds for them
  read    paged.read: a run of positions of each sequence, out of the pages, as dense tensors of values
  attend  paged.attention: attention of the new tokens of each sequence to its keys in the pages: one token of each, a few
          drafted ones, pieces of prompts and single tokens in one batch, a long piece of one prompt

The new tokens of a batch are packed, sequence after sequence. Matrix shapes are the encoder's (1024 <-> 4096), the decoder's
(640 -> 2560, 640 -> 1030), and odd ones.
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


def listed() -> list:
    def gemm(name, m, n, k, **more):
        return {"name": name, "op": "gemm", "m": m, "n": n, "k": k, "group": 128, "scales": "f16", "bias": False, "silu": False,
                "residual": False, "out": "f16", **more}

    def cache(name, op, batch, new, length, **more):
        return {"name": name, "op": op, "batch": batch, "new": new, "length": length, "mixed": False, "kv_heads": 4, "d": 128,
                "page": 16, "dtype": "bf16", **more}

    def attend(name, batch, new, length, **more):
        return cache(name, "attend", batch, new, length, **{"heads": 16, "left": None, **more})

    return [
        # one step of a decoder: a token's row through its input projection
        gemm("gemm_token", 1, 2560, 640, group=64, scales="f32", bias=True),
        # a token's row through the widest matrix of a large decoder
        gemm("gemm_vector", 1, 16384, 4096),
        # a few streams' tokens through a down projection, added to the residual stream; a fine group
        gemm("gemm_13_down", 13, 1024, 4096, group=32, residual=True, out="f32"),
        # a piece of a prompt through the up projection with its activation
        gemm("gemm_prompt", 4000, 4096, 4096, silu=True, bias=True, out="bf16"),
        # the new tokens of 16 streams
        cache("write_tokens", "write", 16, 1, 2000),
        # a prompt of 16000 tokens
        cache("write_prompt", "write", 1, 16000, 16000, kv_heads=8, dtype="f16", page=64),
        # the last tokens of a few short sequences, odd heads
        cache("read_short", "read", 3, 33, 500, kv_heads=5, d=80, dtype="f32"),
        # eight whole sequences, dense, for an operator that takes no pages
        cache("read_whole", "read", 8, 4000, 4000, kv_heads=8, page=32),
        # one token of 16 streams of different ages, each against its own long cache
        attend("attend_tokens", 16, 1, 16000),
        # four drafted tokens of each of eight streams, to the last 1000 and some keys
        attend("attend_drafts", 8, 4, 4000, left=1023, kv_heads=2, heads=8, dtype="f16", page=64),
        # pieces of prompts beside single tokens, odd heads, FP32
        attend("attend_mixed", 10, 250, 1500, mixed=True, kv_heads=3, heads=6, d=80, dtype="f32"),
        # the last piece of a long prompt
        attend("attend_prompt", 1, 2048, 16000, kv_heads=4, page=64),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A whole number in lo .. hi, even over its logarithm."""
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("gemm", "gemm", "write", "read", "attend", "attend"))
    yes = lambda: rng.random() < 0.5  # noqa: E731
    if op == "gemm":
        n, k = rng.choice(SHAPES) if rng.random() < 0.6 else (_spread(rng, 1, 16384), _spread(rng, 1, 4100))
        m = _spread(rng, 1, min(4000, max(1, 4000 * 4096 * 4096 // (n * k)))) if yes() else _spread(rng, 1, 32)
        return {"op": op, "m": m, "n": n, "k": k, "group": rng.choice((32, 64, 128, 256)), "scales": rng.choice(("f32", "f16")),
                "bias": yes(), "silu": yes(), "residual": yes(), "out": rng.choice(("f32", "f16", "bf16"))}
    case = {"op": op, "batch": _spread(rng, 1, 32), "mixed": yes(), "kv_heads": rng.choice((1, 2, 3, 4, 8)),
            "d": rng.choice((64, 80, 128, 128)), "page": rng.choice((16, 32, 64, 128)), "dtype": rng.choice(("f32", "f16", "bf16"))}
    case["length"] = _spread(rng, 1, 16000 if case["batch"] <= 16 else 8000)
    if op != "attend":
        most = max(1, 16000 * 8 // (case["batch"] * case["kv_heads"]))
        return {**case, "new": _spread(rng, 1, min(case["length"], most))}
    case["heads"] = case["kv_heads"] * rng.choice((1, 2, 4) if case["kv_heads"] < 8 else (1, 2))
    most = max(1, 2048 * 16000 * 16 // (case["batch"] * case["length"] * case["heads"] * (4 if case["dtype"] == "f32" else 1)))
    new = rng.choice((1, 1, 4, 0))
    return {**case, "new": min(case["length"], new or _spread(rng, 1, min(2048, most))),
            "left": rng.choice((None, None, _spread(rng, 1, 4096)))}


def spans(case: dict) -> list:
    """(new tokens, length with them) of each sequence: lengths from `length` down to a quarter of it; with "mixed", sequences of
    all new tokens, a single one, half and so on."""
    out = []
    for b in range(case["batch"]):
        length = max(1, case["length"] - 3 * case["length"] * b // (4 * case["batch"]))
        new = case["new"] if not case["mixed"] else 1 if b % 2 else case["new"] >> (b // 2 % 8)
        out.append((max(1, min(new, length)), length))
    return out


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _rows8(x):
    """Float rows as int8 with a scale each."""
    s = (x.abs().amax(-1) / 127).clamp_min(1e-30)
    return torch.round(x / s[..., None]).to(torch.int8), s


def _prepare_gemm(case, g, randn):
    m, n, k, group = case["m"], case["n"], case["k"], case["group"]
    groups = -(-k // group)
    x8, qs = _rows8(randn(m, k) * (0.5 + torch.rand(m, 1, generator=g, device="cuda")))
    q = torch.zeros(1, m, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
    q[0, :, :k] = x8
    dense = torch.zeros(n, groups * group, device="cuda")
    dense[:, :k] = randn(n, k) / math.sqrt(k)
    dense = dense.view(n, groups, group)
    scale = (dense.abs().amax(2) / 7).clamp_min(1e-7).to(DTYPES[case["scales"]])
    weight = torch.round(dense / scale.float()[:, :, None]).clamp_(-8, 7).to(torch.int8).view(n, -1)[:, :k].contiguous()
    state = {"case": case, "q": q, "qs": qs[None], "weight": weight, "scale": scale,
             "bias": 0.1 * randn(n) if case["bias"] else None, "residual": randn(m, n) if case["residual"] else None}
    if own:
        from kea_kernels import int4
        state["packed"] = int4.pack(weight, scale, group)
    return state


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "gemm":
        return _prepare_gemm(case, g, randn)
    hk, d, page, dtype, rows = case["kv_heads"], case["d"], case["page"], DTYPES[case["dtype"]], spans(case)
    # pages in no order, as a pool that sequences come to and leave gives them; entries past a sequence's end name none
    per = -(-max(n for _, n in rows) // page)
    table = torch.full((len(rows), per), -1, dtype=torch.int32, device="cuda")
    used = [-(-n // page) for _, n in rows]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    for b, n in enumerate(used):
        table[b, :n] = order[sum(used[:b]):sum(used[:b + 1])]
    total = sum(n for n, _ in rows)
    state = {"case": case, "table": table, "spans": rows,
             "lengths": torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda"), "offsets": None,
             "starts": torch.tensor([n - new for new, n in rows], dtype=torch.int32, device="cuda")}
    if len({n for n, _ in rows}) > 1:
        state["offsets"] = torch.tensor([sum(n for n, _ in rows[:b]) for b in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
    # what the pages hold: ints as keys and values of a normal distribution give them, and scales of heads and tokens of any size
    ints = lambda: (randn(pages, hk, page, d) * 40).round_().clamp_(-127, 127).to(torch.int8)  # noqa: E731
    scales = lambda: 0.025 * torch.exp(0.3 * randn(pages, hk, page))  # noqa: E731
    state["pages"] = pages4 = (ints(), ints(), scales(), scales())
    if case["op"] == "attend":
        state["q"] = randn(total, case["heads"], d).to(dtype)
    elif case["op"] == "write":
        state["k"], state["v"] = ((randn(total, hk, d) * (0.2 + randn(total, hk, 1).abs())).to(dtype) for _ in range(2))
    if own:
        from kea_kernels import paged
        state["cache"] = paged.Cache(*pages4)
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------------

def run(state: dict):
    case = state["case"]
    if own:
        return _own(case, state)
    return {"gemm": _gemm, "write": _write, "read": _read, "attend": _attend}[case["op"]](case, state)


def _own(case, s):
    if case["op"] == "gemm":
        from kea_kernels import int4
        return int4.gemm(s["q"], s["qs"], s["packed"], s["bias"], silu=case["silu"], residual=s["residual"], residual_factor=0.5,
                         out_dtype=DTYPES[case["out"]])
    from kea_kernels import paged
    if case["op"] == "attend":
        return paged.attention(s["q"], s["cache"], s["table"], s["lengths"], s["offsets"], left=case["left"])
    if case["op"] == "write":
        paged.write(s["cache"], s["k"], s["v"], s["table"], s["lengths"], s["offsets"])
    most = max(n for n, _ in s["spans"])
    return paged.read(s["cache"], s["table"], s["lengths"], most, starts=s["starts"], out_dtype=DTYPES[case["dtype"]])


def _gemm(case, s):
    (n, k), group, groups = s["weight"].shape, case["group"], s["scale"].shape[1]
    w = torch.zeros(n, groups * group, device="cuda")
    w[:, :k] = s["weight"]
    w = (w.view(n, groups, group) * s["scale"].float()[:, :, None]).view(n, -1)[:, :k]
    r = (s["q"][0, :, :k].float() @ w.t()) * s["qs"][0][:, None]
    if s["bias"] is not None:
        r = r + s["bias"]
    if case["silu"]:
        r = r * torch.sigmoid(r)
    if s["residual"] is not None:
        r = s["residual"] + 0.5 * r
    return r.to(DTYPES[case["out"]])


def _places(case, s, b, low, high):
    """Pages and rows in them of the positions low .. high - 1 of sequence b."""
    p = torch.arange(low, high, device="cuda")
    return s["table"][b].long()[p // case["page"]], p % case["page"]


def _write(case, s):
    k, v, ks, vs = s["pages"]
    where = [_places(case, s, b, n - new, n) for b, (new, n) in enumerate(s["spans"])]
    page, row = torch.cat([p for p, _ in where]), torch.cat([r for _, r in where])
    for x, ints, scales in ((s["k"], k, ks), (s["v"], v, vs)):
        x8, sx = _rows8(x.float())
        ints[page, :, row] = x8
        scales[page, :, row] = sx
    return _read(case, s)


def _read(case, s):
    most, dtype = max(n for n, _ in s["spans"]), DTYPES[case["dtype"]]
    p = s["starts"].long()[:, None] + torch.arange(most, device="cuda")                     # [B, most]
    there = p < s["lengths"][:, None]
    entry = (p // case["page"]).clamp_max(s["table"].shape[1] - 1)
    page = s["table"].long().gather(1, entry).clamp_min(0)
    k, v, ks, vs = s["pages"]
    values = lambda c, sc: torch.where(there[:, :, None, None], c[page, :, p % case["page"]].float() * sc[page, :, p % case["page"]][..., None],  # noqa: E731
                                       torch.zeros((), device="cuda")).to(dtype)
    return values(k, ks), values(v, vs)


def _attend(case, s):
    hk, d, group = case["kv_heads"], case["d"], case["heads"] // case["kv_heads"]
    k, v, ks, vs = s["pages"]
    out, at = [], 0
    for b, (new, n) in enumerate(s["spans"]):
        low = 0 if case["left"] is None else max(0, n - new - case["left"])
        page, row = _places(case, s, b, low, n)
        kb, vb = ((c[page, :, row].float() * sc[page, :, row][..., None]).transpose(0, 1).contiguous() for c, sc in ((k, ks), (v, vs)))
        q = s["q"][at:at + new].float().view(new, hk, group, d).permute(1, 2, 0, 3).reshape(hk, group * new, d)
        scores = torch.bmm(q, kb.transpose(1, 2).contiguous()).view(hk, group, new, n - low) * (1 / math.sqrt(d))
        i, j = torch.arange(n - new, n, device="cuda")[:, None], torch.arange(low, n, device="cuda")
        unseen = j > i
        if case["left"] is not None:
            unseen = unseen | (j < i - case["left"])
        scores = scores.masked_fill_(unseen, float("-inf"))
        e = torch.exp_(scores.sub_(scores.amax(-1, keepdim=True)))
        o = torch.bmm(e.view(hk, group * new, n - low), vb).view(hk, group, new, d) / e.sum(-1, keepdim=True)
        out.append(o.permute(2, 0, 1, 3).reshape(new, hk * group, d))
        at += new
    return torch.cat(out).to(s["q"].dtype)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        b = m * k + n * k / 2 + n * -(-k // case["group"]) * size[case["scales"]] + 4 * m + m * n * size[case["out"]]
        return {"bytes": b + 4 * n * case["bias"] + 4 * m * n * case["residual"], "flops": 2 * m * n * k}
    rows, hk, d, e = spans(case), case["kv_heads"], case["d"], size[case["dtype"]]
    total, most = sum(n for n, _ in rows), max(n for n, _ in rows)
    if case["op"] == "attend":
        pairs = keys = 0
        for new, n in rows:
            left = n if case["left"] is None else case["left"]
            keys += min(n, new + left)
            pairs += sum(min(p, left) + 1 for p in range(n - new, n))
        return {"bytes": 2 * total * case["heads"] * d * e + 2 * keys * hk * (d + 4), "flops": 4 * d * case["heads"] * pairs}
    stored, dense = 2 * total * hk * (d + 4), 2 * len(rows) * most * hk * d * e
    if case["op"] == "write":  # tokens in, rows of the cache out, and back as values
        return {"bytes": 2 * total * hk * d * e + 2 * stored + dense, "flops": 8 * total * hk * d}
    return {"bytes": stored + dense, "flops": 2 * total * hk * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["op"] == "gemm":
        w = s["weight"].double() * s["scale"].double().repeat_interleave(case["group"], 1)[:, :case["k"]]
        r = s["q"][0, :, :case["k"]].double().mm(w.t().contiguous()).mul_(s["qs"][0].double()[:, None])
        if case["bias"]:
            r += s["bias"].double()
        if case["silu"]:
            r /= 1 + torch.exp(-r)
        return s["residual"].double() + r / 2 if case["residual"] else r
    hk, d, page, rows = case["kv_heads"], case["d"], case["page"], s["spans"]
    k, v, ks, vs = s["pages"]

    def sequence(c, sc, b, n):  # the first n rows of sequence b, [heads, n, d]
        at = s["table"][b, :-(-n // page)].long()
        return (c[at].double() * sc[at].double()[..., None]).transpose(0, 1).reshape(hk, -1, d)[:, :n]

    if case["op"] == "attend":
        out = torch.zeros(sum(n for n, _ in rows), case["heads"], d, dtype=torch.float64, device="cuda")
        at = 0
        for b, (new, n) in enumerate(rows):
            kb, vb = sequence(k, ks, b, n), sequence(v, vs, b, n)
            for i0 in range(0, new, 512):  # a block of queries
                i = torch.arange(i0, min(i0 + 512, new), device="cuda")
                p, j = (n - new + i)[:, None], torch.arange(n, device="cuda")
                seen = j <= p if case["left"] is None else (j <= p) & (j + case["left"] >= p)
                for h in range(case["heads"]):
                    kv = h * hk // case["heads"]
                    w = s["q"][at + i, h].double().mm(kb[kv].t().contiguous()).div_(math.sqrt(d))
                    out[at + i, h] = torch.where(seen, w, -math.inf).softmax(1).mm(vb[kv])
            at += new
        return out
    most = max(n for n, _ in rows)
    result = []
    for c, sc, name in ((k, ks, "k"), (v, vs, "v")):
        dense = torch.zeros(len(rows), most, hk, d, dtype=torch.float64, device="cuda")
        at = 0
        for b, (new, n) in enumerate(rows):
            if case["op"] == "write":  # (a scale is held in FP32)
                x = s[name][at:at + new].double()
                unit = (x.abs().amax(2, keepdim=True) / 127).float().clamp_min(1e-30).double()
                dense[b, :new] = torch.round(x / unit) * unit
            else:
                dense[b, :new] = sequence(c, sc, b, n)[:, n - new:].transpose(0, 1)
            at += new
        result.append(dense)
    return tuple(result)
