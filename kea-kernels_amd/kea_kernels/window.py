"""Attention within a sliding window and to the first tokens (kea_window_attention, include/kea_block.h): limited context
over long recordings, padded batches, and a few tokens at a time against a cache. Runs on torch's current stream of the
tensors' device, never synchronizes the host, takes its workspace, if it needs one, from torch's allocator, and can be
captured into a graph.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from kea_kernels import _hip

_NO_BOUND = 1 << 30
_MOST = 1 << 30  # tokens of a sequence


def _heads(name: str, t: Tensor, b: int, heads: int | None, d: int, dtype, device) -> None:
    if t.dim() != 4 or t.dtype != dtype or t.device != device or t.shape[0] != b or t.shape[3] != d:
        raise ValueError(f"{name} must be {dtype} [{b}, T, heads, {d}] on {device}, got {t.dtype} {tuple(t.shape)} on "
                         f"{t.device}")
    unit = 16 // t.element_size()
    if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.stride(i) % unit for i in range(3) if t.shape[i] > 1):
        raise ValueError(f"{name} needs contiguous heads that start at multiples of 16 bytes, got strides {t.stride()}")
    if t.shape[1] > _MOST:
        raise ValueError(f"{name} has more than 2^30 tokens")


def _span(t: Tensor) -> tuple[int, int]:
    size = t.element_size()
    return t.data_ptr(), t.data_ptr() + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _describe(t: Tensor) -> "_hip.Heads":
    return _hip.Heads(t.data_ptr(), *(t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)))


def _bound(name: str, v) -> int:
    if v is None:
        return _NO_BOUND
    if int(v) != v or v < 0:
        raise ValueError(f"{name} must be None or a whole number >= 0, got {v!r}")
    return min(int(v), _NO_BOUND)


def _native(*args) -> Tensor | None:
    """attention() in one native call (the same checks on the tensors' fields); None, having launched nothing, where an
    argument is not what it takes: the Python path then checks again and raises or launches."""
    try:
        return _hip.native().window_attention(*args)
    except (AttributeError, TypeError, ValueError):
        return None


def attention(q: Tensor, k: Tensor, v: Tensor, *, left: int | None = None, right: int | None = 0, sinks: int = 0,
              scale: float | None = None, kv_lengths: Tensor | None = None, q_starts: Tensor | None = None,
              out: Tensor | None = None) -> Tensor:
    """out [B, Tq, H, D] = attention of q [B, Tq, H, D] to k, v [B, Tk, Hkv, D], H a multiple of Hkv (query head h reads key
    head h // (H / Hkv)), f32, f16 or bf16, D a multiple of 8 up to 256.

    Query i of sequence b stands at position p = q_starts[b] + i among that sequence's keys 0 .. len - 1, and sees key j < len
    iff j <= p + right and (j >= p - left or j < sinks): a window of `left` keys behind and `right` ahead (None: without
    bound; right = 0 is causal), and the first `sinks` keys. len is kv_lengths[b] (int32 [B] on the device, held to 0 .. Tk;
    None: Tk); q_starts int32 [B] (None: len - Tq, the queries are the last tokens). For padded clips q_starts is zeros and
    kv_lengths the clips' lengths; for tokens against a cache kv_lengths counts them too. Queries that see nothing (or
    scores of -infinity alone), or stand outside 0 .. len - 1 (padding), give zeros. What a query does not see has no part in
    its output, whatever it holds. scale: 1 / sqrt(D) unless given, any finite FP32 number. out must not overlap an input.
    Everything is FP32 up to the output's rounding, but for the softmax's weights of f16 and bf16 inputs, which are rounded to
    their type; the same values as f32 keep them whole."""
    if out is None and (hit := _native(q, k, v, left, right, sinks, scale, kv_lengths, q_starts)) is not None:
        return hit
    if q.dim() != 4 or k.dim() != 4 or q.dtype not in _hip.DTYPES:
        raise ValueError(f"q must be f32, f16 or bf16 [B, Tq, H, D] and k, v [B, Tk, Hkv, D], got {q.dtype} "
                         f"{tuple(q.shape)}, {tuple(k.shape)}")
    (b, tq, h, d), (tk, hk), device = q.shape, k.shape[1:3], q.device
    if d < 8 or d % 8 or d > 256:
        raise ValueError(f"head size {d}: a multiple of 8 from 8 to 256")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"{h} query heads are no multiple of {hk} key heads")
    for name, t in (("q", q), ("k", k), ("v", v)):
        _heads(name, t, b, None, d, q.dtype, device)
    if v.shape != k.shape:
        raise ValueError(f"k is {tuple(k.shape)}, v {tuple(v.shape)}")
    scale = 1 / math.sqrt(d) if scale is None else ctypes.c_float(scale).value
    if not math.isfinite(scale):
        raise ValueError("scale is not a finite FP32 number")
    left, right, sinks = _bound("left", left), _bound("right", right), _bound("sinks", 0 if sinks is None else sinks)
    for name, t in (("kv_lengths", kv_lengths), ("q_starts", q_starts)):
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (b,) or not t.is_contiguous() or t.device != device):
            raise ValueError(f"{name} must be a contiguous int32 tensor [{b}] on {device}")
    if out is not None:
        _heads("out", out, b, h, d, q.dtype, device)
        if out.shape != q.shape:
            raise ValueError(f"out is {tuple(out.shape)}, q {tuple(q.shape)}")
        steps = sorted((out.stride(i), out.shape[i]) for i in range(4) if out.shape[i] > 1)
        if any(s < reach for (s, _), reach in zip(steps[1:], (a * n for a, n in steps))) or any(s < 1 for s, _ in steps):
            raise ValueError(f"out has elements that share memory: strides {out.stride()}")
        others = [t for t in (q, k, v, kv_lengths, q_starts) if t is not None and t.numel()]
        if out.numel() and any(_span(out)[0] < _span(t)[1] and _span(t)[0] < _span(out)[1] for t in others):
            raise ValueError("out overlaps q, k or v, or the lengths or starts")
    _hip.refuse_grad("window.attention", q, k, v, out)
    if out is None:
        out = torch.empty(b, tq, h, d, dtype=q.dtype, device=device)
    if not out.numel():
        return out
    L, code = _hip.lib(), _hip.dtype_code(q.dtype)
    with _hip.on_device(device):
        need = L.kea_window_attention_workspace(code, b, tq, tk, h, hk, d, left, right, sinks)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        rc = L.kea_window_attention(_describe(q), _describe(k), _describe(v), _describe(out), code, b, tq, tk, h, hk, d,
                                    left, right, sinks, scale,
                                    _hip.ptr(kv_lengths), _hip.ptr(q_starts), _hip.ptr(ws), max(need, 0),
                                    _hip.stream_handle(device))
    _hip.check(rc, "kea_window_attention")
    return out
