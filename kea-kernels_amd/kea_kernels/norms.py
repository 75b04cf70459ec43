"""The norms behind one block and before the next, with the block's gate and residual scale, in one pass over the rows
(kea_block_norm, include/kea_block.h). Runs on torch's current stream of the tensors' device, never synchronizes the host and
can be captured into a graph.
"""
from __future__ import annotations

import torch
from torch import Tensor

from kea_kernels import _hip, lowbit

_NO_NORM = _hip.Norm(0, 0, None, None, 0.0)
_ACTS = {"": 0, "sigmoid": 1, "tanh": 2}


def _norm(name: str, norm, d: int, device) -> tuple:
    """(the C description, the parameters, to keep until the launch) of a norm: a LayerNorm has a `bias` (which may be None), an
    RMSNorm has none; `weight` may be None, `eps` None stands for FP32's epsilon as in torch.nn.RMSNorm."""
    if norm is None:
        return _NO_NORM, ()
    kind = 1 if hasattr(norm, "bias") else 2
    shape = getattr(norm, "normalized_shape", (d,))
    if tuple(shape) != (d,):
        raise ValueError(f"{name} normalizes {tuple(shape)}, the rows have {d} elements")
    w, b = norm.weight, getattr(norm, "bias", None)
    for what, t in (("weight", w), ("bias", b)):
        if t is not None and (t.numel() != d or t.device != device or not t.is_contiguous() or t.dtype not in _hip.DTYPES):
            raise ValueError(f"{name}.{what} must be a contiguous f32, f16 or bf16 tensor of {d} elements on {device}")
    if w is not None and b is not None and w.dtype != b.dtype:
        raise ValueError(f"{name}: weight is {w.dtype}, bias {b.dtype}")
    some = w if w is not None else b
    eps = torch.finfo(torch.float32).eps if norm.eps is None else float(norm.eps)
    return _hip.Norm(kind, 0 if some is None else _hip.dtype_code(some.dtype), _hip.ptr(w), _hip.ptr(b), eps), (w, b)


def _rows(name: str, t: Tensor) -> Tensor:
    """[..., d] as rows [M, d] without a copy."""
    if t.dim() < 1 or t.shape[-1] < 1 or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must have rows of contiguous elements, got {tuple(t.shape)} strides {t.stride()}")
    try:
        return t.view(-1, t.shape[-1]) if t.numel() else t.new_empty(0, t.shape[-1])
    except RuntimeError:
        raise ValueError(f"{name}: the leading dimensions do not form rows of one stride, {tuple(t.shape)} strides "
                         f"{t.stride()}") from None


def _stride(t: Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


_NO_PARAMETERS = (0, None, None, 0.0)


def _parameters(norm, d: int) -> tuple:
    """(kind, weight, bias, eps) of a torch.nn norm of d elements whose parameters are its own (LookupError otherwise)."""
    if norm is None:
        return _NO_PARAMETERS
    fields = norm.__dict__
    own = fields["_parameters"]
    if tuple(norm.normalized_shape) != (d,):
        raise LookupError
    kind = 1 if "bias" in own else 2
    # (a bias kept elsewhere makes a LayerNorm too; hasattr on a plain RMSNorm would cost a microsecond)
    if kind == 2 and ("bias" in fields or "bias" in fields["_buffers"] if type(norm) is torch.nn.RMSNorm else hasattr(norm, "bias")):
        raise LookupError
    eps = norm.eps
    return kind, own["weight"], own.get("bias"), torch.finfo(torch.float32).eps if eps is None else eps


def _native(x, block, post, gate, act, factor, pre, quantize, out) -> tuple | None:
    """block_norm() in one native call (the same checks on the tensors' fields); None, having launched nothing, where an
    argument is not what it takes: the Python path then checks again and raises or launches."""
    try:
        d = x.shape[-1]
        return _hip.native().block_norm(x, block, *_parameters(post, d), gate, _ACTS[act], factor, *_parameters(pre, d),
                                        bool(quantize), out)
    except (AttributeError, LookupError, TypeError, ValueError):
        return None


def block_norm(x: Tensor, block: Tensor | None, *, post=None, gate: Tensor | None = None, gate_activation: str = "",
               factor: float = 1.0, pre=None, quantize: bool = False, out: Tensor | None = None) -> tuple:
    """y = x + factor * act(gate) * post(block) and z = pre(y): (y, z), (y, None) without `pre`, and with `quantize`
    (y, q, qs), q int8 [1, M, round_up(d, 16)] and qs FP32 [1, M] the int8 rows of z (of y without `pre`) as
    lowbit.quantize makes one part of them.

    x [..., d] is the residual stream, block [..., d] the output of the block in the same shape, each f32, f16 or bf16; y
    has x's type (`out` receives it if given; it may be x or the block itself), z the block's. post and pre: modules with
    weight, bias and eps (torch.nn.LayerNorm) or weight and eps (torch.nn.RMSNorm); there is no backward, so like the tensors
    their parameters must not require grad while autograd records. gate: [G, d] in the block's type, any
    leading dimensions of G elements, M a multiple of G: M / G rows in turn share a gate row (G = 1 a gate for each channel,
    G = the batch one for each sequence, G = M one for each token), passed through gate_activation ("", "sigmoid", "tanh").
    Everything is FP32 up to one rounding of each output: z is the norm of y before y's rounding. block None (then without
    gate, post and factor): y is x itself and z = pre(x) in x's type."""
    if gate_activation not in _ACTS:
        raise ValueError(f"unsupported gate activation {gate_activation!r}")
    if block is not None and (hit := _native(x, block, post, gate, gate_activation, factor, pre, quantize, out)) is not None:
        return hit
    xr, device, d = _rows("x", x), x.device, x.shape[-1] if x.dim() else 0
    m = xr.shape[0]
    if d > 32768:
        raise ValueError(f"rows of {d} elements, at most 32768")
    for name, t in (("x", x), ("block", block), ("gate", gate), ("out", out)):
        if t is not None and (t.dtype not in _hip.DTYPES or t.device != device):
            raise ValueError(f"{name} must be f32, f16 or bf16 on {device}, got {t.dtype} on {t.device}")
    gr = br = yr = None
    if block is None:
        if gate is not None or post is not None or out is not None or (pre is None and not quantize):
            raise ValueError("without a block there is only the norm of x")
    else:
        if block.shape != x.shape:
            raise ValueError(f"block is {tuple(block.shape)}, x {tuple(x.shape)}")
        br = _rows("block", block)
        if out is not None:
            if out.shape != x.shape or out.dtype != x.dtype:
                raise ValueError("out must have x's shape and type")
            yr = _rows("out", out)
            if m > 1 and yr.stride(0) < d:
                raise ValueError("the rows of out overlap")
            others = [t for t in (xr, br) if t.dtype != yr.dtype or t.data_ptr() != yr.data_ptr() or (
                m > 1 and t.stride(0) != yr.stride(0))] + ([] if gate is None else [_rows("gate", gate)])
            if any(_hip.rows_meet(yr, t) for t in others):
                raise ValueError("out shares memory with another operand (it may be x or the block itself)")
    if gate is not None:
        gr = _rows("gate", gate)
        if gr.shape[1] != d or gr.shape[0] < 1 and m or (m and m % gr.shape[0]) or gate.dtype != block.dtype:
            raise ValueError(f"gate must be [G, {d}] in the block's type with {m} rows a multiple of G, got {gate.dtype} "
                             f"{tuple(gate.shape)}")
    elif gate_activation:
        gate_activation = ""
    _hip.refuse_grad("block_norm", x, block, gate, out)
    pn, keep0 = _norm("post", post, d, device)
    nn, keep1 = _norm("pre", pre, d, device)
    if yr is not None and any(_hip.rows_meet(yr, t.view(1, d)) for t in (*keep0, *keep1) if t is not None):
        raise ValueError("out shares memory with a norm's parameters")
    stream = _hip.stream_handle(device) if m else 0
    _hip.refuse_grad("block_norm", *keep0, *keep1)
    y = x if block is None else torch.empty(x.shape, dtype=x.dtype, device=device) if out is None else out
    if block is not None and yr is None:
        yr = y.view(-1, d) if y.numel() else y.new_empty(0, d)
    zt = x if block is None else block
    z = torch.empty(x.shape, dtype=zt.dtype, device=device) if pre is not None and not quantize else None
    q = qs = None
    ldq = lowbit.round_up(d, 16)
    if quantize:
        q = torch.empty(1, m, ldq, dtype=torch.int8, device=device)
        qs = torch.empty(1, m, dtype=torch.float32, device=device)
    if m:
        with _hip.on_device(device):
            rc = _hip.lib().kea_block_norm(
                xr.data_ptr(), _hip.dtype_code(x.dtype), _stride(xr), _hip.ptr(br), _hip.dtype_code(zt.dtype),
                _stride(br) if br is not None else 0, m, d, pn, _hip.ptr(gr), _stride(gr) if gr is not None else 0,
                m // gr.shape[0] if gr is not None else 1, _ACTS[gate_activation], float(factor),
                _hip.ptr(yr), _stride(yr) if yr is not None else 0, nn, _hip.ptr(z), d, _hip.ptr(q), ldq, _hip.ptr(qs),
                stream)
        _hip.check(rc, "kea_block_norm")
    del keep0, keep1
    return (y, q, qs) if quantize else (y, z)
