"""The int8 x int8 matrix product with a scale for each token and channel (kea_int8_gemm, include/kea_block.h).

For the layers of a model that do not stand 1- or 2-bit weights (the first and last ones, a decoder's): `gemm` multiplies the
int8 rows that lowbit.quantize or norms.block_norm make (one part) with int8 weights [N, K] as they are stored, and applies
the epilogue of lowbit.gemm: scales, bias, SiLU, residual. `Int8Linear` holds such a weight and takes float rows. Calls run
on torch's current stream of the tensors' device, never synchronize the host and can be captured into a graph.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from kea_kernels import _hip, lowbit

_SCALES = (torch.float32, torch.float16)
_OUT = {torch.float32: _hip.F32, torch.float16: _hip.F16, torch.bfloat16: _hip.BF16, torch.int32: 3}
MAX_K = 131071  # sums of k products of two int8 values fit int32
MAX_FEATURES = 8192  # of a row that lowbit.quantize takes


def _vector(name: str, t: Tensor, n: int, device) -> None:
    if not isinstance(t, Tensor) or t.dtype not in _SCALES or t.device != device or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous f32 or f16 tensor of {n} elements on {device}")


def _matrix(name: str, t: Tensor) -> Tensor:
    if t.dtype != torch.int8 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be int8 rows [.., K] with unit column stride, got {t.dtype} {tuple(t.shape)}")
    if t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) % 16) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        raise ValueError(f"{name} rows must start at multiples of 16 bytes (pad_rows gives such a copy)")
    return t


def pad_rows(weight: Tensor) -> Tensor:
    """int8 [N, K] -> the same values as a view [N, K] of rows padded with zeros to a multiple of 16 bytes, as gemm reads
    them (the tensor itself where its rows are such already)."""
    if weight.dtype != torch.int8 or weight.dim() != 2:
        raise ValueError(f"expected int8 [N, K], got {weight.dtype} {tuple(weight.shape)}")
    n, k = weight.shape
    if weight.data_ptr() % 16 == 0 and (k <= 1 or weight.stride(1) == 1) and (n <= 1 or (
            weight.stride(0) % 16 == 0 and weight.stride(0) >= lowbit.round_up(k, 16))):
        end = weight.storage_offset() + (n - 1) * (weight.stride(0) if n > 1 else 0) + lowbit.round_up(k, 16)
        if end <= weight.untyped_storage().nbytes():  # (the last row is read to a multiple of 16 bytes)
            return weight
    rows = torch.zeros(n, lowbit.round_up(k, 16), dtype=torch.int8, device=weight.device)
    rows[:, :k] = weight
    return rows[:, :k]


def _native_gemm(*args) -> Tensor | None:
    """gemm() in one native call (the same checks on the tensors' fields); None, having launched nothing, where an argument is
    not what it takes: the Python path then checks again and raises or launches."""
    try:
        return _hip.native().int8_gemm(*args)
    except (AttributeError, TypeError, ValueError):
        return None


def gemm(q: Tensor, qs: Tensor | None, weight: Tensor, wscale: Tensor | None, bias: Tensor | None = None, *,
         out: Tensor | None = None, out_dtype: torch.dtype = torch.float32, silu: bool = False,
         residual: Tensor | None = None, residual_factor: float = 1.0) -> Tensor:
    """[M, N]: residual + residual_factor * act(qs[m] * wscale[n] * sum_k q[m][k] * weight[n][k] + bias[n]), the sum exact.

    q int8 [1, M, ldq] or [M, ldq], ldq >= K (what lowbit.quantize returns for one part); qs f32 / f16, M elements; weight
    int8 [N, K], rows on multiples of 16 bytes (see pad_rows; bytes of q and weight rows past K may hold anything); wscale
    and bias f32 / f16 [N]; residual FP32 [M, N]. silu: act(r) = r * sigmoid(r), the identity otherwise. out (or a new
    tensor of out_dtype: f32, f16, bf16) receives the result, `out` may be the residual itself. out_dtype torch.int32 (or
    an int32 out) gives the sums alone: qs and wscale may then be None, and there is no bias, activation or residual."""
    if (hit := _native_gemm(q, qs, weight, wscale, bias, out, out_dtype, silu, residual, residual_factor)) is not None:
        return hit
    if q.dim() == 3:
        if q.shape[0] != 1:
            raise ValueError(f"q must hold one activation part, got {q.shape[0]}")
        q = q[0]
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_K or weight.shape[0] < 1:
        raise ValueError(f"weight must be int8 [N, K] with N >= 1 and 1 <= K <= {MAX_K}, got {tuple(weight.shape)}")
    _matrix("q", q)
    _matrix("weight", weight)
    (m, ldq), (n, k), device = q.shape, weight.shape, q.device
    if ldq < k:
        raise ValueError(f"q has rows of {ldq} elements, the weight of {k}")
    for name, t in (("q", q), ("weight", weight)):  # the last row is read to a multiple of 16 bytes
        if t.shape[0] and t.storage_offset() + (t.shape[0] - 1) * t.stride(0) + lowbit.round_up(k, 16) > \
                t.untyped_storage().nbytes():
            raise ValueError(f"{name}: the last row ends inside 16 bytes (pad_rows gives a padded copy)")
    out_dtype = out_dtype if out is None else out.dtype
    if out_dtype not in _OUT:
        raise ValueError(f"unsupported output dtype {out_dtype}")
    if out_dtype == torch.int32:
        if bias is not None or silu or residual is not None:
            raise ValueError("int32 sums take no bias, activation or residual")
        qs = wscale = None
    else:
        _vector("qs", qs, m, device)
        _vector("wscale", wscale, n, device)
    if bias is not None:
        _vector("bias", bias, n, device)
    if residual is not None and (residual.dtype != torch.float32 or tuple(residual.shape) != (m, n)
                                 or (n > 1 and residual.stride(1) != 1) or residual.device != device):
        raise ValueError(f"residual must be FP32 [{m}, {n}] with unit column stride on {device}")
    if out is not None and (tuple(out.shape) != (m, n) or (n > 1 and out.stride(1) != 1) or out.device != device
                            or (m > 1 and out.stride(0) < n)):
        raise ValueError(f"out must be [{m}, {n}] rows with unit column stride on {device}")
    if out is not None:
        same = residual is not None and out.dtype == residual.dtype and out.data_ptr() == residual.data_ptr() and (
            m < 2 or out.stride(0) == residual.stride(0))
        others = [q, weight, *(t.view(1, -1) for t in (qs, wscale, bias) if t is not None)]
        if any(_hip.rows_meet(out, t) for t in (others if same or residual is None else [*others, residual])):
            raise ValueError("out shares memory with another operand (it may be the residual itself)")
    if weight.device != device:
        raise ValueError(f"tensor on {weight.device}, expected {device}")
    _hip.refuse_grad("the int8 GEMM", qs, wscale, bias, residual, out)
    if out is None:
        out = torch.empty(m, n, device=device, dtype=out_dtype)
    if m == 0:
        return out
    L = _hip.lib()
    with _hip.on_device(device):
        code = lambda t: 0 if t is None else _hip.dtype_code(t.dtype)  # noqa: E731
        rc = L.kea_int8_gemm(q.data_ptr(), lowbit.round_up(ldq, 16) if m == 1 else q.stride(0),
                             _hip.ptr(qs), code(qs), weight.data_ptr(),
                             lowbit.round_up(k, 16) if n == 1 else weight.stride(0), _hip.ptr(wscale), code(wscale),
                             _hip.ptr(bias), code(bias), out.data_ptr(), _OUT[out_dtype], n if m == 1 else out.stride(0),
                             _hip.ptr(residual), (n if m == 1 else residual.stride(0)) if residual is not None else 0,
                             float(residual_factor), m, n, k, int(silu), _hip.stream_handle(device))
    _hip.check(rc, "kea_int8_gemm")
    return out


class Int8Linear:
    """One layer with int8 weights: rows [N, K] padded to 16 bytes, FP32 scales and bias, resident on the GPU. A call makes
    one int8 part of its input's rows (lowbit.quantize, with the LayerNorm and SiLU that it fuses) and runs gemm."""

    def __init__(self, weight: Tensor, scale: Tensor, bias: Tensor | None):
        self.weight, self.scale, self.bias = weight, scale, bias
        self.out_features, self.in_features = weight.shape
        self.device = weight.device

    @classmethod
    def prepare(cls, weight: Tensor, scale: Tensor, bias: Tensor | None, device) -> "Int8Linear":
        """int8 weight [N, K], K <= 8192, a scale for each row and an optional bias [N]; makes the only GPU copies."""
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("Int8Linear runs on GPU devices only")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if weight.dtype != torch.int8 or weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_FEATURES or weight.shape[0] < 1:
            raise ValueError(f"weight must be int8 [N, K], K <= {MAX_FEATURES}, got {weight.dtype} {tuple(weight.shape)}")
        for name, t in (("scale", scale), ("bias", bias)):
            if t is not None and (t.numel() != weight.shape[0] or not torch.isfinite(t.float()).all()):
                raise ValueError(f"{name} must be {weight.shape[0]} finite values")
        with torch.no_grad():
            n, k = weight.shape
            rows = torch.zeros(n, lowbit.round_up(k, 16), dtype=torch.int8, device=device)
            rows[:, :k] = weight  # (never the caller's memory)
            return cls(rows[:, :k], scale.to(device=device, dtype=torch.float32, copy=True).contiguous().view(-1),
                       None if bias is None else bias.to(device=device, dtype=torch.float32, copy=True).contiguous().view(-1))

    @classmethod
    def from_dense(cls, weight: Tensor, bias: Tensor | None = None, device="cuda") -> "Int8Linear":
        """A float weight [N, K] rounded to int8 with a scale for each row: max|w| / 127, ties to even."""
        if weight.dim() != 2 or not weight.is_floating_point() or not torch.isfinite(weight).all():
            raise ValueError("weight must be a finite float matrix [N, K]")
        w = weight.detach().float()
        scale = (w.abs().amax(1) / 127).clamp_min(1e-30)
        return cls.prepare(torch.round(w / scale[:, None]).clamp_(-127, 127).to(torch.int8), scale, bias, device)

    def weight_bytes(self) -> int:
        return self.out_features * lowbit.round_up(self.in_features, 16) + self.scale.numel() * 4 + (
            0 if self.bias is None else self.bias.numel() * 4)

    def linear(self, x: Tensor, *, activation: str = "", norm=None, input_activation: str = "",
               out_dtype: torch.dtype = torch.float32) -> Tensor:
        """[..., K] -> [..., N] (FP32 unless out_dtype says otherwise); x f32 or f16."""
        if activation not in ("", "silu"):
            raise ValueError(f"unsupported activation {activation!r}")
        if x.device != self.device:
            raise ValueError(f"input on {x.device}, layer on {self.device}")
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"expected [..., {self.in_features}] input, got {tuple(x.shape)}")
        _hip.refuse_grad("Int8Linear", x, getattr(norm, "weight", None), getattr(norm, "bias", None))
        lead, m = x.shape[:-1], math.prod(x.shape[:-1])
        if m == 0:
            return torch.empty(*lead, self.out_features, device=self.device, dtype=out_dtype)
        xr = x.reshape(-1, x.shape[-2], x.shape[-1]) if x.dim() > 2 else x.view(1, 1, -1) if x.dim() == 1 else x[None]
        with _hip.on_device(x.device):
            q, qs, _ = lowbit.quantize(xr, (xr.stride(0), xr.stride(1), xr.stride(2), max(xr.shape[1], 1)), m,
                                       self.in_features, 1, norm=norm, input_activation=input_activation)
        return gemm(q, qs, self.weight, self.scale, self.bias, out_dtype=out_dtype, silu=activation == "silu").view(
            *lead, self.out_features)
