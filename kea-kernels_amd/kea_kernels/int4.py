"""The int8 x int4 matrix product with a scale for each token and each group of a row's weights (kea_int4_gemm,
include/kea_decode.h).

Between the 1- and 2-bit layers and those of int8.gemm: `pack` lays 4-bit weights [N, K] out for the matrix cores, `gemm`
multiplies the int8 rows that lowbit.quantize or norms.block_norm make (one part) with them, with int8.gemm's epilogue: scales,
bias, SiLU, residual. `Int4Linear` holds such a weight and takes float rows. Calls run on torch's current stream of the tensors'
device, never synchronize the host and can be captured into a graph.
"""
from __future__ import annotations

import math

import torch
from torch import Tensor

from kea_kernels import _hip, lowbit
from kea_kernels.int8 import MAX_FEATURES, _matrix, _vector

_SCALES = (torch.float32, torch.float16)
MAX_K = 1 << 20
MOST_SCALE = 2.0**100


class Weight:
    """4-bit weights [out_features, in_features] as kea_int4_gemm reads them: int32 `words` and `scales` [tiles of 16 rows][groups]
    [16] (f32 or f16), with a scale for each `group` weights of a row. Made by pack."""

    def __init__(self, words: Tensor, scales: Tensor, out_features: int, in_features: int, group: int):
        self.words, self.scales = words, scales
        self.out_features, self.in_features, self.group = out_features, in_features, group

    @property
    def device(self) -> torch.device:
        return self.words.device

    def to(self, device) -> "Weight":
        return Weight(self.words.to(device), self.scales.to(device), self.out_features, self.in_features, self.group)

    def dense(self) -> Tensor:
        """The weights' values in FP32, [N, K]."""
        n, k, tiles = self.out_features, self.in_features, self.scales.shape[0]
        b = self.words.view(torch.uint8).view(tiles, -1, 4, 16, 2, 2, 4)  # [tile, block, j, i, h, u, b]
        v = torch.stack((b & 15, b >> 4), 6).to(torch.int8)               # [tile, block, j, i, h, u, nibble, b]
        v = torch.where(v > 7, v - 16, v).permute(0, 3, 1, 4, 2, 5, 6, 7).reshape(16 * tiles, -1)[:n, :k]
        s = self.scales.float().transpose(1, 2).reshape(16 * tiles, -1)[:n]
        return v.float() * s.repeat_interleave(min(self.group, k), 1)[:, :k]  # (a longer group is all of a row)

    def nbytes(self) -> int:
        return self.words.numel() * 4 + self.scales.numel() * self.scales.element_size()


def _groups(k: int, group: int) -> int:
    if not isinstance(group, int) or group < 32 or group & (group - 1) or group > 1 << 30:
        raise ValueError(f"group must be a power of two of 32 or more, got {group!r}")
    return -(-k // group)


def pack(weight: Tensor, scale: Tensor, group: int) -> Weight:
    """int8 weight [N, K] of values from -8 to 7 and their scales [N, ceil(K / group)] (f32 or f16, finite, up to 2^100 in size, from K =
    8192 on up to 2^113 / K: no sum passes FP32's range), on the tensors' device. Copies; reads the values back once to check them."""
    if weight.dtype != torch.int8 or weight.dim() != 2 or not 1 <= weight.shape[1] <= MAX_K or weight.shape[0] < 1:
        raise ValueError(f"weight must be int8 [N, K], 1 <= K <= {MAX_K}, got {weight.dtype} {tuple(weight.shape)}")
    n, k = weight.shape
    groups = _groups(k, group)
    if scale.dtype not in _SCALES or tuple(scale.shape) != (n, groups) or scale.device != weight.device:
        raise ValueError(f"scale must be f32 or f16 [{n}, {groups}] on {weight.device}, got {scale.dtype} {tuple(scale.shape)} on "
                         f"{scale.device}")
    with torch.no_grad():
        weight, scale = weight.detach(), scale.detach()
        if int(weight.min()) < -8 or int(weight.max()) > 7:
            raise ValueError("weight has values outside -8 .. 7")
        # (the kernel holds 16 times a sum of up to 128 * 8 k products and scales)
        most = min(MOST_SCALE, 2.0**113 / k)
        if not bool((scale.double().abs() <= most).all()):
            raise ValueError(f"scale must be finite values of at most {most:.6g}")
        tiles, blocks = -(-n // 16), -(-k // 128)
        full = torch.zeros(16 * tiles, 128 * blocks, dtype=torch.int8, device=weight.device)
        full[:n, :k] = weight
        # [tile, i, block, h, j, u, nibble, b] -> [tile, block, j, i, h, u, nibble, b]
        full = full.view(tiles, 16, blocks, 2, 4, 2, 2, 4).permute(0, 2, 4, 1, 3, 5, 6, 7).contiguous().view(torch.uint8)
        words = ((full[..., 0, :] & 15) | (full[..., 1, :] << 4)).contiguous().view(torch.int32).view(-1)
        rows = torch.zeros(16 * tiles, groups, dtype=scale.dtype, device=scale.device)
        rows[:n] = scale
        return Weight(words, rows.view(tiles, 16, groups).transpose(1, 2).contiguous(), n, k, group)


def _check_weight(w: Weight) -> None:
    n, k, groups = w.out_features, w.in_features, _groups(w.in_features, w.group)
    tiles, blocks = -(-n // 16), -(-k // 128)
    if n < 1 or not 1 <= k <= MAX_K:
        raise ValueError(f"weight [{n}, {k}]: N >= 1 and 1 <= K <= {MAX_K}")
    if w.words.dtype != torch.int32 or w.words.numel() != tiles * blocks * 256 or not w.words.is_contiguous() or w.words.data_ptr() % 16:
        raise ValueError(f"weight.words must be {tiles * blocks * 256} int32 values aligned to 16 bytes (pack makes them)")
    if w.scales.dtype not in _SCALES or tuple(w.scales.shape) != (tiles, groups, 16) or not w.scales.is_contiguous() \
            or w.scales.data_ptr() % 16 or w.scales.device != w.words.device:
        raise ValueError(f"weight.scales must be f32 or f16 [{tiles}, {groups}, 16] aligned to 16 bytes (pack makes them)")


def _native_gemm(*args) -> Tensor | None:
    """gemm() in one native call (the same checks on the tensors' fields); None, having launched nothing, where an argument is
    not what it takes: the Python path then checks again and raises or launches."""
    try:
        return _hip.native().int4_gemm(*args)
    except (AttributeError, TypeError, ValueError):
        return None


def gemm(q: Tensor, qs: Tensor, weight: Weight, bias: Tensor | None = None, *, out: Tensor | None = None,
         out_dtype: torch.dtype = torch.float32, silu: bool = False, residual: Tensor | None = None,
         residual_factor: float = 1.0) -> Tensor:
    """[M, N]: residual + residual_factor * act(qs[m] * sum_g scale[n][g] * sum_{k in g} q[m][k] * weight[n][k] + bias[n]), a group's
    sum exact, the rest in FP32 with one rounding at the end.

    q int8 [1, M, ldq] or [M, ldq], ldq >= K, rows on multiples of 16 bytes (what lowbit.quantize returns for one part; bytes past
    K may hold anything); qs f32 / f16, M elements; bias f32 / f16 [N]; residual FP32 [M, N]. silu: act(r) = r * sigmoid(r), the
    identity otherwise. out (or a new tensor of out_dtype: f32, f16, bf16) receives the result, `out` may be the residual itself."""
    if (hit := _native_gemm(q, qs, weight.words, weight.scales, weight.out_features, weight.in_features, weight.group, bias, out,
                            out_dtype, silu, residual, residual_factor)) is not None:
        return hit
    if q.dim() == 3:
        if q.shape[0] != 1:
            raise ValueError(f"q must hold one activation part, got {q.shape[0]}")
        q = q[0]
    _check_weight(weight)
    _matrix("q", q)
    (m, ldq), n, k, device = q.shape, weight.out_features, weight.in_features, q.device
    if ldq < k:
        raise ValueError(f"q has rows of {ldq} elements, the weight of {k}")
    if m and q.storage_offset() + (m - 1) * q.stride(0) + lowbit.round_up(k, 16) > q.untyped_storage().nbytes():
        raise ValueError("q: the last row ends inside 16 bytes (int8.pad_rows gives a padded copy)")
    out_dtype = out_dtype if out is None else out.dtype
    if out_dtype not in _hip.DTYPES:
        raise ValueError(f"unsupported output dtype {out_dtype}")
    if weight.device != device:
        raise ValueError(f"weight on {weight.device}, expected {device}")
    _vector("qs", qs, m, device)
    if bias is not None:
        _vector("bias", bias, n, device)
    if residual is not None and (residual.dtype != torch.float32 or tuple(residual.shape) != (m, n)
                                 or (n > 1 and residual.stride(1) != 1) or residual.device != device):
        raise ValueError(f"residual must be FP32 [{m}, {n}] with unit column stride on {device}")
    if out is not None:
        if tuple(out.shape) != (m, n) or (n > 1 and out.stride(1) != 1) or out.device != device or (m > 1 and out.stride(0) < n):
            raise ValueError(f"out must be [{m}, {n}] rows with unit column stride on {device}")
        same = residual is not None and out.dtype == residual.dtype and out.data_ptr() == residual.data_ptr() and (
            m < 2 or out.stride(0) == residual.stride(0))
        others = [q, *(t.view(1, -1) for t in (qs, weight.words, weight.scales, bias) if t is not None)]
        if any(_hip.rows_meet(out, t) for t in (others if same or residual is None else [*others, residual])):
            raise ValueError("out shares memory with another operand (it may be the residual itself)")
    _hip.refuse_grad("the int4 GEMM", qs, weight.scales, bias, residual, out)
    if out is None:
        out = torch.empty(m, n, device=device, dtype=out_dtype)
    if m == 0:
        return out
    L = _hip.lib()
    with _hip.on_device(device):
        code = lambda t: 0 if t is None else _hip.dtype_code(t.dtype)  # noqa: E731
        rc = L.kea_int4_gemm(q.data_ptr(), lowbit.round_up(ldq, 16) if m == 1 else q.stride(0), qs.data_ptr(), code(qs),
                             weight.words.data_ptr(), weight.scales.data_ptr(), code(weight.scales), weight.group,
                             _hip.ptr(bias), code(bias), out.data_ptr(), code(out), n if m == 1 else out.stride(0),
                             _hip.ptr(residual), (n if m == 1 else residual.stride(0)) if residual is not None else 0,
                             float(residual_factor), m, n, k, int(silu), _hip.stream_handle(device))
    _hip.check(rc, "kea_int4_gemm")
    return out


class Int4Linear:
    """One layer with 4-bit weights and a scale for each group of a row's weights, resident on the GPU, with an FP32 bias. A call
    makes one int8 part of its input's rows (lowbit.quantize, with the LayerNorm and SiLU that it fuses) and runs gemm. Rows are f32 or
    f16 and up to 8192 wide, as lowbit.quantize takes them; norms.block_norm makes int8 rows of bf16 and wider ones, which gemm takes."""

    def __init__(self, weight: Weight, bias: Tensor | None):
        self.weight, self.bias = weight, bias
        self.out_features, self.in_features = weight.out_features, weight.in_features
        self.device = weight.device

    @classmethod
    def prepare(cls, weight: Tensor, scale: Tensor, bias: Tensor | None, group: int, device) -> "Int4Linear":
        """int8 weight [N, K] of values from -8 to 7, K <= 8192, scales [N, ceil(K / group)] and an optional bias [N]; makes the
        only GPU copies."""
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("Int4Linear runs on GPU devices only")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if weight.dim() != 2 or weight.shape[1] > MAX_FEATURES:
            raise ValueError(f"weight must be [N, K], K <= {MAX_FEATURES}, got {tuple(weight.shape)}")
        if bias is not None and (bias.numel() != weight.shape[0] or not torch.isfinite(bias.float()).all()):
            raise ValueError(f"bias must be {weight.shape[0]} finite values")
        scale = scale.detach() if scale.dtype in _SCALES else scale.detach().float()
        with torch.no_grad():
            return cls(pack(weight.detach(), scale.to(weight.device), group).to(device),
                       None if bias is None else bias.detach().to(device=device, dtype=torch.float32, copy=True).contiguous().view(-1))

    @classmethod
    def from_dense(cls, weight: Tensor, bias: Tensor | None = None, group: int = 128, device="cuda") -> "Int4Linear":
        """A float weight [N, K] rounded to 4 bits with an FP32 scale for each group of a row: max|w| / 7, ties to even."""
        if weight.dim() != 2 or not weight.is_floating_point() or not torch.isfinite(weight).all() or not weight.numel():
            raise ValueError("weight must be a finite float matrix [N, K]")
        with torch.no_grad():
            n, k = weight.shape
            groups = _groups(k, group)
            span = min(group, k)  # (a longer group is all of a row)
            w = torch.zeros(n, groups * span, device=weight.device)
            w[:, :k] = weight.detach()
            w = w.view(n, groups, span)
            scale = (w.abs().amax(2) / 7).clamp_min(1e-30)
            q = torch.round(w / scale[:, :, None]).clamp_(-7, 7).to(torch.int8).view(n, -1)[:, :k]
        return cls.prepare(q, scale, bias, group, device)

    def weight_bytes(self) -> int:
        return self.weight.nbytes() + (0 if self.bias is None else self.bias.numel() * 4)

    def linear(self, x: Tensor, *, activation: str = "", norm=None, input_activation: str = "",
               out_dtype: torch.dtype = torch.float32) -> Tensor:
        """[..., K] -> [..., N] (FP32 unless out_dtype says otherwise); x f32 or f16."""
        if activation not in ("", "silu"):
            raise ValueError(f"unsupported activation {activation!r}")
        if x.device != self.device:
            raise ValueError(f"input on {x.device}, layer on {self.device}")
        if x.dim() < 1 or x.shape[-1] != self.in_features:
            raise ValueError(f"expected [..., {self.in_features}] input, got {tuple(x.shape)}")
        _hip.refuse_grad("Int4Linear", x, getattr(norm, "weight", None), getattr(norm, "bias", None))
        lead, m = x.shape[:-1], math.prod(x.shape[:-1])
        if m == 0:
            return torch.empty(*lead, self.out_features, device=self.device, dtype=out_dtype)
        xr = x.reshape(-1, x.shape[-2], x.shape[-1]) if x.dim() > 2 else x.view(1, 1, -1) if x.dim() == 1 else x[None]
        with _hip.on_device(x.device):
            q, qs, _ = lowbit.quantize(xr, (xr.stride(0), xr.stride(1), xr.stride(2), max(xr.shape[1], 1)), m,
                                       self.in_features, 1, norm=norm, input_activation=input_activation)
        return gemm(q, qs, self.weight, self.bias, out_dtype=out_dtype, silu=activation == "silu").view(
            *lead, self.out_features)
