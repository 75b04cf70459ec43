"""An int8 key and value cache in pages, and attention over it (kea_paged_write, kea_paged_read, kea_paged_attention,
include/kea_decode.h): for sequences that come, grow and leave at different times and share one pool of memory.

A Cache holds `pages` of page_size positions; a table names each sequence's pages in the order of its positions. The new tokens of
a call are packed, sequence after sequence: `write` puts their keys and values in their places, a scale for each token and head,
`attention` lets them attend to their sequences, themselves included, and `read` gives positions back as dense tensors of values.
Lengths, offsets and tables are read on the device: they may change between replays of a captured call. Calls run on torch's
current stream of the tensors' device and never synchronize the host.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch import Tensor

from kea_kernels import _hip
from kea_kernels.window import _bound, _span

_MOST = 1 << 30  # positions of a sequence, tokens of a call


def _distinct(name: str, t: Tensor, other: Tensor | None = None) -> None:
    """ValueError where two elements of t, or of t and `other` of its shape, share memory."""
    steps = [(t.stride(i), t.shape[i]) for i in range(t.dim()) if t.shape[i] > 1]
    if other is not None:  # one tensor of both, where they lie in each other's span
        if not t.numel() or _span(t)[0] >= _span(other)[1] or _span(other)[0] >= _span(t)[1]:
            return
        if any(n > 1 and a != b for a, b, n in zip(t.stride(), other.stride(), t.shape)):
            raise ValueError(f"{name} lie in the same memory in different orders")
        steps.append((abs(t.data_ptr() - other.data_ptr()) // t.element_size(), 2))
    steps.sort()
    if any(s < 1 for s, _ in steps) or any(s < reach for (s, _), reach in zip(steps[1:], (1 + sum((n - 1) * s for s, n in steps[:i + 1])
                                                                                          for i in range(len(steps))))):
        raise ValueError(f"{name} has elements that share memory: shape {tuple(t.shape)}, strides {t.stride()}")


class Cache:
    """Keys and values as int8 `k`, `v` [pages, kv_heads, page_size, D] with FP32 scales `k_scale`, `v_scale` [pages, kv_heads,
    page_size]: element e of a row stands for k[..., e] * k_scale[...]. page_size is a power of two from 16 to 1024, D a multiple of 16
    up to 256; rows of D are contiguous and start at multiples of 16 bytes, the other dimensions may have any order in memory. Keys and
    values may lie between each other, the codes' memory and the scales' may not. The tensors are the caller's (no copies are made);
    pages need no initial values."""

    def __init__(self, k: Tensor, v: Tensor, k_scale: Tensor, v_scale: Tensor):
        if k.dim() != 4 or k.dtype != torch.int8 or k.shape != v.shape or v.dtype != torch.int8:
            raise ValueError(f"k and v must be int8 [pages, kv_heads, page_size, D], got {k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)}")
        pages, heads, size, d = k.shape
        if size < 16 or size > 1024 or size & (size - 1):
            raise ValueError(f"page size {size}: a power of two from 16 to 1024")
        if d < 16 or d > 256 or d % 16 or not 1 <= heads <= 65535:
            raise ValueError(f"{heads} heads of {d}: at least one, of a multiple of 16 from 16 to 256")
        for name, t in (("k", k), ("v", v)):
            if t.stride(3) != 1 or t.data_ptr() % 16 or any(t.stride(i) % 16 for i in range(3) if t.shape[i] > 1):
                raise ValueError(f"{name} needs contiguous rows that start at multiples of 16 bytes, got strides {t.stride()}")
            _distinct(name, t)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or t.shape != k.shape[:3]:
                raise ValueError(f"{name} must be f32 {tuple(k.shape[:3])}, got {t.dtype} {tuple(t.shape)}")
            _distinct(name, t)
        if any(t.device != k.device for t in (v, k_scale, v_scale)):
            raise ValueError("the cache's tensors are on different devices")
        _distinct("k and v", k, v)
        _distinct("k_scale and v_scale", k_scale, v_scale)
        for t in (k, v):
            for s in (k_scale, v_scale):
                if t.numel() and _span(t)[0] < _span(s)[1] and _span(s)[0] < _span(t)[1]:
                    raise ValueError("codes and scales lie in the same memory")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, d: int, device="cuda") -> "Cache":
        ints = [torch.empty(pages, kv_heads, page_size, d, dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.empty(pages, kv_heads, page_size, device=device) for _ in range(2)]
        return cls(*ints, *scales)

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def head_size(self) -> int:
        return self.k.shape[3]

    @property
    def device(self) -> torch.device:
        return self.k.device

    def nbytes(self) -> int:
        return 2 * self.k.numel() + 8 * self.k_scale.numel()


def _pages(c: Tensor, s: Tensor) -> "_hip.Pages":
    at = lambda t: [t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)]  # noqa: E731
    return _hip.Pages(c.data_ptr(), s.data_ptr(), *at(c), *at(s))


def _index(name: str, t: Tensor, n: int, device) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous int32 tensor [{n}] on {device}")


def _paging(cache: Cache, table: Tensor, kv_lengths: Tensor, q_offsets: Tensor | None, tokens: int) -> "_hip.Paging":
    device = cache.device
    if table.dim() != 2 or table.dtype != torch.int32 or table.device != device or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"table must be int32 [sequences, pages] with unit column stride on {device}, got {table.dtype} {tuple(table.shape)}")
    batch, width = table.shape
    if width * cache.page_size > _MOST:
        raise ValueError(f"table has room for more than 2^30 positions: {width} pages of {cache.page_size}")
    _index("kv_lengths", kv_lengths, batch, device)
    if q_offsets is not None:
        _index("q_offsets", q_offsets, batch + 1, device)
    elif tokens % batch if batch else tokens:
        raise ValueError(f"{tokens} tokens are no multiple of {batch} sequences (q_offsets gives each its own)")
    if tokens >= _MOST or batch >= _MOST:
        raise ValueError("tokens and sequences must be below 2^30")
    return _hip.Paging(table.data_ptr(), kv_lengths.data_ptr(), _hip.ptr(q_offsets), table.stride(0) if batch > 1 else 0, width, batch,
                       cache.pages, cache.page_size, tokens)


def _rows(name: str, t: Tensor, cache: Cache, heads: int | None) -> "_hip.Heads":
    d = cache.head_size
    if t.dim() != 3 or t.dtype not in _hip.DTYPES or t.shape[2] != d or (heads is not None and t.shape[1] != heads) or t.device != cache.device:
        raise ValueError(f"{name} must be f32, f16 or bf16 [tokens, {'heads' if heads is None else heads}, {d}] on {cache.device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    unit = 16 // t.element_size()
    if t.stride(2) != 1 or t.data_ptr() % 16 or any(t.stride(i) % unit for i in range(2) if t.shape[i] > 1):
        raise ValueError(f"{name} needs contiguous heads that start at multiples of 16 bytes, got strides {t.stride()}")
    return _hip.Heads(t.data_ptr(), 0, *(t.stride(i) if t.shape[i] > 1 else 0 for i in range(2)))


def _apart(name: str, written: tuple, others: tuple) -> None:
    for t in written:
        for o in others:
            if o is not None and t.numel() and o.numel() and _span(t)[0] < _span(o)[1] and _span(o)[0] < _span(t)[1]:
                raise ValueError(f"{name} shares memory with another operand")


def write(cache: Cache, k: Tensor, v: Tensor, table: Tensor, kv_lengths: Tensor, q_offsets: Tensor | None = None) -> None:
    """Quantises new tokens' keys and values into the cache. k, v f32, f16 or bf16 [T, kv_heads, D]; table int32 [B, pages of a
    sequence]; kv_lengths int32 [B], with the new tokens; q_offsets int32 [B + 1], ascending: sequence b has the rows q_offsets[b] to
    q_offsets[b + 1] - 1 (None: T / B rows each). The n rows of a sequence of len positions stand at len - n .. len - 1; position p
    goes to row p % page_size of page table[b, p // page_size]. len is held to 0 .. table.shape[1] * page_size.

    A row x of D elements becomes s = max(max|x| / 127, 1e-30), held to the largest number of which 127 s is finite, and rint(x / s);
    one that holds an infinity or NaN becomes s = NaN and zeros, and reads as NaN. Rows of no sequence, positions below 0 and table
    entries outside 0 .. pages - 1 are left out, and no other byte of the cache is written. No two tokens of a call may stand at the same
    place (what is there then is not defined)."""
    if (_native("paged_write", cache, k, v, table, kv_lengths, q_offsets)) is not None:
        return
    heads = cache.kv_heads
    rows = [_rows(name, t, cache, heads) for name, t in (("k", k), ("v", v))]
    if k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k is {k.dtype} {tuple(k.shape)}, v {v.dtype} {tuple(v.shape)}")
    paging = _paging(cache, table, kv_lengths, q_offsets, k.shape[0])
    _apart("the cache", (cache.k, cache.v, cache.k_scale, cache.v_scale), (k, v, table, kv_lengths, q_offsets))
    _hip.refuse_grad("paged.write", k, v, cache.k_scale, cache.v_scale)
    if not k.shape[0] or not table.shape[0]:
        return
    with _hip.on_device(cache.device):
        rc = _hip.lib().kea_paged_write(*rows, _hip.dtype_code(k.dtype), heads, cache.head_size, _pages(cache.k, cache.k_scale),
                                        _pages(cache.v, cache.v_scale), paging, _hip.stream_handle(cache.device))
    _hip.check(rc, "kea_paged_write")


def read(cache: Cache, table: Tensor, kv_lengths: Tensor, length: int, *, starts: Tensor | None = None,
         out_dtype: torch.dtype = torch.float32) -> tuple[Tensor, Tensor]:
    """(k, v), each [B, length, kv_heads, D] of out_dtype (f32, f16, bf16): the values of positions starts[b] + i, 0 <= i < length, of
    every sequence (starts int32 [B], None: 0), integers times scales in FP32, f16 and bf16 rounded from there; zeros for positions
    outside 0 .. kv_lengths[b] - 1 and for table entries outside 0 .. pages - 1."""
    if (hit := _native("paged_read", cache, table, kv_lengths, length, starts, out_dtype)) is not None:
        return hit
    if out_dtype not in _hip.DTYPES:
        raise ValueError(f"unsupported output dtype {out_dtype}")
    if int(length) != length or not 0 <= length <= _MOST:
        raise ValueError(f"length must be a whole number from 0 to 2^30, got {length!r}")
    paging = _paging(cache, table, kv_lengths, None, 0)
    if starts is not None:
        _index("starts", starts, table.shape[0], cache.device)
    _hip.refuse_grad("paged.read", cache.k_scale, cache.v_scale)
    shape = (table.shape[0], int(length), cache.kv_heads, cache.head_size)
    k, v = (torch.empty(shape, dtype=out_dtype, device=cache.device) for _ in range(2))
    if k.numel():
        with _hip.on_device(cache.device):
            rc = _hip.lib().kea_paged_read(_pages(cache.k, cache.k_scale), _pages(cache.v, cache.v_scale), paging, _hip.ptr(starts), int(length),
                                           cache.kv_heads, cache.head_size, k.data_ptr(), v.data_ptr(), _hip.dtype_code(out_dtype),
                                           _hip.stream_handle(cache.device))
        _hip.check(rc, "kea_paged_read")
    return k, v


def attention(q: Tensor, cache: Cache, table: Tensor, kv_lengths: Tensor, q_offsets: Tensor | None = None, *, left: int | None = None,
              scale: float | None = None, out: Tensor | None = None) -> Tensor:
    """out [T, H, D] = attention of the new tokens q [T, H, D] (f32, f16 or bf16; H a multiple of kv_heads, query head h reads key head
    h // (H / kv_heads)) to their sequences' positions in the cache, their own among them: `write` comes first. table, kv_lengths and
    q_offsets as there: the n rows of a sequence of len positions stand at len - n .. len - 1, and the token at position p sees
    position j iff p - left <= j <= p (left None: all before) and the table names a page for it. A token that sees nothing gives
    zeros, and so do rows of no sequence, but in `out`, where those stay as they are. What a token does not see has no part in its
    output, whatever it holds. scale: 1 / sqrt(D) unless given, any finite FP32 number. out must not overlap an input.

    Scores, maxima and sums are FP32 and the codes enter the products exactly; the softmax's weights times the values' scales are
    rounded to FP16 (f32: to two parts, 22 bits; small ones to multiples of 2^-30 of the row's largest), and so are bf16 and f32 queries, after a power of two of each row's own (what is
    below 2^-28 of a row's largest element is lost; f32 keeps 22 bits)."""
    if out is None and (hit := _native("paged_attention", cache, q, table, kv_lengths, q_offsets, left, scale)) is not None:
        return hit
    rows = _rows("q", q, cache, None)
    (tokens, h, d), hk, device = q.shape, cache.kv_heads, cache.device
    if h < 1 or h % hk or h > 65535:
        raise ValueError(f"{h} query heads are no multiple of {hk} key heads")
    paging = _paging(cache, table, kv_lengths, q_offsets, tokens)
    scale = 1 / math.sqrt(d) if scale is None else ctypes.c_float(scale).value
    if not math.isfinite(scale):
        raise ValueError("scale is not a finite FP32 number")
    left = _bound("left", left)
    fill = out is None
    if out is not None:
        _rows("out", out, cache, h)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError(f"out is {out.dtype} {tuple(out.shape)}, q {q.dtype} {tuple(q.shape)}")
        _distinct("out", out)
        _apart("out", (out,), (q, cache.k, cache.v, cache.k_scale, cache.v_scale, table, kv_lengths, q_offsets))
    _hip.refuse_grad("paged.attention", q, cache.k_scale, cache.v_scale, out)
    if out is None:
        out = torch.empty(tokens, h, d, dtype=q.dtype, device=device)
    if not tokens:
        return out
    L, code, batch, width = _hip.lib(), _hip.dtype_code(q.dtype), *table.shape
    with _hip.on_device(device):
        need = L.kea_paged_attention_workspace(code, batch, tokens, width * cache.page_size, h, hk, d, left, q_offsets is not None)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        rc = L.kea_paged_attention(rows, _rows("out", out, cache, h), code, h, hk, d, _pages(cache.k, cache.k_scale),
                                   _pages(cache.v, cache.v_scale), paging, left, scale, fill, _hip.ptr(ws), max(need, 0), _hip.stream_handle(device))
    _hip.check(rc, "kea_paged_attention")
    return out


def _native(name: str, cache: Cache, *args):
    """A call in one native call (the same checks on the tensors' fields); None, having launched nothing, where an argument is not
    what it takes: the Python path then checks again and raises or launches."""
    try:
        return getattr(_hip.native(), name)(cache.k, cache.v, cache.k_scale, cache.v_scale, *args)
    except (AttributeError, TypeError, ValueError):
        return None
