"""paged.attention (kea_paged_attention) against a dense softmax in 64 bits.

Bounds, u = 2^-24, h = 2^-11 half a step of FP16. A score is a product of d terms whose keys are exact, in FP32 with three more
roundings; the queries are off by nothing (f16), by half of FP16's smallest step, 2^-25, where a row's largest element is 2^4 or more, 2^-29 of their row's largest element each (bf16), by that and 2^-22 of themselves
(f32): es = (d + 4) u scale sum |q k| + 3 u |s| + scale 2^-29 max|q| sum|k| + [f32] 2^-22 scale sum |q k|. A weight exp(s - max) is off by
2 es + 8 u of itself, twice, in the sum and in the product; sums over n keys by (n + 24) u; the weights of the product by h (f32: h^2)
of themselves and, where FP16 has no smaller number, by 2^-25 of their unit: the reference stands at most where the largest weight times
the largest value scale that a query sees (rounded up to a power of two) would be 2^7, so that is 2^-31 max w max|v_scale| 127 a key.
The output takes half a step of its type."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

from kea_kernels import _hip, paged
from test_paged_cache import make_table

DEV = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def make(news, lengths, heads, hk, d, size, dtype, g, spread=0.3):
    """q, a cache (on the CPU), the table, lengths and offsets."""
    pages = sum(-(-max(n, 0) // size) for n in lengths) + 2
    table = make_table([max(n, 0) for n in lengths], size, pages, g)
    ints = [torch.randint(-127, 128, (pages, hk, size, d), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [0.02 * torch.exp(spread * torch.randn(pages, hk, size, generator=g)) for _ in range(2)]
    q = torch.randn(sum(news), heads, d, generator=g).to(dtype)
    offsets = torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32)
    return q, paged.Cache(*ints, *scales), table, torch.tensor(lengths, dtype=torch.int32), offsets


def on_gpu(cache):
    return paged.Cache(*(t.to(DEV) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))


def expected(q, cache, table, lengths, offsets, left=None, scale=None):
    """(the output in 64 bits, how far the kernel's may be from it), on the CPU; unseen keys are left out altogether."""
    total, heads, d = q.shape
    hk, size, dtype = cache.kv_heads, cache.page_size, q.dtype
    scale = 1 / math.sqrt(d) if scale is None else scale
    out, err = torch.zeros(total, heads, d, dtype=torch.float64), torch.zeros(total, heads, d, dtype=torch.float64)
    for b in range(len(lengths)):
        first, end = int(offsets[b]), int(offsets[b + 1])
        n, len_ = end - first, min(max(int(lengths[b]), 0), table.shape[1] * size)
        j = torch.arange(len_)
        page = table[b].long()[j // size]
        there = (page >= 0) & (page < cache.pages)
        j, page = j[there], page[there]
        if not n or not len(j):
            continue
        kc, vc = (c[page, :, j % size].double() for c in (cache.k, cache.v))
        ks, vs = (s[page, :, j % size].double() for s in (cache.k_scale, cache.v_scale))
        p = torch.arange(len_ - n, len_)[:, None]
        seen = (j <= p) & (j >= (p - left if left is not None else 0)) & (p >= 0)
        for x in range(heads):
            y = x * hk // heads
            qd = q[first:end, x].double()
            k, v = kc[:, y] * ks[:, y, None], vc[:, y] * vs[:, y, None]
            s, mag = (qd @ k.t()) * scale, (qd.abs() @ k.abs().t()) * abs(scale)
            es = (d + 4) * U * mag + 3 * U * s.abs()
            if dtype != F16:
                es = es + abs(scale) * 2.0**-29 * qd.abs().amax(1, keepdim=True) * k.abs().sum(1)
            if dtype == F32:
                es = es + 2.0**-22 * mag
            es = torch.where(seen, es, torch.zeros(1, dtype=torch.float64)).amax(1, keepdim=True)
            w = torch.nan_to_num(torch.softmax(torch.where(seen, s, torch.tensor(-math.inf, dtype=torch.float64)), 1))
            o, a = w @ v, w @ v.abs()
            rounded = 2.0**-11 if dtype != F32 else 2.0**-22
            most = w.amax(1, keepdim=True) * torch.where(seen, vs[:, y].abs(), torch.zeros(1, dtype=torch.float64)).amax(1, keepdim=True)
            e = a * (4 * es + (len(j) + 40) * U + rounded) * 1.05 + 2.0**-31 * most * (seen.double() @ vc[:, y].abs())
            out[first:end, x], err[first:end, x] = o, e + (o.abs() + e) * HALF_STEP[dtype] + (2.0**-25 if dtype == F16 else 1e-37) * seen.any(1, keepdim=True)
    return out, err


def check(got, want, err):
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    off = (got - want).abs()
    assert (off[err == 0] == 0).all()
    worst = (off / err.clamp_min(1e-300))[err > 0].max().item() if (err > 0).any() else 0.0
    assert worst <= 1, f"{worst:.3g} times the bound"


def run(q, cache, table, lengths, offsets, **kw):
    return paged.attention(q.to(DEV), on_gpu(cache), table.to(DEV), lengths.to(DEV), None if offsets is None else offsets.to(DEV), **kw)


SHAPES = [(4, 4, 64), (8, 2, 128), (6, 2, 80), (1, 1, 16), (3, 3, 256), (16, 1, 48), (33, 1, 128), (5, 5, 208)]
BATCHES = [([1], [1], 16), ([1, 1, 1], [5, 33, 300], 16), ([3, 1, 0, 40], [3, 70, 64, 200], 32), ([100], [100], 16), ([17, 9], [1000, 17], 64),
           ([1, 1], [2500, 1023], 128), ([64, 65, 63, 1, 2], [64, 130, 63, 1, 700], 16), ([300], [900], 256)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news,lengths,size", BATCHES)
def test_new_tokens(news, lengths, size, dtype):
    g = torch.Generator().manual_seed(sum(lengths))
    for i, (heads, hk, d) in enumerate(SHAPES):
        if heads * sum(news) * max(lengths) > 2_000_000 and i % 3:
            continue
        case = make(news, lengths, heads, hk, d, size, dtype, g)
        for left in (None, 0, 1, 31, 40, 500):
            got = run(*case, left=left)
            assert got.shape == case[0].shape and got.dtype == dtype
            check(got, *expected(*case, left=left))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,new,length,heads,hk,d", [(1, 1, 5000, 8, 2, 128), (4, 1, 3000, 4, 4, 64), (16, 1, 700, 16, 4, 128), (8, 4, 1500, 8, 2, 128), (70, 1, 90, 4, 2, 48),
                                                         (2, 9, 2000, 4, 1, 80), (1, 33, 4000, 2, 2, 256), (3, 70, 500, 6, 3, 96)])
def test_as_many_tokens_for_every_sequence(batch, new, length, heads, hk, d, dtype):
    """Without offsets; tables much wider than the sequences."""
    g = torch.Generator().manual_seed(length)
    lengths = [max(new, length - 131 * b) for b in range(batch)]
    q, cache, table, ln, offsets = make([new] * batch, lengths, heads, hk, d, 32, dtype, g)
    wide = torch.full((batch, table.shape[1] * 3), -5, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    for left in (None, 700):
        want = expected(q, cache, table, ln, offsets, left=left)
        check(run(q, cache, table, ln, None, left=left), *want)
        check(run(q, cache, wide, ln, None, left=left), *want)
        check(run(q, cache, wide, ln, offsets, left=left), *want)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news,lengths,heads,hk,d", [([700, 3, 333], [1500, 900, 333], 16, 4, 128), ([1200], [3500], 16, 2, 64), ([1100, 0, 1, 64], [1100, 40, 3300, 2000], 16, 16, 80),
                                                      ([257, 256, 255, 600], [500, 256, 3100, 700], 12, 3, 112)])
def test_many_rows(news, lengths, heads, hk, d, dtype):
    """Enough rows, and room for enough keys, for tiles of 128 and 256 rows."""
    g = torch.Generator().manual_seed(d)
    q, cache, table, ln, offsets = make(news, lengths, heads, hk, d, 16, dtype, g)
    wide = torch.full((len(news), 300), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    wide[0, 5] = -1  # (an entry without a page in front of every row)
    for left in (None, 3000) if d == 128 else (None,):
        check(run(q, cache, wide, ln, offsets, left=left), *expected(q, cache, wide, ln, offsets, left=left))
    if len(news) == 1:
        check(run(q, cache, wide, ln, None), *expected(q, cache, wide, ln, offsets))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_beside_scales_that_are_no_numbers(dtype):
    """Tiles of 256 rows: the last keys hold NaN or the largest scales; rows in front of them keep their bits, those behind are NaN."""
    g = torch.Generator().manual_seed(12)
    q, cache, table, ln, offsets = make([1100], [3400], 16, 4, 128, 16, dtype, g)
    clean = run(q, cache, table, ln, offsets)
    out = torch.full_like(clean, 7.0)
    tail = torch.cat([q, q[:20]])
    got = paged.attention(tail.to(DEV), on_gpu(cache), table.to(DEV), ln.to(DEV), offsets.to(DEV))
    assert torch.equal(got[:1100], clean) and not got[1100:].any()
    paged.attention(q.to(DEV), on_gpu(cache), table.to(DEV), ln.to(DEV), offsets.to(DEV), out=out)
    assert torch.equal(out, clean)
    for bad in (float("nan"), float("inf"), 3e38):
        k_scale, v_scale = cache.k_scale.clone(), cache.v_scale.clone()
        for p in (3390, 3399):
            k_scale[int(table[0, p // 16]), :, p % 16], v_scale[int(table[0, p // 16]), :, p % 16] = bad, bad
        for p in range(3400, -(-3400 // 16) * 16):
            k_scale[int(table[0, p // 16]), :, p % 16], v_scale[int(table[0, p // 16]), :, p % 16] = bad, bad
        got = run(q, paged.Cache(cache.k, cache.v, k_scale, v_scale), table, ln, offsets)
        assert torch.equal(got[:1090], clean[:1090]), bad
        if bad != 3e38:
            assert torch.isnan(got[1090:]).all()


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_tables_lengths_and_offsets_that_leave_rows_empty(dtype):
    """Entries without a page (all of a sequence's, the last, some), lengths of zero, below the new tokens and past the table, rows in
    front of and behind all sequences: zeros in a new tensor, left as they are in out."""
    g = torch.Generator().manual_seed(3)
    for heads, hk, d in ((4, 2, 64), (8, 1, 128)):
        q, cache, table, lengths, offsets = make([3, 5, 40, 2, 6, 9], [200, 0, 150, 64, 3, 70], heads, hk, d, 16, dtype, g)
        table[0, 3], table[0, 12], table[2, 2:5], table[3] = -1, cache.pages, -7, 2**31 - 1
        lengths[5] = 100000
        table[5] = torch.arange(table.shape[1]) % cache.pages
        q = torch.cat([q, q[:7]])
        offsets = offsets + 4
        want, err = expected(q, cache, table, lengths, offsets)
        got = run(q, cache, table, lengths, offsets)
        check(got, want, err)
        assert not got[:4].any() and not got[-3:].any() and not got[7:12].any() and not got[52:54].any()
        out = torch.full((len(q), heads, d + 16), 7.0, dtype=dtype, device=DEV)
        assert run(q, cache, table, lengths, offsets, out=out[..., :d]).data_ptr() == out.data_ptr()
        assert torch.equal(out[4:-3, :, :d], got[4:-3])
        assert bool((out[:4] == 7).all()) and bool((out[-3:] == 7).all()) and bool((out[..., d:] == 7).all())
        for left in (0, 20):
            check(run(q, cache, table, lengths, offsets, left=left), *expected(q, cache, table, lengths, offsets, left=left))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("rows,first,news,lengths,heads,hk,d,dtype", [
    (700, 5, (1, 3, 0, 3), (40, 70, 30, 9), 16, 4, 128, BF16), (300, 0, (2,), (33,), 5, 5, 80, F32), (400, 390, (1, 9), (100, 9), 6, 2, 48, F16),
    (64, 64, (0, 0), (20, 0), 4, 1, 256, F32), (1100, 1, (3, 2), (3200, 3000), 16, 4, 128, F16), (600, 599, (1,), (3100,), 32, 2, 64, F32)])
def test_rows_of_no_sequence_become_zeros(rows, first, news, lengths, heads, hk, d, dtype):
    """Padded batches: rows before the first sequence's and behind the last one's, in tiles of 32 rows and of more."""
    g = torch.Generator().manual_seed(rows)
    q, cache, table, lens, offsets = make(news, lengths, heads, hk, d, 16, dtype, g)
    padded = torch.full((rows, heads, d), math.nan, dtype=dtype)
    padded[first:first + len(q)] = q
    offsets = offsets + first
    want, err = expected(padded, cache, table, lens, offsets)
    old = torch.full((rows, heads, d), math.nan, dtype=dtype, device=DEV)
    args = padded.to(DEV), on_gpu(cache), table.to(DEV), lens.to(DEV), offsets.to(DEV)
    del old  # (its memory may become the output's)
    got = paged.attention(*args)
    outside = torch.ones(rows, dtype=torch.bool)
    outside[first:first + len(q)] = False
    assert (got.cpu()[outside] == 0).all()
    check(got, want, err)
    kept = torch.full_like(got, 7.0)
    paged.attention(*args, out=kept)
    assert (kept.cpu()[outside] == 7).all() and torch.equal(kept.cpu()[~outside], got.cpu()[~outside])


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,length", [(1, 900), (5, 400), (150, 300)])
def test_unseen_keys_have_no_part(new, length, dtype):
    """Scales that are no numbers, or as large as there are, where no token sees them or only some do: nothing changes for the others,
    to the bit; rows that see a NaN scale are NaN."""
    g = torch.Generator().manual_seed(new)
    q, cache, table, lengths, offsets = make([new], [length], 4, 2, 64, 32, dtype, g)
    left = 200
    clean = run(q, cache, table, lengths, offsets, left=left)
    place = lambda p: (int(table[0, p // 32]), slice(None), p % 32)  # noqa: E731
    unused = [i for i in range(cache.pages) if i not in table[0, :-(-length // 32)].tolist()]
    for bad in (float("nan"), float("inf"), -float("inf"), 3e38, 1e-38):
        k_scale, v_scale = cache.k_scale.clone(), cache.v_scale.clone()
        k_scale[unused], v_scale[unused] = bad, bad
        seen_from = 0
        for p in range(length):
            if p < length - new - left or (new > 3 and p == length - 2):  # before every window; or the last but one: two tokens see it
                k_scale[place(p)], v_scale[place(p)] = bad, bad
        for p in range(length, -(-length // 32) * 32):  # behind the sequence, in its last page
            k_scale[place(p)], v_scale[place(p)] = bad, bad
        seen_from = new - 2 if new > 3 else new
        got = run(q, paged.Cache(cache.k, cache.v, k_scale, v_scale), table, lengths, offsets, left=left)
        assert torch.equal(got[:seen_from], clean[:seen_from]), bad
        if not math.isfinite(bad):
            assert torch.isnan(got[seen_from:]).all()


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_values_of_any_size(dtype):
    """Value scales from 1e-30 (rows of zeros and others) to 1e30 side by side, scores up to the hundreds, rows of equal scores, scales of
    zero and below zero."""
    g = torch.Generator().manual_seed(5)
    for new, length in ((1, 700), (20, 333)):
        q, cache, table, lengths, offsets = make([new], [length], 4, 2, 64, 16, dtype, g, spread=2.0)
        check(run(q, cache, table, lengths, offsets), *expected(q, cache, table, lengths, offsets))
        for scale in (0.0, -0.3, 1.0, 1e-20, -0.0, 1e-45):
            check(run(q, cache, table, lengths, offsets, scale=scale), *expected(q, cache, table, lengths, offsets, scale=scale))
        for size in (1e-30, 1e-12, 1e4) if dtype == F16 else (1e-30, 1e-12, 1e4, 1e25):  # all values alike, and zeros among them
            values = torch.full_like(cache.v_scale, size)
            if dtype == F16:
                values = values.clamp(1e-3, 400)
            same = paged.Cache(cache.k, cache.v, cache.k_scale, values)
            check(run(q, same, table, lengths, offsets), *expected(q, same, table, lengths, offsets))
        v, v_scale = cache.v.clone(), cache.v_scale.clone()
        v[::2], v_scale[::2] = 0, 1e-30  # every other page: rows of zeros
        zeros = paged.Cache(cache.k, v, cache.k_scale, v_scale)
        check(run(q, zeros, table, lengths, offsets), *expected(q, zeros, table, lengths, offsets))
        q2 = (q.float() * torch.tensor([1e-3, 30.0, 1.0, 0.0])[:, None]).to(dtype)
        check(run(q2, cache, table, lengths, offsets), *expected(q2, cache, table, lengths, offsets))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_orders_in_memory(dtype):
    """q as a slice of a fused projection, out a slice of something wider, the cache's tensors in other orders, a table with room."""
    g = torch.Generator().manual_seed(6)
    q, cache, table, lengths, offsets = make([30, 1], [90, 200], 4, 2, 64, 16, dtype, g)
    want, err = expected(q, cache, table, lengths, offsets)
    rows = lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)  # noqa: E731
    pairs = torch.stack((cache.k, cache.v), 1).to(DEV)
    for other in (paged.Cache(*(rows(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))),
                  paged.Cache(pairs[:, 0], pairs[:, 1], cache.k_scale.to(DEV), cache.v_scale.to(DEV))):
        fused = torch.full((31, 3, 4, 64), float("nan"), dtype=dtype, device=DEV)
        fused[:, 1] = q.to(DEV)
        wide = torch.full((2, table.shape[1] + 5), 2**31 - 1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table.to(DEV)
        check(paged.attention(fused[:, 1], other, wide[:, :table.shape[1]], lengths.to(DEV), offsets.to(DEV)), want, err)
        out = torch.full((4, 31, 64), 3.0, dtype=dtype, device=DEV).transpose(0, 1)
        check(paged.attention(fused[:, 1], other, wide, lengths.to(DEV), offsets.to(DEV), out=out), want, err)


@pytest.mark.gpu
@torch.inference_mode()
def test_pages_past_32_bits():
    g = torch.Generator().manual_seed(8)
    q, cache, table, lengths, offsets = make([2], [40], 4, 2, 64, 16, F16, g)
    far = torch.empty(((cache.pages - 1) << 30) + 2048, dtype=torch.int8, device=DEV)
    k = far.as_strided(cache.k.shape, (1 << 30, 1024, 64, 1))
    k.copy_(cache.k)
    other = paged.Cache(k, cache.v.to(DEV), cache.k_scale.to(DEV), cache.v_scale.to(DEV))
    got = paged.attention(q.to(DEV), other, table.to(DEV), lengths.to(DEV), offsets.to(DEV))
    assert torch.equal(got, run(q, cache, table, lengths, offsets))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_captured_calls_follow_the_lengths(dtype):
    g = torch.Generator().manual_seed(9)
    q, cache, table, lengths, offsets = make([4, 4, 4], [900, 640, 300], 8, 2, 128, 32, dtype, g)
    dev = on_gpu(cache)
    q, table, lengths, offsets = q.to(DEV), table.to(DEV), lengths.to(DEV), offsets.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.attention(q, dev, table, lengths, offsets)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.attention(q, dev, table, lengths, offsets)
        even = paged.attention(q, dev, table, lengths, left=100)
    for step in range(4):
        q.normal_()
        lengths.copy_(torch.tensor([900 - 200 * step, 100 * step, 300]))
        offsets.copy_(torch.tensor([0, 1 + 2 * step, 9, 9 + step]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, paged.attention(q, dev, table, lengths, offsets))
        assert torch.equal(even, paged.attention(q, dev, table, lengths, left=100))


@pytest.mark.gpu
@torch.inference_mode()
def test_what_write_stores_is_attended_to():
    """Prompts in pieces and single tokens, written and attended to in steps, are one causal attention over the values in the cache."""
    g = torch.Generator().manual_seed(10)
    heads, hk, d, lengths = 6, 3, 64, [150, 33]
    cache = paged.Cache.empty(16, 16, hk, d, DEV)
    table = make_table(lengths, 16, 16, g).to(DEV)
    q, k, v = ([torch.randn(n, h, d, generator=g).half().to(DEV) for n in lengths] for h in (heads, hk, hk))
    done, outs = [0, 0], [[], []]
    for news in ((100, 20), (1, 1), (30, 0), (0, 11), (18, 1), (1, 0)):
        packed = [torch.cat([t[b][done[b]:done[b] + n] for b, n in enumerate(news)]) for t in (q, k, v)]
        done = [x + n for x, n in zip(done, news)]
        ln, off = torch.tensor(done, dtype=torch.int32, device=DEV), torch.tensor([0, news[0], sum(news)], dtype=torch.int32, device=DEV)
        paged.write(cache, packed[1], packed[2], table, ln, off)
        o = paged.attention(packed[0], cache, table, ln, off)
        outs[0].append(o[:news[0]])
        outs[1].append(o[news[0]:])
    assert done == lengths
    ln = torch.tensor(lengths, dtype=torch.int32)
    host = paged.Cache(*(t.cpu() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    host.k_scale.nan_to_num_(0.0)
    host.v_scale.nan_to_num_(0.0)
    want = expected(torch.cat(q).cpu(), host, table.cpu(), ln, torch.tensor([0, lengths[0], sum(lengths)], dtype=torch.int32))
    check(torch.cat(outs[0] + outs[1]), *want)


def cpu_case(d=32):
    cache = paged.Cache.empty(3, 16, 2, d, "cpu")
    return dict(q=torch.zeros(4, 4, d), cache=cache, table=torch.zeros(2, 3, dtype=torch.int32), kv_lengths=torch.zeros(2, dtype=torch.int32),
                q_offsets=torch.zeros(3, dtype=torch.int32))


def test_refusals():
    good = cpu_case()
    q = good["q"]
    for bad in (dict(q=q.double()), dict(q=q[:, :3]), dict(q=q[:, :0]), dict(q=q[..., :16]), dict(q=q[0]), dict(q=torch.zeros(4, 4, 33)[..., 1:]), dict(table=good["table"].long()),
                dict(kv_lengths=good["q_offsets"]), dict(q_offsets=good["kv_lengths"]), dict(q=q[:3], q_offsets=None), dict(left=-1), dict(left=1.5),
                dict(scale=float("nan")), dict(scale=1e39), dict(out=q[:3].clone()), dict(out=q.half()), dict(out=q[:1].expand(4, -1, -1)), dict(), dict(q_offsets=None)):
        with pytest.raises(ValueError):
            paged.attention(**{**good, **bad})
    for out in (q, good["cache"].v.view(-1).view(torch.float32)[:512].view(4, 4, 32), good["cache"].k_scale.view(-1)[:0]):
        with pytest.raises(ValueError):
            paged.attention(**good, out=out)
    with pytest.raises(RuntimeError, match="inference only"):
        paged.attention(**{**good, "q": q.clone().requires_grad_()})


def test_library_refusals():
    L, one = _hip.lib(), 16
    rows, pages = _hip.Heads(one, 0, 128, 32), _hip.Pages(one, one, 1024, 512, 32, 32, 16, 1)
    paging = _hip.Paging(one, one, one, 3, 3, 2, 3, 16, 4)
    assert L.kea_paged_attention_workspace(0, 2, 4, 48, 4, 2, 32, 1 << 30, 1) == 0
    need = L.kea_paged_attention_workspace(0, 1, 1, 16000, 4, 2, 32, 1 << 30, 0)
    assert need > 0 and need % 16 == 0
    for bad in ((3, 2, 4, 48, 4, 2, 32, 0, 1), (0, -1, 4, 48, 4, 2, 32, 0, 1), (0, 2, 4, (1 << 30) + 1, 4, 2, 32, 0, 1), (0, 2, 4, 48, 3, 2, 32, 0, 1),
                (0, 2, 4, 48, 4, 2, 24, 0, 1), (0, 2, 4, 48, 4, 2, 32, -1, 1), (0, 2, 1 << 29, 48, 4096, 2, 32, 0, 1)):
        assert L.kea_paged_attention_workspace(*bad) < 0
    call = lambda q=rows, out=rows, t=0, h=4, hk=2, d=32, k=pages, g=paging, left=0, scale=1.0, ws=None, n=0: L.kea_paged_attention(  # noqa: E731
        q, out, t, h, hk, d, k, pages, g, left, scale, 1, ws, n, None)
    for rc in (call(t=3), call(h=3), call(hk=0), call(d=24), call(left=-1), call(scale=float("inf")), call(q=_hip.Heads(None, 0, 128, 32)),
               call(k=_hip.Pages(one, one, 1 << 40, 1 << 38, 1 << 27, 32, 16, 1)), call(g=_hip.Paging(one, one, one, 3, 3, 2, 3, 24, 4))):
        assert rc == -1
    for rc in (call(q=_hip.Heads(8, 0, 128, 32)), call(out=_hip.Heads(one, 0, 130, 32)), call(k=_hip.Pages(8, one, 1024, 512, 32, 32, 16, 1)), call(ws=ctypes.c_void_p(8))):
        assert rc == -2
    long = _hip.Paging(one, one, None, 1000, 1000, 1, 3, 16, 1)
    assert call(g=long, left=1 << 30) == -4 and call(g=long, left=1 << 30, ws=ctypes.c_void_p(16), n=need // 2 // 16 * 16 if need > 64 else 0) == -4
    assert call(g=_hip.Paging(one, one, one, 3, 3, 2, 3, 16, 0)) == 0
