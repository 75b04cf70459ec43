"""paged.Cache, paged.write and paged.read (kea_paged_write, kea_paged_read): an int8 cache in pages against its definition.

The rule s = max(max|x| / 127, 1e-30) (held to where 127 s is finite), rint(x / s) is FP32 throughout with correctly rounded quotients, as torch's elementary
operations are on the CPU: codes and scales are equal, and so are values read back, c * s rounded once."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kea_kernels import _hip, paged

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
MOST = float.fromhex("0x1.0204060000000p+121")


def rows8(x):
    """Codes and scales of the rows of x, on the CPU."""
    x = x.float()
    good = torch.isfinite(x).all(-1)
    s = (torch.where(good[..., None], x, torch.zeros(())).abs().amax(-1) / 127).clamp(1e-30, MOST)
    c = torch.round(torch.where(good[..., None], x, torch.zeros(())) / s[..., None]).clamp(-127, 127).to(torch.int8)
    return c, torch.where(good, s, torch.tensor(float("nan")))


def make_cache(pages, heads, size, d, g, device=DEV, order="heads"):
    """A cache of known garbage; order: how it lies in memory."""
    if order == "heads":
        ints = [torch.randint(-128, 128, (pages, heads, size, d), generator=g, dtype=torch.int8).to(device) for _ in range(2)]
        scales = [torch.rand(pages, heads, size, generator=g).to(device) for _ in range(2)]
    elif order == "rows":  # positions first, as tokens come
        ints = [torch.randint(-128, 128, (pages, size, heads, d), generator=g, dtype=torch.int8).to(device).transpose(1, 2) for _ in range(2)]
        scales = [torch.rand(pages, size, heads, generator=g).to(device).transpose(1, 2) for _ in range(2)]
    else:  # keys and values of a page side by side
        ints = list(torch.randint(-128, 128, (pages, 2, heads, size, d), generator=g, dtype=torch.int8).to(device).unbind(1))
        scales = list(torch.rand(pages, heads, size, 2, generator=g).to(device).unbind(3))
    return paged.Cache(*ints, *scales)


def make_table(lengths, size, pages, g, width=None):
    """Each sequence's pages, drawn without order; entries past its end name none or anything."""
    width = width or max(-(-n // size) for n in lengths) + 1
    order = torch.randperm(pages, generator=g)
    table, at = torch.full((len(lengths), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(lengths):
        need = -(-n // size)
        table[b, :need] = order[at:at + need]
        table[b, need:] = torch.tensor([-1, 10**9, -(2**31), pages])[(torch.arange(width - need) + b) % 4].int()
        at += need
    return table


def plain(t):
    return t.detach().cpu().clone()


CASES = [([1], [1], 1, 64, 16), ([1, 1, 1], [5, 16, 33], 4, 128, 16), ([7, 0, 40, 1], [40, 9, 40, 100], 2, 80, 32), ([3, 3], [3, 260], 5, 16, 16),
         ([130], [130], 3, 256, 64), ([65, 64, 63], [200, 64, 70], 8, 96, 128), ([2] * 70, [9] * 70, 2, 48, 16)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news,lengths,heads,d,size", CASES)
def test_written_rows_and_nothing_else(news, lengths, heads, d, size, dtype):
    g = torch.Generator().manual_seed(sum(lengths) + d)
    pages = sum(-(-n // size) for n in lengths) + 2
    table = make_table(lengths, size, pages, g)
    total = sum(news)
    k, v = ((torch.randn(total + 3, heads, d, generator=g) * torch.randn(total + 3, heads, 1, generator=g).exp()).to(dtype) for _ in range(2))
    if total > 1:
        k[1, 0] = 0.0
        v[0, heads - 1] = v[0, heads - 1] * 1e-35 if dtype != F16 else 0.0
    offsets = torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32)
    for order in ("heads", "rows", "pairs"):
        cache = make_cache(pages, heads, size, d, g, order=order)
        want = [plain(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        for b, (new, n) in enumerate(zip(news, lengths)):
            for i in range(new):
                p = n - new + i
                page, row = int(table[b, p // size]), p % size
                for x, c, s in ((k, want[0], want[2]), (v, want[1], want[3])):
                    c[page, :, row], s[page, :, row] = rows8(x[int(offsets[b]) + i])
        args = (table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
        if len(set(news)) == 1 and order != "rows":
            paged.write(cache, k[:total].to(DEV), v[:total].to(DEV), *args)
        else:  # rows behind the last sequence's are not read into any
            paged.write(cache, k.to(DEV), v.to(DEV), *args, offsets.to(DEV))
        for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
            assert torch.equal(got.cpu(), w)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("news,lengths,heads,d,size", CASES)
def test_read_gives_the_values(news, lengths, heads, d, size, dtype):
    g = torch.Generator().manual_seed(sum(lengths) + d)
    pages = sum(-(-n // size) for n in lengths) + 2
    table = make_table(lengths, size, pages, g)
    cache = make_cache(pages, heads, size, d, g, order=["heads", "rows", "pairs"][d % 3])
    c = [plain(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    most = max(lengths)
    starts = torch.tensor([(-3, 0, most // 2, most + 5, 2**31 - 1, -(2**31))[b % 6] for b in range(len(lengths))], dtype=torch.int32)
    for st, length in ((None, most + 2), (starts, most), (None, 1)):
        want = torch.zeros(2, len(lengths), length, heads, d, dtype=dtype)
        for b, n in enumerate(lengths):
            for i in range(length):
                p = i + (0 if st is None else int(st[b]))
                if 0 <= p < n:
                    page, row = int(table[b, p // size]), p % size
                    for w, ints, s in ((want[0], c[0], c[2]), (want[1], c[1], c[3])):
                        w[b, i] = (ints[page, :, row].float() * s[page, :, row][:, None]).to(dtype)
        got = paged.read(cache, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), length,
                         starts=None if st is None else st.to(DEV), out_dtype=dtype)
        assert all(torch.equal(x.cpu(), w) for x, w in zip(got, want))


@pytest.mark.gpu
@torch.inference_mode()
def test_bad_entries_lengths_and_offsets_are_left_out():
    """Entries that name no page, lengths past the table or below the new tokens, rows in front of and behind all sequences."""
    g = torch.Generator().manual_seed(4)
    cache = make_cache(6, 2, 16, 32, g)
    want = [plain(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    table = torch.tensor([[0, -1, 3], [6, 1, 2**31 - 1], [4, -(2**31), 5]], dtype=torch.int32)
    lengths, offsets = torch.tensor([40, 14, 1000], dtype=torch.int32), torch.tensor([2, 22, 42, 50], dtype=torch.int32)
    k, v = (torch.randn(60, 2, 32, generator=g) for _ in range(2))
    for b, (n, lo, hi) in enumerate(((40, 2, 22), (14, 22, 42), (48, 42, 50))):
        for t in range(lo, hi):
            p = n - hi + t
            if p >= 0 and 0 <= int(table[b, p // 16]) < 6:
                page, row = int(table[b, p // 16]), p % 16
                want[0][page, :, row], want[2][page, :, row] = rows8(k[t])
                want[1][page, :, row], want[3][page, :, row] = rows8(v[t])
    paged.write(cache, k.to(DEV), v.to(DEV), table.to(DEV), lengths.to(DEV), offsets.to(DEV))
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), want):
        assert torch.equal(got.cpu(), w)
    values = paged.read(cache, table.to(DEV), lengths.to(DEV), 60)
    for b, n in enumerate((40, 14, 48)):
        for p in range(60):
            page = int(table[b, p // 16]) if p < n else -1
            w = want[0][page, :, p % 16].float() * want[2][page, :, p % 16][:, None] if 0 <= page < 6 else torch.zeros(2, 32)
            assert torch.equal(values[0][b, p].cpu(), w)
    # lengths below zero, a table without columns, no sequences, no tokens
    before = [plain(t) for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    paged.write(cache, k.to(DEV), v.to(DEV), table.to(DEV), -lengths.to(DEV), offsets.to(DEV))
    paged.write(cache, k.to(DEV), v.to(DEV), table[:, :0].to(DEV), lengths.to(DEV), offsets.to(DEV))
    paged.write(cache, k[:0].to(DEV), v[:0].to(DEV), table[:0].to(DEV), lengths[:0].to(DEV))
    paged.write(cache, k[:0].to(DEV), v[:0].to(DEV), table.to(DEV), lengths.to(DEV))
    paged.write(cache, k.to(DEV), v.to(DEV), table.to(DEV), lengths.to(DEV), torch.tensor([60, 60, 70, 2**31 - 1], dtype=torch.int32, device=DEV))
    for got, w in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        assert torch.equal(got.cpu(), w)
    assert not paged.read(cache, table[:, :0].to(DEV), lengths.to(DEV), 4)[0].any()
    assert paged.read(cache, table[:0].to(DEV), lengths[:0].to(DEV), 4)[0].shape == (0, 4, 2, 32)
    assert paged.read(cache, table.to(DEV), lengths.to(DEV), 0)[1].shape == (3, 0, 2, 32)
    none = paged.Cache.empty(0, 16, 2, 32, DEV)
    paged.write(none, k.to(DEV), v.to(DEV), table.to(DEV), lengths.to(DEV), offsets.to(DEV))
    assert not paged.read(none, table.to(DEV), lengths.to(DEV), 30)[0].any()
    assert not paged.attention(k.to(DEV), none, table.to(DEV), lengths.to(DEV), offsets.to(DEV)).any()
    assert not paged.attention(k.to(DEV), cache, table[:, :0].to(DEV), lengths.to(DEV), offsets.to(DEV)).any()


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_no_numbers_and_of_any_size(dtype):
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.randn(8, 1, 64, generator=torch.Generator().manual_seed(5)).to(dtype)
    x[1, 0, 5], x[2, 0, 63], x[3, 0, 0] = float("inf"), float("nan"), -float("inf")
    x[4] = (x[4].float().clamp(-1, 1) * big).to(dtype)
    x[5] = (x[5].float() * small).to(dtype)
    x[6, 0, 1:] = 0.0
    cache = paged.Cache.empty(1, 16, 1, 64, DEV)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([8], dtype=torch.int32, device=DEV)
    paged.write(cache, x.to(DEV), -x.to(DEV), table, lengths)
    c, s = rows8(x)
    assert torch.equal(cache.k[0, 0, :8].cpu(), c[:, 0]) and torch.equal(cache.v[0, 0, :8].cpu(), -c[:, 0])
    assert torch.equal(cache.k_scale[0, 0, :8].cpu().nan_to_num(-1.0), s[:, 0].nan_to_num(-1.0))
    k, v = paged.read(cache, table, lengths, 8, out_dtype=dtype)
    assert torch.isnan(k[0, 1:4]).all() and torch.isnan(v[0, 1:4]).all() and torch.isfinite(k[0, 4:]).all()
    # a value is within half a step of its row, and half a step of the type
    off, step = (k[0].cpu().double() - x.double()).abs(), x.double().abs().amax(2, keepdim=True) / 254
    tiny = 5e-31 if dtype != F16 else 2.0**-24
    assert bool((off[[0, 4, 5, 6, 7]] <= (step * 1.0001 + x.double().abs() * torch.finfo(dtype).eps + tiny)[[0, 4, 5, 6, 7]]).all())


@pytest.mark.gpu
@torch.inference_mode()
def test_views_of_a_fused_projection_and_far_pages():
    """k and v as slices of wider rows; pages whose bytes lie past 2^31."""
    g = torch.Generator().manual_seed(6)
    fused = torch.randn(5, 6, 64, generator=g).half()
    dev = fused.to(DEV)
    store = torch.empty(2, 2 * 16 * 64, dtype=torch.int8, device=DEV)
    far = torch.empty((1 << 31) + 4096, dtype=torch.int8, device=DEV)
    k = far.as_strided((2, 2, 16, 64), (1 << 31, 1024, 64, 1))
    scale = torch.empty(2, 2, 16, device=DEV)
    cache = paged.Cache(k, store.view(2, 2, 16, 64), scale, torch.empty_like(scale))
    table, lengths = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), torch.tensor([19], dtype=torch.int32, device=DEV)
    paged.write(cache, dev[:, 2:4], dev[:, 4:], table, lengths)
    got = paged.read(cache, table, lengths, 5, starts=torch.tensor([14], dtype=torch.int32, device=DEV))
    for x, y in ((fused[:, 2:4], got[0][0]), (fused[:, 4:], got[1][0])):
        c, s = rows8(x)
        assert torch.equal(y.cpu(), c.float() * s[..., None])


@pytest.mark.gpu
@torch.inference_mode()
def test_captured_calls_follow_the_lengths():
    g = torch.Generator().manual_seed(7)
    cache = make_cache(20, 2, 16, 64, g)
    table = make_table([100, 100], 16, 20, g).to(DEV)
    lengths, offsets = torch.tensor([4, 4], dtype=torch.int32, device=DEV), torch.tensor([0, 2, 4], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(6, 2, 64, generator=g).to(DEV) for _ in range(2))
    paged.write(cache, k, v, table, lengths, offsets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.write(cache, k, v, table, lengths, offsets)
        out = paged.read(cache, table, lengths, 50)
    for step in range(4):
        k.normal_()
        lengths.copy_(torch.tensor([5 + 7 * step, 30 + step], dtype=torch.int32))
        offsets.copy_(torch.tensor([0, 1 + step, 4 + step // 2], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = paged.read(cache, table, lengths, 50)
        assert all(torch.equal(x, y) for x, y in zip(out, want))
        n, last = 30 + step, 4 + step // 2 - (1 + step)
        c, s = rows8(k[1 + step:4 + step // 2].cpu())
        assert torch.equal(out[0][1, n - last:n].cpu(), c.float() * s[..., None])


def cpu_cache(pages=3, heads=2, size=16, d=32):
    return paged.Cache.empty(pages, size, heads, d, "cpu")


def test_cache_refusals():
    i, s = torch.zeros(3, 2, 16, 32, dtype=torch.int8), torch.zeros(3, 2, 16)
    paged.Cache(i, i.clone(), s, s.clone())
    for bad in (lambda: paged.Cache(i.float(), i.clone(), s, s.clone()), lambda: paged.Cache(i, i[:2], s, s.clone()), lambda: paged.Cache(i[0], i[0].clone(), s, s.clone()),
                lambda: paged.Cache(i, i.clone(), s.half(), s.clone()), lambda: paged.Cache(i, i.clone(), s, s[:2]), lambda: paged.Cache(i, i, s, s.clone()),
                lambda: paged.Cache(i, i.clone(), s, s), lambda: paged.Cache(i[:1].expand(3, -1, -1, -1), i.clone(), s, s.clone()),
                lambda: paged.Cache(i.transpose(2, 3), i.clone().transpose(2, 3), torch.zeros(3, 2, 32), torch.ones(3, 2, 32)),
                lambda: paged.Cache(i, i.clone(), s[:1].expand(3, -1, -1), s.clone()), lambda: cpu_cache(size=12), lambda: cpu_cache(size=8),
                lambda: cpu_cache(size=2048), lambda: cpu_cache(d=24), lambda: cpu_cache(d=272), lambda: cpu_cache(heads=0)):
        with pytest.raises(ValueError):
            bad()


def test_keys_and_values_that_share_memory_are_refused():
    b, s = torch.zeros(6, 2, 16, 32, dtype=torch.int8), torch.zeros(6, 2, 16)
    for k, v in ((b[::2], b[1::2]), (b[:3], b[3:]), (b.view(3, 2, 2, 16, 32)[:, 0], b.view(3, 2, 2, 16, 32)[:, 1])):
        paged.Cache(k, v, s[:3], s[3:])
    paged.Cache(b[:3], b[3:], s[::2], s[1::2])
    for k, v, ks, vs in ((b[:3], b[2:5], s[:3], s[3:]), (b[:3], b[3:], s[:3], s[1:4]), (b[:3], b[::2], s[:3], s[3:]),
                         (b[:3].transpose(1, 2).reshape(3, 2, 16, 32), b[3:], b.view(-1)[:3 * 2 * 16 * 4].view(torch.float32).view(3, 2, 16), b[3:].view(-1)[:3 * 2 * 16 * 4].view(torch.float32).view(3, 2, 16))):
        with pytest.raises(ValueError):
            paged.Cache(k, v, ks, vs)


def test_call_refusals():
    c = cpu_cache()
    x, table, lengths, offsets = torch.zeros(4, 2, 32), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    w = lambda **kw: paged.write(*{**dict(cache=c, k=x, v=x, table=table, kv_lengths=lengths, q_offsets=offsets), **kw}.values())  # noqa: E731
    for bad in (dict(k=x.double()), dict(k=x[:, :1]), dict(v=x[:3]), dict(v=x.half()), dict(k=x[..., :16]), dict(k=x[0]), dict(table=table.long()),
                dict(table=table[0]), dict(table=table.t().contiguous().t()[:, :2]), dict(kv_lengths=lengths[:1]), dict(kv_lengths=lengths.long()),
                dict(q_offsets=lengths), dict(k=x[:3], v=x[:3], q_offsets=None), dict(table=table[:0], kv_lengths=lengths[:0], q_offsets=None),
                dict(k=torch.zeros(4, 2, 33)[..., 1:]), dict(), dict(q_offsets=None)):  # (the last two: tensors on the CPU)
        with pytest.raises(ValueError):
            w(**bad)
    with pytest.raises(ValueError, match="shares memory"):
        w(k=c.k.view(-1).view(torch.float32)[:256].view(4, 2, 32))
    for bad in (dict(length=-1), dict(length=1.5), dict(length=2**31), dict(out_dtype=torch.int8), dict(starts=offsets), dict(starts=lengths.long()),
                dict(kv_lengths=offsets), dict()):
        with pytest.raises(ValueError):
            paged.read(**{**dict(cache=c, table=table, kv_lengths=lengths, length=4), **bad})
    with pytest.raises(ValueError, match="2\\^30"):
        paged.read(cpu_cache(size=1024, d=16), torch.empty(1, (1 << 20) + 1, dtype=torch.int32), lengths[:1], 4)
    with pytest.raises(RuntimeError, match="inference only"):
        w(k=x.clone().requires_grad_())


def test_library_refusals():
    L, one, odd = _hip.lib(), 16, 8
    heads, pages = _hip.Heads(one, 0, 64, 32), _hip.Pages(one, one, 1024, 512, 32, 32, 16, 1)
    paging = lambda **kw: _hip.Paging(*{**dict(table=one, kv_lengths=one, q_offsets=one, table_stride=3, table_width=3, batch=2, pages=3, page_size=16,  # noqa: E731
                                               tokens=4), **kw}.values())
    write = lambda k=heads, t=0, hk=2, d=32, p=pages, g=None: L.kea_paged_write(k, k, t, hk, d, p, p, g or paging(), None)  # noqa: E731
    read = lambda p=pages, g=None, n=4, k=one, t=0, s=None: L.kea_paged_read(p, p, g or paging(), s, n, 2, 32, k, k, t, None)  # noqa: E731
    for rc in (write(t=3), write(hk=0), write(d=24), write(d=272), write(g=paging(batch=-1)), write(g=paging(tokens=-1)), write(g=paging(page_size=12)),
               write(g=paging(page_size=8)), write(g=paging(page_size=2048)), write(g=paging(table_width=1 << 28)), write(g=paging(q_offsets=None, tokens=3)),
               write(g=paging(kv_lengths=None)), write(g=paging(table=None)), write(p=_hip.Pages(None, one, 1024, 512, 32, 32, 16, 1)),
               write(k=_hip.Heads(None, 0, 64, 32)), read(t=5), read(n=-1), read(n=(1 << 30) + 1), read(k=None)):
        assert rc == -1
    for rc in (write(k=_hip.Heads(odd, 0, 64, 32)), write(k=_hip.Heads(one, 0, 66, 32)), write(k=_hip.Heads(one, 0, -64, 32)),
               write(p=_hip.Pages(odd, one, 1024, 512, 32, 32, 16, 1)), write(p=_hip.Pages(one, 18, 1024, 512, 32, 32, 16, 1)),
               write(p=_hip.Pages(one, one, 1032, 512, 32, 16, 8, 1)), write(g=paging(table=18)), read(k=odd), read(s=ctypes.c_void_p(18))):
        assert rc == -2
    assert write(g=paging(tokens=0)) == 0 and read(n=0) == 0 and write(g=paging(batch=0, tokens=0)) == 0
