"""The paged cache's calls on batches of no sequence and of very many."""
from __future__ import annotations

import pytest
import torch

from kea_kernels import paged
from test_paged_attention import DEV, TYPES


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 7, 9, 300, 2000])
def test_attention_of_no_sequence(tokens, dtype):
    """All rows are of no sequence: zeros in a new tensor, left as they are in out."""
    cache = paged.Cache.empty(4, 16, 2, 64, DEV)
    table, none, at = torch.zeros(0, 300, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    q = torch.ones(tokens, 8, 64, dtype=dtype, device=DEV)
    for t in (table, table[:, :0]):
        assert not paged.attention(q, cache, t, none, at).any()
        out = torch.full_like(q, 7.0)
        assert paged.attention(q, cache, t, none, at, out=out) is out
        torch.cuda.synchronize()
        assert bool((out == 7).all())


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("batch", [500, 65535, 65536, 70001, 131071])
def test_very_many_sequences(batch):
    """write, read and attention of one token of each, with offsets and without; every seventh sequence has none, or no page."""
    g = torch.Generator().manual_seed(batch)
    k, v = (torch.randn(batch, 1, 16, generator=g).to(DEV) for _ in range(2))
    table = torch.randperm(batch, generator=g).int()[:, None].to(DEV)
    lengths = torch.ones(batch, dtype=torch.int32, device=DEV)
    table[3::7], lengths[5::7] = -1, 0
    cache = paged.Cache.empty(batch, 16, 1, 16, DEV)
    paged.write(cache, k, v, table, lengths)
    there = (table[:, 0] >= 0) & (lengths > 0)
    page = table[there, 0].long()
    want_k, want_v = (torch.zeros(batch, 1, 16, device=DEV) for _ in range(2))
    want_k[there] = cache.k[page, 0, :1].float() * cache.k_scale[page, 0, :1, None]
    want_v[there] = cache.v[page, 0, :1].float() * cache.v_scale[page, 0, :1, None]
    assert float((want_k[there] - k[there]).abs().max()) < 0.05  # (half a step: 1 / 254 of a row's largest)
    for start in (None, torch.zeros(batch, dtype=torch.int32, device=DEV)):
        got = paged.read(cache, table, lengths, 2, starts=start)
        assert torch.equal(got[0][:, 0], want_k) and torch.equal(got[1][:, 0], want_v) and not got[0][:, 1].any() and not got[1][:, 1].any()
    out = paged.attention(k, cache, table, lengths)
    assert float((out - want_v).abs().max()) < 1e-6 * 5  # (one key: its value, in 22 bits, of numbers below 2^3)
    at = torch.arange(batch + 1, dtype=torch.int32, device=DEV)
    assert torch.equal(paged.attention(k, cache, table, lengths, at), out)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale[page, :, 0], cache.v_scale[page, :, 0])]
    paged.write(cache, k, v, table, lengths, at)
    assert all(torch.equal(x, y) for x, y in zip(before, (cache.k, cache.v, cache.k_scale[page, :, 0], cache.v_scale[page, :, 0])))
