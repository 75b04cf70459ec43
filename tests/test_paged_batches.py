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
