"""int4.pack, Weight and gemm at the ends of their range."""
from __future__ import annotations

import pytest
import torch

from kea_kernels import int4

DEV = "cuda"


@pytest.mark.parametrize("k", [1, 8192, 8193, 1 << 15, 1 << 20])
def test_scales_with_which_a_sum_could_pass_fp32_are_refused(k):
    """16 times a sum (as the kernel holds it) is at most 16 * 128 * 8 k times the largest scale: 2^14 k 2^113 / k = 2^127."""
    w, most = torch.zeros(1, k, dtype=torch.int8), min(2.0**100, 2.0**113 / k)
    below = torch.tensor(most, dtype=torch.float64).to(torch.float32)
    while float(below) > most:
        below = torch.nextafter(below, torch.zeros(()))
    groups = -(-k // 128)
    int4.pack(w, below.expand(1, groups), 128)
    int4.pack(w, -below.expand(1, groups), 128)
    for bad in (below * 1.001, -below * 1.001):
        scales = torch.ones(1, groups)
        scales[0, -1] = bad
        with pytest.raises(ValueError, match="scale"):
            int4.pack(w, scales, 128)


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("m,n,k", [(1, 20, 8192), (3, 17, 1 << 15), (1, 16, 1 << 20), (130, 64, 1 << 15)])
@pytest.mark.parametrize("group", [32, 64, 128, 1024])
def test_the_largest_sums(m, n, k, group):
    """Every product the largest there is: 2^30 2^93 and the like, brought back by the rows' scales."""
    most = min(2.0**100, 2.0**113 / k)
    q, w = torch.full((1, m, k), -128, dtype=torch.int8, device=DEV), torch.full((n, k), -8, dtype=torch.int8, device=DEV)
    p = int4.pack(w, torch.full((n, -(-k // group)), most, device=DEV), group)
    got = int4.gemm(q, torch.full((1, m), 2.0**-100, device=DEV), p)
    assert torch.equal(got, torch.full((m, n), 1024.0 * k * most * 2.0**-100, device=DEV))  # (powers of two: every sum is exact)


def test_groups_far_longer_than_a_row_take_no_memory():
    """A group is any power of two up to 2^30: what a row of 100 does not have is not made."""
    g = torch.Generator().manual_seed(1)
    w, s = torch.randint(-8, 8, (40, 100), generator=g, dtype=torch.int8), torch.rand(40, 1, generator=g)
    assert torch.equal(int4.pack(w, s, 1 << 30).dense(), w.float() * s)


@pytest.mark.gpu
@torch.inference_mode()
def test_layers_of_groups_far_longer_than_a_row():
    g = torch.Generator().manual_seed(2)
    w, x = torch.randn(70, 100, generator=g), torch.randn(5, 100, generator=g).to(DEV)
    long, short = (int4.Int4Linear.from_dense(w, group=group, device=DEV) for group in (1 << 30, 128))
    assert torch.equal(long.weight.dense(), short.weight.dense()) and torch.equal(long.linear(x), short.linear(x))
