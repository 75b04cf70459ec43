"""paged.attention where scales, queries and scores lie far apart, against a softmax in 64 bits.

Bounds as in test_paged_attention, but for what FP16 takes from the weights: the reference of a row's weights stands where the largest
product of a weight and its own key's value scale that the row sees is at least 2^6, and half of FP16's smallest step is 2^-25:
2^-31 max_j(w_j |v_scale_j|) a code. No key enters it by its value scale alone."""
from __future__ import annotations

import math

import pytest
import torch

from kea_kernels import paged
from test_paged_attention import BF16, DEV, F16, F32, HALF_STEP, TYPES, U, on_gpu

ROUNDED = {F32: 2.0**-22, F16: 2.0**-11, BF16: 2.0**-11}


def one_sequence(n, length, heads, hk, d, dtype, g, room=None):
    """q of n new tokens, a cache of `length` positions, its table with room for `room`, and the lengths."""
    pages = -(-length // 16)
    table = torch.full((1, -(-(room or length) // 16)), -1, dtype=torch.int32)
    table[0, :pages] = torch.randperm(pages, generator=g).int()
    ints = [torch.randint(-127, 128, (pages, hk, 16, d), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [torch.full((pages, hk, 16), 0.01) for _ in range(2)]
    return torch.randn(n, heads, d, generator=g).to(dtype), paged.Cache(*ints, *scales), table, torch.tensor([length], dtype=torch.int32)


def place(table, p):
    """Where position p's rows are: the first three indices of a cache's tensors."""
    return table[0].long()[p // 16], slice(None), p % 16


def expected(q, cache, table, lengths, scale=None, exact_scores=False):
    """(the output in 64 bits, how far the kernel's may be from it). exact_scores: the softmax is one key's but for nothing, whatever
    the rounding of scores."""
    (n, heads, d), hk, length = q.shape, cache.kv_heads, int(lengths[0])
    scale = 1 / math.sqrt(d) if scale is None else scale
    at = place(table, torch.arange(length))
    kc, vc, ks, vs = (t[at].double() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))  # [length, hk, ...]
    seen = torch.arange(length) <= torch.arange(length - n, length)[:, None]
    out, err = torch.zeros(n, heads, d, dtype=torch.float64), torch.zeros(n, heads, d, dtype=torch.float64)
    for x in range(heads):
        y = x * hk // heads
        qd, k, v = q[:, x].double(), kc[:, y] * ks[:, y, None], vc[:, y] * vs[:, y, None]
        s, mag = (qd @ k.t()) * scale, (qd.abs() @ k.abs().t()) * abs(scale)
        es = (d + 4) * U * mag + 3 * U * s.abs() + (2.0**-22 * mag if q.dtype == F32 else 0)
        if q.dtype != F16:
            es = es + abs(scale) * 2.0**-29 * qd.abs().amax(1, keepdim=True) * k.abs().sum(1)
        es = torch.zeros(n, 1, dtype=torch.float64) if exact_scores else torch.where(seen, es, 0.0).amax(1, keepdim=True)
        w = torch.softmax(torch.where(seen, s, -math.inf), 1)
        out[:, x] = w @ v
        e = (w @ v.abs()) * (4 * es + (length + 40) * U + ROUNDED[q.dtype]) * 1.05
        err[:, x] = e + 2.0**-31 * (w * vs[:, y].abs()).amax(1, keepdim=True) * (seen.double() @ vc[:, y].abs())
    return out, err + (out.abs() + err) * HALF_STEP[q.dtype] + (2.0**-25 if q.dtype == F16 else 1e-37)


def check(got, want, err):
    got = got.cpu().double()
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / err).max().item()
    assert worst <= 1, f"{worst:.3g} times the bound"


def run(q, cache, table, lengths, **kw):
    return paged.attention(q.to(DEV), on_gpu(cache), table.to(DEV), lengths.to(DEV), **kw)


# (new tokens, length, room of the table): tiles of 32 rows, and of 128 and 256
KERNELS = [(1, 96, None), (5, 200, None), (1000, 1100, 4800)]


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,length,room", KERNELS)
@pytest.mark.parametrize("d", [64, 128])
def test_large_values_without_weight_take_no_digits(d, n, length, room, dtype):
    """One key has all the weight; its neighbours, 2^65 times lighter, have value scales up to 2^34 times its own."""
    g = torch.Generator().manual_seed(d + n)
    q, cache, table, lengths = one_sequence(n, length, 16, 4, d, dtype, g, room)
    q = (torch.randint(0, 2, (1, 1, d), generator=g) * 2.0 - 1).expand(n, 16, d).contiguous().to(dtype)
    cache.k.zero_()
    cache.k[place(table, 40)] = (100 * q[0, :1]).to(torch.int8)
    cache.k_scale.fill_(45 / (100 * math.sqrt(d)))  # (the score is 45, e^45 = 2^65)
    cache.v_scale.fill_(2.0**-10)
    for ratio in (12, 16, 20, 24, 28, 31, 34):
        for p in range(32, 64):
            cache.v_scale[place(table, p)] = 2.0 ** (-10 if p == 40 else ratio - 10 - p % 3)
        check(run(q, cache, table, lengths), *expected(q, cache, table, lengths, exact_scores=True))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,length,room", KERNELS)
@pytest.mark.parametrize("spread", [4, 24, 60])
def test_value_scales_of_every_size_side_by_side(spread, n, length, room, dtype):
    """Each key has a scale of its own, powers of two `spread` apart, zeros among them, and scores that are within some 2^20."""
    g = torch.Generator().manual_seed(spread + n)
    q, cache, table, lengths = one_sequence(n, length, 16, 4, 80, dtype, g, room)
    top = 6 if dtype == F16 else spread / 2
    cache.v_scale.copy_(torch.exp2(top - spread * torch.rand(cache.v_scale.shape, generator=g)))
    check(run(q, cache, table, lengths), *expected(q, cache, table, lengths))
    cache.v_scale[torch.rand(cache.v_scale.shape, generator=g) < 0.2] = 0.0
    check(run(q, cache, table, lengths), *expected(q, cache, table, lengths))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,length,room", [(1, 2500, None), (5, 3000, None), (1000, 1100, 4800)])
def test_values_near_the_largest_numbers(n, length, room, dtype):
    """Values up to 2^127: the light keys, 2^-16 of the heaviest one each, keep their part in the sum; beside them, and in other parts of
    the keys, rows of zeros with the smallest scale; a weight of 2^-130 with a value of 2^127."""
    g = torch.Generator().manual_seed(n)
    q, cache, table, lengths = one_sequence(n, length, 16, 4, 64, dtype, g, room)
    q = (torch.randint(0, 2, (1, 1, 64), generator=g) * 2.0 - 1).expand(n, 16, 64).contiguous().to(dtype)
    towards = (100 * q[0, :1]).to(torch.int8)
    cache.k.zero_()
    cache.k[place(table, 40)] = towards
    cache.k_scale.fill_(11.1 / 800)  # (e^11.1 = 2^16)
    cache.v_scale.fill_(2.0**120)
    check(run(q, cache, table, lengths), *expected(q, cache, table, lengths))
    cache.v_scale.fill_(1e-30)
    check(run(q, cache, table, lengths), *expected(q, cache, table, lengths))
    cache.k.zero_()
    cache.v[:, :, 8:] = 0
    for p in range(32):
        cache.v_scale[place(table, p)] = 2.0**120
    check(run(q, cache, table, lengths), *expected(q, cache, table, lengths))
    cache.v_scale.fill_(2.0**-10)
    cache.k[:] = towards[0]
    cache.k_scale.fill_(90.0 / 800)  # (e^90 = 2^130)
    for p in range(32):
        cache.k[place(table, p)] = 0
        cache.v_scale[place(table, p)] = 2.0**120
    check(run(q, cache, table, lengths), *expected(q, cache, table, lengths))


@pytest.mark.gpu
@torch.inference_mode()
def test_a_sum_of_2_to_the_30_weights():
    """One token of 2^30 positions that share two pages, with the smallest value scale: the first page of every part has the weights 1, all
    others 2^4.5."""
    cache = paged.Cache(*(torch.zeros(2, 1, 1024, 16, dtype=torch.int8, device=DEV) for _ in range(2)), torch.full((2, 1, 1024), 4.5 * math.log(2) / 100, device=DEV),
                        torch.full((2, 1, 1024), 1e-30, device=DEV))
    cache.k[1, ..., 0], cache.v[0], cache.v[1] = 100, 50, 100
    table = torch.ones(1, 1 << 20, dtype=torch.int32, device=DEV)
    table[0, ::1 << 14] = 0
    q = torch.zeros(1, 1, 16, device=DEV)
    q[..., 0] = 1.0
    out = paged.attention(q, cache, table, torch.tensor([1 << 30], dtype=torch.int32, device=DEV), scale=1.0)
    first = 64 / (1 << 20)
    want = 1e-30 * (50 * first + 100 * 2**4.5 * (1 - first)) / (first + 2**4.5 * (1 - first))
    # FP32 sums of equal numbers: of 2^18 blocks a wave, off by half a step each; products and sum, of 16 (32) weights a block
    assert bool(((out.double() - want).abs() <= want * 2 * (2**18 + 40) * U).all())


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,length,room", KERNELS)
def test_scores_of_any_size(n, length, room, dtype):
    """Scores of up to 2^100, one of them the largest by far: its value comes out, whatever its scale and the others' are."""
    g = torch.Generator().manual_seed(n)
    q, cache, table, lengths = one_sequence(n, length, 16, 4, 64, dtype, g, room)
    q = (torch.randint(0, 2, (1, 1, 64), generator=g) * 2.0 - 1).expand(n, 16, 64).contiguous().to(dtype)
    cache.k[:] = (60 * q[0, :1]).to(torch.int8)
    cache.k[place(table, 70)] = (100 * q[0, :1]).to(torch.int8)
    for own, others in ((-10, -10), (-10, 8), (8, -20), (-20, 20), (100, -100), (-90, 100)):
        if dtype == F16 and abs(own) > 10:
            continue
        cache.v_scale.fill_(2.0**others)
        cache.v_scale[place(table, 70)] = 2.0**own
        for scale in (1.0, 2.0**14, 2.0**20, 2.0**30, 2.0**97):
            check(run(q, cache, table, lengths, scale=scale), *expected(q, cache, table, lengths, scale=scale, exact_scores=True))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,length,room", KERNELS)
def test_queries_keys_and_scales_of_every_size(n, length, room, dtype):
    """Powers of two on the queries, the keys' scales and `scale` that cancel: the same scores."""
    g = torch.Generator().manual_seed(n)
    q, cache, table, lengths = one_sequence(n, length, 16, 4, 64, dtype, g, room)
    k_scale = cache.k_scale * torch.exp(0.3 * torch.randn(cache.k_scale.shape, generator=g))
    for of_q, of_k, of_scale in ([(0, 0, 0), (-8, -90, 98), (8, 110, -118), (0, -95, 95), (4, 117, -121), (-6, 8, -2), (0, -64, 64)] if dtype == F16 else
                                 [(0, 0, 0), (-126, 0, 126), (-120, 0, 120), (-138, 120, 18), (-124, 122, 2), (-100, 100, 0), (120, -90, -30), (125, 0, -125),
                                  (100, -96, -4), (90, 30, -120)]):
        cache.k_scale.copy_(k_scale * 2.0**of_k)
        scaled, scale = (q.double() * 2.0**of_q).to(dtype), 2.0 ** (of_scale - 3)
        check(run(scaled, cache, table, lengths, scale=scale), *expected(scaled, cache, table, lengths, scale=scale))


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,length,room", [(6, 200, None), (33, 97, None), (1000, 1100, 4800)])
@pytest.mark.parametrize("spread", [1, 24, 200])
def test_rows_keep_their_bits_beside_keys_that_they_do_not_see(spread, n, length, room, dtype):
    """The last four keys, which the last tokens see, hold NaN, infinities, the largest, smallest and ordinary scales: nothing changes for
    the tokens before them, whatever the other keys' scales are."""
    g = torch.Generator().manual_seed(spread + n)
    q, cache, table, lengths = one_sequence(n, length, 16, 4, 64, dtype, g, room)
    top = 6 if dtype == F16 else min(spread / 2, 100)
    cache.v_scale.copy_(torch.exp2(top - spread * torch.rand(cache.v_scale.shape, generator=g)))
    clean = run(q, cache, table, lengths)
    check(clean, *expected(q, cache, table, lengths))
    for bad in (math.nan, math.inf, 3e38, 2.0**120, 1e-30, 0.0, 1e-45):
        k_scale, v_scale = cache.k_scale.clone(), cache.v_scale.clone()
        for p in range(length - 4, length):
            v_scale[place(table, p)] = bad
            if not 0 < bad < 1e30:
                k_scale[place(table, p)] = bad
        assert torch.equal(run(q, paged.Cache(cache.k, cache.v, k_scale, v_scale), table, lengths)[:-4], clean[:-4]), bad


@pytest.mark.gpu
@torch.inference_mode()
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seed", range(12))
def test_mixtures(seed, dtype):
    """Heads of 16 to 256, value scales of several sizes in runs and alone, scores of several sizes."""
    g = torch.Generator().manual_seed(100 + seed)
    pick = lambda *c: c[int(torch.randint(0, len(c), (1,), generator=g))]  # noqa: E731
    n, length = pick((1, 40), (1, 3000), (7, 700), (40, 333), (1000, 1100))
    room, d = pick(None, 4800), pick(16, 64, 128, 128, 208, 256)
    q, cache, table, lengths = one_sequence(n, length, 16, pick(1, 4, 16), d, dtype, g, room)
    at = place(table, torch.arange(length))
    low, high = (-16, 6) if dtype == F16 else (-140, 118)
    run_of = pick(1, 5, 40, 300)
    power = torch.randint(low, high, (-(-length // run_of), cache.kv_heads), generator=g).repeat_interleave(run_of, 0)[:length]
    if pick(0, 1):  # (most keys alike)
        power = torch.where(torch.rand(power.shape, generator=g) < 0.9, -5, power)
    cache.v_scale[at] = torch.exp2(power.float() + torch.rand(power.shape, generator=g))
    scale = pick(1.0, 0.125, 8.0)
    check(run(q, cache, table, lengths, scale=scale), *expected(q, cache, table, lengths, scale=scale))
