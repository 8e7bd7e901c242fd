"""4-bit values over long contexts of like weight: the products' sums must not drift away from results that get smaller and smaller."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import PagedCache, _quantise, sdpa_paged
from test_gpu_paged import TINY, _cache, _heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("n", [8192, 131072, 524288])
@pytest.mark.parametrize("N", [1, 4, 8])                       # of 4 heads: products of 8, 16 and 32 rows
def test_sums_over_long_contexts(D, dtype, n, N):
    """512 sequences over the same pages: every one is more than a CTA's share, a quarter of it a warp's sum.

    With weights p of about 1 / n and values step (c - 7.5) + middle: between two takings of the offset a sum grows to 31 step of
    the weights in 16 products (32 at D = 64), each cut off by 2^-23 of it at most; over all of them 16 * 31 * 2^-23 step.
    What is left are sums about zero: of j of n values of N(0, 1), less than 6 sqrt(j) / n each, so 6 / sqrt(n) at most, over
    n / 64 steps of 2^-23.  Then the weights' parts, 2^-16 of 31 step in a sum of n random ones, 6 / sqrt(n) of it (32 rows: one
    part, 2^-8 of 8 step); the exponential's 2^-21 and the scores' errors (below 2^-18, queries are 0.01 N(0, 1)) of such sums' magnitude,
    of random sign too; the middles' fp32 sums 2^-23 in n / 8 additions of a lane, rounded to nearest: 6 sqrt(n / 8) 2^-24; the result's rounding."""
    seqs = R.Sequences([n], 64)
    cache = _cache(seqs, 1, D, dtype, 4, garbage=False)
    q = 0.01 * _heads((512, 4, N, D), dtype, 3)
    out = sdpa_paged(q, cache, seqs.table.expand(512, -1), seqs.lengths.expand(512))
    k, _ = R.values(cache, "k", seqs, 0, n)
    v, step = R.values(cache, "v", seqs, 0, n)
    root, top = n ** 0.5, float(step.max())
    weight = 2.0 ** -8 * 8 * top if N == 8 else 2.0 ** -16 * 31 * top
    for b, h in ((0, 0), (17, 3), (511, 2)):
        for i in range(N):
            seen = n - N + i + 1
            want = torch.softmax(q[b, h, i].double() @ k[0, :seen].T * D ** -0.5, -1) @ v[0, :seen]
            bound = R.half_step(dtype) * want.abs() + 2.0 ** -23 * ((32 if D == 64 else 16) * 31 * top + n / 64 * 6 / root) \
                + 6 / root * (weight + 2.0 ** -17) + 6 * (n / 8) ** 0.5 * 2.0 ** -24 / root
            R.close(out[b, h, i], want, 1.01 * bound, TINY[dtype])


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("N", [1, 4])
def test_sums_of_rows_with_one_large_element(D, dtype, N):
    """Element 3 of every value row is about 20, so that the codes of the others are small ones: their sums are as far from the middle
    as the offset.  The bound is as above, where a sum is of j values between -1/2 and 15 1/2 steps about the columns' mean: the
    large element's column drifts by n / 64 steps of 2^-23 of its 20, and the others by as much of a step, their mean being off
    the columns' mean by what the large one adds, 20 / D, and their own below 1."""
    n = 131072
    seqs = R.Sequences([n], 64)
    gen = torch.Generator(device="cuda").manual_seed(1)
    k, v = (torch.randn(seqs.pages, 1, 64, D, device="cuda", generator=gen) for _ in range(2))
    v[..., 3] = 20 + 0.1 * v[..., 3]
    (k, ks), (v, vs) = (_quantise(t.to(dtype)) for t in (k, v))
    cache = PagedCache(k, v, k_scales=ks, v_scales=vs, dtype=dtype)
    q = 0.01 * _heads((512, 4, N, D), dtype, 3)
    out = sdpa_paged(q, cache, seqs.table.expand(512, -1), seqs.lengths.expand(512))
    k, _ = R.values(cache, "k", seqs, 0, n)
    v, step = R.values(cache, "v", seqs, 0, n)
    root, top = n ** 0.5, float(step.max())
    for b, h in ((0, 0), (17, 3), (511, 2)):
        for i in range(N):
            seen = n - N + i + 1
            want = torch.softmax(q[b, h, i].double() @ k[0, :seen].T * D ** -0.5, -1) @ v[0, :seen]
            drift = n / 64 * (want.abs() + 20 / D + 1)
            bound = R.half_step(dtype) * want.abs() + 2.0 ** -23 * ((32 if D == 64 else 16) * 31 * top + drift) \
                + 6 / root * (2.0 ** -16 * 31 * top + 2.0 ** -15) + 6 * (n / 8) ** 0.5 * 2.0 ** -24 * 20 / root
            R.close(out[b, h, i], want, 1.01 * bound, TINY[dtype])
