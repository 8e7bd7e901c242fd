"""4-bit values near the end of fp32's range: sums of a column are within it, and no sum over columns may leave it."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import PagedCache, _quantise, sdpa_paged
from test_gpu_paged import TINY, _heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [1, 4, 8])                       # of 4 heads: products of 8, 16 and 32 rows
@pytest.mark.parametrize("D", [32, 128])
def test_large_values_stay_finite(N, D):
    """40 keys of weights up to 2^8 and steps of 2^113: 40 * 2^8 * 31 * 2^113 is below 2^127 / 2, and 128 columns of it are not."""
    seqs = R.Sequences([40, 33], 16)
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(seqs.pages, 1, 16, D, device="cuda", generator=gen) for _ in range(2))
    (k, ks), (v, vs) = _quantise(k.bfloat16()), _quantise((v * 2.0 ** 115).clamp(-(2.0 ** 117), 2.0 ** 117).bfloat16())
    cache = PagedCache(k, v, k_scales=ks, v_scales=vs, dtype=torch.bfloat16)
    q = 0.1 * _heads((2, 4, N, D), torch.bfloat16, 1)
    want, bound = R.attention(q, cache, seqs)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths), want, bound, TINY[torch.bfloat16])
