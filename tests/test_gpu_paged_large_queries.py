"""Queries near the end of fp32's range, with a scale that makes their scores ordinary ones."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import sdpa_paged
from test_gpu_paged import TINY, _cache, _heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N", [1, 3, 8, 40])                   # 4 heads share keys: products of 8, 16 and 32 rows, tiles of 128
@pytest.mark.parametrize("size", [116, 117, 118, 119, 120])
@pytest.mark.parametrize("lengths", [[700, 40], [9000, 40]])   # (long: in parts that are added afterwards)
def test_their_scores_keep_their_size(bits, N, size, lengths):
    """The elements are below 4 * 2^size and the sums of 64 products with keys of N(0, 1), some eight times that, below 2^127."""
    D = 64
    seqs = R.Sequences(lengths, 32)
    cache = _cache(seqs, 2, D, torch.bfloat16, bits)
    q = _heads((2, 8, N, D), torch.bfloat16, 5).clamp(-3.5, 3.5) * 2.0 ** size
    scale = 2.0 ** (-size - 3)
    want, bound = R.attention(q, cache, seqs, scale=scale, unpacked=bits == 4 and N == 40)     # (160 rows of 4 bits)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, scale=scale), want, bound, TINY[torch.bfloat16])
