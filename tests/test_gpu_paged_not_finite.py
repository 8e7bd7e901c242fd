"""NaN and infinities that a row of the paged attention meets make it NaN, however many rows there are, and reach no other row."""

import math

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import sdpa_paged
from test_gpu_paged import _cache, _heads

pytestmark = pytest.mark.gpu

# a few rows (products of 8, 16 and 32), tiles with their keys divided, packed heads, and tiles that are finished where they are
SHAPES = [(2, 4, 1, 1), (2, 4, 1, 3), (2, 4, 1, 8), (2, 4, 4, 40), (2, 4, 1, 40), (2, 16, 16, 300), (5, 16, 16, 130)]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("B,Hq,Hkv,N", SHAPES)
@pytest.mark.parametrize("what", ["query", "key", "infinite key"])
def test_rows_that_meet_it_are_nan_and_no_others(bits, D, dtype, B, Hq, Hkv, N, what):
    n = 500
    seqs = R.Sequences([n] * B, 32)
    cache = _cache(seqs, Hkv, D, dtype, bits)
    q = _heads((B, Hq, N, D), dtype, 2).abs().contiguous()
    G, at = Hq // Hkv, n - (N + 1) // 2                          # a position that half of the rows see
    bad = torch.zeros(B, Hq, N, dtype=torch.bool, device="cuda")
    if what == "query":
        q[1, 0, N // 2, 3] = math.nan
        bad[1, 0, N // 2] = True
    else:
        page, row = seqs.table[1, at // 32].long(), at % 32
        value = math.nan if what == "key" else math.inf
        if bits == 16:
            cache.k[page, 0, row] = 0
            cache.k[page, 0, row, 5] = value
        else:
            cache.k_scales[page, 0, row, 1] = value              # (the zero, and with it the row)
        bad[1, :G, at - (n - N) :] = True
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths)
    assert torch.equal(out.isnan().any(-1), bad)
    assert out[bad].isnan().all() and out[~bad].isfinite().all()


@pytest.mark.parametrize("B,Hq,Hkv,N", SHAPES)
def test_rows_behind_the_new_ones_are_zero_whatever_their_queries_hold(B, Hq, Hkv, N):
    seqs = R.Sequences([500] * B, 32)
    cache = _cache(seqs, Hkv, 64, torch.bfloat16, 16)
    q = _heads((B, Hq, N, 64), torch.bfloat16, 2).contiguous()
    counts = torch.full((B,), N // 2, dtype=torch.int32, device="cuda")
    q[:, :, N // 2 :] = math.nan
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts)
    assert not out[:, :, N // 2 :].any() and out.isfinite().all()
