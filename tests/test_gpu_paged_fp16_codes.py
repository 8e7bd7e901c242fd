"""An fp16 cache in 4 bits keeps fp16's bits: up to 64 rows only the result is rounded, as up to 16 rows elsewhere."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import sdpa_paged
from flashbob_b200.rotary import Rotary
from test_paged_two_parts import TINY, _call, expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("N,Hq,Hkv", [(17, 1, 1), (5, 4, 1), (5, 28, 4), (16, 2, 2), (11, 3, 1), (8, 32, 4), (2, 32, 1), (63, 2, 2), (64, 1, 1)])
@pytest.mark.parametrize("turn", [False, True])
def test_up_to_64_rows(D, N, Hq, Hkv, turn):
    rotary = Rotary(D) if turn else None
    q, cache, seqs = _call("cuda", 4, torch.float16, D, N, Hq, Hkv, rotary, B=8)
    want, bound = expected(q, cache, seqs, rotary)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, rotary=rotary), want, bound, TINY[torch.float16])
