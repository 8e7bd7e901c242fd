"""Many rows over 4-bit pages under a table with room for far more positions than there are: too many to unpack."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import sdpa_paged
from flashbob_b200.rotary import Rotary
from test_gpu_paged import TINY, _cache, _heads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,Hq,Hkv,counts", [(65, 8, 8, [65, 1, 0, 33]), (130, 8, 8, None), (33, 16, 8, [33, 32, 1, 0]), (20, 24, 8, None), (11, 56, 8, [11, 3, 1, 8])])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("kw", [dict(), dict(window_size=50), dict(is_causal=False)])
def test_many_rows_under_a_table_of_great_room(N, Hq, Hkv, counts, D, dtype, kw):
    lengths = [500, 130, 131, 1040]
    # 2 x 4 sequences x 8 heads x D elements of 2 bytes for every position: over 1 GiB with this room
    room = (1 << 30) // (2 * 4 * Hkv * D * 2) // 16 + 8
    seqs = R.Sequences(lengths, 16, room=room)
    cache = _cache(seqs, Hkv, D, dtype, 4)
    q = _heads((4, Hq, N, D), dtype, 5)
    rotary = None if "is_causal" in kw else Rotary(D)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, rotary=rotary, **kw)
    want, bound = R.attention(q, cache, seqs, counts, rotary=rotary, **kw)
    R.close(out, want, bound, TINY[dtype])
    # (the rows fit the largest products: with less room they are unpacked and take tiles, to the same result within both roundings)
    near = R.Sequences(lengths, 16)
    near.table = seqs.table[:, : near.table.shape[1]].contiguous()
    other = sdpa_paged(q, cache, near.table, seqs.lengths, counts=counts, rotary=rotary, **kw)
    want, more = R.attention(q, cache, seqs, counts, rotary=rotary, unpacked=True, **kw)
    R.close(other, want, more, TINY[dtype])
