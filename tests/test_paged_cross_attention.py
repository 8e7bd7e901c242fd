"""Attention without `is_causal`: queries have no position among the keys, so there may be more of them than keys."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import PagedCache, _quantise, sdpa_paged

LENGTHS = [5, 0, 700, 64, 1]


def _compare(device, bits, N, Hq, Hkv, D, dtype, counts):
    seqs = R.Sequences(LENGTHS, 16, device=device)
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(seqs.pages, Hkv, 16, D, generator=gen).to(dtype).to(device) for _ in range(2))
    if bits == 4:
        (k, ks), (v, vs) = (_quantise(t) for t in (k, v))
        cache = PagedCache(k, v, k_scales=ks, v_scales=vs, dtype=dtype)
    else:
        cache = PagedCache(k, v)
    q = torch.randn(len(LENGTHS), Hq, N, D, generator=gen).to(dtype).to(device)
    if counts is not None:
        counts = torch.tensor(counts, dtype=torch.int32, device=device)
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, is_causal=False)
    want, bound = R.attention(q, cache, seqs, counts, is_causal=False, unpacked=bits == 4)
    R.close(out, want, bound, 2.0 ** -25)
    assert not out[1].any()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,counts", [(1, None), (9, None), (9, [9, 9, 9, 0, 5]), (100, None)])
def test_on_the_cpu(bits, N, counts):
    _compare("cpu", bits, N, 4, 2, 32, torch.bfloat16, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,counts", [(1, None), (9, None), (9, [9, 9, 9, 0, 5]), (100, None), (300, [300, 300, 1, 299, 300])])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 2, 64, torch.bfloat16), (16, 16, 128, torch.float16)])
def test_on_the_gpu(bits, N, counts, Hq, Hkv, D, dtype):
    _compare("cuda", bits, N, Hq, Hkv, D, dtype, counts)


def test_causal_calls_keep_their_limit():
    seqs = R.Sequences([5], 16, device="cpu")
    cache = PagedCache.allocate(seqs.pages, 1, 16, 32, device="cpu")
    q = torch.zeros(1, 1, 9, 32, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="out of range"):
        sdpa_paged(q, cache, seqs.table, seqs.lengths)
    with pytest.raises(ValueError, match="out of range"):
        sdpa_paged(q, cache, seqs.table, seqs.lengths, is_causal=False, counts=torch.tensor([10], dtype=torch.int32))
