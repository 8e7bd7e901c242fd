"""Sequences whose length or number of new tokens is out of range: reported, and neither read nor written."""

import pytest
import torch

import paged_reference as R
from flashbob_b200 import _lib, ops
from flashbob_b200.paged import PagedCache, append_kv, read_kv, sdpa_paged
from flashbob_b200.rotary import Rotary
from test_gpu_paged import _cache, _heads

pytestmark = pytest.mark.gpu

# (length, new tokens) with room for 112 positions; `more` than the call's N rows
WRONG = [(-1, 0), (113, 1), (113, 0), (1 << 30, 1), ((1 << 31) - 1, 8), (-(1 << 31), 1), (3, 5), (20, -1), (20, -(1 << 31)), (100, "more"), (113, "more")]


def _batch(bits, garbage=False):
    """Three sequences of 100 positions; the middle one's whole row of the page table holds pages of the cache."""
    seqs = R.Sequences([100, 100, 100], 16)
    cache = _cache(seqs, 2, 64, torch.bfloat16, bits, garbage=garbage)
    return seqs, cache, ("k", "v") if bits == 16 else ("k", "v", "k_scales", "v_scales")


def _spoil(seqs, counts, length, count, n):
    seqs.lengths[1] = length
    counts[1] = n + 1 if count == "more" else count


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("length,count", WRONG)
def test_their_rows_are_not_written(bits, length, count):
    seqs, cache, names = _batch(bits)
    twin = PagedCache(cache.k.clone(), cache.v.clone(), **({} if bits == 16 else dict(k_scales=cache.k_scales.clone(), v_scales=cache.v_scales.clone(),
                                                                                       dtype=cache.dtype)))
    k, v = (_heads((3, 2, 8, 64), torch.bfloat16, s) for s in (3, 4))
    counts = torch.tensor([1, 0, 2], dtype=torch.int32, device="cuda")
    append_kv(k, v, twin, seqs.table, seqs.lengths, counts=counts, rotary=Rotary(64))        # nothing new in the middle
    _spoil(seqs, counts, length, count, 8)
    with pytest.raises(_lib.BobSm100Error, match="length"):
        append_kv(k, v, cache, seqs.table, seqs.lengths, counts=counts, rotary=Rotary(64))
    ops.check_device_status()
    for name in names:
        assert torch.equal(getattr(cache, name), getattr(twin, name)), name


def _replayed(call, spoil):
    """The results of a call captured while all is well and replayed after `spoil`."""
    before, ops._CHECK_STATUS = ops._CHECK_STATUS, False        # (waiting for the stream is no part of a graph)
    try:
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        spoil()
        for t in out:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
    finally:
        ops._CHECK_STATUS = before
    with pytest.raises(_lib.BobSm100Error, match="length"):
        ops.check_device_status()
    return out


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N", [1, 8, 40, 300])                 # a few rows, and tiles of them
@pytest.mark.parametrize("length,count", WRONG)
def test_their_attention_is_zero_and_the_others_are_untouched(bits, N, length, count):
    seqs, cache, _ = _batch(bits)
    q = _heads((3, 4, N, 64), torch.bfloat16, 2)
    counts = torch.tensor([1, 0, min(N, 100)], dtype=torch.int32, device="cuda")
    want = sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, rotary=Rotary(64))
    (out,) = _replayed(lambda: (sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, rotary=Rotary(64)),),
                       lambda: _spoil(seqs, counts, length, count, N))
    assert not out[1].any()
    assert torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("length", [-1, 113, 1 << 30, -(1 << 31)])
def test_they_read_as_zeros(bits, length):
    seqs, cache, _ = _batch(bits)
    want = read_kv(cache, seqs.table, seqs.lengths, 100)
    out = _replayed(lambda: read_kv(cache, seqs.table, seqs.lengths, 100), lambda: seqs.lengths[1:2].fill_(length))
    for a, b in zip(out, want):
        assert not a[1].any()
        assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
