"""The paged cache on the CPU: its plain route against the formulas in 64 bits, and everything that is refused."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import PagedCache, append_kv, read_kv, sdpa_paged
from flashbob_b200.rotary import Rotary


def _filled(lengths, bits, dtype=torch.bfloat16, H=2, D=32, page=16):
    seqs = R.Sequences(lengths, page, device="cpu")
    cache = PagedCache.allocate(seqs.pages, H, page, D, dtype=dtype, bits=bits, device="cpu")
    gen = torch.Generator().manual_seed(4)
    n = max(1, *lengths)
    k, v = (torch.randn(len(lengths), H, n, D, generator=gen).to(dtype) for _ in range(2))
    append_kv(k, v, cache, seqs.table, seqs.lengths, counts=seqs.lengths, rotary=Rotary(D))
    return seqs, cache, k, v


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(), dict(window_size=7), dict(is_causal=False), dict(scale=0.5)])
def test_append_read_and_attention(bits, dtype, kw):
    lengths = [37, 0, 16, 1]
    seqs, cache, k, v = _filled(lengths, bits, dtype)
    for b, n in enumerate(lengths):
        at = torch.arange(n)
        for which, x in (("k", R.turned(k[b, :, :n], at, Rotary(32))), ("v", v[b, :, :n].double())):
            got, step = R.values(cache, which, seqs, b, n)
            off = (got - x).abs()
            # 16 bits: one rounding (and fp32 below it); 4 bits: half a step more
            assert (off <= R.half_step(dtype) * x.abs() + 1e-6 + (0 if step is None else 0.51 * step)).all()
    for t, which in zip(read_kv(cache, seqs.table, seqs.lengths, 40), ("k", "v")):
        for b, n in enumerate(lengths):
            assert not t[b, :, n:].any()
            want, _ = R.values(cache, which, seqs, b, n)
            assert ((t[b, :, :n].double() - want).abs() <= 1.001 * R.half_step(dtype) * want.abs() + 1e-6).all()
    q = torch.randn(4, 6, 5, 32, generator=torch.Generator().manual_seed(9)).to(dtype)
    counts = torch.tensor([5, 0, 2, 1], dtype=torch.int32)
    rotary = None if "is_causal" in kw else Rotary(32)
    want, bound = R.attention(q, cache, seqs, counts, rotary=rotary, **kw)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, rotary=rotary, **kw), want, bound, 2.0 ** -25)


def test_pages_that_are_none_are_refused_within_reach_and_ignored_elsewhere():
    seqs, cache, k, v = _filled([40, 20], 16)
    q, new = torch.zeros(2, 2, 1, 32, dtype=torch.bfloat16), torch.zeros(2, 2, 1, 32, dtype=torch.bfloat16)
    for entry in (-1, seqs.pages, 1 << 30):
        kept, seqs.table[0, 1] = seqs.table[0, 1].clone(), entry
        with pytest.raises(ValueError, match="page table"):
            sdpa_paged(q, cache, seqs.table, seqs.lengths)
        with pytest.raises(ValueError, match="page table"):
            read_kv(cache, seqs.table, seqs.lengths, 40)
        sdpa_paged(q, cache, seqs.table, seqs.lengths, window_size=8)        # keys 32 ... 39
        read_kv(cache, seqs.table, seqs.lengths, 16)
        append_kv(new, new, cache, seqs.table, seqs.lengths)
        seqs.table[0, 1] = kept
        kept, seqs.table[1, 1] = seqs.table[1, 1].clone(), entry
        before = cache.k.clone()
        with pytest.raises(ValueError, match="page table"):
            append_kv(new + 1, new, cache, seqs.table, seqs.lengths)
        assert torch.equal(before, cache.k)                                  # nothing was written
        seqs.table[1, 1] = kept


@pytest.mark.parametrize("length,count", [(-1, 0), (49, 1), (3, 5), (20, -1), (20, 9)])
def test_lengths_and_counts_out_of_range_are_refused(length, count):
    seqs, cache, _, _ = _filled([40, 20], 16)                                # room for 48
    seqs.lengths[0] = length
    counts = torch.tensor([count, 1], dtype=torch.int32)
    x = torch.zeros(2, 2, 8, 32, dtype=torch.bfloat16)
    for call in (lambda: sdpa_paged(x, cache, seqs.table, seqs.lengths, counts=counts), lambda: append_kv(x, x, cache, seqs.table, seqs.lengths, counts=counts)):
        with pytest.raises(ValueError, match="out of range"):
            call()


def test_invalid_caches():
    z = torch.zeros
    good = z(3, 2, 16, 32, dtype=torch.bfloat16)
    codes, scales = z(3, 2, 16, 16, dtype=torch.uint8), z(3, 2, 16, 2)
    PagedCache(good, good.clone())
    PagedCache(codes, codes.clone(), k_scales=scales, v_scales=scales.clone(), dtype=torch.float16)
    for args, kw, error in [
        ((good.float().numpy(), good), {}, TypeError), ((good, good[0]), {}, ValueError), ((good, good[:2]), {}, ValueError),
        ((good, good.half()), {}, TypeError), ((good.float(), good.float()), {}, TypeError), ((good, good), dict(dtype=torch.float16), TypeError),
        ((good[:0], good[:0]), {}, ValueError), ((z(3, 2, 24, 32).bfloat16(),) * 2, {}, ValueError), ((z(3, 2, 8, 32).bfloat16(),) * 2, {}, ValueError),
        ((z(3, 2, 16, 48).bfloat16(),) * 2, {}, ValueError), ((good.clone().requires_grad_(), good), {}, ValueError),
        ((z(3, 2, 16, 36).bfloat16()[..., :32],) * 2, {}, ValueError), ((z(3, 2, 16, 64).bfloat16()[..., ::2],) * 2, {}, ValueError),
        ((good[:1].expand(3, 2, 16, 32), good), {}, ValueError), ((good, good), dict(k_scales=scales), ValueError),
        ((good, good), {}, ValueError), ((codes, codes.clone()), dict(k_scales=scales, v_scales=scales, dtype=torch.float16), ValueError),
        ((good, good), dict(k_scales=scales, v_scales=scales), TypeError), ((codes, codes), {}, TypeError),
        ((codes, codes), dict(k_scales=scales, v_scales=scales), TypeError),
        ((codes, codes), dict(k_scales=scales.half(), v_scales=scales.half(), dtype=torch.float16), TypeError),
        ((codes, codes), dict(k_scales=scales[:2], v_scales=scales, dtype=torch.float16), ValueError),
    ]:
        with pytest.raises(error):
            PagedCache(*args, **kw)
    with pytest.raises(ValueError):
        PagedCache.allocate(3, 2, 16, 32, bits=8, device="cpu")
    with pytest.raises(TypeError):
        PagedCache.allocate(3, 2, 16.0, 32, device="cpu")
    with pytest.raises(TypeError):
        PagedCache.allocate(3, 2, 16, 32, dtype=torch.float32, device="cpu")
    cache = PagedCache.allocate(3, 2, 16, 32, bits=4, device="cpu")
    assert (cache.pages, cache.kv_heads, cache.page_size, cache.head_dim, cache.bits) == (3, 2, 16, 32, 4)


def test_invalid_calls():
    seqs, cache, _, _ = _filled([40, 20], 16)
    x, t, n = torch.zeros(2, 2, 3, 32, dtype=torch.bfloat16), seqs.table, seqs.lengths
    counts = torch.ones(2, dtype=torch.int32)
    for call, error in [
        (lambda: append_kv(x, x, "cache", t, n), TypeError), (lambda: append_kv(x, x[:, :, :2], cache, t, n), ValueError),
        (lambda: append_kv(x[:, :1], x[:, :1], cache, t, n), ValueError), (lambda: append_kv(x.half(), x.half(), cache, t, n), TypeError),
        (lambda: append_kv(x[..., :16], x[..., :16], cache, t, n), ValueError), (lambda: append_kv(x, x, cache, t.long(), n), TypeError),
        (lambda: append_kv(x, x, cache, t, n.long()), TypeError), (lambda: append_kv(x, x, cache, t, n.tolist()), TypeError),
        (lambda: append_kv(x, x, cache, t, n[:1]), ValueError), (lambda: append_kv(x, x, cache, t[:1], n), ValueError),
        (lambda: append_kv(x, x, cache, t[0], n), ValueError), (lambda: append_kv(x, x, cache, t[:, :0], n), ValueError),
        (lambda: append_kv(x, x, cache, t, n, counts=counts.long()), TypeError), (lambda: append_kv(x, x, cache, t, n, counts=counts[:1]), ValueError),
        (lambda: append_kv(x, x, cache, t, n, counts=3), TypeError), (lambda: append_kv(x, x, cache, t, n, rotary=Rotary(64)), ValueError),
        (lambda: append_kv(x, x, cache, t, n, rotary=1), TypeError), (lambda: append_kv(x[:, :, :0], x[:, :, :0], cache, t, n), ValueError),
        (lambda: append_kv(x.clone().requires_grad_(), x, cache, t, n), NotImplementedError),
        (lambda: sdpa_paged(x[:, :1], cache, t, n), ValueError), (lambda: sdpa_paged(x.repeat(1, 33, 1, 1), cache, t, n), NotImplementedError),
        (lambda: sdpa_paged(x.clone().requires_grad_(), cache, t, n), NotImplementedError), (lambda: sdpa_paged(x, cache, t, n, scale=0.0), ValueError),
        (lambda: sdpa_paged(x, cache, t, n, scale="1"), TypeError), (lambda: sdpa_paged(x, cache, t, n, window_size=-1), ValueError),
        (lambda: sdpa_paged(x, cache, t, n, window_size=1.0), TypeError), (lambda: sdpa_paged(x, cache, t, n, is_causal=1), TypeError),
        (lambda: sdpa_paged(x, cache, t, n, is_causal=False, window_size=3), NotImplementedError),
        (lambda: sdpa_paged(x, cache, t, n, is_causal=False, rotary=Rotary(32)), ValueError), (lambda: sdpa_paged(x[0], cache, t, n), ValueError),
        (lambda: sdpa_paged(x[:1], cache, t, n), ValueError), (lambda: read_kv(cache, t, n, 0), ValueError), (lambda: read_kv(cache, t, n, 2.0), TypeError),
        (lambda: read_kv(cache, t, n, True), TypeError), (lambda: read_kv(x, t, n, 4), TypeError),
    ]:
        with pytest.raises(error):
            call()
    with torch.no_grad():
        sdpa_paged(x.clone().requires_grad_(), cache, t, n)
