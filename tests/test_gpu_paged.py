"""Appending to the paged cache, reading it back and attention over it, against the formulas in 64 bits."""

import math

import pytest
import torch

import paged_reference as R
from flashbob_b200 import _lib, ops
from flashbob_b200.interface import sdpa_bob
from flashbob_b200.paged import PagedCache, _quantise, append_kv, read_kv, sdpa_paged
from flashbob_b200.rotary import Rotary, apply_rotary

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def _cache(seqs, heads, D, dtype, bits, seed=0, garbage=True):
    """A cache whose sequences hold N(0, 1) rows and everything else, behind a sequence and in unused pages, NaN."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    k, v = (torch.randn(seqs.pages, heads, seqs.page_size, D, device="cuda", generator=gen).to(dtype) for _ in range(2))
    if bits == 4:
        (k, ks), (v, vs) = (_quantise(t) for t in (k, v))
        cache = PagedCache(k, v, k_scales=ks, v_scales=vs, dtype=dtype)
    else:
        cache = PagedCache(k, v)
    if garbage:
        keep = torch.zeros(seqs.pages, seqs.page_size, dtype=torch.bool, device="cuda")
        for b, n in enumerate(seqs.lengths.tolist()):
            at = torch.arange(n, device="cuda")
            keep[seqs.table[b].long()[at // seqs.page_size], at % seqs.page_size] = True
        for t in ((cache.k, cache.v) if bits == 16 else (cache.k_scales, cache.v_scales)):
            t.masked_fill_(~keep[:, None, :, None], math.nan)
    return cache


def _heads(shape, dtype, seed, layout="bnhd"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, N, D = shape
    if layout == "bnhd":
        return torch.randn(B, N, H, D, device="cuda", generator=gen).to(dtype).transpose(1, 2)
    return torch.randn(shape, device="cuda", generator=gen).to(dtype)


def _check(lengths, counts, N, Hq, Hkv, D, dtype, bits, page, **kw):
    seqs = R.Sequences(lengths, page, seed=len(lengths))
    cache = _cache(seqs, Hkv, D, dtype, bits)
    q = _heads((len(lengths), Hq, N, D), dtype, 5)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, **kw)
    assert out.is_contiguous() and out.dtype == dtype and out.shape == q.shape
    want, bound = R.attention(q, cache, seqs, counts, **kw)
    R.close(out, want, bound, TINY[dtype])
    return q, cache, seqs, counts, out


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,page", [(32, 16), (64, 32), (128, 16), (128, 256)])
@pytest.mark.parametrize("lengths", [[1], [0, 17, 0, 64, 65, 0], [700, 3, 1500, 33]])
def test_one_new_token_per_sequence(bits, dtype, D, page, lengths):
    counts = [min(n, 1) for n in lengths]
    _check(lengths, counts, 1, 8, 2, D, dtype, bits, page, rotary=Rotary(D))


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (7, 1), (6, 2), (32, 1), (16, 2), (40, 2)])
@pytest.mark.parametrize("N", [1, 3])
def test_groups_of_heads(bits, Hq, Hkv, N):
    _check([130, 1030], None, N, Hq, Hkv, 64, torch.bfloat16, bits, 16)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,counts", [(2, [2, 1, 0]), (5, [5, 3, 1]), (33, [33, 7, 32]), (130, [129, 1, 130]), (257, [200, 5, 257])])
@pytest.mark.parametrize("kw", [dict(), dict(window_size=1), dict(window_size=40), dict(is_causal=False), dict(scale=0.3)])
@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_several_new_tokens(bits, N, counts, kw, D, dtype):
    rotary = None if kw.get("is_causal") is False else Rotary(D, rotary_dim=D // 2, interleaved=D == 64)
    lengths = [max(200, N), 5, 1111]
    _check(lengths, [min(n, c) for n, c in zip(lengths, counts)], N, 8, 2, D, dtype, bits, 32, rotary=rotary, **kw)


@pytest.mark.parametrize("page", [16, 64, 128, 1024])
@pytest.mark.parametrize("kw", [dict(), dict(window_size=100), dict(is_causal=False)])
@pytest.mark.parametrize("D,dtype", [(32, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16)])
def test_chunks_over_pages_of_every_size(page, kw, D, dtype):
    """More rows than fit a tile, sequences that end inside, at and behind one, more items than SMs."""
    lengths, counts = [1300, 128, 129, 700, 0, 257, 640], [300, 128, 1, 129, 0, 256, 0]
    _check(lengths, counts, 300, 8, 4, D, dtype, 16, page, **kw)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("D", [32, 128])
def test_whole_prompts(bits, D):
    """Every row is new: the first one sees one key."""
    lengths = [300, 1, 129]
    _check(lengths, lengths, 300, 4, 1, D, torch.bfloat16, bits, 16, rotary=Rotary(D))


@pytest.mark.parametrize("bits", [16, 4])
def test_many_sequences_and_long_ones(bits):
    """More sequences than a warp has lanes, and one that takes most of the work."""
    lengths = [(37 * i) % 90 for i in range(70)]
    lengths[41] = 20000
    _check(lengths, [min(n, 1) for n in lengths], 1, 4, 2, 64, torch.bfloat16, bits, 64)


@pytest.mark.parametrize("bits", [16, 4])
def test_one_long_sequence_in_many_parts(bits):
    _check([40000], None, 1, 8, 1, 128, torch.float16, bits, 128, rotary=Rotary(128, scaling="yarn", factor=8.0, original_length=4096))


@pytest.mark.parametrize("rotary", [dict(rotary_dim=2), dict(rotary_dim=6), dict(rotary_dim=12, interleaved=True), dict(rotary_dim=16), dict(rotary_dim=64),
                                    dict(rotary_dim=50), dict(rotary_dim=24), dict(scaling="linear", factor=2.0), dict(scaling="ntk", factor=4.0, interleaved=True)])
@pytest.mark.parametrize("bits", [16, 4])
def test_forms_of_rotation_in_append_and_attention(rotary, bits):
    D, dtype = 64, torch.float16
    rotary = Rotary(D, **rotary)
    lengths, counts = [90, 40, 257], [3, 40, 0]
    seqs = R.Sequences(lengths, 32)
    cache = _cache(seqs, 2, D, dtype, bits)
    _append_and_compare(cache, seqs, counts, 40, dtype, rotary)
    q = _heads((3, 4, 40, D), dtype, 8)
    c = torch.tensor(counts, dtype=torch.int32, device="cuda")
    want, bound = R.attention(q, cache, seqs, c, rotary=rotary)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=c, rotary=rotary), want, bound, TINY[dtype])


def _check_codes(cache, which, seqs, b, n, c, rows):
    """The last c rows of a sequence are the 16-bit `rows` in 4 bits: bit by bit those of plain fp32 arithmetic, whose step is
    off by 2^-24 and whose quotient, of at most 15, by 2^-24 more: half a step and 15 * 2^-23 of one from the row at most."""
    codes, scales = _quantise(rows)
    assert torch.equal(seqs.rows(getattr(cache, which), b, n)[:, n - c :], codes)
    assert torch.equal(seqs.rows(getattr(cache, which + "_scales"), b, n)[:, n - c :], scales)
    got, step = R.values(cache, which, seqs, b, n)
    assert ((got[:, n - c :] - rows.double()).abs() <= step[:, n - c :] * (0.5 + 15 * 2.0 ** -23) + 2.0 ** -149).all()


def _append_and_compare(cache, seqs, counts, N, dtype, rotary, layout="bnhd"):
    k, v = (_heads((len(counts), cache.kv_heads, N, cache.head_dim), dtype, s, layout) for s in (11, 12))
    for b, c in enumerate(counts):
        k[b, :, c:] = math.nan                                   # padding is not looked at
        v[b, :, c:] = math.nan
    names = ("k", "v") if cache.bits == 16 else ("k", "v", "k_scales", "v_scales")
    before = {n: getattr(cache, n).clone() for n in names}
    append_kv(k, v, cache, seqs.table, seqs.lengths, counts=torch.tensor(counts, dtype=torch.int32, device="cuda"), rotary=rotary)
    new = torch.zeros(seqs.pages, seqs.page_size, dtype=torch.bool, device="cuda")
    u = R.half_step(dtype)
    for b, c in enumerate(counts):
        n = int(seqs.lengths[b])
        at = torch.arange(n - c, n, device="cuda")
        new[seqs.table[b].long()[at // seqs.page_size], at % seqs.page_size] = True
        for which, x in (("k", k[b, :, :c]), ("v", v[b, :, :c])):
            got, _ = R.values(cache, which, seqs, b, n)
            got = got[:, n - c :]
            want = R.turned(x, at, rotary) if which == "k" else x.double()
            if cache.bits == 16:
                # one rounding; in fp32 three more per element of a turned pair, of at most |a| + |b|
                exact = want.to(dtype).double()
                if which == "v":
                    assert torch.equal(got, exact)
                else:
                    pair = x.double().abs().amax(-1, keepdim=True) * 2 * (1 if rotary is None else rotary.attention_factor)
                    R.close(got, want, u * want.abs() + 4 * 2.0 ** -24 * pair, TINY[dtype])
            elif c:
                _check_codes(cache, which, seqs, b, n, c, want.to(dtype))
    same = ~new[:, None, :, None]
    for n in names:
        a, b_ = getattr(cache, n), before[n]
        assert torch.equal(torch.where(same, a, torch.zeros_like(a)).nan_to_num(7.0) if a.is_floating_point() else torch.where(same, a, 0),
                           torch.where(same, b_, torch.zeros_like(b_)).nan_to_num(7.0) if a.is_floating_point() else torch.where(same, b_, 0)), n


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("counts,N", [([1, 1, 1, 1], 1), ([100, 0, 33, 64], 100), ([7, 1, 3, 2], 9)])
def test_append(bits, dtype, D, counts, N):
    lengths = [100, 20, 4000, 64]
    seqs = R.Sequences(lengths, 16)
    cache = _cache(seqs, 3, D, dtype, bits)
    _append_and_compare(cache, seqs, counts, N, dtype, Rotary(D), "bnhd" if N == 9 else "bhnd")


@pytest.mark.parametrize("bits", [16, 4])
def test_append_of_many_rows_takes_several_heads_per_thread(bits):
    seqs = R.Sequences([4001, 3999], 64)
    cache = _cache(seqs, 10, 128, torch.bfloat16, bits, garbage=False)
    _append_and_compare(cache, seqs, [4001, 3998], 4001, torch.bfloat16, Rotary(128))
    k, v = read_kv(cache, seqs.table, seqs.lengths, 4001)
    for b, n in enumerate((4001, 3999)):
        for t, which in ((k, "k"), (v, "v")):
            want, _ = R.values(cache, which, seqs, b, n)
            R.close(t[b, :, :n], want, 1.001 * R.half_step(torch.bfloat16) * want.abs() + 2.0 ** -20, 0)
            assert not t[b, :, n:].any()


def test_rows_of_equal_and_of_extreme_elements_in_4_bits():
    """No range: the step is 1 and the row exact.  Elements at a code's border go to the even code, as in plain arithmetic."""
    D, dtype = 64, torch.float16
    seqs = R.Sequences([6], 16)
    cache = _cache(seqs, 1, D, dtype, 4)
    rows = torch.zeros(6, D)
    rows[0] = -2.5
    rows[1] = 0.0
    rows[2] = torch.arange(D).remainder(31) * 0.5                # steps of 1: every half is a border
    rows[3] = torch.linspace(-65504, 65504, D)
    rows[4, 0], rows[4, 1:] = 6e-8, 0.0                          # the smallest number there is
    rows[5] = torch.linspace(0, 1, D)
    x = rows.to(dtype).cuda().view(1, 1, 6, D)
    append_kv(x, x, cache, seqs.table, seqs.lengths)
    for which in ("k", "v"):
        _check_codes(cache, which, seqs, 0, 6, 6, x[0])
    got, _ = R.values(cache, "v", seqs, 0, 6)
    assert torch.equal(got[0, 0], torch.full((D,), -2.5, dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_row_that_is_not_finite_reads_as_not_finite_and_no_other(value):
    seqs = R.Sequences([40], 16)
    cache = _cache(seqs, 1, 64, torch.bfloat16, 4)
    x = _heads((1, 1, 40, 64), torch.bfloat16, 1, "bhnd").clone()
    x[0, 0, 7, 3] = value
    append_kv(x, x, cache, seqs.table, seqs.lengths)
    for t in read_kv(cache, seqs.table, seqs.lengths, 40):
        bad = ~t[0, 0].isfinite()
        assert bad[7].any() and not bad[:7].any() and not bad[8:].any()


@pytest.mark.parametrize("bits", [16, 4])
def test_other_layouts_of_cache_and_rows(bits):
    """Pages of [page_size, heads, D] storage, one allocation for keys and values, expanded queries, a strided page table."""
    D, H, dtype = 64, 2, torch.bfloat16
    seqs = R.Sequences([70, 9], 16)
    plain = _cache(seqs, H, D, dtype, bits, garbage=False)
    both = torch.zeros(seqs.pages, 2, 16, H, plain.k.shape[3], dtype=plain.k.dtype, device="cuda")
    kw = {}
    if bits == 4:
        scales = torch.zeros(seqs.pages, 16, H, 2, 2, device="cuda")
        kw = dict(k_scales=scales[:, :, :, 0].transpose(1, 2), v_scales=scales[:, :, :, 1].transpose(1, 2), dtype=dtype)
    other = PagedCache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), **kw)
    for n in ("k", "v") + (("k_scales", "v_scales") if bits == 4 else ()):
        getattr(other, n).copy_(getattr(plain, n))
    k = _heads((2, H, 4, D), dtype, 3)
    v = _heads((2, 1, 4, D), dtype, 4, "bhnd").expand(2, H, 4, D)
    q = _heads((2, 1, 4, D), dtype, 6, "bhnd").expand(2, 6, 4, D)
    wide = torch.full((2, 2 * seqs.table.shape[1]), -1, dtype=torch.int32, device="cuda")
    wide[:, ::2] = seqs.table
    for cache, table in ((plain, seqs.table), (other, wide[:, ::2])):
        append_kv(k, v, cache, table, seqs.lengths, rotary=Rotary(D))
    a = sdpa_paged(q, plain, seqs.table, seqs.lengths, rotary=Rotary(D))
    b = sdpa_paged(q, other, wide[:, ::2], seqs.lengths, rotary=Rotary(D))
    assert torch.equal(a, b)
    for x, y in zip(read_kv(plain, seqs.table, seqs.lengths, 70), read_kv(other, wide[:, ::2], seqs.lengths, 70)):
        assert torch.equal(x, y)
    odd = torch.zeros(2, 6, 4, D + 4, dtype=dtype, device="cuda")[..., :D]       # rows that start at no multiple of 16 bytes
    odd.copy_(q)
    assert torch.equal(sdpa_paged(odd, plain, seqs.table, seqs.lengths, rotary=Rotary(D)), a)


@pytest.mark.parametrize("rotary", [None, Rotary(64)])
def test_many_expanded_queries(rotary):
    seqs = R.Sequences([300, 200], 16)
    cache = _cache(seqs, 2, 64, torch.bfloat16, 16)
    q = _heads((2, 1, 90, 64), torch.bfloat16, 6, "bhnd").expand(2, 4, 90, 64)
    a = sdpa_paged(q, cache, seqs.table, seqs.lengths, rotary=rotary)
    assert torch.equal(a, sdpa_paged(q.contiguous(), cache, seqs.table, seqs.lengths, rotary=rotary))
    want, bound = R.attention(q, cache, seqs, rotary=rotary)
    R.close(a, want, bound, 0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Hq,Hkv,N,lengths", [(14, 2, 33, [900, 0, 40]), (8, 8, 129, [4000]), (32, 1, 3, [50, 777]), (6, 2, 64, [64] * 5), (4, 1, 260, [3000, 260])])
@pytest.mark.parametrize("kw", [dict(), dict(window_size=70), dict(is_causal=False)])
def test_rows_packed_and_keys_divided(bits, Hq, Hkv, N, lengths, kw):
    """Several heads in a tile of rows, a head's keys divided between CTAs, 4-bit caches unpacked: every way through the tiles,
    with sequences without queries and rows behind them."""
    counts = [max(0, min(n, N - 5 * (b % 2))) for b, n in enumerate(lengths)]
    for D, dtype, page in ((64, torch.bfloat16, 16), (128, torch.float16, 256)):
        rotary = None if "is_causal" in kw else Rotary(D, interleaved=D == 64)
        _check(lengths, counts, N, Hq, Hkv, D, dtype, bits, page, rotary=rotary, **kw)


@pytest.mark.parametrize("bits", [16, 4])
def test_many_rows_over_other_layouts_and_freed_pages(bits):
    """Tiles over [page, row, head, element] storage; pages before the window are none any more."""
    D, H, dtype = 64, 2, torch.bfloat16
    seqs = R.Sequences([1000, 150], 32)
    plain = _cache(seqs, H, D, dtype, bits)
    names = ("k", "v") if bits == 16 else ("k", "v", "k_scales", "v_scales")
    turned = [getattr(plain, n).transpose(1, 2).contiguous().transpose(1, 2) for n in names]
    other = PagedCache(*turned[:2], **(dict(k_scales=turned[2], v_scales=turned[3], dtype=dtype) if bits == 4 else {}))
    q = _heads((2, 4, 100, D), dtype, 2)
    want, bound = R.attention(q, plain, seqs, window_size=60, rotary=Rotary(D))
    seqs.table[0, : (1000 - 100 - 59) // 32] = -5
    a = sdpa_paged(q, plain, seqs.table, seqs.lengths, window_size=60, rotary=Rotary(D))
    R.close(a, want, bound, 0)
    assert torch.equal(a, sdpa_paged(q, other, seqs.table, seqs.lengths, window_size=60, rotary=Rotary(D)))


@pytest.mark.parametrize("bits,pages", [(16, 64000), (4, 256000)])
def test_offsets_of_more_than_32_bits(bits, pages):
    """Keys and values of 8.4 GB each: rows written, read and attended to at both ends."""
    D, H, page, lengths = 128, 8, 64, [3000, 65, 700]
    seqs = R.Sequences(lengths, page, extra_pages=pages)
    cache = PagedCache.allocate(seqs.pages, H, page, D, dtype=torch.bfloat16, bits=bits)
    page_bytes = cache.k.stride(0) * cache.k.element_size()
    assert int(seqs.table.max()) * page_bytes > 2 ** 32 > int(seqs.table.clamp(min=0).min()) * page_bytes
    k, v = (_heads((3, H, 3000, D), torch.bfloat16, seed) for seed in (1, 2))
    append_kv(k, v, cache, seqs.table, seqs.lengths, counts=seqs.lengths)
    got = read_kv(cache, seqs.table, seqs.lengths, 3000)
    for which, x, y in (("k", k, got[0]), ("v", v, got[1])):
        for b, n in enumerate(lengths):
            rows, _ = R.values(cache, which, seqs, b, n)
            assert torch.equal(y[b, :, :n], rows.to(y.dtype)) if bits == 4 else torch.equal(y[b, :, :n], x[b, :, :n])
    for N, counts in ((1, [1, 1, 1]), (40, [40, 40, 33])):
        q = _heads((3, 2 * H, N, D), torch.bfloat16, 5)
        counts = torch.tensor(counts, dtype=torch.int32, device="cuda")
        want, bound = R.attention(q, cache, seqs, counts)
        R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts), want, bound, TINY[torch.bfloat16])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,Hq,Hkv,counts,D,dtype", [(1030, 2, 2, [1030, 7, 0, 900], 64, torch.float16), (300, 8, 2, [300, 1, 0, 257], 128, torch.bfloat16), (1100, 1, 1, None, 32, torch.bfloat16)])
@pytest.mark.parametrize("kw", [dict(), dict(window_size=100), dict(is_causal=False)])
@pytest.mark.parametrize("room", [200, 1000])                 # pages that the table has room for: more than are in use
def test_many_rows_over_pages_of_16(bits, N, Hq, Hkv, counts, D, dtype, kw, room):
    lengths = [1500, 40, 0, 1203] if counts else [2000, 1100]
    seqs = R.Sequences(lengths, 16, room=room, seed=3)
    cache = _cache(seqs, Hkv, D, dtype, bits)
    q = _heads((len(lengths), Hq, N, D), dtype, 5)
    counts = None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda")
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts, **kw)
    want, bound = R.attention(q, cache, seqs, counts, unpacked=bits == 4, **kw)
    R.close(out, want, bound, TINY[dtype])


def test_in_inference_mode():
    with torch.inference_mode():
        seqs = R.Sequences([20], 16)
        cache = PagedCache.allocate(seqs.pages, 1, 16, 64)
        x = _heads((1, 1, 20, 64), torch.bfloat16, 1)
        q, k = apply_rotary(x, x, Rotary(64))
        append_kv(x, x, cache, seqs.table, seqs.lengths, rotary=Rotary(64))
        assert torch.equal(read_kv(cache, seqs.table, seqs.lengths, 20)[0], k)
    append_kv(x.clone(), x.clone(), cache, seqs.table, seqs.lengths, rotary=Rotary(64))
    with torch.no_grad():
        out = sdpa_paged(x.clone(), cache, seqs.table, seqs.lengths, rotary=Rotary(64))
    want, bound = R.attention(x, cache, seqs, rotary=Rotary(64))
    R.close(out, want, bound, 0)


def test_pages_shared_between_sequences():
    """Two sequences with a common prefix read the same pages."""
    seqs = R.Sequences([100, 100, 60], 16)
    seqs.table[1, :5] = seqs.table[0, :5]
    seqs.table[2, :] = seqs.table[0, :7]
    cache = _cache(seqs, 2, 64, torch.bfloat16, 16)
    q = _heads((3, 4, 1, 64), torch.bfloat16, 2)
    want, bound = R.attention(q, cache, seqs)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths), want, bound, 0)


@pytest.mark.parametrize("bits", [16, 4])
def test_pages_before_the_window_are_never_looked_at(bits):
    seqs = R.Sequences([1000, 400], 16)
    cache = _cache(seqs, 2, 64, torch.bfloat16, bits)
    q = _heads((2, 4, 3, 64), torch.bfloat16, 2)
    want, bound = R.attention(q, cache, seqs, window_size=100)
    for b, n in enumerate((1000, 400)):
        seqs.table[b, : (n - 3 - 99) // 16] = 1 << 30                            # freed: no pages any more
        page, row = seqs.table[b, (n - 3 - 99) // 16].long(), (n - 3 - 99) % 16  # in the window's first page, before it
        for t in ((cache.k, cache.v) if bits == 16 else (cache.k_scales, cache.v_scales)):
            t[page, :, :row] = math.inf
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, window_size=100), want, bound, 0)


@pytest.mark.parametrize("bits", [16, 4])
def test_scores_of_any_size(bits):
    """A key that takes all the probability, late or early, and scores around -1e4."""
    D, dtype = 64, torch.bfloat16
    seqs = R.Sequences([500, 500, 500], 32)
    cache = _cache(seqs, 1, D, dtype, 16)
    x = _heads((3, 1, 500, D), dtype, 9, "bhnd").clone()
    x[0, 0, 3] *= 40
    x[1, 0, 490] *= 40
    x[2] -= 30
    v = _heads((3, 1, 500, D), dtype, 10, "bhnd")
    if bits == 4:
        cache = PagedCache.allocate(seqs.pages, 1, 32, D, dtype=dtype, bits=4)
    append_kv(x, v, cache, seqs.table, seqs.lengths)
    q = _heads((3, 4, 1, D), dtype, 2).abs() * 4
    want, bound = R.attention(q, cache, seqs, scale=1.0)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, scale=1.0), want, bound, 0)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 40, 2.0 ** 120])
@pytest.mark.parametrize("N", [1, 3, 8, 40, 300])             # 4 heads share keys: products of 8, 16 and 32 rows, tiles of 128
def test_scores_of_any_size_give_the_largest_all_the_weight(bits, size, N):
    """fp32 scores of up to 2^123, whose products with log2 e are not to leave the largest anything but 2^0."""
    D, n, j = 64, 3000, 1234
    seqs = R.Sequences([n], 64)
    x, v = (_heads((1, 1, n, D), torch.bfloat16, seed, "bhnd").clamp(-3, 3) for seed in (9, 10))
    x[0, 0, j, 0] = 8
    cache = PagedCache.allocate(seqs.pages, 1, 64, D, dtype=torch.bfloat16, bits=bits)
    append_kv(x, v, cache, seqs.table, seqs.lengths)
    q = torch.zeros(1, 4, N, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = size
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths)[0]
    rows, step = R.values(cache, "v", seqs, 0, n)
    want = rows[0, j].expand_as(out)
    # 16 bits: the product with 1 is the value.  4 bits: the probability times the scale in two parts of 8 bits, 2^-18, times
    # a code of 16 to 31, and the sums' fp32 roundings, which are smaller; then one rounding of the result.
    # 32 rows of 4 bits: the probability times the scale is one part of 8 bits, off by 2^-9 of it, and meets the code less 8
    # (16 + c - 24, from -8 to 7), with the 8 added in fp32.
    # Tiles: the values are unpacked to 16 bits first, another 2^-9 of theirs.
    parts = 8 * 2.0 ** -9 if N == 8 else 1.01 * 31 * 2.0 ** -17
    more = R.half_step(out.dtype) * want.abs() if N > 16 else 0
    bound = 0 if bits == 16 else R.half_step(out.dtype) * want.abs() + (parts + 2.0 ** -18) * step[0, j] + 1.01 * more
    assert ((out.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N", [1, 3, 8, 40])
@pytest.mark.parametrize("size,scale", [(2.0 ** -120, 1.0), (1.0, 2.0 ** -120), (2.0 ** -60, 2.0 ** -80), (2.0 ** 100, 2.0 ** -100)])
def test_small_queries_and_scales(bits, N, size, scale):
    D = 64
    seqs = R.Sequences([700, 40], 32)
    cache = _cache(seqs, 2, D, torch.bfloat16, bits)
    q = _heads((2, 8, N, D), torch.bfloat16, 5) * size
    want, bound = R.attention(q, cache, seqs, scale=scale, unpacked=bits == 4 and N == 40)     # (160 rows of 4 bits)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, scale=scale), want, bound, TINY[torch.bfloat16])


def test_an_infinite_score_makes_its_row_nan_and_no_other():
    seqs = R.Sequences([300, 300], 16)
    cache = _cache(seqs, 1, 64, torch.bfloat16, 16)
    page, row = seqs.table[0, 33 // 16].long(), 33 % 16
    cache.k[page, 0, row] = 0
    cache.k[page, 0, row, 0] = math.inf
    q = _heads((2, 4, 1, 64), torch.bfloat16, 2).abs()
    q[:, 1::2] = -q[:, 1::2]
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths)
    assert out[0, 0::2].isnan().all() and out[0, 1::2].isfinite().all() and out[1].isfinite().all()


@pytest.mark.parametrize("N", [1, 4, 40])
def test_an_infinite_value_reaches_its_column_and_no_other(N):
    seqs = R.Sequences([300, 300], 16)
    cache = _cache(seqs, 1, 64, torch.bfloat16, 16)
    page, row = seqs.table[0, 33 // 16].long(), 33 % 16
    cache.v[page, 0, row, 5] = -math.inf
    q = _heads((2, 4, N, 64), torch.bfloat16, 2)
    out = sdpa_paged(q, cache, seqs.table, seqs.lengths)
    assert (out[0, ..., 5] == -math.inf).all()
    out[0, ..., 5] = 0
    assert out.isfinite().all()


def test_generation_step_by_step_equals_one_attention_over_the_whole():
    """Prompts, then tokens one at a time, against the operator for contiguous tensors on the whole sequences."""
    B, Hq, Hkv, D, dtype = 3, 8, 2, 64, torch.bfloat16
    prompts, steps = [37, 5, 80], 6
    rotary = Rotary(D, scaling="yarn", factor=2.0, original_length=64)
    total = [n + steps for n in prompts]
    q, k, v = (_heads((B, H, max(total), D), dtype, s) for H, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))
    seqs = R.Sequences(total, 16)
    cache = PagedCache.allocate(seqs.pages, Hkv, 16, D, dtype=dtype)
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    at = [torch.stack([t[b, :, :max(prompts)] for b in range(B)]) for t in (q, k, v)]
    append_kv(at[1], at[2], cache, seqs.table, lengths, counts=lengths, rotary=rotary)
    outs = [sdpa_paged(at[0], cache, seqs.table, lengths, counts=lengths, rotary=rotary)]
    for i in range(steps):
        lengths += 1
        new = [torch.stack([t[b, :, prompts[b] + i : prompts[b] + i + 1] for b in range(B)]) for t in (q, k, v)]
        append_kv(new[1], new[2], cache, seqs.table, lengths, rotary=rotary)
        outs.append(sdpa_paged(new[0], cache, seqs.table, lengths, rotary=rotary))
    tq, tk = apply_rotary(q, k, rotary)
    for b in range(B):
        n = prompts[b]
        whole = sdpa_bob(tq[b : b + 1, :, : total[b]], tk[b : b + 1, :, : total[b]], v[b : b + 1, :, : total[b]], is_causal=True)
        got = torch.cat([outs[0][b, :, :n]] + [o[b] for o in outs[1:]], 1)
        # both round every probability and the result: 2 (2^-8 sum p |v| + 2^-8 |out|), |v| < 5 and the sum's scale 0.8
        torch.testing.assert_close(got.float(), whole[0].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
        assert not outs[0][b, :, n:].any()
    kk, vv = read_kv(cache, seqs.table, lengths, max(total))
    for b in range(B):
        assert torch.equal(kk[b, :, : total[b]], tk[b, :, : total[b]]) and torch.equal(vv[b, :, : total[b]], v[b, :, : total[b]])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("Hq", [8, 64])                     # a few rows of a KV head, and enough for tiles
def test_a_captured_step_follows_lengths_and_pages_and_repeats_bits(bits, Hq):
    B, Hkv, D, dtype = 4, 2, 128, torch.bfloat16
    seqs = R.Sequences([900, 30, 64, 1], 32, room=40)
    cache = _cache(seqs, Hkv, D, dtype, bits, garbage=False)
    rotary = Rotary(D)
    q, k, v = (_heads((B, H, 1, D), dtype, s) for H, s in ((Hq, 1), (Hkv, 2), (Hkv, 3)))

    def step():
        append_kv(k, v, cache, seqs.table, seqs.lengths, rotary=rotary)
        return sdpa_paged(q, cache, seqs.table, seqs.lengths, rotary=rotary)

    before, ops._CHECK_STATUS = ops._CHECK_STATUS, False        # (waiting for the stream is no part of a graph)
    try:
        eager = step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        graph.replay()
        assert torch.equal(captured, eager)
        seqs.lengths.copy_(torch.tensor([3, 29, 60, 500], dtype=torch.int32))
        seqs.table.copy_(torch.randint(0, seqs.pages, seqs.table.shape, dtype=torch.int32))
        # (distinct pages for the new rows)
        for b, n in enumerate((3, 29, 60, 500)):
            seqs.table[b, (n - 1) // 32] = b
            seqs.table[b, : (n - 1) // 32] = torch.arange(4, 4 + (n - 1) // 32, dtype=torch.int32)
        graph.replay()
        got = captured.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step())
        for _ in range(5):
            graph.replay()
            assert torch.equal(captured, got)
    finally:
        ops._CHECK_STATUS = before


def test_two_streams_at_once():
    lengths = [3000, 77, 1024, 9]
    seqs = R.Sequences(lengths, 16)
    caches = [_cache(seqs, 2, 64, torch.float16, bits, seed=bits) for bits in (16, 4)]
    q = _heads((4, 8, 2, 64), torch.float16, 4)
    alone = [sdpa_paged(q, c, seqs.table, seqs.lengths) for c in caches]
    torch.cuda.synchronize()
    before, ops._CHECK_STATUS = ops._CHECK_STATUS, False
    try:
        streams = [torch.cuda.Stream() for _ in caches]
        got = [[], []]
        for _ in range(20):
            for i, (s, c) in enumerate(zip(streams, caches)):
                with torch.cuda.stream(s):
                    got[i].append(sdpa_paged(q, c, seqs.table, seqs.lengths))
        torch.cuda.synchronize()
    finally:
        ops._CHECK_STATUS = before
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])


def test_work_behind_a_call_waits_for_all_of_it():
    """The call's second kernel starts early; what the stream runs next must see every result."""
    seqs = R.Sequences([30000], 64)
    cache = _cache(seqs, 8, 128, torch.bfloat16, 16)
    q = _heads((1, 32, 1, 128), torch.bfloat16, 4)
    lone = R.Sequences([128] * 64, 64)
    small = _cache(lone, 8, 128, torch.bfloat16, 16)
    ql = _heads((64, 8, 1, 128), torch.bfloat16, 4)
    before, ops._CHECK_STATUS = ops._CHECK_STATUS, False
    try:
        for args in ((q, cache, seqs.table, seqs.lengths), (ql, small, lone.table, lone.lengths)):
            want = sdpa_paged(*args)
            torch.cuda.synchronize()
            for _ in range(30):
                assert torch.equal(sdpa_paged(*args) * 1, want)
    finally:
        ops._CHECK_STATUS = before


# ---- what only the GPU can find out ---------------------------------------------------------------------------
# (entries outside the cache and lengths outside the table are skipped by the kernels' own checks)
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("entry", [-1, 1 << 30, -(1 << 31)])
def test_a_page_outside_the_cache_is_reported_and_not_read(bits, entry):
    seqs = R.Sequences([100, 100], 16)
    cache = _cache(seqs, 2, 64, torch.bfloat16, bits, garbage=False)
    q = _heads((2, 4, 1, 64), torch.bfloat16, 2)
    k, v = (_heads((2, 2, 1, 64), torch.bfloat16, s) for s in (3, 4))
    names = ("k", "v") if bits == 16 else ("k", "v", "k_scales", "v_scales")
    for where, call in ((2, lambda: sdpa_paged(q, cache, seqs.table, seqs.lengths)), (2, lambda: read_kv(cache, seqs.table, seqs.lengths, 100)),
                        (6, lambda: append_kv(k, v, cache, seqs.table, seqs.lengths))):
        kept = seqs.table[0, where].clone()
        seqs.table[0, where] = entry
        saved = [getattr(cache, n)[seqs.table[0, 3].long()].clone() for n in names]
        with pytest.raises(_lib.BobSm100Error, match="page table"):
            call()
        assert all(torch.equal(a, getattr(cache, n)[seqs.table[0, 3].long()]) for a, n in zip(saved, names))
        seqs.table[0, where] = kept
    ops.check_device_status()
    want, bound = R.attention(q, cache, seqs)                    # the other sequence's token was appended all the same
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths), want, bound, 0)


@pytest.mark.parametrize("length,count", [(-1, 0), (113, 1), (1 << 30, 1), (3, 5), (20, -1), (20, 9)])
def test_lengths_and_counts_out_of_range_are_reported(length, count):
    seqs = R.Sequences([100, 100], 16)                           # room for 112
    cache = _cache(seqs, 2, 64, torch.bfloat16, 16, garbage=False)
    seqs.table[0] = torch.arange(7, dtype=torch.int32)
    q = _heads((2, 4, 8, 64), torch.bfloat16, 2)
    k, v = (_heads((2, 2, 8, 64), torch.bfloat16, s) for s in (3, 4))
    seqs.lengths[0] = length
    counts = torch.tensor([count, 1], dtype=torch.int32, device="cuda")
    for call in (lambda: sdpa_paged(q, cache, seqs.table, seqs.lengths, counts=counts), lambda: append_kv(k, v, cache, seqs.table, seqs.lengths, counts=counts)):
        with pytest.raises(_lib.BobSm100Error, match="length"):
            call()
    ops.check_device_status()


def test_writes_count_as_changes_of_the_cache():
    seqs = R.Sequences([4], 16)
    cache = PagedCache.allocate(seqs.pages, 1, 16, 32)
    weight = torch.ones((), device="cuda", requires_grad=True)
    y = (weight * cache.k.float()).sum() + (weight * cache.k).sum()
    x = _heads((1, 1, 4, 32), torch.bfloat16, 1)
    append_kv(x, x, cache, seqs.table, seqs.lengths)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
