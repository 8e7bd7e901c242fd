"""Up to 16 rows only the result of the paged attention is rounded to 16 bits: turned queries and probabilities are held in two parts.

Sequences of a few keys whose values nearly cancel: the result is small against its terms, so that its own rounding no longer
hides one of a probability or of a query."""

import math

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import PagedCache, append_kv, sdpa_paged
from flashbob_b200.rotary import Rotary

TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def _call(device, bits, dtype, D, N, Hq, Hkv, rotary, B=24):
    """(q, cache, sequences): B sequences of N + 1 to N + 3 keys; half of the values nearly the negative of the others."""
    gen = torch.Generator().manual_seed(0)
    lengths = [N + 1 + b % 3 for b in range(B)]
    seqs = R.Sequences(lengths, 16, device=device)
    cache = PagedCache.allocate(seqs.pages, Hkv, 16, D, dtype=dtype, bits=bits, device=device)
    n = max(lengths)
    k = torch.randn(B, Hkv, 1, D, generator=gen) + 0.05 * torch.randn(B, Hkv, n, D, generator=gen)         # nearly one key
    v = torch.randn(B, Hkv, 1, D, generator=gen) * torch.tensor([1.0, -1.0]).repeat(n)[:n, None] * (1 + 0.02 * torch.randn(B, Hkv, n, 1, generator=gen))
    k, v = (t.to(dtype).to(device) for t in (k, v))
    append_kv(k, v, cache, seqs.table, seqs.lengths, counts=seqs.lengths, rotary=rotary)
    q = (2 * torch.randn(B, Hq, N, D, generator=gen)).to(dtype).to(device)
    return q, cache, seqs


def _rounded(x, dtype):
    return x.to(dtype).double()


def expected(q, cache, seqs, rotary, lost=None):
    """(out, bound) in 64 bits.  lost: "probabilities" or "queries" rounded once to 16 bits, as a kernel without second parts has them.

    u: half a step of the type.  Two parts leave u^2 of a value (fp16 also 2^-25, half the smallest number, of a query's
    element; of a probability, which is 1 where the reference is, 2^-25 too).  A turned element is off by the angle, 4.3e-7 at most, the sine's and the cosine's
    4.3e-7 and 4e-7 and fp32 roundings: 2^-19 of |a| + |b| covers them.  That moves a score by scale err . |k|; the score's own fp32 sum by
    (D / 16 + 4) 2^-23 of its sum of magnitudes, in 4 bits of those that the scale and the zero enter with.  The exponential, with its
    argument's rounding, 2^-21 and 2^-23 of the argument.  Sums of n / 16 + 16 steps of 2^-23.  4 bits: probability times scale is two bf16 parts,
    2^-16 of it, and meets codes of 16 to 31; the zero and 7.5 scales are added in fp32.  Then the result's rounding.
    """
    B, Hq, N, D = q.shape
    G, tau, u = Hq // cache.kv_heads, D ** -0.5, R.half_step(q.dtype)
    four = cache.bits == 4
    up = 2.0 ** -8 if four else u
    floor = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n = int(seqs.lengths[b])
        k, _ = R.values(cache, "k", seqs, b, n)
        v, vstep = R.values(cache, "v", seqs, b, n)
        kmag, vmag = k.abs(), v.abs()
        if four:
            ks, vs = (seqs.rows(getattr(cache, w + "_scales"), b, n).double() for w in ("k", "v"))
            kmag = 15 * ks[..., :1] + ks[..., 1:].abs()
            vmag = 38.5 * vs[..., :1] + vs[..., 1:].abs()
        position = torch.arange(n - N, n, device=q.device)
        keep = position[:, None] >= torch.arange(n, device=q.device)
        x = R.turned(q[b], position, rotary)
        err = u * u * x.abs() + floor
        if four:
            err = err + 2.0 ** -22 * x.abs() + 2.0 ** -38 * x.abs().amax(-1, keepdim=True)
        if rotary is not None:
            assert not rotary.interleaved and rotary.rotary_dim == D
            a = q[b].double().abs()
            err = err + 2.0 ** -19 * (a + a.roll(D // 2, -1))
        if lost == "queries":
            x = _rounded(x, q.dtype)
        for h in range(Hq):
            kh, vh, km, vm = k[h // G], v[h // G], kmag[h // G].expand(n, D), vmag[h // G].expand(n, D)
            s = (x[h] @ kh.T * tau).masked_fill(~keep, -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            p = e / e.sum(-1, keepdim=True)
            if lost == "probabilities":
                if four:
                    weight = e * vstep[h // G].T                     # what the codes, from 16 on, are multiplied by
                    codes = (vh - vs[h // G][:, 1:]) / vs[h // G][:, :1]
                    out[b, h] = (e @ vh + (_rounded(weight, torch.bfloat16) - weight) @ (16 + codes)) / e.sum(-1, keepdim=True)
                else:
                    out[b, h] = _rounded(e, q.dtype) @ vh / e.sum(-1, keepdim=True)
            else:
                out[b, h] = p @ vh
            d = tau * (err[h] @ kh.abs().T) + (D / 16 + 4) * 2.0 ** -23 * tau * (x[h].abs() @ km.T) + 2.0 ** -21
            d = d + 2.0 ** -23 * (s - s.amax(-1, keepdim=True)).abs()
            d = d.masked_fill(~keep, 0.0).amax(-1, keepdim=True)
            mag = p @ vm
            bound[b, h] = 1.01 * (u * out[b, h].abs() + (up * up + (n / 16 + 16) * 2.0 ** -23) * mag + floor * (keep.double() @ vm)
                                  + torch.expm1(2 * d) * (p @ vh.abs() + out[b, h].abs()))
    return out, bound


FORMS = [(1, 4, 1), (1, 8, 8), (2, 4, 1), (3, 4, 1), (2, 8, 1), (16, 2, 2)]        # new tokens, heads: products of 8 rows, and of 16


# (not fp16 queries over 4 bits: what their second part holds is less than what a probability's two bf16 parts lose)
@pytest.mark.parametrize("lost,dtype,bits", [("probabilities", torch.bfloat16, 16), ("probabilities", torch.float16, 16), ("probabilities", torch.bfloat16, 4),
                                             ("probabilities", torch.float16, 4), ("queries", torch.bfloat16, 16), ("queries", torch.float16, 16),
                                             ("queries", torch.bfloat16, 4)])
def test_the_bound_notices_a_part_that_is_lost(lost, dtype, bits):
    rotary = Rotary(64)
    q, cache, seqs = _call("cpu", bits, dtype, 64, 1, 4, 1, rotary, B=60)
    want, bound = expected(q, cache, seqs, rotary)
    with pytest.raises(AssertionError, match="off, by up to"):
        R.close(expected(q, cache, seqs, rotary, lost=lost)[0].to(dtype), want, bound, TINY[dtype])
    R.close(want.to(dtype), want, bound, TINY[dtype])


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("N,Hq,Hkv", FORMS)
def test_on_the_cpu(bits, N, Hq, Hkv):
    q, cache, seqs = _call("cpu", bits, torch.bfloat16, 64, N, Hq, Hkv, Rotary(64))
    want, bound = expected(q, cache, seqs, Rotary(64))
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, rotary=Rotary(64)), want, bound, TINY[torch.bfloat16])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("N,Hq,Hkv", FORMS)
@pytest.mark.parametrize("turn", [False, True])
def test_on_the_gpu(bits, dtype, D, N, Hq, Hkv, turn):
    rotary = Rotary(D) if turn else None
    q, cache, seqs = _call("cuda", bits, dtype, D, N, Hq, Hkv, rotary)
    want, bound = expected(q, cache, seqs, rotary)
    R.close(sdpa_paged(q, cache, seqs.table, seqs.lengths, rotary=rotary), want, bound, TINY[dtype])
