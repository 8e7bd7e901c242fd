"""Tensors that are contiguous and yet start where no 16-byte access may, or have odd strides along dimensions of one entry."""

import pytest
import torch

import paged_reference as R
from flashbob_b200.paged import PagedCache, append_kv, read_kv, sdpa_paged
from flashbob_b200.rotary import Rotary, apply_rotary
from test_gpu_paged import _cache, _heads

pytestmark = pytest.mark.gpu


def _shifted(t):
    """t's values one element into a buffer."""
    out = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    assert out.is_contiguous() and out.data_ptr() % 16
    return out.copy_(t)


def _odd_strides(t):
    """t [1, 1, 1, D] as a row of a wider buffer whose rows have no multiple of 8 elements."""
    out = torch.empty(1, 1, 5, t.shape[3] + 4, dtype=t.dtype, device=t.device)[:, :, :1, : t.shape[3]]
    assert out.is_contiguous() and out.stride(2) % 8 and out.data_ptr() % 16 == 0
    return out.copy_(t)


@pytest.mark.parametrize("form,shape", [(_shifted, (2, 4, 33, 64)), (_shifted, (1, 1, 1, 64)), (_odd_strides, (1, 1, 1, 64))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rotation_and_its_gradient(form, shape, dtype):
    rotary = Rotary(64)
    q, k, uq, uk = (_heads(shape, dtype, s, "bhnd") for s in (1, 2, 3, 4))
    plain = [t.clone().requires_grad_() for t in (q, k)]
    other = [form(t).requires_grad_() for t in (q, k)]
    want, got = apply_rotary(*plain, rotary, offset=9), apply_rotary(*other, rotary, offset=9)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for a, b in zip(torch.autograd.grad(want, plain, (uq, uk)), torch.autograd.grad(got, other, (form(uq), form(uk)))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("form,B,H,N", [(_shifted, 2, 2, 5), (_shifted, 2, 2, 150), (_odd_strides, 1, 1, 1)])
def test_append_and_attention(bits, form, B, H, N):
    D, dtype = 64, torch.bfloat16
    seqs = R.Sequences([200] * B, 16)
    k, v, q = (_heads((B, H, N, D), dtype, s, "bhnd") for s in (1, 2, 3))
    outs = []
    for change in (lambda t: t, form):
        cache = _cache(seqs, H, D, dtype, bits, garbage=False)
        append_kv(change(k), change(v), cache, seqs.table, seqs.lengths, rotary=Rotary(D))
        outs.append((sdpa_paged(change(q), cache, seqs.table, seqs.lengths, rotary=Rotary(D)), sdpa_paged(change(q), cache, seqs.table, seqs.lengths),
                     *read_kv(cache, seqs.table, seqs.lengths, 200)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N", [1, 150])
def test_a_cache_of_one_head_with_a_stride_of_zero_along_it(N):
    seqs = R.Sequences([300], 16)
    plain = _cache(seqs, 1, 64, torch.bfloat16, 16)
    k, v = (torch.as_strided(t, t.shape, (t.stride(0), 0, t.stride(2), 1)) for t in (plain.k, plain.v))
    q = _heads((1, 2, N, 64), torch.bfloat16, 3)
    assert torch.equal(sdpa_paged(q, PagedCache(k, v), seqs.table, seqs.lengths), sdpa_paged(q, plain, seqs.table, seqs.lengths))
