"""Rotary positions on the CPU: frequencies, values, gradients, and what is refused."""

import math

import pytest
import torch

import paged_reference as R
from flashbob_b200 import _lib
from flashbob_b200.rotary import Rotary, apply_rotary


@pytest.mark.parametrize("form", [dict(), dict(interleaved=True), dict(rotary_dim=6), dict(rotary_dim=6, interleaved=True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values(form, dtype):
    rotary = Rotary(16, **form)
    gen = torch.Generator().manual_seed(0)
    q, k = torch.randn(2, 4, 9, 16, generator=gen).to(dtype), torch.randn(2, 2, 9, 16, generator=gen).to(dtype)
    for got, x in zip(apply_rotary(q, k, rotary, offset=5), (q, k)):
        want = R.turned(x, torch.arange(5, 14), rotary)
        # one rounding of the result, and in fp32 those of sine, cosine, products and sum
        assert ((got.double() - want).abs() <= R.half_step(dtype) * want.abs() + 6 * 2.0 ** -24 * 2 * x.abs().max()).all()
        assert torch.equal(got[..., rotary.rotary_dim :], x[..., rotary.rotary_dim :])
    positions = torch.tensor([[3], [10]]) + torch.arange(9)
    got, none = apply_rotary(q, None, rotary, positions=positions)
    assert none is None
    assert torch.equal(got[1], apply_rotary(q, None, rotary, offset=10)[0][1])


def test_gradients_of_two_orders_against_differences():
    rotary = Rotary(8, scaling="yarn", factor=2.0, original_length=32)
    x = torch.randn(1, 2, 5, 8, dtype=torch.float32, generator=torch.Generator().manual_seed(1)).requires_grad_()
    u = torch.randn(1, 2, 5, 8, generator=torch.Generator().manual_seed(2)).requires_grad_()
    (g,) = torch.autograd.grad(apply_rotary(x, None, rotary)[0], x, u, create_graph=True)
    want = R.turned(u, torch.arange(5), rotary, inverse=True)
    torch.testing.assert_close(g.detach().double(), want, rtol=1e-6, atol=1e-6)
    d = torch.randn(1, 2, 5, 8, generator=torch.Generator().manual_seed(3))
    (h,) = torch.autograd.grad(g, u, d)
    # the map is linear: y(x + d) - y(x) is its derivative
    torch.testing.assert_close(h, (apply_rotary(x + d, None, rotary)[0] - apply_rotary(x, None, rotary)[0]).detach(), rtol=1e-5, atol=1e-5)


def test_frequencies():
    plain = Rotary(64).frequencies
    assert plain[0] == 1.0 and math.isclose(plain[31], 10000 ** (-62 / 64))
    assert Rotary(64, scaling="linear", factor=4.0).frequencies == tuple(f / 4 for f in plain)
    ntk = Rotary(64, scaling="ntk", factor=4.0).frequencies
    assert ntk[0] == 1.0 and math.isclose(ntk[31], plain[31] / 4)
    yarn = Rotary(64, scaling="yarn", factor=4.0, original_length=4096)
    assert yarn.frequencies[0] == 1.0 and math.isclose(yarn.frequencies[31], plain[31] / 4) and math.isclose(yarn.attention_factor, 0.1 * math.log(4) + 1)
    for i, f in enumerate(yarn.frequencies):
        turns = 4096 * plain[i] / (2 * math.pi)
        assert f == plain[i] if turns > 45 else plain[i] / 4 * 0.999 <= f <= plain[i]
    given = Rotary(64, rotary_dim=4, frequencies=(0.5, -7.0), attention_factor=2.0)
    assert given.frequencies == (0.5, -7.0)


def test_packed_turns_are_fractions_of_a_turn():
    packed = _lib.Rotary.from_buffer_copy(Rotary(128, rotary_dim=8, frequencies=(0.0, math.pi, 2 * math.pi, -math.pi / 2))._packed)
    assert packed.pairs == 4
    for got, want in zip(packed.turns, (0.0, 0.5, 0.0, -0.25)):
        off = (got - int(want * 2 ** 64)) % 2 ** 64
        assert min(off, 2 ** 64 - off) < 2 ** 13            # math.pi itself is off by 1.2e-16


@pytest.mark.parametrize("kw,error", [
    (dict(head_dim=1.5), TypeError), (dict(head_dim=True), TypeError), (dict(head_dim=-4), ValueError), (dict(head_dim=0), ValueError),
    (dict(rotary_dim=0), ValueError), (dict(rotary_dim=7), ValueError), (dict(rotary_dim=130), ValueError), (dict(rotary_dim=66), ValueError),
    (dict(theta=0.0), ValueError), (dict(theta=math.inf), ValueError), (dict(theta="1"), TypeError), (dict(theta=True), TypeError),
    (dict(interleaved=1), TypeError), (dict(scaling="cubic"), ValueError), (dict(factor=0.0), ValueError), (dict(factor=math.nan), ValueError),
    (dict(scaling="yarn", factor=2.0), ValueError), (dict(scaling="yarn", factor=2.0, original_length=0), ValueError),
    (dict(scaling="yarn", factor=2.0, original_length=64, theta=1.0), ValueError), (dict(scaling="ntk", factor=2.0, rotary_dim=2), ValueError),
    (dict(frequencies=(1.0,)), ValueError), (dict(frequencies=[math.nan] * 32), ValueError), (dict(frequencies=[1.0] * 32, scaling="linear"), ValueError),
    (dict(attention_factor=0.0), ValueError), (dict(attention_factor=math.nan), ValueError),
])
def test_invalid_rotations(kw, error):
    with pytest.raises(error):
        Rotary(**{"head_dim": 64, **kw})


def test_invalid_calls():
    r = Rotary(8)
    q, k = torch.randn(2, 4, 5, 8), torch.randn(2, 2, 5, 8)
    for args, kw, error in [
        ((q.numpy(), k, r), {}, TypeError), ((q, k.numpy(), r), {}, TypeError), ((q, k, None), {}, TypeError), ((q, k, "r"), {}, TypeError),
        ((q[0], k, r), {}, ValueError), ((q[:, :, :0], k[:, :, :0], r), {}, ValueError), ((q, k[:, :, :4], r), {}, ValueError),
        ((q, k[:1], r), {}, ValueError), ((q, k.bfloat16(), r), {}, ValueError), ((q.double(), k.double(), r), {}, TypeError),
        ((q, k, Rotary(16)), {}, ValueError), ((q, k, r), dict(offset=-1), ValueError), ((q, k, r), dict(offset=1.0), TypeError),
        ((q, k, r), dict(offset=2 ** 62), ValueError), ((q, k, r), dict(positions=[0, 1, 2, 3, 4]), TypeError),
        ((q, k, r), dict(positions=torch.arange(5.0)), TypeError), ((q, k, r), dict(positions=torch.arange(4)), ValueError),
        ((q, k, r), dict(positions=torch.zeros(1, 5, dtype=torch.int32)), ValueError), ((q, k, r), dict(positions=torch.arange(5), offset=1), ValueError),
    ]:
        with pytest.raises(error):
            apply_rotary(*args, **kw)


def test_transformations_that_would_take_it_for_something_else_are_refused():
    import torch.autograd.forward_ad as fwAD

    r, q = Rotary(8), torch.randn(1, 1, 3, 8)
    with pytest.raises(NotImplementedError):
        torch.func.vmap(lambda x: apply_rotary(x, None, r)[0])(q[None])
    with pytest.raises(NotImplementedError):
        torch.jit.trace(lambda x: apply_rotary(x, None, r)[0], q)
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        apply_rotary(fwAD.make_dual(q, q), None, r)
