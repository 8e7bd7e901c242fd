"""Rotary positions on the GPU: values, gradients of every order, positions near and far, layouts, captured calls."""

import pytest
import torch

import paged_reference as R
from flashbob_b200 import ops
from flashbob_b200.interface import sdpa_bob
from flashbob_b200.rotary import Rotary, apply_rotary

pytestmark = pytest.mark.gpu

FORMS = [dict(), dict(interleaved=True), dict(rotary_dim=16), dict(rotary_dim=2), dict(rotary_dim=10), dict(rotary_dim=18, interleaved=True), dict(rotary_dim=28), dict(rotary_dim=8),
         dict(scaling="yarn", factor=4.0, original_length=512), dict(scaling="ntk", factor=2.0), dict(scaling="linear", factor=8.0, theta=500.0)]
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}


def _heads(shape, dtype, seed, layout="bhnd", grad=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, N, D = shape
    t = torch.randn((B, N, H, D) if layout == "bnhd" else shape, device="cuda", generator=gen).to(dtype)
    return (t.transpose(1, 2) if layout == "bnhd" else t).requires_grad_(grad)


def _compare(got, x, positions, rotary, inverse=False):
    """One rounding of the result; in fp32 the sine and cosine (2 steps each, and the angle's 2^-30), two products and a
    sum, together below 6 half steps of the pair's two elements, both at most the row's largest."""
    want = torch.stack([R.turned(x[b], positions[b], rotary, inverse) for b in range(x.shape[0])])
    pair = 2 * rotary.attention_factor * x.detach().double().abs().amax(-1, keepdim=True)
    R.close(got.detach(), want, R.half_step(x.dtype) * want.abs() + 6 * 2.0 ** -24 * pair, TINY[x.dtype])
    assert torch.equal(got[..., rotary.rotary_dim :], x[..., rotary.rotary_dim :])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("B,Hq,Hkv,N,layout", [(1, 1, 1, 1, "bhnd"), (3, 5, 2, 77, "bnhd"), (2, 8, 2, 1, "bnhd")])
def test_values(form, dtype, D, B, Hq, Hkv, N, layout):
    rotary = Rotary(D, **form)
    q, k = _heads((B, Hq, N, D), dtype, 1, layout), _heads((B, Hkv, N, D), dtype, 2, layout)
    a, b = apply_rotary(q, k, rotary, offset=1000)
    assert a.is_contiguous() and b.is_contiguous() and a.dtype == dtype
    positions = torch.arange(1000, 1000 + N, device="cuda").expand(B, N)
    _compare(a, q, positions, rotary)
    _compare(b, k, positions, rotary)


@pytest.mark.parametrize("form", [dict(), dict(interleaved=True), dict(rotary_dim=20)])
def test_many_rows_take_several_heads_per_thread(form):
    rotary = Rotary(128, **form)
    q, k = _heads((2, 9, 4099, 128), torch.bfloat16, 1, "bnhd"), _heads((2, 2, 4099, 128), torch.bfloat16, 2, "bnhd")
    for t, x in zip(apply_rotary(q, k, rotary), (q, k)):
        _compare(t, x, torch.arange(4099, device="cuda").expand(2, 4099), rotary)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", ["n", "bn", "strided", "expanded"])
def test_positions(wide, shape):
    rotary = Rotary(64)
    x = _heads((2, 3, 40, 64), torch.float16, 1)
    gen = torch.Generator().manual_seed(3)
    top = 2 ** 31 - 1 if wide == torch.int32 else 2 ** 40
    p = torch.randint(-top if wide == torch.int32 else 0, top, (2, 40), generator=gen).to(wide).cuda()
    p[0, 0] = 0
    if shape == "n":
        p = p[0].contiguous()
    elif shape == "strided":
        p = torch.stack((p, p - p), -1)[..., 0]
    elif shape == "expanded":
        p = p[:1].expand(2, 40)
    got, none = apply_rotary(x, None, rotary, positions=p)
    assert none is None
    # at 2^40 the reference's angle itself is rounded, by 2^-53 of 2^40 radians
    want = torch.stack([R.turned(x[b], p.expand(2, 40)[b], rotary) for b in range(2)])
    pair = 2 * x.double().abs().amax(-1, keepdim=True)
    R.close(got, want, 2.0 ** -11 * want.abs() + (6 * 2.0 ** -24 + 2.0 ** -13) * pair, 2.0 ** -25)
    assert torch.equal(apply_rotary(x, None, rotary, offset=2 ** 61)[0], apply_rotary(x, None, rotary, positions=torch.arange(40, device="cuda") + 2 ** 61)[0])


@pytest.mark.parametrize("form", [dict(), dict(interleaved=True, rotary_dim=32), dict(rotary_dim=12, scaling="yarn", factor=2.0, original_length=128)])
@pytest.mark.parametrize("which", ["both", "q", "k", "one"])
def test_gradients_of_three_orders(form, which):
    """The gradient is the rotation back; its own gradient the rotation, and so on."""
    rotary, D, dtype = Rotary(64, **form), 64, torch.bfloat16
    q, k = _heads((2, 4, 33, D), dtype, 1, "bnhd", which != "k"), _heads((2, 2, 33, D), dtype, 2, "bhnd", which in ("both", "k"))
    positions = (torch.arange(33, device="cuda") * 3 + torch.tensor([[0], [50]], device="cuda")).to(torch.int32)
    a, b = apply_rotary(q, None if which == "one" else k, rotary, positions=positions)
    outs = [(a, q)] if which in ("q", "one") else [(b, k)] if which == "k" else [(a, q), (b, k)]
    if which == "q":
        assert b.grad_fn is None or not k.requires_grad
    ups = [_heads(x.shape, dtype, 10 + i, "bnhd", True) for i, (_, x) in enumerate(outs)]
    first = torch.autograd.grad([t for t, _ in outs], [x for _, x in outs], ups, create_graph=True)
    for g, u in zip(first, ups):
        _compare(g, u, positions.long(), rotary, inverse=True)
    dirs = [_heads(x.shape, dtype, 20 + i, "bhnd", True) for i, (_, x) in enumerate(outs)]
    second = torch.autograd.grad(first, ups, dirs, create_graph=True)
    for g, u in zip(second, dirs):
        _compare(g, u, positions.long(), rotary)
    last = [_heads(x.shape, dtype, 30 + i) for i, (_, x) in enumerate(outs)]
    for g, u in zip(torch.autograd.grad(second, dirs, last), last):
        _compare(g, u, positions.long(), rotary, inverse=True)


def test_gradients_against_differences():
    """<u, y(x + h d)> - <u, y(x - h d)> over 2 h: the map is linear, so only the 16-bit roundings are left."""
    rotary = Rotary(32, interleaved=True)
    x, d, u = (_heads((1, 2, 9, 32), torch.float16, s) for s in (1, 2, 3))
    x = (x * 16).round() / 16
    d = (d * 16).round() / 16                                    # x +- d are exact
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(apply_rotary(leaf, None, rotary)[0], leaf, u)
    plus, minus = (apply_rotary(x + s * d, None, rotary)[0].double() for s in (1, -1))
    got, want = (g.double() * d.double()).sum(), (u.double() * (plus - minus)).sum() / 2
    # 2^-11 of every y and of every element of g
    slack = 2.0 ** -11 * (u.double().abs() * (plus.abs() + minus.abs())).sum() / 2 + 2.0 ** -11 * (g.double().abs() * d.double().abs()).sum()
    assert (got - want).abs() <= slack


def test_expanded_inputs_and_gradients_that_are_missing_or_expanded():
    rotary = Rotary(64)
    base = _heads((1, 1, 20, 64), torch.bfloat16, 1).requires_grad_()
    a, b = apply_rotary(base.expand(3, 4, 20, 64), base.expand(3, 2, 20, 64), rotary)
    a.sum().backward()                                           # an expanded gradient for q, none for k
    one = torch.ones(20, 64, device="cuda")
    want = 12 * R.turned(one, torch.arange(20, device="cuda"), rotary, inverse=True)
    # each of the 12 equal parts is rounded, and so is their sum
    torch.testing.assert_close(base.grad[0, 0].double(), want, rtol=2.0 ** -7, atol=12 * 2.0 ** -22)
    assert torch.equal(a[0, 0], a[2, 3])
    positions = torch.arange(20, device="cuda")
    kept = apply_rotary(base, None, rotary, positions=positions)[0].sum()
    kept.backward()
    with pytest.raises(RuntimeError, match="second time"):       # its positions are released with the graph
        kept.backward()


def test_attention_with_positions_has_second_gradients():
    """A Hessian-vector product through rotation and attention, against both in 64 bits by plain autograd."""
    D, dtype = 64, torch.bfloat16
    rotary = Rotary(D)
    q, k, v = (_heads((1, 2, 96, D), dtype, s, grad=True) for s in (1, 2, 3))
    dirs = [_heads((1, 2, 96, D), dtype, s) for s in (4, 5, 6)]

    def hvp(leaves, rotate, attend, dirs):
        a, b = rotate(leaves[0], leaves[1])
        loss = attend(a, b, leaves[2]).to(torch.float64).square().sum()
        first = torch.autograd.grad(loss, leaves, create_graph=True)
        return torch.autograd.grad(first, leaves, dirs)

    got = hvp((q, k, v), lambda a, b: apply_rotary(a, b, rotary), lambda a, b, c: sdpa_bob(a, b, c, is_causal=True), dirs)
    f = torch.tensor(rotary.frequencies, dtype=torch.float64, device="cuda")
    angle = torch.arange(96, device="cuda").double()[:, None] * f

    def plain(x):
        a, b = x[..., :32], x[..., 32:]
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    def attend(a, b, c):
        s = (a @ b.transpose(-1, -2) / 8).masked_fill(torch.ones(96, 96, dtype=torch.bool, device="cuda").triu(1), -torch.inf)
        return torch.softmax(s, -1) @ c

    wide = tuple(t.detach().double().requires_grad_() for t in (q, k, v))
    want = hvp(wide, lambda a, b: (plain(a), plain(b)), attend, [t.double() for t in dirs])
    for g, w in zip(got, want):
        # operands, first gradients and results are rounded to bf16 on the way: about six roundings of 2^-8 (one to
        # two thirds of it on average) add up in quadrature to 1.2e-2 at most
        assert float((g.double() - w).norm() / w.norm()) < 1.2e-2


def test_captured_forward_and_backward_beside_a_living_eager_graph():
    rotary = Rotary(128)
    q, k = _heads((2, 4, 50, 128), torch.bfloat16, 1, grad=True), _heads((2, 2, 50, 128), torch.bfloat16, 2, grad=True)
    up = [_heads(t.shape, torch.bfloat16, 5) for t in (q, k)]
    before, ops._CHECK_STATUS = ops._CHECK_STATUS, False
    try:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = apply_rotary(q, k, rotary)                   # its graph lives on
            want = torch.autograd.grad(eager, (q, k), up, retain_graph=True)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = apply_rotary(q, k, rotary)
            grads = torch.autograd.grad(out, (q, k), up)
        graph.replay()
        torch.cuda.synchronize()
    finally:
        ops._CHECK_STATUS = before
    for a, b in zip((*out, *grads), (*eager, *want)):
        assert torch.equal(a, b)


def test_positions_changed_in_place_are_noticed():
    q = _heads((1, 2, 8, 64), torch.bfloat16, 1, grad=True)
    positions = torch.arange(8, device="cuda")
    out, _ = apply_rotary(q, None, Rotary(64), positions=positions)
    positions += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_forward_mode_tangents_of_a_gradient_are_refused():
    import torch.autograd.forward_ad as fwAD

    q = _heads((1, 1, 4, 32), torch.bfloat16, 1, grad=True)
    out, _ = apply_rotary(q, None, Rotary(32))
    with fwAD.dual_level():
        u = fwAD.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, q, u)
