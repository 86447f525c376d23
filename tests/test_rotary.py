"""Rotation by position against the formula in 64 bits: types, both orders of pairs, part of a head, odd sizes and strides,
far and negative positions, scaled frequencies, in place; its gradient against the formula's and against differences."""

import copy
import math
import pickle
import struct

import pytest
import torch

import libcertex_b200 as certex
from libcertex_b200.paged import _frequencies

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
# smallest step of a type, halved: what a rounding to a subnormal number may be off by
TINY = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}


def turned(x, positions, rotary, inverse=False):
    """(value, sum of the magnitudes that each value is made of) in 64 bits on the CPU."""
    x, positions = x.detach().cpu().double(), positions.cpu().double()
    r = rotary.rotary_dim
    a = positions[:, None, None] * torch.tensor(rotary.frequencies, dtype=torch.float64)
    c, s = rotary.magnitude * a.cos(), rotary.magnitude * a.sin() * (-1 if inverse else 1)
    i = torch.arange(r // 2)
    lo, hi = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + r // 2)
    y, size = x.clone(), torch.zeros_like(x)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    size[..., lo] = size[..., hi] = rotary.magnitude * (x[..., lo].abs() + x[..., hi].abs())
    return y, size


def close(got, x, positions, rotary, inverse=False):
    """A sine or cosine is off by at most 2^-20 (16-bit types: the angle's product with pi, 2 * 2^-24 * pi, and the hardware's
    sine, 2^-20.9) or 2^-21 (float32: the angle's rounding, 2^-25 * pi, and sincospif, 2 * 2^-24, and the products' and the
    sum's roundings). The angle of the formula, position * w in 64 bits, is itself rounded, by 2^-53 * position * w: 2^-22 at
    2^31 where w is 1, but 7.5 times that for a pair that adds 7.5 a position; the kernel's by position * 2^-64 turns."""
    want, size = turned(x, positions, rotary, inverse)
    t = got.dtype
    angle = (2.0**-21 if t == torch.float32 else 2.0**-19.4) + 2.0**-52 * positions.abs().max().item() * max(map(abs, rotary.frequencies))
    tolerance = size * angle + (HALF_STEP[t] * 1.01) * want.abs() + TINY[t]
    off = (got.cpu().double() - want).abs() - tolerance
    assert off.max() <= 0 if off.numel() else True, float(off.max())


def test_frequencies_of_every_scaling():
    r, n = 64, 4096
    w = _frequencies(r, 1e4, None, 1.0, n, None, None)
    assert w[0] == 1.0 and math.isclose(w[-1], 1e4 ** (-62 / 64))
    assert _frequencies(r, 1e4, "linear", 4.0, n, None, None) == [f / 4 for f in w]
    ntk = _frequencies(r, 1e4, "ntk", 4.0, n, None, None)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], w[-1] / 4)  # the slowest pair is stretched by the whole factor
    for kind, high in (("wavelength", 4), ("yarn", 32)):
        z = _frequencies(r, 1e4, kind, 8.0, n, None, None)
        share = [a / b for a, b in zip(z, w)]
        assert share[0] == 1.0 and math.isclose(share[-1], 1 / 8) and all(a >= b - 1e-12 for a, b in zip(share, share[1:]))
        assert all(s == 1.0 for s, f in zip(share, w) if n * f / (2 * math.pi) > high * 1.4)
        assert all(math.isclose(s, 1 / 8) for s, f in zip(share, w) if n * f / (2 * math.pi) < 0.7)


@pytest.mark.parametrize("kwargs", [dict(head_dim=7), dict(head_dim=8, rotary_dim=3), dict(head_dim=8, rotary_dim=10), dict(head_dim=8, rotary_dim=0),
                                    dict(head_dim=8, scaling="cubic"), dict(head_dim=8, base=0.0), dict(head_dim=8, factor=-1.0, scaling="linear"),
                                    dict(head_dim=8, frequencies=[1.0]), dict(head_dim=8, frequencies=[1.0, 2.0, math.nan, 4.0]),
                                    dict(head_dim=2, scaling="ntk", factor=2.0), dict(head_dim=8, scaling="yarn", low=3.0, high=2.0)])
def test_plans_that_make_no_sense_are_refused(kwargs):
    with pytest.raises(ValueError):
        certex.Rotary(**kwargs, device="cpu")


def test_rows_on_the_host_are_refused():
    plan = certex.Rotary(8, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        plan(torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,heads,dim,r", [(1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 80, 80), (17, 3, 96, 32), (2, 2, 20, 6), (1000, 1, 64, 16),
                                           (5, 13, 256, 128), (2500, 20, 128, 128), (7, 9, 26, 26)])
def test_against_the_formula(n, heads, dim, r, interleaved, dtype):
    g = torch.Generator(device="cuda").manual_seed(n * dim)
    x = torch.randn((n, heads, dim), generator=g, device="cuda").to(dtype)
    positions = torch.randint(0, 200_000, (n,), generator=g, device="cuda", dtype=torch.int32)
    plan = certex.Rotary(dim, r, interleaved=interleaved)
    y = plan(x, positions)
    close(y, x, positions, plan)
    assert torch.equal(y[..., r:], x[..., r:])
    close(plan(x, positions.long(), inverse=True), x, positions, plan, inverse=True)
    before = x.clone()
    assert plan(x, positions, out=x) is x and torch.equal(x, y) and not torch.equal(before, y)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("ntk", 2.0), ("wavelength", 8.0), ("yarn", 16.0)])
def test_scaled_frequencies_and_far_positions(scaling, factor):
    plan = certex.Rotary(128, scaling=scaling, factor=factor, base=5e5)
    x = torch.randn((9, 2, 128), device="cuda")
    for at in ([0, 1, 2, 3, 4095, 4096, 131_071, 1_000_000, 10_000_000], [-1, -2, -131_072, 2**31 - 1, -(2**31), 7, 8, 9, 10]):
        positions = torch.tensor(at, device="cuda")
        close(plan(x, positions), x, positions, plan)
        close(plan(x, positions.int()), x, positions, plan)
    fast = certex.Rotary(4, frequencies=[7.5, -0.3])  # more than a turn a position, and backwards
    close(fast(x[:, :, :4], positions), x[:, :, :4], positions, fast)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views(dtype):
    """Heads out of one projection, rows that do not begin on 16 bytes, one head for all, axes in another order, a
    view with the negative bit."""
    plan = certex.Rotary(64, 32)
    positions = torch.arange(11, device="cuda", dtype=torch.int32) * 977
    qkv = torch.randn((11, 12, 64), device="cuda").to(dtype)
    flat = torch.randn((11 * 3 * 64 + 1,), device="cuda").to(dtype)
    for x in (qkv[:, 8:], qkv[:, ::5], flat[1:].view(11, 3, 64), qkv[:, :1].expand(11, 4, 64), qkv.transpose(0, 1)[:11, :11].transpose(0, 1)[:, 3:],
              qkv.transpose(1, 2)[:, :12].transpose(1, 2)[..., None].expand(11, 12, 12, 6).reshape(11, 12, 72)[..., :64], torch._neg_view(qkv)):
        close(plan(x, positions), x, positions, plan)
    out = torch.full((11, 30, 64), 7.0, device="cuda").to(dtype)
    plan(qkv, positions, out=out[:, 10:22])
    close(out[:, 10:22], qkv, positions, plan)
    assert bool((out[:, :10] == 7).all()) and bool((out[:, 22:] == 7).all())


@pytest.mark.gpu
def test_nothing_to_turn_and_refusals():
    plan = certex.Rotary(64)
    x, p = torch.randn((4, 2, 64), device="cuda"), torch.arange(4, device="cuda")
    assert plan(x[:0], p[:0]).shape == (0, 2, 64) and plan(x[:, :0], p).shape == (4, 0, 64)
    for bad in (lambda: plan(x[0], p), lambda: plan(x[..., :32], p), lambda: plan(x, p[:3]), lambda: plan(x, p.float()), lambda: plan(x, p.cpu()),
                lambda: plan(x.double(), p), lambda: plan(x.int(), p), lambda: plan(x, p, out=x[:3]), lambda: plan(x, p, out=x.half()),
                lambda: plan(x[:2], p[:2], out=x[1:3]), lambda: plan(x, p, out=x[:, :1].expand(4, 2, 64)), lambda: plan(x.cpu(), p)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="gradient"):
        plan(x.clone().requires_grad_(), p, out=torch.empty_like(x))


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradient(dtype, interleaved):
    plan = certex.Rotary(48, 32, interleaved=interleaved, scaling="yarn", factor=4.0)
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((6, 3, 48), generator=g, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
    p = torch.tensor([0, 1, 50, 4000, 99_999, 3], device="cuda")
    (dx,) = torch.autograd.grad(plan(x, p), x, dy)
    close(dx, dy, p, plan, inverse=True)  # the formula's: the transpose of a rotation turns back
    (dx,) = torch.autograd.grad(plan(x, p).sum(), x)  # a gradient that is one number, expanded
    close(dx, torch.ones_like(dy), p, plan, inverse=True)
    if dtype == torch.float32:
        # differences: the map is linear, so a step of any length has the exact slope; what is left is the rounding of two
        # values of up to 40, 2 * 2^-24 * 40 * 1.2 of each, over a step of 32
        h = torch.randn(x.shape, generator=g, device="cuda")
        with torch.no_grad():
            slope = ((plan(x + 16 * h, p) - plan(x - 16 * h, p)).double() * dy.double()).sum() / 32
        (dx,) = torch.autograd.grad(plan(x, p), x, dy)
        want = (dx.double() * h.double()).sum()
        assert abs(slope - want) <= 2 * 2.0**-21 * (dy.double().abs() * (x.double().abs() + 16 * h.double().abs()).amax()).sum() / 16
    # a second derivative: the gradient with respect to dy is the rotation itself
    dy.requires_grad_()
    (dx,) = torch.autograd.grad(plan(x, p), x, dy, create_graph=True)
    (ddy,) = torch.autograd.grad(dx, dy, x.detach())
    close(ddy, x, p, plan)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    plan = certex.Rotary(128)
    x, p = torch.randn((64, 8, 128), device="cuda").half(), torch.arange(64, device="cuda", dtype=torch.int32)
    want = plan(x, p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = plan(x, p)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = plan(x, p)
    x.copy_(x.flip(0))
    p.add_(100)
    graph.replay()
    assert torch.equal(y, plan(x, p)) and not torch.equal(y, want)


@pytest.mark.gpu
def test_a_captured_training_step():
    """Forward and gradient in one graph, replayed on other inputs."""
    plan = certex.Rotary(32, interleaved=True)
    x = torch.randn((50, 4, 32), device="cuda").requires_grad_()
    dy, p = torch.randn((50, 4, 32), device="cuda"), torch.randint(0, 9999, (50,), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            torch.autograd.grad(plan(x, p), x, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = plan(x, p)
        (dx,) = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        x.mul_(2)
        p.add_(7)
    graph.replay()
    close(y.detach(), x, p, plan)
    close(dx, dy, p, plan, inverse=True)


@pytest.mark.gpu
def test_gradient_of_an_input_that_is_shared():
    """One head for all query heads, one row for all positions: the gradients add up; and an input that is used twice."""
    plan = certex.Rotary(16)
    p = torch.tensor([3, 70, 4096], device="cuda")
    dy = torch.randn((3, 5, 16), device="cuda")
    turned_back = turned(dy, p, plan, inverse=True)[0]
    for shape in ((3, 1, 16), (1, 5, 16), (1, 1, 16)):
        x = torch.randn(shape, device="cuda", requires_grad=True)
        (dx,) = torch.autograd.grad(plan(x.expand(3, 5, 16), p), x, dy)
        want = turned_back
        for axis in (0, 1):
            if shape[axis] == 1:
                want = want.sum(axis, keepdim=True)
        # up to 15 values of up to 6, each off by 2^-21 of its terms, and their sum's roundings
        assert dx.shape == x.shape and float((dx.cpu().double() - want).abs().max()) <= 15 * 12 * 2.0**-21
    x = torch.randn((3, 5, 16), device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(plan(x, p) + plan(x, -p), x, dy)
    want = turned_back + turned(dy, -p, plan, inverse=True)[0]
    assert float((dx.cpu().double() - want).abs().max()) <= 2 * 12 * 2.0**-21


def test_copies_of_a_plan_have_their_own_memory():
    plan = certex.Rotary(16, 8, interleaved=True, magnitude=0.5, device="cpu")
    for twin in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan)), copy.copy(plan)):
        at, r, interleaved, magnitude = struct.unpack("3qd", twin._plan)
        assert at == twin._turns.data_ptr() and (r, interleaved, magnitude) == (8, 1, 0.5)
        assert torch.equal(twin._turns, plan._turns) and twin.device == plan.device and twin._index == plan._index
    assert copy.deepcopy(plan)._turns.data_ptr() != plan._turns.data_ptr()


@pytest.mark.gpu
def test_forward_mode():
    """The rotation is linear: its derivative along dx is the rotation of dx, by the same kernel."""
    plan = certex.Rotary(16, 8)
    x, dx = torch.randn((2, 5, 3, 16), device="cuda")
    positions = torch.arange(5, device="cuda")
    for inverse in (False, True):
        with torch.autograd.forward_ad.dual_level():
            y, dy = torch.autograd.forward_ad.unpack_dual(plan(torch.autograd.forward_ad.make_dual(x, dx), positions, inverse=inverse))
            assert torch.equal(y, plan(x, positions, inverse=inverse)) and torch.equal(dy, plan(dx, positions, inverse=inverse))
            cache = certex.PagedCache(1, 8, 3, 16, dtype=torch.float32)
            table = torch.zeros((1, 1), device="cuda", dtype=torch.int32)
            with pytest.raises(ValueError, match="gradient"):
                cache.append(torch.autograd.forward_ad.make_dual(x, dx), x, table, positions, torch.zeros_like(positions, dtype=torch.int32))
            with pytest.raises(ValueError, match="gradient"):
                plan(torch.autograd.forward_ad.make_dual(x, dx), positions, out=torch.empty_like(x))
