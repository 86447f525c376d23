"""Sines and cosines of the float32 rotation, each to a part of itself: near whole quarters of a turn, at small angles and far positions, against
angles that are reduced in 70 digits."""

import decimal
import math

import pytest
import torch

import libcertex_b200 as certex

PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628621")


def sin_cos(position, w):
    """Of position * w, both to a few parts in 2^53 of themselves: the nearest quarter of a turn is taken off in 70 digits."""
    with decimal.localcontext(prec=70):
        angle = decimal.Decimal(position) * decimal.Decimal(w)
        n = int((angle / (PI / 2)).to_integral_value())
        r = float(angle - n * PI / 2)
    s, c = math.sin(r), math.cos(r)
    return ((s, c), (c, -s), (-s, -c), (-c, s))[n % 4]


def test_the_oracle_agrees_with_64_bits():
    for position, w in ((0, 1.0), (1, 1e-9), (7, 0.3), (-5, 1.1), (12, -2.9), (3, math.pi / 2), (100, 0.01)):
        s, c = sin_cos(position, w)
        assert abs(s - math.sin(position * w)) < 1e-13 and abs(c - math.cos(position * w)) < 1e-13


@pytest.mark.gpu
def test_the_inverse_is_the_transpose():
    """It undoes the rotation up to the square of the magnitude: a value is a sum of two products at most, twice, each off by 2^-21.4 and the
    roundings of products and sum, 2^-23 together, of the sizes of what it is made of, 4 times the largest of the row."""
    x, y = torch.randn((2, 40, 3, 64), device="cuda")
    p = torch.arange(40, device="cuda") * 977
    for plan in (certex.Rotary(64), certex.Rotary(64, 32, scaling="yarn", factor=16.0), certex.Rotary(64, magnitude=0.5, interleaved=True)):
        back = plan(plan(x, p), p, inverse=True)
        r, m = plan.rotary_dim, plan.magnitude
        off = 2 * 4 * m * m * (2.0**-21.4 + 2.0**-23) * float(x.abs().max())
        assert float((back[..., :r].double() - m * m * x[..., :r].double()).abs().max()) <= off and torch.equal(back[..., r:], x[..., r:])
        # <R x, y> = <x, R' y>
        left, right = (plan(x, p).double() * y.double()).sum(), (x.double() * plan(y, p, inverse=True).double()).sum()
        assert abs(float(left - right)) <= 2 * 2 * m * (2.0**-21.4 + 2.0**-23) * x.numel() * float(x.abs().max() * y.abs().max())


@pytest.mark.gpu
def test_transforms_of_functions_are_refused():
    """torch.func's transforms wrap their tensors: the kernels cannot read those, and say so."""
    plan, x, p = certex.Rotary(16), torch.randn((5, 2, 16), device="cuda"), torch.arange(5, device="cuda")
    for call in (lambda: torch.func.grad(lambda z: plan(z, p).sum())(x), lambda: torch.func.jvp(lambda z: plan(z, p), (x,), (x,)),
                 lambda: torch.func.vmap(lambda z: plan(z, p))(x[None]), lambda: torch.func.vmap(lambda z: plan(x, z))(p[None])):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim", [256, 250])
def test_sines_to_a_part_of_themselves(dim, interleaved):
    """The unit vector (1, 0) turned by a is (cos a, sin a), in float32: the rest of the angle after whole quarters is a sum of two rounded
    parts, 1.5 * 2^-24 of itself; the sine is a rounded sum of pi t and terms that are a tenth of it at most, 1 + 0.5, and what the series leaves
    out is 0.1; the cosine, at least 0.7, a rounded sum of 1 and terms of 0.3 at most, 1 + 1.3. A magnitude comes on top, 1: 2^-21.4 is 6 *
    2^-24. The frequency is rounded too, by 2^-65 of a turn a position."""
    pairs = dim // 2
    g = torch.Generator().manual_seed(dim)
    # from 2^-24 to 2 radians a position, quarters of a turn, and numbers right beside them
    w = [2.0 ** (-24 + 25 * i / (pairs - 1)) for i in range(pairs)]
    w[3::16] = [math.pi / 2 * (1 + k * 2.0**-30) for k in range(len(w[3::16]))]
    w[5::16] = [-f for f in w[5::16]]
    plan = certex.Rotary(dim, frequencies=w, interleaved=interleaved)
    positions = torch.cat([torch.arange(0, 12), torch.tensor([-1, -2, 63, 4097, 131_071, 1_000_003, 2**31 - 1, -(2**31)]), torch.randint(0, 200_000, (12,), generator=g)])
    x = torch.zeros((len(positions), 1, dim))
    x[..., slice(0, None, 2) if interleaved else slice(0, pairs)] = 1
    got = plan(x.cuda(), positions.cuda())[:, 0].cpu().double()
    cos, sin = (got[:, 0::2], got[:, 1::2]) if interleaved else (got[:, :pairs], got[:, pairs:])
    for i, p in enumerate(positions.tolist()):
        want = torch.tensor([sin_cos(p, f) for f in w], dtype=torch.float64)
        for have, v in ((sin[i], want[:, 0]), (cos[i], want[:, 1])):
            off = v.abs() * 2.0**-21.4 + 2.0**-150 + abs(p) * 2.0**-64 * math.pi
            far = (have - v).abs() - off
            j = int(far.argmax())
            assert float(far[j]) <= 0, (p, w[j], float(have[j]), float(v[j]))
