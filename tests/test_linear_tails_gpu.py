"""GELU and its slope far from zero, where a bound that is not relative to the value says nothing.

z is a grid of numbers of the type, so that it is exact.  Tolerances, relative: with e = exp(-z^2 / 2) = 2^(-0.72 z^2), the exponent is rounded three times (z^2, the constant, their
product), 2^-24 of 0.72 z^2 each, which moves e by 3 * 2^-24 * 0.72 * ln 2 * z^2 < 2^-23 z^2 of itself; the quotient by e, exponential and reciprocal 2^-17
in all.  In 16 bits half a step more.  Beyond |z| = 13.1 e is below 2^-126 and taken for zero: an error below 2^-120."""
import math

import pytest

from test_linear_gpu import ACT, KIND, TYPE, capi, check, half_step, ptr, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def grid(kind, low, high, n):
    return torch.linspace(low, high, n, device="cuda", dtype=torch.float64).to(TYPE[kind])


def tail(x):
    return 0.5 * torch.special.erfc(x / math.sqrt(2))


def density(z):
    return torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


# a few tokens in each of their forms, tiles, K ranges
@pytest.mark.parametrize("T,n,m", [(1, 8, 4000), (12, 8, 4000), (31, 40, 4000), (40, 8, 4000), (300, 72, 1001), (70, 8192, 136)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_gelu(kind, T, n, m):
    for low, high in ((-14, -3), (-6, 0), (-1e-2, 1e-2), (0, 14)):
        z = grid(kind, low, high, m)
        x, w = torch.zeros((T, n), device="cuda", dtype=TYPE[kind]), torch.zeros((m, n), device="cuda", dtype=TYPE[kind])
        x[:, -1], w[:, -1] = 1, z
        y = torch.zeros((T, m), device="cuda", dtype=TYPE[kind])
        check(capi.load_library().ts2_op_linear_forward(0, stream(), KIND[kind], ACT["gelu"], T, n, m, ptr(x), n, ptr(w), n, None, None, m, ptr(y), m, None, m))
        z64 = z.double()
        want = torch.where(z64 < 0, z64 * tail(-z64), z64 * (1 - tail(z64)))
        off = (y.double() - want).abs() - half_step(kind, want) - 1.01 * ((2.0 ** -17 + 2.0 ** -23 * z64 ** 2) * z64.abs() * tail(z64.abs()) + 2.0 ** -22 * want.abs()) - 2.0 ** -120
        assert off.max() <= 0, (low, z[off.argmax() % m].item(), off.max().item())


# rows without 16-byte alignment take other loads
@pytest.mark.parametrize("m", [4096, 4001])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_slope_of_gelu(kind, m):
    """of one token dbias is the unrounded dz, and dw = dz x is dz rounded"""
    for low, high in ((-14, -3), (-6, 0), (-1e-2, 1e-2), (0, 14)):
        z = grid(kind, low, high, m).view(1, m)
        dy, x = torch.ones((1, m), device="cuda", dtype=TYPE[kind]), torch.ones((1, 8), device="cuda", dtype=TYPE[kind])
        dw, db = torch.zeros((m, 8), device="cuda"), torch.zeros(m, device="cuda")
        check(capi.load_library().ts2_op_linear_backward(0, stream(), KIND[kind], ACT["gelu"], 1, 8, m, ptr(dy), m, ptr(z), m, ptr(x), 8, None, 8, None, 8, KIND["f32"], ptr(dw), 8,
                                                         ptr(db)))
        z64 = z[0].double()
        part = tail(z64.abs()) - z64.abs() * density(z64)  # the slope at -|z|
        want = torch.where(z64 < 0, part, 1 - part)
        off = 1.01 * ((2.0 ** -17 + 2.0 ** -23 * z64 ** 2) * (tail(z64.abs()) + z64.abs() * density(z64)) + 2.0 ** -23 * want.abs()) + 2.0 ** -120
        assert ((db - want).abs() <= off).all(), (low, z64[((db - want).abs() - off).argmax()].item())
        assert ((dw.double() - want[:, None]).abs() <= (off + half_step(kind, want))[:, None]).all()
