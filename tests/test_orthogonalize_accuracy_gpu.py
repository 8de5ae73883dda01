"""How near ts2_op_orthogonalize comes to its formula before the result is rounded to bf16, for matrices of every kind: few
rows, few directions, few rows that hold anything, falling spectra.

What is measured.  The result is out = bf16(w + d) where w is the formula in float64 and d the error looked for.  Rounding to
a grid is a step function whose steps lie anywhere with regard to w, so the mean of |bf16(w + d) - bf16(w)| is the mean of |d|:
`error` is the sum of these differences over the sum of |w|, over enough elements that single steps do not count.

Limit.  The operands are in two fp16 halves: each value to 2^-22 of itself.  These roundings alone (the formula in float64 with every
operand as two halves) carry a matrix of the kinds below 1.1e-5 at most (one direction in 8 x 8), mostly less than 1e-6; what they
leave is passed on by the polynomial, whose slope is up to 4.2.  The sums are fp32, of K / 16 terms
that may each be cut off (2^-23): for K up to 8192 as much as 2^-14 of a sum of one sign and 2^-17 on average, which moves every
singular value alike and is passed on with a slope below 4.  4 x 2^-17 x sqrt(5 steps) + 1e-5 = 8e-5: 1e-4."""
import ml_dtypes
import numpy as np
import pytest

from test_orthogonalize_gpu import COEF, TYPE, exact, run

pytestmark = pytest.mark.gpu

LIMIT = 1e-4


def rank(rows, cols, k):
    return lambda rng: rng.standard_normal((rows, k)) @ rng.standard_normal((k, cols))


def sparse(rows, cols, k):
    """k rows that hold something"""
    def make(rng):
        g = np.zeros((rows, cols))
        g[rng.permutation(rows)[:k]] = rng.standard_normal((k, cols))
        return g
    return make


def falling(rows, cols, power):
    def make(rng):
        n = min(rows, cols)
        return (rng.standard_normal((rows, n)) / np.sqrt(n) * np.arange(1, n + 1) ** -float(power)) @ rng.standard_normal((n, cols))
    return make


def error(got, want):
    near = want.astype(ml_dtypes.bfloat16).astype(np.float64)
    return np.abs(got - near).sum() / np.abs(want).sum()


def check(make, batch, kind="f32", steps=5, coef=COEF, limit=LIMIT):
    g = np.stack([make(np.random.default_rng(100 + s)) for s in range(batch)]).astype(TYPE[kind])
    got = run(kind, g, coef, steps)
    want = np.stack([exact(m, coef, steps) for m in g])
    off = error(got, want)
    assert off <= limit, f"{off:.1e}"
    # the whole distance, of every matrix: that and the rounding, at most 2^-8 of every element (2^-8 / sqrt(3) would be the mean square
    # of many, which four elements need not keep: 0.3990, 0.5599, 0.5643 and 0.4074 are 0.6, 1.3, 1.8 and 0.8 thousandths off the grid)
    for o, w in zip(got, want):
        assert np.linalg.norm(o - w) <= (2 * limit + 2.0 ** -8) * np.linalg.norm(w)


# matrices that one CTA or a cluster holds, and larger ones
SMALL = {"2x2": (rank(2, 2, 2), 400), "3x50": (rank(3, 50, 3), 40), "300x2": (rank(300, 2, 2), 20), "4x64": (rank(4, 64, 4), 40), "6x20": (rank(6, 20, 6), 60),
         "rank 1 of 8x8": (rank(8, 8, 1), 100), "rank 1 of 32x32": (rank(32, 32, 1), 40), "rank 1 of 64x256": (rank(64, 256, 1), 10),
         "rank 1 of 600x100": (rank(600, 100, 1), 4), "rank 2 of 40x60": (rank(40, 60, 2), 20), "rank 3 of 128x4000": (rank(128, 4000, 3), 1),
         "2 rows of 100x120": (sparse(100, 120, 2), 20), "128x256": (rank(128, 256, 128), 2), "128x384": (rank(128, 384, 128), 2),
         "1/k^2, 90x900": (falling(90, 900, 2), 2)}


@pytest.mark.parametrize("name", SMALL)
def test_matrices_that_a_cluster_holds(name):
    check(*SMALL[name])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("name", ["4x64", "rank 1 of 64x256", "rank 2 of 40x60"])
def test_types_of_matrices_that_a_cluster_holds(name, kind):
    check(*SMALL[name], kind=kind)


@pytest.mark.parametrize("coef,steps", [(COEF, 1), (COEF, 2), ((1.875, -1.25, 0.375), 8), ((1.5, -0.5, 0.0), 12)])
def test_other_coefficients_of_matrices_that_a_cluster_holds(coef, steps):
    check(falling(100, 300, 1), 3, coef=coef, steps=steps)


# products through memory: whole and half tiles, divided K, rows that are not a tile, more of K than a cluster holds
LARGE = {"130x140": (rank(130, 140, 130), 3), "rank 1 of 200x300": (rank(200, 300, 1), 2), "rank 4 of 700x260": (rank(700, 260, 4), 2),
         "2 rows of 1000x400": (sparse(1000, 400, 2), 2), "1/k^2, 512x1024": (falling(512, 1024, 2), 1), "1/k, 300x2500": (falling(300, 2500, 1), 1),
         "20x6300": (rank(20, 6300, 20), 2), "rank 1 of 7000x64": (rank(7000, 64, 1), 1), "rank 2 of 30 of 200x264": (rank(200, 264, 2), 30),
         "1500x1100": (falling(1500, 1100, 0.5), 1)}


@pytest.mark.parametrize("name", LARGE)
def test_products_through_memory(name):
    check(*LARGE[name])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("name", ["130x140", "rank 4 of 700x260"])
def test_types_of_products_through_memory(name, kind):
    check(*LARGE[name], kind=kind)


@pytest.mark.parametrize("coef,steps", [(COEF, 1), (COEF, 2), ((1.875, -1.25, 0.375), 8), ((1.5, -0.5, 0.0), 12)])
def test_other_coefficients_of_products_through_memory(coef, steps):
    check(falling(300, 280, 1), 1, coef=coef, steps=steps)


@pytest.mark.parametrize("batch,rows,cols", [(1, 8192, 1100), (2, 2100, 8192)])
def test_long_sums(batch, rows, cols):
    """K of 8192, in ranges and in one piece; the formula in float64 on the device"""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(rows)
    g = torch.randn((batch, rows, cols), device="cuda", generator=gen) + 0.1 * torch.randn((batch, rows, 8), device="cuda", generator=gen) @ \
        torch.randn((batch, 8, cols), device="cuda", generator=gen)
    x = g.double()
    x /= torch.linalg.matrix_norm(x)[:, None, None]
    x = x.transpose(1, 2) if rows > cols else x
    for _ in range(5):
        a = x @ x.transpose(1, 2)
        x = COEF[0] * x + (COEF[1] * a + COEF[2] * a @ a) @ x
    x = (x.transpose(1, 2) if rows > cols else x).cpu().numpy()
    assert error(run("f32", g.cpu().numpy()), x) <= LIMIT
