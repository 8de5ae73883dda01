"""ts2_op_linear_backward with gradients that are not finite or leave the type's range: weight gradients and dbias in fp32 show it, and nothing else is touched.

One element (token t, output j) of dy is bad.  Row j of dw and element j of dbias sum over it; row t of dx, too.  All else is as without it, to the bit, since sums of
other rows and columns never meet it."""
import pytest

from test_linear_gpu import ACT, KIND, LAYOUTS, TYPE, capi, check, ptr, rows, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

INF, NAN = float("inf"), float("nan")
# tiles that are not full, several tiles, K ranges
SIZES = [(40, 72, 96), (300, 333, 335), (5000, 24, 40)]


def backward(kind, act, T, n, m, layout, bad, at):
    gen = torch.Generator(device="cuda").manual_seed(T)
    t = TYPE[kind]
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)
    x, w = randn(T, n).abs() + 0.5, randn(m, n).abs() + 0.5
    dy, z = randn(T, m), randn(T, m)
    z[at] = 1.5  # a slope above one in GELU and SiLU
    out = []
    for value in (1.0, bad):
        dy[at] = value
        a = [rows(v.to(t), layout) for v in (dy, z, x, w)]
        dx, dw, db = rows(torch.zeros((T, n), device="cuda", dtype=t), layout), torch.zeros((m, n), device="cuda"), torch.zeros(m, device="cuda")
        check(capi.load_library().ts2_op_linear_backward(0, stream(), KIND[kind], ACT[act], T, n, m, a[0].ptr, a[0].ld, a[1].ptr if act != "none" else None, a[1].ld, a[2].ptr, a[2].ld,
                                                         a[3].ptr, a[3].ld, dx.ptr, dx.ld, KIND["f32"], ptr(dw), n, ptr(db)))
        assert dx.around_is_kept()
        out.append((dx.t.clone(), dw, db))
    return out


@pytest.mark.parametrize("layout", ["tight", "odd base"])
@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("T,n,m", SIZES)
def test_bad_gradients_show(T, n, m, bad, kind, act, layout):
    at = (T - 3, m // 2)
    (dx0, dw0, db0), (dx, dw, db) = backward(kind, act, T, n, m, layout, bad, at)
    same = lambda v: torch.isnan(v).all() if bad != bad else (v == bad).all()
    assert same(dw[at[1]]) and same(db[at[1]])
    if bad != bad:
        assert torch.isnan(dx[at[0]]).all()
    else:  # fp16 results saturate
        assert (dx[at[0]] == (bad if kind == "bf16" else (65504 if bad > 0 else -65504))).all()
    others, tokens = torch.arange(m, device="cuda") != at[1], torch.arange(T, device="cuda") != at[0]
    assert torch.equal(dw[others], dw0[others]) and torch.equal(db[others], db0[others]) and torch.equal(dx[tokens], dx0[tokens])


@pytest.mark.parametrize("T,n,m", SIZES)
@pytest.mark.parametrize("act,slope", [("gelu", 1.1275), ("silu", 1.0410)])
def test_products_beyond_fp16_show(T, n, m, act, slope):
    """dy act'(z) of 65504 times the slope at 1.5 is no fp16 number: dw is infinite, dbias what it is"""
    at = (T - 3, m // 2)
    (dx0, dw0, db0), (dx, dw, db) = backward("f16", act, T, n, m, "tight", 65504.0, at)
    assert torch.isinf(dw[at[1]]).all() and abs(db[at[1]] - db0[at[1]] - (65504 - 1) * slope).item() < 1e-3 * 65504
    others = torch.arange(m, device="cuda") != at[1]
    assert torch.equal(dw[others], dw0[others])


# a few tokens in each of their forms, tiles, K ranges; rows without 16-byte alignment
@pytest.mark.parametrize("T,n,m", [(4, 64, 96), (13, 64, 96), (31, 40, 33), (40, 64, 96), (300, 333, 335), (70, 8192, 136)])
@pytest.mark.parametrize("layout", ["tight", "odd base"])
@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_inputs_that_are_not_finite(kind, act, T, n, m, layout):
    """a token's x of inf, NaN and -inf: act of it, by the formula (-inf / inf of SiLU is none), and every other token as it was"""
    gen = torch.Generator(device="cuda").manual_seed(T)
    t = TYPE[kind]
    xs = torch.randn((T, n), device="cuda", generator=gen)
    w = rows((torch.randn((m, n), device="cuda", generator=gen).abs() + 0.5).to(t), layout)
    out = []
    for bad in (False, True):
        if bad:
            xs[0, n // 2], xs[1, 0], xs[2, n - 1] = INF, NAN, -INF
        x, y, z = rows(xs.to(t), layout), rows(torch.zeros((T, m), device="cuda", dtype=t), layout), rows(torch.zeros((T, m), device="cuda", dtype=t), layout)
        check(capi.load_library().ts2_op_linear_forward(0, stream(), KIND[kind], ACT[act], T, n, m, x.ptr, x.ld, w.ptr, w.ld, None, None, m, y.ptr, y.ld, z.ptr, z.ld))
        assert y.around_is_kept() and z.around_is_kept()
        out.append((y.t.clone(), z.t.clone()))
    (y0, z0), (y, z) = out
    assert torch.equal(y[3:], y0[3:]) and torch.equal(z[3:], z0[3:])
    most = INF if kind == "bf16" else 65504.0  # fp16 results saturate
    assert (z[0] == most).all() and torch.isnan(z[1]).all() and (z[2] == -most).all()
    assert (y[0] == most).all() and torch.isnan(y[1]).all()
    if act == "silu":
        assert torch.isnan(y[2]).all()
    else:
        assert (y[2] == (-most if act == "none" else 0)).all()
