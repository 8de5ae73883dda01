"""The orthogonalised update (ts2_op_orthogonalize) against its formula in float64.

Tolerance: `modelled` computes the formula in float64 with the roundings that the kernels make (X and the diagonal of B in 32 bits, the
operands of the three products in fp16), which says how far these roundings alone carry a result; another order of fp32 sums moves single
roundings, so a right kernel is within twice that of the formula, and the final rounding to bf16 adds 2^-8 of an element at most
(relative L2: 2^-8 / sqrt(3), the mean square of a uniform error)."""
import ctypes as C

import ml_dtypes
import numpy as np
import pytest

from tscale2_b200 import capi
from tscale2_b200.device import DeviceBuffer, check, sync

pytestmark = pytest.mark.gpu

KIND = {"f32": capi.OUT_F32, "f16": capi.OUT_F16, "bf16": capi.OUT_BF16}
TYPE = {"f32": np.float32, "f16": np.float16, "bf16": ml_dtypes.bfloat16}
COEF = (3.4445, -4.7750, 2.0315)


def exact(g, coef=COEF, steps=5, rounded=False):
    def half(v, s):
        return (v * s).astype(np.float16).astype(np.float64) / s if rounded else v

    x = g.astype(np.float64)
    norm = np.linalg.norm(x)
    x = x / norm if norm else x
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    for _ in range(steps):
        h = half(x, 2.0 ** 14)
        a = half(h @ h.T, 2.0 ** 12)
        b = coef[1] * a + coef[2] * (a @ a)
        d = np.diag(b).copy() if rounded else np.zeros(len(b))
        x = (coef[0] + d)[:, None] * x + half(b - np.diag(d), 2.0 ** 11) @ h
    return x.T if tall else x


def modelled(g, coef=COEF, steps=5):
    return exact(g, coef, steps, rounded=True)


def spectrum(rows, cols, power, seed):
    """a matrix whose singular values fall off as 1 / k^power"""
    rng = np.random.default_rng(seed)
    n = min(rows, cols)
    s = np.arange(1, n + 1) ** -float(power)
    return (rng.standard_normal((rows, n)) / np.sqrt(n) * s) @ rng.standard_normal((n, cols))


def run(kind, g, coef=COEF, steps=5, scale=1.0, ld=None, out_ld=None, gap=0, offset=0):
    lib = capi.load_library()
    b, r, c = g.shape
    ld, out_ld = ld or c, out_ld or c
    t = TYPE[kind]
    flat = np.full(offset + b * (r * ld + gap), 5, t)
    for i in range(b):
        at = offset + i * (r * ld + gap)
        flat[at:at + r * ld].reshape(r, ld)[:, :c] = g[i]
    G = DeviceBuffer.from_numpy(flat.view(np.uint8))
    O = DeviceBuffer.from_numpy(np.full(offset + b * (r * out_ld + gap), 5, ml_dtypes.bfloat16).view(np.uint8))
    check(lib.ts2_op_orthogonalize(0, None, KIND[kind], G.ptr + offset * flat.itemsize, ld, r * ld + gap, b, r, c, (C.c_float * 3)(*coef), steps, scale,
                                   O.ptr + offset * 2, out_ld, r * out_ld + gap))
    sync()
    flat = O.download(O.nbytes, np.uint8).view(ml_dtypes.bfloat16)
    assert (flat[:offset] == 5).all()
    out = []
    for i in range(b):
        at = offset + i * (r * out_ld + gap)
        rows = flat[at:at + r * out_ld].reshape(r, out_ld)
        assert (rows[:, c:] == 5).all() and (flat[at + r * out_ld:at + r * out_ld + gap] == 5).all()
        out.append(rows[:, :c].astype(np.float64))
    return np.stack(out)


def near(got, g, coef=COEF, steps=5, scale=1.0):
    want = exact(g, coef, steps) * scale
    size = np.linalg.norm(want)
    model = np.linalg.norm(modelled(g, coef, steps) * scale - want)
    off = np.linalg.norm(got - want)
    assert off <= 2 * model + (2.0 ** -8 / 3 ** 0.5) * size, (off / size, model / size)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (9, 1), (16, 16), (17, 200), (128, 256), (200, 70), (130, 129), (333, 1000), (700, 260)])
def test_against_the_formula(kind, rows, cols):
    g = np.stack([spectrum(rows, cols, p, rows + p) for p in (0, 1)]).astype(TYPE[kind])
    got = run(kind, g)
    for o, m in zip(got, g):
        near(o, m)


@pytest.mark.parametrize("power", [0, 1, 2, 3])
@pytest.mark.parametrize("rows,cols", [(256, 512), (512, 512), (640, 300)])
def test_small_singular_values_are_carried(power, rows, cols):
    g = spectrum(rows, cols, power, power)[None].astype(np.float32)
    near(run("f32", g)[0], g[0])


def test_one_large_matrix():
    g = spectrum(1500, 1100, 0.5, 3)[None].astype(np.float32)
    near(run("f32", g)[0], g[0])


@pytest.mark.parametrize("kind,batch,rows,cols", [("f32", 2, 100, 385), ("bf16", 1, 700, 33), ("f32", 3, 128, 900), ("f16", 1, 1999, 128), ("f32", 1, 5, 3100),
                                                  ("f32", 1, 128, 6144), ("f32", 1, 6145, 120)])
def test_long_rows_on_clusters_of_every_size(kind, batch, rows, cols):
    g = np.stack([spectrum(rows, cols, 0.5, s) for s in range(batch)]).astype(TYPE[kind])
    got = run(kind, g)
    for o, m in zip(got, g):
        near(o, m)


@pytest.mark.parametrize("batch,rows,cols", [(1, 300, 2500), (30, 200, 264), (13, 520, 300), (1, 2000, 140)])
def test_products_of_few_and_of_many_tiles(batch, rows, cols):
    """one matrix whose K is divided, and more matrices than are worked on at a time"""
    g = np.stack([spectrum(rows, cols, 0.5, s) for s in range(batch)]).astype(np.float32)
    got = run("f32", g, steps=6)
    for i in {0, batch // 2, batch - 1}:
        near(got[i], g[i], steps=6)


@pytest.mark.parametrize("batch,rows,cols", [(1, 64, 64), (5, 96, 160), (40, 128, 100), (3, 300, 128), (17, 256, 256)])
def test_a_batch_is_its_matrices_one_by_one(batch, rows, cols):
    g = np.stack([spectrum(rows, cols, 0.5, s) for s in range(batch)]).astype(np.float32)
    together = run("f32", g)
    for i in (0, batch // 2, batch - 1):
        near(together[i], g[i])
        assert np.array_equal(run("f32", g[i:i + 1])[0], together[i])


@pytest.mark.parametrize("coef,steps", [(COEF, 1), (COEF, 2), (COEF, 10), ((1.875, -1.25, 0.375), 8), ((1.5, -0.5, 0.0), 12), ((2.0, -1.5, 0.5), 6)])
def test_other_coefficients_and_steps(coef, steps):
    for rows, cols in ((100, 140), (300, 280)):
        g = spectrum(rows, cols, 0.5, steps)[None].astype(np.float32)
        near(run("f32", g, coef, steps)[0], g[0], coef, steps)


def test_the_singular_values_come_near_to_one():
    """the polynomial's own range after five steps for what starts above 0.02 of the norm: [0.68, 1.21] (evaluated on a grid)"""
    g = spectrum(128, 384, 0, 1)[None].astype(np.float32)
    s = np.linalg.svd(run("f32", g)[0], compute_uv=False)
    start = np.linalg.svd(g[0].astype(np.float64), compute_uv=False) / np.linalg.norm(g[0].astype(np.float64))
    for _ in range(5):
        start = COEF[0] * start + COEF[1] * start ** 3 + COEF[2] * start ** 5
    assert s.max() < start.max() + 0.01 and s.min() > start.min() - 0.01


@pytest.mark.parametrize("kind,ld,out_ld,gap,offset", [("f32", 171, 160, 3, 1), ("f16", 161, 173, 1, 1), ("bf16", 168, 168, 8, 8), ("f32", 160, 161, 0, 0)])
def test_pitches_strides_and_offsets(kind, ld, out_ld, gap, offset):
    g = np.stack([spectrum(144, 160, 0.5, s) for s in range(3)]).astype(TYPE[kind])
    got = run(kind, g, ld=ld, out_ld=out_ld, gap=gap, offset=offset)
    for o, m in zip(got, g):
        near(o, m)


def test_the_scale_of_the_input_does_not_matter():
    g = spectrum(128, 192, 0.5, 4)
    for s in (1e-30, 1e-3, 1e30):
        m = (g * s).astype(np.float32)
        near(run("f32", m[None], scale=0.25)[0], m, scale=0.25)


def test_zeros_stay_zeros_and_bad_values_stay_in_their_matrix():
    rng = np.random.default_rng(5)
    g = rng.standard_normal((5, 130, 140)).astype(np.float32)
    g[1] = 0
    g[2, 7, 9] = np.nan
    g[3, 100, 3] = np.inf
    got = run("f32", g)
    assert (got[1] == 0).all() and np.isnan(got[2]).all() and np.isnan(got[3]).all()
    for i in (0, 4):
        near(got[i], g[i])


def test_a_matrix_of_one_row_or_one_element():
    g = np.zeros((1, 1, 300), np.float32)
    g[0, 0, 17] = -4
    near(run("f32", g)[0], g[0])
    near(run("f32", -g.transpose(0, 2, 1))[0], -g[0].T)


def test_the_same_matrix_for_a_whole_batch():
    lib = capi.load_library()
    g = spectrum(100, 90, 0, 6).astype(np.float32)
    G, O = DeviceBuffer.from_numpy(g), DeviceBuffer(3 * g.size * 2)
    check(lib.ts2_op_orthogonalize(0, None, capi.OUT_F32, G.ptr, 90, 0, 3, 100, 90, (C.c_float * 3)(*COEF), 5, 1.0, O.ptr, 90, 9000))
    sync()
    out = O.download((3, 100, 90), np.uint16).view(ml_dtypes.bfloat16).astype(np.float64)
    assert np.array_equal(out[0], out[1]) and np.array_equal(out[0], out[2])
    near(out[0], g)


@pytest.mark.parametrize("rows,cols", [(128, 128), (500, 260)])
def test_in_place(rows, cols):
    lib = capi.load_library()
    g = np.stack([spectrum(rows, cols, 0, s) for s in range(2)]).astype(ml_dtypes.bfloat16)
    want = run("bf16", g)
    G = DeviceBuffer.from_numpy(g.view(np.uint8))
    check(lib.ts2_op_orthogonalize(0, None, capi.OUT_BF16, G.ptr, cols, rows * cols, 2, rows, cols, (C.c_float * 3)(*COEF), 5, 1.0, G.ptr, cols, rows * cols))
    sync()
    assert np.array_equal(G.download(g.nbytes, np.uint8).view(ml_dtypes.bfloat16).reshape(g.shape).astype(np.float64), want)


@pytest.mark.parametrize("batch,rows,cols", [(1, 96, 300), (2, 700, 900), (9, 260, 140)])
def test_the_same_call_gives_the_same_bits(batch, rows, cols):
    g = np.stack([spectrum(rows, cols, 0.5, s) for s in range(batch)]).astype(np.float32)
    first = run("f32", g)
    for _ in range(3):
        assert np.array_equal(run("f32", g), first)


def test_two_streams_and_captured_graphs():
    import torch
    lib = capi.load_library()
    sets = []
    for seed, (b, r, c) in enumerate([(2, 300, 200), (1, 128, 500), (2, 300, 200)]):
        g = np.stack([spectrum(r, c, 0.5, seed + i) for i in range(b)]).astype(np.float32)
        sets.append(dict(shape=(b, r, c), host=g, g=torch.from_numpy(g).cuda(), o=torch.zeros((b, r, c), device="cuda", dtype=torch.bfloat16),
                         s=torch.cuda.Stream()))
    torch.cuda.synchronize()

    def call(st):
        b, r, c = st["shape"]
        check(lib.ts2_op_orthogonalize(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), capi.OUT_F32, st["g"].data_ptr(), c, r * c, b, r, c,
                                       (C.c_float * 3)(*COEF), 5, 1.0, st["o"].data_ptr(), c, r * c))

    def verify():
        sync()
        for st in sets:
            for o, m in zip(st["o"].float().cpu().numpy(), st["host"]):
                near(o, m)
            st["o"].zero_()
        torch.cuda.synchronize()

    for _ in range(3):
        for st in sets:
            with torch.cuda.stream(st["s"]):
                call(st)
    verify()
    graphs = []
    for st in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(st)
        graphs.append(g)
    for _ in range(3):
        for st, g in zip(sets, graphs):
            with torch.cuda.stream(st["s"]):
                g.replay()
    verify()
