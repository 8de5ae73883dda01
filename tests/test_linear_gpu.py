"""ts2_op_linear_forward and _backward against the formula in float64.

Tolerances, per element.  A result of a 16-bit type is rounded once: half a step, eps / 2 of it (and half of the smallest subnormal step for
fp16).  The products of 16-bit operands are exact in fp32; sums of K of them on the tensor cores are cut off rather than rounded, at
most a step 2^-23 of what has been added up for every 8 terms and 8 more for the ends and the joins of K ranges: (K / 8 + 8) 2^-23 sum |x w|.  Activations move an
error of z on with a slope of at most 1.13 and add 2^-21 (1 + |z|) of their own (their functions are good to 2^-22 where the sum of a few terms is formed).  dz is
rounded to the operands' type before its two products: eps / 2 sum |dz w|.  dbias sums fp32 numbers in T / 16 + 40 steps or fewer: (T / 16 + 40) 2^-24 sum |dz|."""
import ctypes as C

import pytest

from tscale2_b200 import capi
from tscale2_b200.device import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPE = {"f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f16": capi.OUT_F16, "bf16": capi.OUT_BF16, "f32": capi.OUT_F32, "f32_add": capi.OUT_F32_ADD}
ACT = {"none": capi.ACT_NONE, "relu": capi.ACT_RELU, "gelu": capi.ACT_GELU, "silu": capi.ACT_SILU}
F = torch.nn.functional
ACT64 = {"none": lambda z: z, "relu": torch.relu, "gelu": F.gelu, "silu": F.silu}
# one token, fewer than a tile, tiles and one more, sizes that no 16-byte access divides; few and many tiles, short and long sums
SIZES = [(1, 1, 1), (1, 256, 512), (2, 333, 7), (7, 64, 130), (16, 2048, 264), (17, 1000, 24), (32, 4096, 40), (33, 100, 1001), (129, 1024, 64), (300, 2048, 768), (513, 72, 520),
         (1030, 4104, 256), (2049, 520, 2056)]


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def ptr(t):
    return None if t is None else t.data_ptr()


class Rows:
    """[rows][cols] inside a larger array: a pitch, a first element, and what lies around them, which has to stay"""

    def __init__(self, values, pad=0, first=0):
        rows, cols = values.shape
        self.ld = cols + pad
        self.flat = torch.full((first + rows * self.ld + 64,), 7.0, device="cuda", dtype=values.dtype)
        self.t = self.flat.as_strided((rows, cols), (self.ld, 1), first)
        self.t.copy_(values)
        self.keep = self.flat.clone()

    @property
    def ptr(self):
        return self.t.data_ptr()

    def around_is_kept(self):
        now = self.flat.clone()
        now.as_strided(self.t.shape, (self.ld, 1), self.t.storage_offset()).copy_(self.keep.as_strided(self.t.shape, (self.ld, 1), self.t.storage_offset()))
        return torch.equal(now, self.keep)


LAYOUTS = {"tight": (0, 0), "pitch": (8, 16), "odd pitch": (3, 0), "odd base": (8, 1)}


def rows(values, layout):
    return Rows(values, *LAYOUTS[layout])


def near(got, want, tol):
    off = (got.double() - want).abs() - tol
    assert torch.isfinite(got.double()).all()
    assert off.max().item() <= 0, (off.max().item(), int((off > 0).sum()), got.shape)


def half_step(kind, want):
    if kind == "f32":
        return want.abs() * 2.0 ** -24
    return want.abs() * torch.finfo(TYPE[kind]).eps / 2 + (2.0 ** -25 if kind == "f16" else 0)


def forward(kind, act, T, n, m, bias=True, residual=True, kept=True, layout="tight", seed=0, in_place=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)
    t = TYPE[kind]
    x, w = rows(randn(T, n).to(t), layout), rows((randn(m, n) / n ** 0.5).to(t), layout)
    b = randn(m + 1)[1:] if layout == "odd base" else randn(m)
    r = rows(randn(T, m).to(t), layout)
    y = r if in_place else rows(torch.zeros((T, m), device="cuda", dtype=t), layout)
    z = rows(torch.zeros((T, m), device="cuda", dtype=t), layout)
    r64 = r.t.double().clone()
    check(capi.load_library().ts2_op_linear_forward(0, stream(), KIND[kind], ACT[act], T, n, m, x.ptr, x.ld, w.ptr, w.ld, ptr(b) if bias else None,
                                                    r.ptr if residual else None, r.ld, y.ptr, y.ld, z.ptr if kept else None, z.ld))
    x64, w64 = x.t.double(), w.t.double()
    z64 = x64 @ w64.T + (b.double() if bias else 0)
    y64 = ACT64[act](z64) + (r64 if residual else 0)
    sums = (n / 8 + 8) * 2.0 ** -23 * (x64.abs() @ w64.abs().T + 3)
    near(y.t, y64, half_step(kind, y64) + 1.01 * (1.13 * sums + 2.0 ** -21 * (1 + z64.abs())))
    assert y.around_is_kept()
    if kept:
        near(z.t, z64, half_step(kind, z64) + 1.01 * sums)
        assert z.around_is_kept()
    for a in (x, w):
        assert torch.equal(a.flat, a.keep)


@pytest.mark.parametrize("T,n,m", SIZES)
@pytest.mark.parametrize("kind,act", [("f16", "gelu"), ("bf16", "silu"), ("bf16", "none"), ("f16", "relu")])
def test_forward(T, n, m, kind, act):
    forward(kind, act, T, n, m, seed=T + n + m)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("T,n,m", [(1, 77, 90), (5, 512, 136), (32, 264, 1000), (200, 333, 335), (1030, 600, 264)])
def test_forward_layouts(T, n, m, layout):
    forward("bf16", "gelu", T, n, m, layout=layout, seed=T)
    forward("f16", "none", T, n, m, layout=layout, seed=T, bias=False, kept=False)


@pytest.mark.parametrize("T", [1, 9, 40, 700])
@pytest.mark.parametrize("bias,residual,kept", [(a, b, c) for a in (0, 1) for b in (0, 1) for c in (0, 1)])
def test_forward_with_and_without(T, bias, residual, kept):
    forward("f16", "silu", T, 192, 328, bias, residual, kept, seed=T)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("T,n,m", [(1, 256, 264), (20, 256, 264), (600, 256, 520), (70, 8192, 136)])
def test_residual_in_place(T, n, m, layout):
    forward("bf16", "none", T, n, m, layout=layout, seed=1, in_place=True)


def backward(kind, act, T, n, m, dw_kind=None, layout="tight", seed=0, wants=("dx", "dw", "dbias")):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen)
    t, dw_kind = TYPE[kind], dw_kind or kind
    x, w, dy, z = rows(randn(T, n).to(t), layout), rows((randn(m, n) / n ** 0.5).to(t), layout), rows(randn(T, m).to(t), layout), rows(randn(T, m).to(t), layout)
    dx = rows(torch.zeros((T, n), device="cuda", dtype=t), layout)
    dw = rows(randn(m, n).to(TYPE.get(dw_kind, torch.float32)), layout)
    old = dw.t.double().clone() if dw_kind == "f32_add" else 0
    db = torch.full((m + 2,), 7.0, device="cuda")
    check(capi.load_library().ts2_op_linear_backward(0, stream(), KIND[kind], ACT[act], T, n, m, dy.ptr, dy.ld, z.ptr if act != "none" else None, z.ld,
                                                     x.ptr if "dw" in wants else None, x.ld, w.ptr if "dx" in wants else None, w.ld,
                                                     dx.ptr if "dx" in wants else None, dx.ld, KIND[dw_kind], dw.ptr if "dw" in wants else None, dw.ld,
                                                     ptr(db[1:]) if "dbias" in wants else None))
    z64 = z.t.double().requires_grad_(True)
    d64 = torch.autograd.grad(ACT64[act](z64), z64, dy.t.double())[0] if act != "none" else dy.t.double()
    # of dz: its functions, and the rounding before the products
    own = 2.0 ** -20 * dy.t.double().abs() if act not in ("none", "relu") else 0 * d64
    dz_off = own + (half_step(kind, d64) if act != "none" else 0)
    x64, w64 = x.t.double(), w.t.double()
    if "dx" in wants:
        want = d64 @ w64
        near(dx.t, want, half_step(kind, want) + 1.01 * (dz_off @ w64.abs() + (m / 8 + 8) * 2.0 ** -23 * (d64.abs() @ w64.abs())))
        assert dx.around_is_kept()
    if "dw" in wants:
        want = d64.T @ x64 + old
        near(dw.t, want, half_step("f32" if dw_kind == "f32_add" else dw_kind, want) +
             1.01 * (dz_off.T @ x64.abs() + (T / 8 + 8) * 2.0 ** -23 * (d64.abs().T @ x64.abs())))
        assert dw.around_is_kept()
    if "dbias" in wants:
        near(db[1:-1], d64.sum(0), 1.01 * (own.sum(0) + (T / 16 + 40) * 2.0 ** -24 * d64.abs().sum(0)))
    assert db[0] == 7 and db[-1] == 7
    for a in (x, w, dy, z):
        assert torch.equal(a.flat, a.keep)


@pytest.mark.parametrize("T,n,m", SIZES)
@pytest.mark.parametrize("kind,act", [("f16", "gelu"), ("bf16", "silu"), ("bf16", "none"), ("f16", "relu")])
def test_backward(T, n, m, kind, act):
    backward(kind, act, T, n, m, seed=T + n + m)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("T,n,m", [(1, 77, 90), (200, 333, 335), (1030, 600, 264)])
@pytest.mark.parametrize("dw_kind", ["bf16", "f32", "f32_add"])
def test_backward_layouts(T, n, m, layout, dw_kind):
    backward("bf16", "gelu", T, n, m, dw_kind, layout, seed=T)
    backward("bf16", "none", T, n, m, dw_kind, layout, seed=T)


@pytest.mark.parametrize("wants", [("dx",), ("dw",), ("dbias",), ("dx", "dbias"), ("dw", "dbias"), ("dx", "dw"), ()])
@pytest.mark.parametrize("act", ["none", "silu"])
def test_backward_of_some(wants, act):
    backward("f16", act, 500, 136, 264, wants=wants)


@pytest.mark.parametrize("dw_kind", ["f16", "f32", "f32_add"])
def test_long_sums_of_few_tiles(dw_kind):
    """many tokens and a small matrix: K ranges"""
    backward("f16", "none", 40000, 96, 40, dw_kind)
    backward("f16", "gelu", 9000, 513, 260, dw_kind)


def test_no_tokens():
    lib = capi.load_library()
    w = torch.ones((8, 16), device="cuda", dtype=torch.float16)
    check(lib.ts2_op_linear_forward(0, stream(), KIND["f16"], ACT["none"], 0, 16, 8, None, 16, ptr(w), 16, None, None, 8, None, 8, None, 8))
    for kind, dtype, left in (("f16", torch.float16, 0), ("f32", torch.float32, 0), ("f32_add", torch.float32, 7)):
        dw, db = torch.full((8, 20), 7.0, device="cuda", dtype=dtype), torch.full((8,), 7.0, device="cuda")
        check(lib.ts2_op_linear_backward(0, stream(), KIND["f16"], ACT["gelu"], 0, 16, 8, None, 8, None, 8, None, 16, ptr(w), 16, None, 16, KIND[kind], ptr(dw), 20,
                                         ptr(db)))
        assert (dw[:, :16] == left).all() and (dw[:, 16:] == 7).all() and (db == 0).all()


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_backward_against_differences(act):
    """the gradient of sum(dy y) along random directions, by central differences of the formula in float64"""
    gen = torch.Generator(device="cuda").manual_seed(5)
    randn = lambda *s: torch.randn(s, device="cuda", generator=gen, dtype=torch.float64)
    T, n, m = 96, 72, 40
    x, w, b, dy = randn(T, n).half(), (randn(m, n) / 8).half(), randn(m).float(), randn(T, m).half()
    z = (x.double() @ w.double().T + b.double()).half()
    dx, dw, db = torch.zeros_like(x), torch.zeros((m, n), device="cuda"), torch.zeros(m, device="cuda")
    check(capi.load_library().ts2_op_linear_backward(0, stream(), KIND["f16"], ACT[act], T, n, m, ptr(dy), m, ptr(z), m, ptr(x), n, ptr(w), n, ptr(dx), n,
                                                     KIND["f32"], ptr(dw), n, ptr(db)))
    f = lambda x, w, b: (ACT64[act](x @ w.T + b) * dy.double()).sum()
    for of in range(3):
        base = [x.double(), w.double(), b.double()]
        d = randn(*base[of].shape)
        e = 1e-5
        up, down = ([a + s * e * d if i == of else a for i, a in enumerate(base)] for s in (1, -1))
        want = (f(*up) - f(*down)) / (2 * e)
        got = ((dx, dw, db)[of].double() * d).sum()
        # z and dz are rounded to fp16: 2^-11 each of terms that add up like independent ones; a kink of relu passed by z's rounding moves one dy in 2^-9
        size = ((dx, dw, db)[of].double() ** 2 * d ** 2).sum().sqrt() + (dy.double() ** 2).sum().sqrt()
        assert abs(got - want) < 8 * 2.0 ** -9 * size, (of, got, want)


def test_infinities_and_nans_stay_where_they_are():
    T, n, m = 40, 64, 96
    x = torch.zeros((T, n), device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    x[3, 0], x[5, 0], x[7, 0] = float("inf"), float("nan"), float("-inf")
    w = torch.ones((m, n), device="cuda", dtype=torch.bfloat16)
    w[:, 1:] = 0
    for act in ("relu", "gelu"):
        y = torch.zeros((T, m), device="cuda", dtype=torch.bfloat16)
        check(capi.load_library().ts2_op_linear_forward(0, stream(), KIND["bf16"], ACT[act], T, n, m, ptr(x[:, :1]), n, ptr(w), n, None, None, m, ptr(y), m, None, m))
        # 0 * inf in the other columns of x makes none: they are zeros times zeros
        assert torch.isnan(y[5]).all() and (y[3] == float("inf")).all() and (y[7] == 0).all()
        rest = [i for i in range(T) if i not in (3, 5, 7)]
        assert torch.isfinite(y[rest]).all()


def test_fp16_saturates():
    x = torch.full((3, 64), 200.0, device="cuda", dtype=torch.float16)
    y, z = torch.zeros((3, 8), device="cuda", dtype=torch.float16), torch.zeros((3, 8), device="cuda", dtype=torch.float16)
    check(capi.load_library().ts2_op_linear_forward(0, stream(), KIND["f16"], ACT["relu"], 3, 64, 8, ptr(x), 64, ptr(x.repeat(3, 1)), 64, None, None, 8, ptr(y), 8, ptr(z), 8))
    assert (y == 65504).all() and (z == 65504).all()


@pytest.mark.parametrize("T", [3, 100, 2000])
def test_same_bits_on_another_stream_and_replayed(T):
    n, m = 520, 264
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w, dy = (torch.randn(s, device="cuda", generator=gen).half() for s in ((T, n), (m, n), (T, m)))
    lib = capi.load_library()

    def step(out):
        y, z, dx, dw, db = out
        check(lib.ts2_op_linear_forward(0, stream(), KIND["f16"], ACT["gelu"], T, n, m, ptr(x), n, ptr(w), n, ptr(bias), None, m, ptr(y), m, ptr(z), m))
        check(lib.ts2_op_linear_backward(0, stream(), KIND["f16"], ACT["gelu"], T, n, m, ptr(dy), m, ptr(z), m, ptr(x), n, ptr(w), n, ptr(dx), n, KIND["f32"], ptr(dw), n,
                                         ptr(db)))

    bias = torch.randn(m, device="cuda", generator=gen)
    outs = [[torch.zeros(s, device="cuda", dtype=d) for s, d in (((T, m), torch.half), ((T, m), torch.half), ((T, n), torch.half), ((m, n), torch.float32), ((m,), torch.float32))]
            for _ in range(4)]
    step(outs[0])
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        step(outs[1])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, o in zip(graphs, outs[2:]):
        with torch.cuda.graph(g, stream=other):
            step(o)
    for _ in range(3):
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
    torch.cuda.synchronize()
    for o in outs[1:]:
        for a, b in zip(outs[0], o):
            assert torch.equal(a, b)


def test_beyond_32_bit_offsets():
    """a pitch of a million elements and a few thousand rows"""
    T, n, m, pitch = 2200, 40, 24, 1_000_000
    flat = torch.zeros(T * pitch, device="cuda", dtype=torch.float16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, y, z, dy, dx = (flat.as_strided((T, k), (pitch, 1), 64 * i) for i, k in enumerate((n, m, m, m, n)))
    x.copy_(torch.randn((T, n), device="cuda", generator=gen))
    dy.copy_(torch.randn((T, m), device="cuda", generator=gen))
    w = torch.randn((m, n), device="cuda", generator=gen).half()
    dw = torch.zeros((m, n), device="cuda", dtype=torch.float16)
    lib = capi.load_library()
    check(lib.ts2_op_linear_forward(0, stream(), KIND["f16"], ACT["relu"], T, n, m, ptr(x), pitch, ptr(w), n, None, None, m, ptr(y), pitch, ptr(z), pitch))
    check(lib.ts2_op_linear_backward(0, stream(), KIND["f16"], ACT["relu"], T, n, m, ptr(dy), pitch, ptr(z), pitch, ptr(x), pitch, ptr(w), n, ptr(dx), pitch, KIND["f16"],
                                     ptr(dw), n, None))
    z64 = x.double() @ w.double().T
    near(z, z64, half_step("f16", z64) + 2.0 ** -19 * (x.double().abs() @ w.double().abs().T))
    dz = dy.double() * (z > 0)
    near(dx, dz @ w.double(), half_step("f16", dz @ w.double()) + 2.0 ** -19 * (dz.abs() @ w.double().abs()))
    want = dz.T @ x.double()
    near(dw, want, half_step("f16", want) + (T / 8 + 8) * 2.0 ** -23 * (dz.abs().T @ x.double().abs()))


def test_more_than_32_bits_of_outputs():
    """2.3e9 results, kept ones and gradients: the last rows, and dw over all of them"""
    T, n, m = 290_001, 64, 8000
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w = torch.randn((T, n), device="cuda", generator=gen).bfloat16(), (torch.randn((m, n), device="cuda", generator=gen) / 8).bfloat16()
    y, z = (torch.zeros((T, m), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    lib = capi.load_library()
    check(lib.ts2_op_linear_forward(0, stream(), KIND["bf16"], ACT["relu"], T, n, m, ptr(x), n, ptr(w), n, None, None, m, ptr(y), m, ptr(z), m))
    tail = slice(T - 300, T)
    z64 = x[tail].double() @ w.double().T
    off = 20 * 2.0 ** -23 * (x[tail].double().abs() @ w.double().abs().T)
    near(z[tail], z64, half_step("bf16", z64) + off)
    near(y[tail], z64.clamp(min=0), half_step("bf16", z64) + off)
    dx, dw = torch.zeros_like(x), torch.zeros((m, n), device="cuda")
    check(lib.ts2_op_linear_backward(0, stream(), KIND["bf16"], ACT["relu"], T, n, m, ptr(y), m, ptr(z), m, ptr(x), n, ptr(w), n, ptr(dx), n, KIND["f32"], ptr(dw), n, None))
    want = y[tail].double() @ w.double()  # dz = y where z > 0, and y is zero elsewhere
    near(dx[tail], want, half_step("bf16", want) + (m / 8 + 8) * 2.0 ** -23 * (y[tail].double().abs() @ w.double().abs()))
    cols = slice(m - 40, m)
    want = y[:, cols].double().T @ x.double()
    near(dw[cols], want, half_step("f32", want) + (T / 8 + 8) * 2.0 ** -23 * (y[:, cols].double().abs().T @ x.double().abs()))


@pytest.mark.parametrize("layout", ["tight", "odd pitch", "odd base"])
@pytest.mark.parametrize("n", [1, 2, 3, 31, 63, 64, 65, 510, 511, 512, 513, 1022, 1023, 1024, 1025, 2048])
def test_rows_that_are_copied_end_anywhere(n, layout):
    """rows at an odd pitch or base come in as words, 512 elements at a time"""
    forward("f16", "none", 40, n, 24, layout=layout, seed=n, bias=False, residual=False, kept=False)
    backward("f16", "none", 70, n, 40, layout=layout, seed=n)
    backward("bf16", "silu", 40, 30, n, layout=layout, seed=n)
