"""ts2_op_adamw against the formula in float64.

Tolerances.  fp32 moments: m = b1 m + c1 g has three roundings of its terms, v as well: 2^-22 of the sum of their sizes.  param: its own product and sum, 2^-23
of it, and the update's functions, 2^-20 of the update.  The copy is half a step of its type from param.  Moments in 8 bits are defined
to the bit."""
import ctypes as C

import numpy as np
import pytest

from tscale2_b200 import capi
from tscale2_b200.device import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KIND = {"f32": capi.OUT_F32, "f16": capi.OUT_F16, "bf16": capi.OUT_BF16, "none": capi.OUT_F32}
B1, B2 = float(np.float32(0.9)), float(np.float32(0.999))
RATE, EPS = float(np.float32(1e-3)), float(np.float32(1e-8))
M64 = (1 << 64) - 1


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def mix64(x):
    x = (x + 0x9E3779B97F4A7C15) & M64
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & M64
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & M64
    return x ^ (x >> 31)


def uniforms(n, seed, step, i):
    key = mix64(mix64((seed + step) & M64) ^ i) & 0xFFFFFFFF
    x = (np.arange(n, dtype=np.uint64) * 0x9E3779B1 + key).astype(np.uint32)
    x = (x ^ (x >> np.uint32(16))) * np.uint32(0x85EBCA6B)
    x = (x ^ (x >> np.uint32(13))) * np.uint32(0xC2B2AE35)
    x = x ^ (x >> np.uint32(16))
    return (x >> np.uint32(16)) / 65536.0, (x & np.uint32(0xFFFF)) / 65536.0


E4M3 = np.array([(m if e == 0 else (8 + m) * 2.0 ** (e - 1)) * 2.0 ** -9 for e in range(16) for m in range(8)])


def decode(codes, scale):
    v = E4M3[codes & 127] * np.where(codes > 127, -1.0, 1.0)
    return v * np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127)).repeat(32)[:len(codes)]


def encode(x, u, second):
    n = len(x)
    a = np.zeros(-(-n // 32) * 32)
    a[:n] = np.abs(x)
    top = a.reshape(-1, 32).max(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(top > 0, np.clip(np.floor(np.log2(top)) - 7, -127, 127), -127)
    bad = ~np.isfinite(top)
    scale = np.where(bad, 255, e + 127).astype(np.uint8)
    y = a / 2.0 ** np.where(bad, 0, e).repeat(32)
    y = np.where(bad.repeat(32), 0, y)[:n]
    step = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    q = np.floor(y / step + u) * step
    if second:
        q = np.where((y > 0) & (q == 0), 2.0 ** -9, q)
    codes = np.searchsorted(E4M3[:127], q)
    assert (E4M3[codes] == q).all()
    return (codes + np.where((np.asarray(x) < 0) & ~bad.repeat(32)[:n], 128, 0)).astype(np.uint8), scale


class Tensor:
    def __init__(self, n, gen, grad="f32", bits=32, copy="none", rate=1.0, decay=0.1, off=0, size=1.0):
        new = lambda k, d: torch.zeros(k + off + 9, device="cuda", dtype=d)
        cut = lambda a, k=n: a[off:off + k]
        randn = lambda: torch.randn(n, device="cuda", generator=gen)
        self.n, self.bits, self.rate, self.decay, self.off = n, bits, float(np.float32(rate)), float(np.float32(decay)), off
        self.all = {"param": new(n, torch.float32), "grad": new(n, TYPE[grad])}
        state = torch.float32 if bits == 32 else torch.uint8
        self.all["m"], self.all["v"] = new(n, state), new(n, state)
        nb = -(-n // 32)
        if bits == 8:
            self.all["m_scale"], self.all["v_scale"] = new(nb, torch.uint8), new(nb, torch.uint8)
        if copy != "none":
            self.all["copy"] = new(n, TYPE[copy])
        self.view = {k: cut(a, nb if "scale" in k else n) for k, a in self.all.items()}
        self.view["param"].copy_(randn())
        self.view["grad"].copy_(size * randn())
        if bits == 32:
            self.view["m"].copy_(0.5 * size * randn())
            self.view["v"].copy_(0.3 * size * size * torch.rand(n, device="cuda", generator=gen))
        else:
            rows = torch.exp(2 * torch.randn(nb, device="cuda", generator=gen)).repeat_interleave(32)[:n]
            for k, x in (("m", 0.5 * size * rows * randn()), ("v", 0.3 * (size * rows) ** 2 * torch.rand(n, device="cuda", generator=gen))):
                c, s = encode(x.double().cpu().numpy(), 0.5, k == "v")
                self.view[k].copy_(torch.from_numpy(c))
                self.view[k + "_scale"].copy_(torch.from_numpy(s))
        for k, a in self.all.items():  # what lies around has to stay
            a[:off], a[off + self.view[k].numel():] = 5, 5

    def record(self, r):
        for k in ("param", "grad", "m", "v", "m_scale", "v_scale", "copy"):
            setattr(r, k, self.view[k].data_ptr() if k in self.view and self.n else None)
        r.n, r.rate, r.decay = self.n, self.rate, self.decay

    def host(self):
        return {k: a.double().cpu().numpy() if a.is_floating_point() else a.cpu().numpy() for k, a in self.view.items()}


def table_of(tensors):
    table = (capi.AdamwTensor * max(1, len(tensors)))()
    for r, t in zip(table, tensors):
        t.record(r)
    return table


def call(tensors, grad, bits, copy, step=7, scale=0.5, dev=None, seed=11, table=None):
    table = table if table is not None else table_of(tensors)
    check(capi.load_library().ts2_op_adamw(0, stream(), KIND[grad], bits, KIND[copy], C.cast(table, C.c_void_p), len(tensors), RATE, B1, B2, EPS, step, scale,
                                           None if dev is None else dev.data_ptr(), seed))


def verify(tensors, grad, bits, copy, step=7, scale=0.5, dev=None, seed=11):
    before = [t.host() for t in tensors]
    call(tensors, grad, bits, copy, step, scale, dev, seed)
    torch.cuda.synchronize()
    factor = np.float32(np.float32(scale) * np.float32(1 if dev is None else dev.item()))
    for i, (t, o) in enumerate(zip(tensors, before)):
        now = t.host()
        with np.errstate(invalid="ignore", over="ignore"):
            g = (o["grad"].astype(np.float32) * factor).astype(np.float64)
            if bits == 32:
                m0, v0 = o["m"], o["v"]
            else:
                m0, v0 = decode(o["m"], o["m_scale"]), decode(o["v"], o["v_scale"])
            m, v = B1 * m0 + (1 - B1) * g, B2 * v0 + (1 - B2) * g * g
            if bits == 32:
                assert (np.abs(now["m"] - m) <= 2.0 ** -22 * (np.abs(B1 * m0) + np.abs((1 - B1) * g)) + 1e-44).all()
                assert (np.abs(now["v"] - v) <= 2.0 ** -22 * v + 1e-44).all()
            else:
                u = uniforms(t.n, seed, step, i)
                for k, x, uu in (("m", m, u[0]), ("v", v, u[1])):
                    code, s = encode(x, uu, k == "v")
                    assert np.array_equal(now[k + "_scale"], s), (k, i)
                    # a double that a compiler sums in another order may round another way once in 2^40
                    assert np.array_equal(now[k], code), (k, i, (now[k] != code).nonzero()[0][:5])
            r = RATE * t.rate
            up = r * m / (1 - B1 ** step) / (np.sqrt(v / (1 - B2 ** step)) + EPS)
            # m's two terms may cancel: m is off by its own roundings of them, 2^-22 of their sizes, and the update by as much of what they would make
            terms = r * (np.abs(B1 * m0) + np.abs((1 - B1) * g)) / (1 - B1 ** step) / (np.sqrt(v / (1 - B2 ** step)) + EPS)
            want = o["param"] * (1 - r * t.decay) - up
            fine = np.isfinite(want)
            assert np.array_equal(fine, np.isfinite(now["param"]))
            assert (np.abs(now["param"] - want) <= 2.0 ** -23 * (np.abs(want) + np.abs(o["param"])) + 2.0 ** -20 * np.abs(up) + 2.0 ** -22 * terms)[fine].all()
            if "copy" in now:
                tiny = 2.0 ** -25 if copy == "f16" else 0
                p = now["param"]
                assert (np.abs(now["copy"] - p) <= torch.finfo(TYPE[copy]).eps / 2 * np.abs(p) + tiny)[fine].all()
        for k, a in t.all.items():
            n = t.view[k].numel()
            assert (a[:t.off].double() == 5).all() and (a[t.off + n:].double() == 5).all(), k


SIZES = [1, 2, 31, 32, 33, 127, 1000, 4095, 4096, 4097, 12289, 100_003]


@pytest.mark.parametrize("off", [0, 1, 2, 4])
@pytest.mark.parametrize("grad,copy", [("f32", "none"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("bits", [32, 8])
def test_step(bits, grad, copy, off):
    gen = torch.Generator(device="cuda").manual_seed(bits + off)
    ts = [Tensor(n, gen, grad, bits, copy, off=off, rate=1 + 0.1 * i, decay=0.01 * i) for i, n in enumerate(SIZES)]
    verify(ts, grad, bits, copy)
    verify(ts, grad, bits, copy, step=8)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [0, 1, 32, 33, 129, 400, 401, 1000])
def test_many_tensors(bits, count):
    gen = torch.Generator(device="cuda").manual_seed(count)
    sizes = np.random.default_rng(count).integers(0, 300, count)
    verify([Tensor(int(n), gen, "bf16", bits, "f16") for n in sizes], "bf16", bits, "f16")


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_elements_and_without_copies(bits):
    gen = torch.Generator(device="cuda").manual_seed(1)
    ts = [Tensor(n, gen, "f32", bits, "bf16") for n in (0, 50, 0, 0, 5000, 0)]
    ts[4].view.pop("copy"), ts[4].all.pop("copy")
    verify(ts, "f32", bits, "bf16")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("step", [1, 2, 1000, 10 ** 9])
@pytest.mark.parametrize("scale,dev", [(1.0, None), (-1.0, 0.25), (2.0 ** -12, 3.0)])
def test_steps_and_scales(bits, step, scale, dev):
    gen = torch.Generator(device="cuda").manual_seed(1)
    d = None if dev is None else torch.tensor([dev], device="cuda")
    verify([Tensor(n, gen, "f32", bits) for n in (640, 33)], "f32", bits, "none", step, scale, d, seed=(1 << 64) - 3)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size", [1e-12, 1e-6, 1e6, 1e15])
def test_sizes_of_gradients(bits, size):
    gen = torch.Generator(device="cuda").manual_seed(1)
    verify([Tensor(2000, gen, "f32", bits, size=size)], "f32", bits, "none")


def test_first_step_from_zero_bytes():
    gen = torch.Generator(device="cuda").manual_seed(1)
    t = Tensor(1000, gen, "f32", 8)
    for k in ("m", "v", "m_scale", "v_scale"):
        t.view[k].zero_()
    t.view["grad"][100:200] = 0
    verify([t], "f32", 8, "none", step=1)
    assert (t.view["m"][128:160] == 0).all() and (t.view["v"][128:160] == 0).all()


def test_a_gradient_that_is_not_finite():
    gen = torch.Generator(device="cuda").manual_seed(1)
    for bits in (32, 8):
        for bad in (float("nan"), float("inf"), float("-inf")):
            t = Tensor(256, gen, "f32", bits)
            t.view["grad"][40] = bad
            before = t.view["param"].clone()
            call([t], "f32", bits, "none")
            p = t.view["param"]
            assert not torch.isfinite(p[40]) and torch.isfinite(p[:40]).all() and torch.isfinite(p[41:]).all() and (p[:40] != before[:40]).any()
            t.view["grad"][40] = 0
            call([t], "f32", bits, "none")
            p = t.view["param"]
            gone = slice(32, 64) if bits == 8 else slice(40, 41)
            assert torch.isnan(p[gone]).all() and torch.isfinite(p).sum() == 256 - (32 if bits == 8 else 1)


def test_slow_averages_move_as_their_expectation():
    """without gradients v falls by a thousandth a step, which is far below a step of e4m3: after 500 steps the mean over many elements is 0.999^500 of what it
    was.  A step's rounding moves a value by a step s of it with odds of about 0.001 / s, a variance of 0.001 s < 1.3e-4 (relative); over 500 steps and
    32768 elements the mean's deviation is below sqrt(500 * 1.3e-4 / 32768) = 1.4e-3: six of them"""
    gen = torch.Generator(device="cuda").manual_seed(1)
    t = Tensor(32768, gen, "f32", 8)
    t.view["grad"].zero_()
    x = np.full(32768, 3.0)
    code, s = encode(x, 0.5, True)
    t.view["v"].copy_(torch.from_numpy(code)), t.view["v_scale"].copy_(torch.from_numpy(s))
    table = table_of([t])
    for k in range(500):
        call([t], "f32", 8, "none", step=k + 1, table=table)
    now = decode(t.view["v"].cpu().numpy(), t.view["v_scale"].cpu().numpy())
    assert abs(now.mean() / (3.0 * B2 ** 500) - 1) < 6 * 1.4e-3


def test_same_bits_on_another_stream_and_replayed():
    gen = torch.Generator(device="cuda").manual_seed(1)
    for bits in (32, 8):
        sets = []
        for _ in range(3):
            gen.manual_seed(4)
            sets.append([Tensor(n, gen, "bf16", bits, "bf16", off=o) for n, o in ((10_000, 0), (777, 3), (64, 0))])
        for step in (5, 5):
            call(sets[0], "bf16", bits, "bf16", step)
        torch.cuda.synchronize()
        other, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(other):
            for step in (5, 5):
                call(sets[1], "bf16", bits, "bf16", step)
        with torch.cuda.graph(g, stream=other):
            call(sets[2], "bf16", bits, "bf16", 5)  # the table may go after the call
        g.replay()
        g.replay()
        torch.cuda.synchronize()
        for s in sets[1:]:
            for a, b in zip(sets[0], s):
                assert all(torch.equal(a.view[k], b.view[k]) for k in a.view)


def test_elements_beyond_32_bits():
    """a tensor of 2^31 elements and some: its last ones, and the ones on both sides of 2^31"""
    n, seed, step = (1 << 31) + 1000, 5, 3
    gen = torch.Generator(device="cuda").manual_seed(1)
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    m, v = (torch.zeros(n, device="cuda", dtype=torch.uint8) for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 32), device="cuda", dtype=torch.uint8) for _ in range(2))
    at = [(1 << 31) - 64, n - 40]
    parts = [slice(a, min(n, a + 128)) for a in at]
    for s in parts:
        g[s] = torch.randn(s.stop - s.start, device="cuda", generator=gen)
    table = (capi.AdamwTensor * 1)()
    t = table[0]
    t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.copy, t.n, t.rate, t.decay = *(x.data_ptr() for x in (p, g, m, v, ms, vs)), None, n, 1.0, 0.0
    check(capi.load_library().ts2_op_adamw(0, stream(), KIND["bf16"], 8, KIND["none"], C.cast(table, C.c_void_p), 1, RATE, B1, B2, EPS, step, 1.0, None, seed))
    key = mix64(mix64((seed + step) & M64) ^ 0) & 0xFFFFFFFF
    for s in parts:
        first = s.start // 32 * 32
        w = slice(first, s.stop)
        grad = g[w].double().cpu().numpy()
        x = ((np.arange(w.start, w.stop, dtype=np.uint64) * 0x9E3779B1 + key) & 0xFFFFFFFF).astype(np.uint32)
        x = (x ^ (x >> np.uint32(16))) * np.uint32(0x85EBCA6B)
        x = (x ^ (x >> np.uint32(13))) * np.uint32(0xC2B2AE35)
        x = x ^ (x >> np.uint32(16))
        for state, scale, now, u, second in ((m, ms, (1 - B1) * grad, x >> np.uint32(16), False), (v, vs, (1 - B2) * grad * grad, x & np.uint32(0xFFFF), True)):
            code, sc = encode(now, u / 65536.0, second)
            assert np.array_equal(state[w].cpu().numpy(), code)
            assert np.array_equal(scale[first // 32:-(-w.stop // 32)].cpu().numpy(), sc)
        want = -RATE * (1 - B1) * grad / (1 - B1 ** step) / (np.sqrt((1 - B2) * grad * grad / (1 - B2 ** step)) + EPS)
        assert (np.abs(p[w].double().cpu().numpy() - want) <= 2.0 ** -20 * np.abs(want)).all()
    assert (p[: 1 << 20] == 0).all() and (p[1 << 30: (1 << 30) + (1 << 20)] == 0).all()
