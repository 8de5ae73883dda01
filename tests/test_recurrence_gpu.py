"""The gated linear recurrence (ts2_op_recurrence_forward / _backward) against its formula in float64, element by element.

Tolerance: with e = exp(-gate), a kernel that computes in fp32 has e to 2^-22 (the exponential) + 1.5 |gate| 2^-24 (its rounded
argument), so a and 1 - a to r = 2^-22 + 1.5 |gate| 2^-24 + 2^-22 (sum, quotient, product), and one step of the recurrence adds at
most (r + 2^-23) of the magnitudes that it sums.  Folding groups of nodes into maps before they are applied multiplies the same
factors in another order: twice that.  The bound goes through the recurrence itself (`slack`), and the rounding of the result to
its type adds half a step.  fp16: values below the normal range have an absolute half step of 2^-25."""
import ctypes as C

import ml_dtypes
import numpy as np
import pytest

from tscale2_b200 import capi
from tscale2_b200.device import DeviceBuffer, check, sync

pytestmark = pytest.mark.gpu

KIND = {"f32": capi.OUT_F32, "f16": capi.OUT_F16, "bf16": capi.OUT_BF16}
TYPE = {"f32": np.float32, "f16": np.float16, "bf16": ml_dtypes.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def sigmoid(g):
    return 1 / (1 + np.exp(-g))


def rate(g):
    return 2 * (2.0 ** -21 + 1.5 * np.abs(g) * 2.0 ** -24 + 2.0 ** -23)


def forward(gate, x, ptr, h0):
    """h, h_last and how far fp32 may be off them"""
    g, x = gate.astype(np.float64), x.astype(np.float64)
    a, k, r = sigmoid(g), sigmoid(-g), rate(np.where(np.isfinite(g), g, 0))
    h, slack, big = np.zeros_like(g), np.zeros_like(g), np.zeros_like(g)
    n = len(ptr) - 1
    last, last_slack = np.zeros((n, g.shape[1])), np.zeros((n, g.shape[1]))
    for s in range(n):
        now = h0[s].astype(np.float64) if h0 is not None else np.zeros(g.shape[1])
        mag, off = np.abs(now), np.zeros(g.shape[1])
        for t in range(ptr[s], ptr[s + 1]):
            now = a[t] * now + k[t] * x[t]
            mag = a[t] * mag + k[t] * np.abs(x[t])
            off = a[t] * off + r[t] * mag
            h[t], slack[t], big[t] = now, off, mag
        last[s], last_slack[s] = now, off + 2.0 ** -24 * mag
    return h, last, slack, last_slack


def backward(gate, x, h, ptr, h0, dh, dh_last):
    g, x, h, dh = (v.astype(np.float64) for v in (gate, x, h, dh))
    a, k, r = sigmoid(g), sigmoid(-g), rate(g)
    dgate, dx, sg, sx = (np.zeros_like(g) for _ in range(4))
    n = len(ptr) - 1
    dh0, s0 = np.zeros((n, g.shape[1])), np.zeros((n, g.shape[1]))
    for s in range(n):
        f = dh_last[s].astype(np.float64) if dh_last is not None else np.zeros(g.shape[1])
        mag, off = np.abs(f), np.zeros(g.shape[1])
        for t in range(ptr[s + 1] - 1, ptr[s] - 1, -1):
            e = dh[t] + f
            mag = np.abs(dh[t]) + mag
            off = off + 2.0 ** -23 * mag
            before = h[t - 1] if t > ptr[s] else (h0[s].astype(np.float64) if h0 is not None else 0 * e)
            w = before - x[t]
            dx[t], sx[t] = k[t] * e, k[t] * (off + 2 * r[t] * mag)
            dgate[t], sg[t] = a[t] * k[t] * w * e, a[t] * k[t] * np.abs(w) * (off + 4 * r[t] * mag)
            f, off, mag = a[t] * e, a[t] * off + r[t] * a[t] * mag, a[t] * mag
        dh0[s], s0[s] = f, off + 2.0 ** -24 * mag
    return dgate, dx, dh0, sg, sx, s0


def near(got, want, slack, kind):
    got = got.astype(np.float64)
    tol = slack + HALF_STEP[kind] * (np.abs(want) + slack) + (2.0 ** -25 if kind == "f16" else 0)
    worst = np.max((np.abs(got - want) - tol), initial=-1.0)
    assert worst <= 0, f"{worst:.3e} beyond the bound"


class Case:
    """Host arrays and their copies on the device, rows of `pitch` elements from an element offset on; what lies between and
    outside of the rows holds a pattern that has to survive."""

    def __init__(self, kind, T, D, ptr, carry, seed, pitch=None, offset=0, low=-3.0, high=6.0):
        rng = np.random.default_rng(seed)
        self.kind, self.T, self.D, self.t = kind, T, D, TYPE[kind]
        self.ptr = np.asarray(ptr, np.int32)
        self.n = len(ptr) - 1
        self.pitch, self.offset = pitch or D, offset
        self.gate = rng.uniform(low, high, (T, D)).astype(self.t)
        self.x = rng.standard_normal((T, D)).astype(self.t)
        self.h0 = rng.standard_normal((self.n, D)).astype(np.float32) if carry else None
        self.dh = rng.standard_normal((T, D)).astype(self.t)
        self.dh_last = rng.standard_normal((self.n, D)).astype(np.float32) if carry else None

    def put(self, a):
        flat = np.full(self.offset + max(self.T, 1) * self.pitch, 7, self.t)
        if a is not None:
            flat[self.offset:self.offset + self.T * self.pitch].reshape(self.T, self.pitch)[:, :self.D] = a
        return DeviceBuffer.from_numpy(flat.view(np.uint8))

    def at(self, buf):
        return buf.ptr + self.offset * np.dtype(self.t).itemsize

    def get(self, buf):
        flat = buf.download(buf.nbytes, np.uint8).view(self.t)
        rows = flat[self.offset:self.offset + self.T * self.pitch].reshape(self.T, self.pitch)
        assert (flat[:self.offset] == 7).all() and (rows[:, self.D:] == 7).all()
        lo, hi = int(self.ptr[0]), int(self.ptr[-1])
        assert (rows[:lo] == 7).all() and (rows[hi:] == 7).all(), "nodes outside of the sequences were written"
        return rows[:, :self.D]

    def forward(self, stream=None, null_ptr=False):
        lib = capi.load_library()
        f = lambda a: None if a is None else DeviceBuffer.from_numpy(a)
        g, x, h, p, h0 = self.put(self.gate), self.put(self.x), self.put(None), DeviceBuffer.from_numpy(self.ptr), f(self.h0)
        last = DeviceBuffer.from_numpy(np.full((self.n, self.D), 7, np.float32)) if self.h0 is not None else None
        check(lib.ts2_op_recurrence_forward(0, stream, KIND[self.kind], self.at(g), self.pitch, self.at(x), self.pitch, self.T, self.D, self.n,
                                            None if null_ptr else p.ptr, h0 and h0.ptr, self.at(h), self.pitch, last and last.ptr))
        sync()
        return self.get(h), last and last.download((self.n, self.D), np.float32)

    def backward(self, h, null_ptr=False):
        lib = capi.load_library()
        f = lambda a: None if a is None else DeviceBuffer.from_numpy(a)
        g, x, hh, dh, dg, dx = (self.put(a) for a in (self.gate, self.x, h, self.dh, None, None))
        p, h0, dl = DeviceBuffer.from_numpy(self.ptr), f(self.h0), f(self.dh_last)
        dh0 = DeviceBuffer.from_numpy(np.full((self.n, self.D), 7, np.float32)) if self.h0 is not None else None
        check(lib.ts2_op_recurrence_backward(0, None, KIND[self.kind], self.at(g), self.pitch, self.at(x), self.pitch, self.at(hh), self.pitch,
                                             self.T, self.D, self.n, None if null_ptr else p.ptr, h0 and h0.ptr, self.at(dh), self.pitch,
                                             dl and dl.ptr, self.at(dg), self.pitch, self.at(dx), self.pitch, dh0 and dh0.ptr))
        sync()
        return self.get(dg), self.get(dx), dh0 and dh0.download((self.n, self.D), np.float32)

    def verify(self, null_ptr=False):
        want, want_last, slack, last_slack = forward(self.gate, self.x, self.ptr, self.h0)
        h, last = self.forward(null_ptr=null_ptr)
        lo, hi = int(self.ptr[0]), int(self.ptr[-1])
        near(h[lo:hi], want[lo:hi], slack[lo:hi], self.kind)
        if last is not None:
            near(last, want_last, last_slack, "f32")
        given = want.astype(self.t)
        dg, dx, dh0, sg, sx, s0 = backward(self.gate, self.x, given, self.ptr, self.h0, self.dh, self.dh_last)
        got = self.backward(given, null_ptr=null_ptr)
        near(got[0][lo:hi], dg[lo:hi], sg[lo:hi], self.kind)
        near(got[1][lo:hi], dx[lo:hi], sx[lo:hi], self.kind)
        if dh0 is not None and got[2] is not None:
            near(got[2], dh0, s0, "f32")


def cut(T, n, seed, first=0, pad=0):
    rng = np.random.default_rng(seed)
    inner = np.sort(rng.integers(first, T - pad + 1, n - 1))
    return [first, *inner.tolist(), T - pad]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,D,n,carry", [(1, 1, 1, True), (2, 64, 1, False), (17, 130, 1, True), (128, 64, 1, True), (129, 96, 2, True),
                                         (1000, 33, 5, True), (777, 200, 40, True), (2500, 64, 3, False), (300, 768, 1, False)])
def test_against_the_formula(kind, T, D, n, carry):
    Case(kind, T, D, cut(T, n, T + D), carry, seed=T * D).verify()


@pytest.mark.parametrize("kind,T,D,n,carry", [("f16", 20000, 24, 30, True), ("bf16", 20000, 23, 3, True), ("f32", 15000, 22, 1, True),
                                              ("f16", 9000, 130, 400, False), ("f32", 12000, 65, 1, False)])
def test_long_arrays_in_segments(kind, T, D, n, carry):
    Case(kind, T, D, cut(T, n, n + D, first=3, pad=5), carry, seed=T + D).verify()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_one_sequence_without_a_table(kind):
    Case(kind, 500, 70, [0, 500], True, seed=3).verify(null_ptr=True)


@pytest.mark.parametrize("T,D", [(513, 256), (1, 300), (64, 65)])
def test_every_token_its_own_sequence(T, D):
    Case("f16", T, D, list(range(T + 1)), True, seed=T).verify()


def test_empty_sequences_pass_their_state_on():
    ptr = [0] * 40 + [3, 3, 3] + [64] * 70 + [65, 200] + [200] * 5
    Case("f32", 200, 66, ptr, True, seed=8).verify()


def test_no_tokens_at_all():
    c = Case("f16", 0, 50, [0, 0, 0], True, seed=1)
    _, last = c.forward()
    assert np.array_equal(last, c.h0)
    _, _, dh0 = c.backward(np.zeros((0, 50), np.float16))
    assert np.array_equal(dh0, c.dh_last)
    one = Case("f16", 0, 50, [0, 0], True, seed=2)
    _, last = one.forward(null_ptr=True)
    assert np.array_equal(last, one.h0)


@pytest.mark.parametrize("kind,pitch,offset", [("f16", 260, 0), ("f16", 257, 0), ("bf16", 256, 1), ("f32", 300, 3), ("f32", 258, 2)])
def test_pitches_and_offsets(kind, pitch, offset):
    Case(kind, 321, 256, cut(321, 4, 5), True, seed=pitch, pitch=pitch, offset=offset).verify()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_nodes_outside_of_the_sequences_are_left_alone(kind):
    Case(kind, 700, 72, cut(700, 6, 2, first=37, pad=101), True, seed=6).verify()


def test_extreme_gates():
    """decays of exactly 0 and 1, gates beyond the exponential's range"""
    c = Case("f32", 300, 64, [0, 300], True, seed=4)
    c.gate[::7] = 200.0
    c.gate[1::7] = -200.0
    c.gate[2::7] = np.inf
    c.gate[3::7] = -np.inf
    c.gate[4::7] = 88.0
    with np.errstate(over="ignore"):
        want, _, slack, _ = forward(c.gate, c.x, c.ptr, c.h0)
    h, _ = c.forward()
    near(h, want, slack + 1e-30, "f32")


def test_nothing_leaks_from_one_sequence_into_the_next():
    """NaN and infinities of a sequence stay in it, forward and backward"""
    ptr = cut(900, 7, 11)
    clean, dirty = Case("f32", 900, 64, ptr, True, seed=9), Case("f32", 900, 64, ptr, True, seed=9)
    bad = range(ptr[2], ptr[3])
    dirty.x[bad[0]] = np.nan
    dirty.gate[bad[-1]] = np.nan
    dirty.x[bad[len(bad) // 2]] = np.inf
    dirty.dh[bad[-1]] = np.inf
    dirty.dh_last[2] = np.nan
    dirty.h0[2] = np.inf
    keep = np.ones(900, bool)
    keep[list(bad)] = False
    a, b = clean.forward(), dirty.forward()
    assert np.array_equal(a[0][keep], b[0][keep]) and np.array_equal(np.delete(a[1], 2, 0), np.delete(b[1], 2, 0))
    assert np.isnan(b[0][bad[0]:bad[-1] + 1]).all() and np.isnan(b[1][2]).all()
    ga, gb = clean.backward(a[0]), dirty.backward(b[0])
    for u, v in zip(ga[:2], gb[:2]):
        assert np.array_equal(u[keep], v[keep])
    assert np.array_equal(np.delete(ga[2], 2, 0), np.delete(gb[2], 2, 0))


def test_fp16_results_saturate():
    c = Case("f16", 40, 64, [0, 40], True, seed=5, low=5, high=8)
    c.h0[:] = 1e6
    h, last = c.forward()
    assert np.isfinite(h.astype(np.float32)).all() and (h[0] == 65504).all() and last.max() > 65504


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_the_same_call_gives_the_same_bits(kind):
    c = Case(kind, 3000, 640, cut(3000, 5, 1), True, seed=2)
    runs = [c.forward() for _ in range(3)]
    back = [c.backward(runs[0][0]) for _ in range(3)]
    for r in runs[1:]:
        assert r[0].tobytes() == runs[0][0].tobytes() and r[1].tobytes() == runs[0][1].tobytes()
    for r in back[1:]:
        assert all(u.tobytes() == v.tobytes() for u, v in zip(r, back[0]))


def test_gradients_against_differences():
    """directional derivatives of sum(w h) + sum(u h_last) by central differences in float64, of the formula"""
    ptr = cut(150, 4, 7)
    c = Case("f32", 150, 16, ptr, True, seed=12)
    h = forward(c.gate, c.x, c.ptr, c.h0)[0].astype(np.float32)
    dg, dx, dh0 = c.backward(h)
    rng = np.random.default_rng(0)
    vg, vx, v0 = (rng.standard_normal(a.shape) for a in (c.gate, c.x, c.h0))

    def loss(eps):
        hh, last, _, _ = forward(c.gate.astype(np.float64) + eps * vg, c.x.astype(np.float64) + eps * vx, c.ptr, c.h0.astype(np.float64) + eps * v0)
        return (c.dh * hh).sum() + (c.dh_last * last).sum()

    numeric = (loss(1e-5) - loss(-1e-5)) / 2e-5
    ours = (dg * vg).sum() + (dx * vx).sum() + (dh0 * v0).sum()
    size = np.sqrt((dg.astype(np.float64) ** 2).sum() + (dx.astype(np.float64) ** 2).sum() + (dh0.astype(np.float64) ** 2).sum())
    # fp32 gradients and a rounded h: 2^-22 of the gradient's norm each; differences in float64: 1e-9
    assert abs(numeric - ours) < 4 * 2.0 ** -22 * size * np.sqrt(vg.size) ** 0.5 + 1e-6


def test_rows_beyond_32_bit_offsets():
    """rows so far apart that element offsets pass 2^31"""
    import torch
    T, D, pitch = 2200, 48, 1_000_001
    ptr = np.array([0, 900, T], np.int32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    flat = [torch.empty(T * pitch, device="cuda", dtype=torch.float16) for _ in range(3)]
    rows = [f.as_strided((T, D), (pitch, 1)) for f in flat]
    for r in rows[:2]:
        r.copy_(torch.randn((T, D), device="cuda", generator=gen))
    p = torch.from_numpy(ptr).cuda()
    check(capi.load_library().ts2_op_recurrence_forward(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), capi.OUT_F16, rows[0].data_ptr(),
                                                        pitch, rows[1].data_ptr(), pitch, T, D, 2, p.data_ptr(), None, rows[2].data_ptr(), pitch,
                                                        None))
    want, _, slack, _ = forward(rows[0].cpu().numpy(), rows[1].cpu().numpy(), ptr, None)
    near(rows[2].cpu().numpy(), want, slack, "f16")


def test_other_streams_and_a_captured_graph():
    """on a stream of its own behind the work that makes its inputs, and replayed from a graph with new inputs"""
    import torch
    lib = capi.load_library()
    T, D = 1500, 200
    ptr = torch.tensor([0, 700, T], dtype=torch.int32, device="cuda")
    gate, x, h, h2 = (torch.zeros((T, D), device="cuda", dtype=torch.bfloat16) for _ in range(4))

    def call(out, stream):
        check(lib.ts2_op_recurrence_forward(0, C.c_void_p(stream.cuda_stream), capi.OUT_BF16, gate.data_ptr(), D, x.data_ptr(), D, T, D, 2,
                                            ptr.data_ptr(), None, out.data_ptr(), D, None))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gate.copy_(torch.randn((T, D), device="cuda") + 2)
        x.copy_(torch.randn((T, D), device="cuda"))
        call(h, side)
    side.synchronize()
    near(h.float().cpu().numpy(), *forward(gate.float().cpu().numpy(), x.float().cpu().numpy(), ptr.cpu().numpy(), None)[::2], "bf16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(h2, torch.cuda.current_stream())
    for seed in range(2):
        x.copy_(torch.randn((T, D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        call(h, torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert torch.equal(h, h2)


def test_two_streams_at_once_and_captured_graphs_of_long_arrays():
    """arrays in segments, whose maps lie in scratch: calls on two streams share nothing, and two captured graphs replay side by side"""
    import torch
    lib = capi.load_library()
    sets = []
    for seed, (T, D, n) in enumerate([(9000, 130, 3), (7000, 64, 1)]):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)
        st = dict(T=T, D=D, n=n, s=torch.cuda.Stream(), gate=randn(T, D) + 2, x=randn(T, D), dh=randn(T, D), h0=randn(n, D),
                  ptr=torch.tensor([T * i // n for i in range(n + 1)], dtype=torch.int32, device="cuda"))
        st.update({k: torch.zeros((T, D), device="cuda") for k in ("h", "dgate", "dx")}, h_last=torch.zeros((n, D), device="cuda"),
                  dh0=torch.zeros((n, D), device="cuda"))
        sets.append(st)
    outs = ("h", "h_last", "dgate", "dx", "dh0")

    def call(st):
        s, D = C.c_void_p(torch.cuda.current_stream().cuda_stream), st["D"]
        p = {k: v.data_ptr() for k, v in st.items() if torch.is_tensor(v)}
        check(lib.ts2_op_recurrence_forward(0, s, capi.OUT_F32, p["gate"], D, p["x"], D, st["T"], D, st["n"], p["ptr"], p["h0"], p["h"], D, p["h_last"]))
        check(lib.ts2_op_recurrence_backward(0, s, capi.OUT_F32, p["gate"], D, p["x"], D, p["h"], D, st["T"], D, st["n"], p["ptr"], p["h0"], p["dh"], D,
                                             None, p["dgate"], D, p["dx"], D, p["dh0"]))

    want = []
    for st in sets: # one after the other; the forward result is compared with the formula elsewhere
        torch.cuda.synchronize()
        call(st)
        torch.cuda.synchronize()
        near(st["h"].cpu().numpy(), *forward(st["gate"].cpu().numpy(), st["x"].cpu().numpy(), st["ptr"].cpu().numpy(), st["h0"].cpu().numpy())[::2], "f32")
        want.append({k: st[k].clone() for k in outs})

    def verify():
        torch.cuda.synchronize()
        for st, w in zip(sets, want):
            for k in outs:
                assert torch.equal(st[k], w[k]), k
                st[k].zero_()
        torch.cuda.synchronize()

    for st in sets:
        for k in outs:
            st[k].zero_()
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
