"""The load-balance term of a router, its counts and its gradient (ts2_op_moe_balance_forward / _backward) against the
formulas in float64.

Tolerances.  A probability is exp(l - max) over a sum of E of them: the difference is exact to 2^-24 of itself, which its
exponential turns into |l - max| 2^-24, expf is within 2 units (2^-22), the sum and the quotient add (log2(32) + E / 32 + 2) 2^-24.
Column means add the same number of roundings as a lane adds rows, at most rows / 8 + 64.  The gradient is p (f - sum p f) with
f exact to 2^-24: its error is at most p (rate of p twice + 2^-22) (|f| + sum p |f|).  Types of 16 bits add half a step."""
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


def formula(logits, ids, mask, E, k):
    l = logits.astype(np.float64)
    on = np.ones(len(l), bool) if mask is None else mask != 0
    l = np.where(on[:, None], l, 0.0)
    m = l.max(1, keepdims=True) if len(l) else np.zeros((0, 1))
    nothing = ~np.isfinite(m) & (m < 0)
    d = l - np.where(nothing, 0, m)
    p = np.exp(d)
    s = p.sum(1, keepdims=True)
    p = np.where(nothing, 0, p / np.where(s == 0, 1, s)) * on[:, None]
    n = int(on.sum())
    chosen = ids[on]
    chosen = chosen[(chosen >= 0) & (chosen < E)]
    counts = np.bincount(chosen.ravel(), minlength=E)
    prob = p.sum(0) / n if n else np.zeros(E)
    loss = E / (k * n) * (counts * prob).sum() if n else 0.0
    rate = (np.abs(np.where(np.isfinite(d), d, 0)) + 4 + 5 + E / 32 + 2) * 2.0 ** -24
    return p, counts, prob, loss, n, rate


def gradient(p, counts, n, E, k, dloss, rate):
    unit = dloss * E / (k * n * n) if n else 0.0
    f = (counts - n * k / E) * unit
    dot = (p * f).sum(1, keepdims=True)
    return p * (f - dot), p * (2 * rate.max(1, keepdims=True) + 2.0 ** -22) * (np.abs(f) + (p * np.abs(f)).sum(1, keepdims=True))


def make(kind, T, E, k, masked, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    logits = (rng.standard_normal((T, E)) * spread + rng.standard_normal(E)).astype(TYPE[kind])
    ids = np.argsort(-logits.astype(np.float32), axis=1, kind="stable")[:, :k].astype(np.int32)
    mask = (rng.random(T) < 0.7).astype(np.uint8) if masked else None
    return logits, np.ascontiguousarray(ids), mask


def pitched(a, pitch, offset, fill=3):
    T, E = a.shape
    flat = np.full(offset + max(T, 1) * pitch, fill, a.dtype)
    flat[offset:offset + T * pitch].reshape(T, pitch)[:, :E] = a
    return DeviceBuffer.from_numpy(flat.view(np.uint8)), offset * a.dtype.itemsize


def run(kind, logits, ids, mask, k, dloss=0.25, scale=1.0, pitch=None, offset=0, add=None):
    lib = capi.load_library()
    T, E = logits.shape
    pitch = pitch or E
    L, at = pitched(logits, pitch, offset)
    I, M = DeviceBuffer.from_numpy(ids if ids.size else np.zeros(1, np.int32)), None if mask is None else DeviceBuffer.from_numpy(mask)
    counts, prob, loss = (DeviceBuffer.from_numpy(np.full(n, 9, t)) for n, t in ((E + 1, np.int32), (E, np.float32), (1, np.float32)))
    check(lib.ts2_op_moe_balance_forward(0, None, KIND[kind], L.ptr + at, pitch, T, E, k, I.ptr, M and M.ptr, counts.ptr, prob.ptr, loss.ptr))
    out, oat = pitched(np.full((T, E), 3, TYPE[kind]) if add is None else add, pitch, offset)
    up = DeviceBuffer.from_numpy(np.array([dloss], np.float32)) if dloss is not None else None
    check(lib.ts2_op_moe_balance_backward(0, None, KIND[kind], L.ptr + at, pitch, T, E, k, M and M.ptr, counts.ptr, up and up.ptr, scale, out.ptr + oat,
                                          pitch, add is not None))
    sync()
    flat = out.download(out.nbytes, np.uint8).view(TYPE[kind])
    rows = flat[offset:offset + T * pitch].reshape(T, pitch)
    assert (flat[:offset] == 3).all() and (rows[:, E:] == 3).all()
    return counts.download(E + 1, np.int32), prob.download(E, np.float32), loss.download(1, np.float32)[0], rows[:, :E]


def verify(kind, logits, ids, mask, k, dloss=0.25, scale=1.0, **kw):
    T, E = logits.shape
    p, counts, prob, loss, n, rate = formula(logits, ids, mask, E, k)
    c, pr, lo, dl = run(kind, logits, ids, mask, k, dloss, scale, **kw)
    assert np.array_equal(c[:E], counts) and c[E] == n
    r = (rate.max() if len(rate) else 0) + (T / 8 + 64) * 2.0 ** -24
    assert (np.abs(pr - prob) <= prob * r + 1e-37).all()
    assert abs(lo - loss) <= loss * (r + 2.0 ** -23)
    want, slack = gradient(p, counts, n, E, k, (1.0 if dloss is None else dloss) * scale, rate)
    tiny = 2.0 ** -25 if kind == "f16" else 1e-37
    assert (np.abs(dl.astype(np.float64) - want) <= slack + HALF_STEP[kind] * (np.abs(want) + slack) + tiny).all()
    return dl


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,E,k,masked", [(1, 1, 1, False), (40, 2, 1, False), (512, 8, 2, False), (333, 16, 4, True), (1000, 7, 3, True),
                                          (2048, 32, 2, True), (5000, 128, 8, True), (700, 65, 6, False), (300, 256, 8, False), (100, 515, 4, True),
                                          (64, 1024, 8, True), (20000, 24, 6, True)])
def test_against_the_formula(kind, T, E, k, masked):
    logits, ids, mask = make(kind, T, E, k, masked, T + E)
    # 16-bit gradients as large as such a type holds well
    verify(kind, logits, ids, mask, k, dloss=0.25 if kind == "f32" else 64.0 * T)


@pytest.mark.parametrize("kind,T,E,k,masked", [("f32", 6000, 1000, 4, True), ("bf16", 5000, 1024, 8, False), ("f16", 9000, 512, 8, True),
                                               ("bf16", 4000, 515, 3, True), ("f32", 3000, 64, 40, True), ("f16", 2500, 1, 1, True)])
def test_rows_of_every_width_over_many_clusters(kind, T, E, k, masked):
    logits, ids, mask = make(kind, T, E, k, masked, T + E)
    verify(kind, logits, ids, mask, k, dloss=0.25 if kind == "f32" else 64.0 * T)


@pytest.mark.parametrize("kind,pitch,offset", [("f32", 32, 0), ("f32", 36, 4), ("f32", 33, 1), ("f16", 40, 8), ("f16", 41, 0), ("bf16", 48, 3)])
def test_pitches_and_offsets(kind, pitch, offset):
    logits, ids, mask = make(kind, 777, 32, 2, True, pitch)
    verify(kind, logits, ids, mask, 2, dloss=1000.0, pitch=pitch, offset=offset)


def test_no_token_counts():
    logits, ids, _ = make("f32", 100, 16, 2, False, 3)
    dl = verify("f32", logits, ids, np.zeros(100, np.uint8), 2)
    assert (dl == 0).all()
    c, pr, lo, dl = run("f32", logits[:0], ids[:0], None, 2)
    assert (c == 0).all() and (pr == 0).all() and lo == 0 and dl.size == 0


def test_masked_tokens_hold_anything():
    """NaN, infinities and impossible ids of tokens that do not count change nothing, and their gradient is zero"""
    logits, ids, mask = make("f32", 400, 24, 2, True, 5)
    a = run("f32", logits, ids, mask, 2)
    off = np.flatnonzero(mask == 0)
    logits[off[0::3]], logits[off[1::3]], logits[off[2::3]] = np.nan, np.inf, -np.inf
    ids[off] = 2 ** 31 - 1
    b = run("f32", logits, ids, mask, 2, dloss=0.25)
    for u, v in zip(a, b):
        assert np.asarray(u).tobytes() == np.asarray(v).tobytes()
    assert (b[3][off] == 0).all()
    inf = run("f32", logits, ids, mask, 2, dloss=np.inf)[3]
    assert (inf[off] == 0).all()


def test_closed_experts_and_rows_without_any():
    """-inf logits have no probability and no gradient; a row of nothing but -inf counts as a token and has neither"""
    logits, ids, _ = make("f32", 300, 12, 2, False, 6)
    logits[:, 5] = -np.inf
    logits[10] = -np.inf
    logits[11] = np.finfo(np.float32).min  # the lowest finite value everywhere is an even row
    ids[12] = -1  # a choice that was not made
    ids[13, 1] = 12
    dl = verify("f32", logits, ids, None, 2)
    assert (np.delete(dl[:, 5], 11) == 0).all() and (dl[10] == 0).all()  # expert 5 is open to row 11


def test_a_nan_row_spoils_itself_and_the_means_only():
    logits, ids, _ = make("f32", 100, 16, 2, False, 7)
    clean = run("f32", logits, ids, None, 2)
    logits[50, 3] = np.nan
    logits[60, 2] = np.inf
    c, pr, lo, dl = run("f32", logits, ids, None, 2)
    assert np.array_equal(c, clean[0]) and np.isnan(lo) and np.isnan(pr).all()
    assert np.isnan(dl[50]).all() and np.isnan(dl[60, 2])
    keep = np.delete(np.arange(100), [50, 60])
    assert np.array_equal(dl[keep], clean[3][keep])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_adds_to_a_gradient(kind):
    logits, ids, mask = make(kind, 200, 40, 4, True, 8)
    base = np.random.default_rng(1).standard_normal((200, 40)).astype(TYPE[kind])
    alone = run(kind, logits, ids, mask, 4, dloss=2000.0, scale=-0.5)[3]
    both = run(kind, logits, ids, mask, 4, dloss=2000.0, scale=-0.5, add=base)[3]
    want = base.astype(np.float64) + alone.astype(np.float64)
    # the sum is rounded once, the plain gradient once more
    tol = HALF_STEP[kind] * (np.abs(want) + 2 * np.abs(alone.astype(np.float64)))
    assert (np.abs(both.astype(np.float64) - want) <= tol + 1e-37).all()
    assert np.array_equal(both[mask == 0], base[mask == 0])


def test_without_a_loss_gradient_the_scale_alone():
    logits, ids, _ = make("f32", 128, 8, 2, False, 9)
    verify("f32", logits, ids, None, 2, dloss=None, scale=-3.0)


def test_an_even_load_is_one_and_has_a_small_gradient():
    E, T = 16, 1600
    logits = np.zeros((T, E), np.float32)
    ids = (np.arange(T)[:, None] + np.array([0, 5])).astype(np.int32) % E
    c, pr, lo, dl = run("f32", logits, ids, None, 2)
    assert (c[:E] == T * 2 // E).all() and lo == 1.0 and (dl == 0).all()


def test_gradient_against_differences():
    """central differences of the formula in float64 along random directions, the counts held"""
    E, k, T = 12, 3, 50
    logits, ids, mask = make("f32", T, E, k, True, 10)
    dl = run("f32", logits, ids, mask, k, dloss=1.0)[3].astype(np.float64)
    rng = np.random.default_rng(2)
    for _ in range(4):
        v = rng.standard_normal((T, E))
        f = [formula(logits.astype(np.float64) + s * 1e-5 * v, ids, mask, E, k)[3] for s in (1, -1)]
        numeric = (f[0] - f[1]) / 2e-5
        # central differences: 1e-10 x the third derivative, 1e-16 / 1e-5 rounding
        assert abs(numeric - (dl * v).sum()) < 1e-5 * np.linalg.norm(dl) * np.linalg.norm(v) / np.sqrt(T * E) + 1e-9


def test_counts_summed_over_ranks_give_each_its_rows():
    """two halves of a batch with their counts added: the gradient of the whole batch's loss"""
    lib = capi.load_library()
    E, k, T = 16, 2, 600
    logits, ids, mask = make("f32", T, E, k, True, 11)
    p, counts, _, _, n, rate = formula(logits, ids, mask, E, k)
    want, slack = gradient(p, counts, n, E, k, 1.0, rate)
    total = DeviceBuffer.from_numpy(np.append(counts, n).astype(np.int32))
    for a, b in ((0, 250), (250, T)):
        L, M, out = DeviceBuffer.from_numpy(logits[a:b]), DeviceBuffer.from_numpy(mask[a:b]), DeviceBuffer((b - a) * E * 4)
        check(lib.ts2_op_moe_balance_backward(0, None, capi.OUT_F32, L.ptr, E, b - a, E, k, M.ptr, total.ptr, None, 1.0, out.ptr, E, 0))
        sync()
        got = out.download((b - a, E), np.float32)
        assert (np.abs(got - want[a:b]) <= slack[a:b] + 2.0 ** -24 * np.abs(want[a:b]) + 1e-37).all()


@pytest.mark.parametrize("T,E,k", [(70000, 16, 2), (9000, 130, 4)])
def test_the_same_call_gives_the_same_bits(T, E, k):
    logits, ids, mask = make("f32", T, E, k, True, 12)
    a = run("f32", logits, ids, mask, k)
    for _ in range(2):
        b = run("f32", logits, ids, mask, k)
        assert all(np.asarray(u).tobytes() == np.asarray(v).tobytes() for u, v in zip(a, b))


def test_rows_beyond_32_bit_offsets():
    import torch
    T, E, k, pitch = 3000, 16, 2, 800_000
    flat = torch.empty(T * pitch, device="cuda", dtype=torch.bfloat16)
    rows = flat.as_strided((T, E), (pitch, 1))
    rows.copy_(torch.randn((T, E), device="cuda"))
    logits = rows.float().cpu().numpy()
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :k].astype(np.int32).copy()
    I = torch.from_numpy(ids).cuda()
    counts, prob, loss = torch.zeros(E + 1, device="cuda", dtype=torch.int32), torch.zeros(E, device="cuda"), torch.zeros(1, device="cuda")
    s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    lib = capi.load_library()
    check(lib.ts2_op_moe_balance_forward(0, s, capi.OUT_BF16, rows.data_ptr(), pitch, T, E, k, I.data_ptr(), None, counts.data_ptr(), prob.data_ptr(),
                                         loss.data_ptr()))
    check(lib.ts2_op_moe_balance_backward(0, s, capi.OUT_BF16, rows.data_ptr(), pitch, T, E, k, None, counts.data_ptr(), None, 1e4, rows.data_ptr() + 64,
                                          pitch, 0))
    p, want_counts, _, _, n, rate = formula(logits, ids, None, E, k)
    assert np.array_equal(counts.cpu().numpy()[:E], want_counts)
    want, slack = gradient(p, want_counts, n, E, k, 1e4, rate)
    got = flat.as_strided((T, E), (pitch, 1), 32).float().cpu().numpy()
    assert (np.abs(got - want) <= slack + 2.0 ** -8 * (np.abs(want) + slack)).all()


def test_two_streams_at_once_and_captured_graphs():
    """calls on two streams share nothing; two captured graphs replay side by side"""
    import torch
    lib = capi.load_library()
    T, E, k = 30000, 32, 2
    sets = []
    for seed in range(2):
        logits, ids, _ = make("f32", T, E, k, False, seed)
        st = dict(l=torch.from_numpy(logits).cuda(), i=torch.from_numpy(ids).cuda(), c=torch.zeros(E + 1, dtype=torch.int32, device="cuda"),
                  p=torch.zeros(E, device="cuda"), o=torch.zeros(1, device="cuda"), s=torch.cuda.Stream())
        _, counts, prob, loss, n, _ = formula(logits, ids, None, E, k)
        st.update(counts=counts, loss=loss)
        sets.append(st)
    torch.cuda.synchronize()

    def call(st):
        check(lib.ts2_op_moe_balance_forward(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), capi.OUT_F32, st["l"].data_ptr(), E, T, E, k,
                                             st["i"].data_ptr(), None, st["c"].data_ptr(), st["p"].data_ptr(), st["o"].data_ptr()))

    def verify_sets():
        torch.cuda.synchronize()
        for st in sets:
            assert np.array_equal(st["c"].cpu().numpy()[:E], st["counts"]) and abs(st["o"].item() - st["loss"]) < 1e-5 * st["loss"]
            st["c"].zero_(), st["o"].zero_()
        torch.cuda.synchronize()

    for _ in range(5):
        for st in sets:
            with torch.cuda.stream(st["s"]):
                call(st)
    verify_sets()
    graphs = []
    for st in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(st)
        graphs.append(g)
    for _ in range(5):
        for st, g in zip(sets, graphs):
            with torch.cuda.stream(st["s"]):
                g.replay()
    verify_sets()
