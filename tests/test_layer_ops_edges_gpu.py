"""Calls at the edges of what the recurrence and the orthogonalised update allow, on each of the forms that they take: one token a
sequence in every type, offsets beyond 32 bits, carried gradients in a captured pass, zeros, NaN, infinities and extreme scales in
matrices of one CTA, of clusters and of products through memory.  Tolerances are those of the tests of each operator."""
import ctypes as C

import ml_dtypes
import numpy as np
import pytest

import test_orthogonalize_gpu as orth
import test_recurrence_gpu as rec
from tscale2_b200 import capi
from tscale2_b200.device import check, sync

pytestmark = pytest.mark.gpu


# ---- recurrence ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,D", [(1, 768), (64, 256), (256, 130), (257, 65), (1000, 33)])
def test_one_token_a_sequence(kind, T, D):
    rec.Case(kind, T, D, list(range(T + 1)), True, seed=T + D).verify()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_sequences_of_a_few_tokens_and_of_none(kind):
    rng = np.random.default_rng(2)
    ptr = np.concatenate([[2], 2 + np.cumsum(rng.integers(0, 5, 700))])
    rec.Case(kind, int(ptr[-1]) + 3, 70, ptr.tolist(), True, seed=4).verify()


def test_backward_recurrence_beyond_32_bit_offsets():
    """six arrays side by side in rows that are a million elements apart"""
    import torch
    T, D, pitch, n = 2200, 48, 1_000_001, 2
    ptr = np.array([0, 900, T], np.int32)
    flat = torch.empty(T * pitch, device="cuda", dtype=torch.float16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    rows = [flat.as_strided((T, D), (pitch, 1), 100 * i) for i in range(6)]  # gate, x, h, dh, dgate, dx
    for r in rows[:4]:
        r.copy_(torch.randn((T, D), device="cuda", generator=gen))
    p = torch.from_numpy(ptr).cuda()
    h0, dl = torch.randn((n, D), device="cuda", generator=gen), torch.randn((n, D), device="cuda", generator=gen)
    dh0 = torch.zeros((n, D), device="cuda")
    at = [r.data_ptr() for r in rows]
    check(capi.load_library().ts2_op_recurrence_backward(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), capi.OUT_F16, at[0], pitch, at[1], pitch,
                                                         at[2], pitch, T, D, n, p.data_ptr(), h0.data_ptr(), at[3], pitch, dl.data_ptr(), at[4], pitch,
                                                         at[5], pitch, dh0.data_ptr()))
    host = [r.cpu().numpy() for r in rows]
    dgate, dx, want0, sg, sx, s0 = rec.backward(host[0], host[1], host[2], ptr, h0.cpu().numpy(), host[3], dl.cpu().numpy())
    rec.near(host[4], dgate, sg, "f16")
    rec.near(host[5], dx, sx, "f16")
    rec.near(dh0.cpu().numpy(), want0, s0, "f32")


@pytest.mark.parametrize("T,D", [(300, 66), (9000, 72)])
def test_carried_states_and_gradients_in_a_captured_step(T, D):
    """forward and backward pass with states in and out, captured, then replayed with other inputs next to eager calls of the same"""
    import torch
    lib = capi.load_library()
    n = 3
    ptr = torch.tensor([0, T // 5, T // 5, T], dtype=torch.int32, device="cuda")
    new = lambda *s: torch.zeros(s, device="cuda")
    gate, x, dh, h0, dl = new(T, D), new(T, D), new(T, D), new(n, D), new(n, D)
    outs = [[new(T, D), new(n, D), new(T, D), new(T, D), new(n, D)] for _ in range(2)]  # h, h_last, dgate, dx, dh0

    def step(o):
        s, p = C.c_void_p(torch.cuda.current_stream().cuda_stream), [t.data_ptr() for t in o]
        check(lib.ts2_op_recurrence_forward(0, s, capi.OUT_F32, gate.data_ptr(), D, x.data_ptr(), D, T, D, n, ptr.data_ptr(), h0.data_ptr(), p[0], D, p[1]))
        check(lib.ts2_op_recurrence_backward(0, s, capi.OUT_F32, gate.data_ptr(), D, x.data_ptr(), D, p[0], D, T, D, n, ptr.data_ptr(), h0.data_ptr(),
                                             dh.data_ptr(), D, dl.data_ptr(), p[2], D, p[3], D, p[4]))

    step(outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs[1])
    for seed in range(2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for t in (gate, x, dh, h0, dl):
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
        graph.replay()
        step(outs[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        a = [t.cpu().numpy() for t in (gate, x, ptr, h0)]
        h, last, slack, last_slack = rec.forward(*a)
        rec.near(outs[1][0].cpu().numpy(), h, slack, "f32")
        rec.near(outs[1][1].cpu().numpy(), last, last_slack, "f32")
        dgate, dx, dh0, sg, sx, s0 = rec.backward(a[0], a[1], outs[1][0].cpu().numpy(), a[2], a[3], dh.cpu().numpy(), dl.cpu().numpy())
        rec.near(outs[1][2].cpu().numpy(), dgate, sg, "f32")
        rec.near(outs[1][3].cpu().numpy(), dx, sx, "f32")
        rec.near(outs[1][4].cpu().numpy(), dh0, s0, "f32")


# ---- orthogonalised update -------------------------------------------------------------------------------------------

FORMS = [(100, 140), (300, 90), (128, 900), (1999, 128), (130, 140), (300, 200), (520, 1300), (64, 6200)]


@pytest.mark.parametrize("rows,cols", FORMS)
def test_zeros_and_bad_values_on_every_form(rows, cols):
    rng = np.random.default_rng(rows)
    g = rng.standard_normal((6, rows, cols)).astype(np.float32)
    g[1] = 0
    g[2, rows // 2, cols // 3] = np.nan
    g[3, rows - 1, cols - 1] = np.inf  # in the last CTA's columns only
    g[4, 0, 0] = -np.inf
    got = orth.run("f32", g)
    assert (got[1] == 0).all() and all(np.isnan(got[i]).all() for i in (2, 3, 4))
    for i in (0, 5):
        orth.near(got[i], g[i])


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e30, 1e34])
@pytest.mark.parametrize("rows,cols", FORMS)
def test_extreme_scales_on_every_form(rows, cols, scale):
    g = (orth.spectrum(rows, cols, 0.5, 4) * scale).astype(np.float32)
    orth.near(orth.run("f32", g[None], scale=0.25)[0], g, scale=0.25)


@pytest.mark.parametrize("rows,cols", [(2200, 100), (2200, 140)])
def test_rows_of_matrices_beyond_32_bit_offsets(rows, cols):
    """a matrix and its update side by side in rows that are a million elements apart"""
    import torch
    pitch = 1_000_003
    flat = torch.empty(rows * pitch, device="cuda", dtype=torch.bfloat16)
    g, o = (flat.as_strided((rows, cols), (pitch, 1), 1000 * i) for i in range(2))
    g.copy_(torch.from_numpy(orth.spectrum(rows, cols, 0.5, 1)))
    check(capi.load_library().ts2_op_orthogonalize(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), capi.OUT_BF16, g.data_ptr(), pitch, 0, 1, rows,
                                                   cols, (C.c_float * 3)(*orth.COEF), 5, 1.0, o.data_ptr(), pitch, 0))
    orth.near(o.float().cpu().numpy().astype(np.float64), g.float().cpu().numpy())


@pytest.mark.parametrize("rows,cols", [(100, 90), (140, 150)])
def test_matrices_of_a_batch_beyond_32_bit_offsets(rows, cols):
    import torch
    stride = (1 << 31) + 24
    flat = torch.empty(stride + 100_000, device="cuda", dtype=torch.bfloat16)
    g, o = (flat.as_strided((2, rows, cols), (stride, cols, 1), 40_000 * i) for i in range(2))
    host = np.stack([orth.spectrum(rows, cols, 0.5, s) for s in range(2)]).astype(ml_dtypes.bfloat16)
    g.copy_(torch.from_numpy(host.astype(np.float32)))
    check(capi.load_library().ts2_op_orthogonalize(0, C.c_void_p(torch.cuda.current_stream().cuda_stream), capi.OUT_BF16, g.data_ptr(), cols, stride, 2,
                                                   rows, cols, (C.c_float * 3)(*orth.COEF), 5, 1.0, o.data_ptr(), cols, stride))
    sync()
    for a, b in zip(o.float().cpu().numpy().astype(np.float64), host):
        orth.near(a, b)
