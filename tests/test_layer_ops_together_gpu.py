"""The recurrence, the router's balance and the orthogonalised update as one training step uses them, between the library's own
contractions and routing: a recurrent mixing layer in front of a router whose only loss is the balance of its experts.

    gate = x Wg, value = x Wv;  h = recurrence(gate, value);  logits = h Wr;  choices = ts2_moe_route;  loss = balance
    and back: d logits, d h, d gate, d value, the gradients of Wg and Wv, and both updates orthogonalised as one batch

against the same step in float64 with the choices given.  Tolerance: five fp16 roundings (half a step 2^-11 each, relative to an
element) lie between the inputs and a weight gradient, where a sum over tokens averages them; the recurrence passes an error of a
gate on with a factor of at most 1 / (1 - a) of a few.  2^-11 x 5 x 4 = 1e-2 of the gradients' norm.  The orthogonalised update is
held to that of the gradient it was given (test_orthogonalize_gpu.py has its tolerance), and to growing along the exact gradient as
a matrix with singular values of at least 0.6 does."""
import ctypes as C

import ml_dtypes
import numpy as np
import pytest

from tscale2_b200 import capi
from tscale2_b200.device import DeviceBuffer, check, sync

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)


def rel(a, b):
    return np.linalg.norm(a.astype(np.float64) - b) / np.linalg.norm(b)


def test_a_step_of_a_recurrent_layer_with_a_balanced_router():
    lib = capi.load_library()
    rng = np.random.default_rng(3)
    T, D, E, k = 1024, 256, 128, 2
    ptr = np.array([0, 300, 301, 700, T], np.int32)
    x = rng.standard_normal((T, D)).astype(np.float16)
    wg, wv = ((rng.standard_normal((D, D)) / np.sqrt(D)).astype(np.float16) for _ in range(2))
    wr = (rng.standard_normal((E, D)) * 0.5).astype(np.float16)  # [out][in], as all matrices here
    up = lambda a: DeviceBuffer.from_numpy(a)
    half = lambda *s: DeviceBuffer(2 * int(np.prod(s)))
    get = lambda b, *s: b.download(s, np.float16).astype(np.float64)
    X, WG, WV, WR, P = up(x), up(wg), up(wv), up(wr), up(ptr)
    gate, value, h, logits, dlogits, dh, dgate, dvalue = (half(T, n) for n in (D, D, D, E, E, D, D, D))
    F16, OUT16 = capi.PREC_F16, capi.OUT_F16
    for w, o in ((WG, gate), (WV, value)):
        check(lib.ts2_gemm_tn(0, None, F16, OUT16, T, D, D, X.ptr, D, w.ptr, D, o.ptr, D, 1.0, None, None))
    check(lib.ts2_op_recurrence_forward(0, None, OUT16, gate.ptr, D, value.ptr, D, T, D, len(ptr) - 1, P.ptr, None, h.ptr, D, None))
    check(lib.ts2_gemm_tn(0, None, F16, OUT16, T, E, D, h.ptr, D, WR.ptr, D, logits.ptr, E, 1.0, None, None))
    sync()
    host_logits = get(logits, T, E).astype(np.float32)
    ids, weights = np.zeros((T, k), np.int32), np.zeros((T, k), np.float32)
    check(lib.ts2_moe_route(0, host_logits.ctypes.data, T, E, k, ids.ctypes.data, weights.ctypes.data))
    I = up(ids)
    counts, prob, loss = DeviceBuffer(4 * (E + 1)), DeviceBuffer(4 * E), DeviceBuffer(4)
    check(lib.ts2_op_moe_balance_forward(0, None, OUT16, logits.ptr, E, T, E, k, I.ptr, None, counts.ptr, prob.ptr, loss.ptr))
    scale = 4096.0  # fp16 gradients
    check(lib.ts2_op_moe_balance_backward(0, None, OUT16, logits.ptr, E, T, E, k, None, counts.ptr, None, scale, dlogits.ptr, E, 0))
    wrt = up(np.ascontiguousarray(wr.T))
    check(lib.ts2_gemm_dx(0, None, F16, OUT16, T, D, E, dlogits.ptr, wrt.ptr, dh.ptr, 1.0, None, None))
    check(lib.ts2_op_recurrence_backward(0, None, OUT16, gate.ptr, D, value.ptr, D, h.ptr, D, T, D, len(ptr) - 1, P.ptr, None, dh.ptr, D, None,
                                         dgate.ptr, D, dvalue.ptr, D, None))
    grads = DeviceBuffer(4 * 2 * D * D)  # both matrices' gradients, one behind the other
    ws = DeviceBuffer(max(16, lib.ts2_gemm_dw_workspace_bytes(T, D, D)))
    for i, d in enumerate((dgate, dvalue)):
        check(lib.ts2_gemm_dw(0, None, F16, capi.OUT_F32, T, D, D, d.ptr, X.ptr, grads.ptr + 4 * i * D * D, 1.0, ws.ptr, ws.nbytes))
    update = half(2, D, D)
    check(lib.ts2_op_orthogonalize(0, None, capi.OUT_F32, grads.ptr, D, D * D, 2, D, D, (C.c_float * 3)(*COEF), 5, 0.2, update.ptr, D, D * D))
    sync()

    # float64
    xd, g, v = x.astype(np.float64), x.astype(np.float64) @ wg.T.astype(np.float64), x.astype(np.float64) @ wv.T.astype(np.float64)
    a, hd = 1 / (1 + np.exp(-g)), np.zeros((T, D))
    starts = set(ptr[:-1].tolist())
    for t in range(T):
        hd[t] = (1 - a[t]) * v[t] + (0 if t in starts else a[t] * hd[t - 1])
    l = hd @ wr.T.astype(np.float64)
    assert rel(get(logits, T, E), l) < 1e-2
    p = np.exp(l - l.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    c = np.bincount(ids.ravel(), minlength=E)
    assert np.array_equal(counts.download(E + 1, np.int32), np.append(c, T))
    want_loss = E / (k * T * T) * (c * p.sum(0)).sum()
    assert abs(loss.download(1, np.float32)[0] - want_loss) < 1e-2 * want_loss
    dl = scale * E / (k * T * T) * p * (c - (p * c).sum(1, keepdims=True))
    dhd, e, dg, dv = dl @ wr.astype(np.float64), np.zeros(D), np.zeros((T, D)), np.zeros((T, D))
    for t in range(T - 1, -1, -1):
        e = dhd[t] + (0 if t + 1 in starts or t == T - 1 else e)
        before = 0 if t in starts else hd[t - 1]
        dg[t], dv[t] = a[t] * (1 - a[t]) * (before - v[t]) * e, (1 - a[t]) * e
        e = a[t] * e
    want = [d.T @ xd for d in (dg, dv)]
    got = grads.download((2, D, D), np.float32)
    out = update.download((2, D, D), np.uint16).view(ml_dtypes.bfloat16).astype(np.float64)
    for i in range(2):
        assert rel(got[i], want[i]) < 1e-2
        s = got[i].astype(np.float64)
        s /= np.linalg.norm(s)
        for _ in range(5):
            q = s @ s.T
            s = COEF[0] * s + (COEF[1] * q + COEF[2] * q @ q) @ s
        assert rel(out[i], 0.2 * s) < 1.5e-3 + 2.0 ** -8 / 3 ** 0.5  # the update of the gradient it was given
        # and it goes uphill as the exact gradient does: <U V^T-like, G> is the sum of the singular values times about one
        assert (out[i] * want[i]).sum() > 0.2 * 0.6 * np.linalg.svd(want[i], compute_uv=False).sum()
