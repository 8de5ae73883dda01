"""What ts2_op_recurrence_*, ts2_op_moe_balance_* and ts2_op_orthogonalize refuse.  Arguments are looked at before the device is,
so this runs anywhere: a call that is refused never touches the GPU."""
import ctypes as C

import pytest

from tscale2_b200 import capi

P = 0x7000  # a pointer that is never followed
F32, F16, BF16 = capi.OUT_F32, capi.OUT_F16, capi.OUT_BF16


@pytest.fixture(scope="module")
def lib():
    return capi.load_library()


FORWARD = dict(device=0, stream=None, type=F16, gate=P, gate_ld=8, x=P, x_ld=8, T=4, D=8, n_seq=2, ptr=P, h0=P, h=P, h_ld=8, h_last=P)
BACKWARD = dict(device=0, stream=None, type=F16, gate=P, gate_ld=8, x=P, x_ld=8, h=P, h_ld=8, T=4, D=8, n_seq=2, ptr=P, h0=P, dh=P, dh_ld=8,
                dh_last=P, dgate=P, dgate_ld=8, dx=P, dx_ld=8, dh0=P)
BALANCE = dict(device=0, stream=None, type=F32, logits=P, ld=8, T=4, E=8, k=2, ids=P, mask=P, counts=P, prob=P, loss=P)
GRADIENT = dict(device=0, stream=None, type=F32, logits=P, ld=8, T=4, E=8, k=2, mask=P, counts=P, dloss=P, scale=1.0, dl=P, dl_ld=8, add=0)
ORTH = dict(device=0, stream=None, type=F32, g=P, ld=8, g_stride=64, batch=2, rows=8, cols=8, coef=(C.c_float * 3)(3.4445, -4.775, 2.0315), steps=5,
            scale=1.0, out=P, out_ld=8, out_stride=64)
NAN, BIG = float("nan"), 1 << 31


def refused(lib, name, args, rc=capi.TS2_ERR_INVALID_ARG, **change):
    a = {**args, **change}
    assert set(change) <= set(args)
    assert getattr(lib, name)(*a.values()) == rc, change
    assert name.split("_op_")[1].split("_")[0].encode() in lib.ts2_last_error(None)


@pytest.mark.parametrize("change", [dict(type=1), dict(type=7), dict(type=-1), dict(T=-1), dict(T=(1 << 30) + 1), dict(D=0), dict(D=-5), dict(D=65535 * 64 + 1), dict(n_seq=-1), dict(n_seq=(1 << 30) + 1),
                                    dict(ptr=None), dict(gate=None), dict(x=None), dict(h=None), dict(gate_ld=7), dict(x_ld=7), dict(h_ld=7),
                                    dict(gate_ld=BIG), dict(gate=P + 1), dict(x=P + 1), dict(h=P + 1), dict(h0=P + 2), dict(h_last=P + 2),
                                    dict(ptr=P + 1), dict(type=F32, x=P + 2)])
def test_recurrence_forward(lib, change):
    refused(lib, "ts2_op_recurrence_forward", FORWARD, **change)


@pytest.mark.parametrize("change", [dict(type=1), dict(T=-1), dict(D=0), dict(n_seq=-1), dict(ptr=None), dict(gate=None), dict(x=None), dict(h=None),
                                    dict(dh=None), dict(dgate=None), dict(dx=None), dict(dh_ld=7), dict(dgate_ld=7), dict(dx_ld=7), dict(h_ld=7),
                                    dict(dh=P + 1), dict(dgate=P + 1), dict(dx=P + 1), dict(dh0=P + 2), dict(dh_last=P + 2), dict(h0=P + 1)])
def test_recurrence_backward(lib, change):
    refused(lib, "ts2_op_recurrence_backward", BACKWARD, **change)


@pytest.mark.parametrize("change", [dict(type=1), dict(T=-1), dict(E=0), dict(k=0), dict(k=9), dict(logits=None), dict(ids=None), dict(counts=None), dict(prob=None),
                                    dict(loss=None), dict(ld=7), dict(ld=BIG), dict(logits=P + 2), dict(ids=P + 1), dict(counts=P + 2),
                                    dict(prob=P + 1), dict(loss=P + 2), dict(T=1 << 30, k=2), dict(T=(1 << 30) + 1)])
def test_balance_forward(lib, change):
    refused(lib, "ts2_op_moe_balance_forward", BALANCE, **change)


@pytest.mark.parametrize("change", [dict(type=1), dict(T=-1), dict(E=0), dict(k=0), dict(k=9), dict(logits=None), dict(counts=None), dict(dl=None), dict(dl_ld=7),
                                    dict(ld=7), dict(dl=P + 2), dict(logits=P + 2), dict(counts=P + 1), dict(dloss=P + 2)])
def test_balance_backward(lib, change):
    refused(lib, "ts2_op_moe_balance_backward", GRADIENT, **change)


@pytest.mark.parametrize("change", [dict(type=1), dict(batch=-1), dict(batch=65536), dict(rows=0), dict(cols=0), dict(rows=(1 << 20) + 1),
                                    dict(cols=(1 << 20) + 1), dict(coef=None), dict(steps=0), dict(steps=65), dict(g=None), dict(out=None), dict(ld=7),
                                    dict(out_ld=7), dict(g=P + 2), dict(out=P + 1), dict(g_stride=-1), dict(out_stride=63)])
def test_orthogonalize(lib, change):
    refused(lib, "ts2_op_orthogonalize", ORTH, **change)


# Singular values of G / |G| lie in [0, 1].  (4, 0, 0) takes 1 to 4 > 3.9; (12, -12, c): 12 s (1 - s^2) is 4.6 at s = 0.577 although it is 0 at 1, and
# so is (12, -12, 1e-30), whose other extremum is at 1e15; (0, 32, 0): B = 32; (2, 0, 0) leaves the range in the second step; (-4, 0, 0) as (4, 0, 0)
@pytest.mark.parametrize("coef,steps", [((4, 0, 0), 1), ((12, -12, 0), 1), ((12, -12, 1e-30), 1), ((12, -12, -1e-30), 2), ((0, 32, 0), 1), ((0, 0, -32), 1),
                                        ((2, 0, 0), 2), ((-4, 0, 0), 1), ((NAN, 0, 0), 1), ((1, NAN, 0), 1), ((1, 0, NAN), 1),
                                        ((float("inf"), 0, 0), 1), ((1, 3e38, -3e38), 1), ((1.05, 0, 0), 64)])
def test_orthogonalize_refuses_coefficients_that_leave_the_range_of_fp16(lib, coef, steps):
    refused(lib, "ts2_op_orthogonalize", ORTH, rc=capi.TS2_ERR_UNSUPPORTED, coef=(C.c_float * 3)(*coef), steps=steps)
