"""What ts2_op_linear_*, ts2_op_moe_route_* and ts2_op_adamw refuse.  Arguments are looked at before the device is, so this runs
anywhere: a call that is refused never touches the GPU."""
import ctypes as C

import pytest

from test_layer_ops_cpu import BIG, NAN, P, lib  # noqa: F401
from tscale2_b200 import capi

F32, F32_ADD, F16, BF16 = capi.OUT_F32, capi.OUT_F32_ADD, capi.OUT_F16, capi.OUT_BF16
INF = float("inf")
FORWARD = dict(device=0, stream=None, type=F16, act=capi.ACT_GELU, T=4, n=8, m=16, x=P, x_ld=8, w=P, w_ld=8, bias=P, res=P, res_ld=16, y=P + 64, y_ld=16, z=P,
               z_ld=16)
BACKWARD = dict(device=0, stream=None, type=F16, act=capi.ACT_GELU, T=4, n=8, m=16, dy=P, dy_ld=16, z=P, z_ld=16, x=P, x_ld=8, w=P, w_ld=8, dx=P, dx_ld=8,
                dw_kind=F32, dw=P, dw_ld=8, dbias=P)
ROUTE = dict(device=0, stream=None, type=F32, score=capi.SCORE_SOFTMAX, logits=P, ld=8, T=4, E=8, k=2, bias=P, groups=4, kept=2, top=2, renorm=1, scale=1.0,
             mask=P, ids=P, weights=P)
ROUTE_BACK = dict(device=0, stream=None, type=F32, score=capi.SCORE_SIGMOID, logits=P, ld=8, T=4, E=8, k=2, renorm=1, scale=1.0, mask=P, ids=P, dweights=P,
                  dl=P, dl_ld=8, add=0)


def refused(lib, name, args, rc=capi.TS2_ERR_INVALID_ARG, **change):  # noqa: F811
    assert set(change) <= set(args)
    assert getattr(lib, name)(*{**args, **change}.values()) == rc, change
    assert name.encode() in lib.ts2_last_error(None)


@pytest.mark.parametrize("change", [dict(type=F32), dict(type=F32_ADD), dict(type=-1), dict(act=-1), dict(act=4), dict(T=-1), dict(T=(1 << 30) + 1), dict(n=0),
                                    dict(m=0), dict(n=(1 << 20) + 1), dict(m=(1 << 20) + 1), dict(T=1 << 30, m=1 << 20, y_ld=1 << 20, z_ld=1 << 20, res_ld=1 << 20),
                                    dict(x=None), dict(w=None), dict(y=None), dict(x_ld=7), dict(w_ld=7), dict(y_ld=15), dict(z_ld=15), dict(res_ld=15),
                                    dict(x_ld=BIG), dict(x=P + 1), dict(w=P + 1), dict(y=P + 1), dict(z=P + 1), dict(res=P + 1), dict(bias=P + 2),
                                    dict(res=P + 64, res_ld=24)])
def test_linear_forward(lib, change):  # noqa: F811
    refused(lib, "ts2_op_linear_forward", FORWARD, **change)


@pytest.mark.parametrize("change", [dict(type=F32), dict(act=-1), dict(act=4), dict(T=-1), dict(n=0), dict(m=0), dict(dy=None), dict(z=None), dict(x=None),
                                    dict(w=None), dict(dy_ld=15), dict(z_ld=15), dict(x_ld=7), dict(w_ld=7), dict(dx_ld=7), dict(dw_ld=7), dict(dw_kind=BF16),
                                    dict(dw_kind=7), dict(dw=P + 2), dict(dw=P + 1, dw_kind=F16), dict(dx=P + 1), dict(dbias=P + 2), dict(z=P + 1)])
def test_linear_backward(lib, change):  # noqa: F811
    refused(lib, "ts2_op_linear_backward", BACKWARD, **change)


@pytest.mark.parametrize("change", [dict(type=1), dict(score=-1), dict(score=2), dict(T=-1), dict(T=(1 << 30) + 1), dict(E=0), dict(k=0), dict(k=9), dict(logits=None),
                                    dict(ids=None), dict(weights=None), dict(ld=7), dict(ld=BIG), dict(logits=P + 2), dict(bias=P + 1), dict(ids=P + 2),
                                    dict(weights=P + 1), dict(groups=0), dict(groups=3), dict(groups=16), dict(kept=0), dict(kept=5), dict(top=0), dict(top=3),
                                    dict(groups=8), dict(k=5), dict(kept=1, k=3), dict(scale=NAN), dict(scale=INF)])
def test_route_forward(lib, change):  # noqa: F811
    refused(lib, "ts2_op_moe_route_forward", ROUTE, **change)


@pytest.mark.parametrize("change", [dict(type=1), dict(score=2), dict(T=-1), dict(E=0), dict(k=0), dict(k=9), dict(logits=None), dict(ids=None), dict(dweights=None),
                                    dict(dl=None), dict(ld=7), dict(dl_ld=7), dict(logits=P + 2), dict(ids=P + 2), dict(dweights=P + 2), dict(dl=P + 2),
                                    dict(scale=-INF)])
def test_route_backward(lib, change):  # noqa: F811
    refused(lib, "ts2_op_moe_route_backward", ROUTE_BACK, **change)


@pytest.mark.parametrize("E,k,groups", [(1025, 1, 1), (4096, 8, 8), (64, 33, 1), (64, 2, 64)])
def test_route_limits(lib, E, k, groups):  # noqa: F811
    refused(lib, "ts2_op_moe_route_forward", ROUTE, rc=capi.TS2_ERR_UNSUPPORTED, E=E, ld=E, k=k, groups=groups, kept=groups, top=1)
    if groups < 64:
        refused(lib, "ts2_op_moe_route_backward", ROUTE_BACK, rc=capi.TS2_ERR_UNSUPPORTED, E=E, ld=E, dl_ld=E, k=k)


def adamw_args(n=2, **change):
    a = dict(device=0, stream=None, grad_type=BF16, bits=8, copy_type=F16, tensors=None, n=n, rate=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, step=1, scale=1.0,
             scale_dev=P, seed=1)
    t = dict(param=P, grad=P, m=P, v=P, m_scale=P, v_scale=P, copy=P, n=5, rate=1.0, decay=0.1)
    table = (capi.AdamwTensor * max(1, n))()
    for i in range(n):
        for k, v in {**t, **(change.pop("tensor", {}) if i == n - 1 else {})}.items():
            setattr(table[i], k, v)
    a["tensors"] = C.cast(table, C.c_void_p)
    a.update(change)
    return a, table


@pytest.mark.parametrize("change", [dict(grad_type=1), dict(bits=16), dict(bits=0), dict(copy_type=1), dict(copy_type=F32), dict(tensors=None), dict(n=-1),
                                    dict(rate=NAN), dict(rate=INF), dict(beta1=1.0), dict(beta1=-0.1), dict(beta1=NAN), dict(beta2=1.0), dict(beta2=NAN),
                                    dict(eps=0.0), dict(eps=1e-39), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF), dict(step=0), dict(step=-3), dict(scale=NAN),
                                    dict(scale_dev=P + 2)] +
                         [dict(tensor=t) for t in (dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(m_scale=None), dict(v_scale=None),
                                                   dict(param=P + 2), dict(grad=P + 1), dict(copy=P + 1), dict(n=-1), dict(n=(1 << 40) + 1), dict(n=1 << 40),
                                                   dict(rate=NAN), dict(decay=INF))])
def test_adamw(lib, change):  # noqa: F811
    n = change.pop("n", None)
    a, keep = adamw_args(**change)
    if n is not None:
        a["n"] = n
    refused(lib, "ts2_op_adamw", a)


@pytest.mark.parametrize("tensor", [dict(m=P + 2), dict(v=P + 1), dict(grad=P + 2)])
def test_adamw_32_bit_moments_are_floats(lib, tensor):  # noqa: F811
    a, keep = adamw_args(bits=32, grad_type=F32, tensor=tensor)
    refused(lib, "ts2_op_adamw", a)


def test_the_table_of_tensors_has_the_header_s_layout():
    assert C.sizeof(capi.AdamwTensor) == 72 and capi.AdamwTensor.n.offset == 56 and capi.AdamwTensor.rate.offset == 64
