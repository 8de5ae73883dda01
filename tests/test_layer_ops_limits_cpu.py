"""Limits that the header states are looked at before the device is, as all other arguments are: a refused call never touches the
GPU."""
import pytest

from test_layer_ops_cpu import BALANCE, BF16, F16, F32, GRADIENT, P, lib, refused  # noqa: F401
from tscale2_b200 import capi


@pytest.mark.parametrize("type_", [F32, F16, BF16])
@pytest.mark.parametrize("E,k", [(1025, 1), (1025, 1025), (4096, 8), (1 << 20, 2)])
def test_more_experts_than_a_router_may_have(lib, type_, E, k):  # noqa: F811
    refused(lib, "ts2_op_moe_balance_forward", BALANCE, rc=capi.TS2_ERR_UNSUPPORTED, type=type_, ld=E, E=E, k=k)
    refused(lib, "ts2_op_moe_balance_backward", GRADIENT, rc=capi.TS2_ERR_UNSUPPORTED, type=type_, ld=E, E=E, k=k, dl=P, dl_ld=E)
