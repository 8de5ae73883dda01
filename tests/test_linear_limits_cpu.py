"""The largest dense layers: ceil(T / 128) * ceil(d / 64) has to be below 2^30, d the larger of in_dim and out_dim.  Calls on the refused side of that border;
arguments are looked at before the device is."""
import pytest

from test_layer_ops_cpu import lib  # noqa: F401
from test_layer_ops_more_cpu import BACKWARD, FORWARD, refused

M = 1 << 20


@pytest.mark.parametrize("T,d", [(1 << 30, 8129), (1 << 30, 8192), (1 << 29, 16321), ((1 << 30) - 127, 8129), ((1 << 23) - 127, M), (1 << 23, M - 63)])
def test_tokens_times_columns(lib, T, d):  # noqa: F811
    assert -(-T // 128) * -(-d // 64) >= 1 << 30
    for n, m in ((d, 16), (16, d)):
        refused(lib, "ts2_op_linear_forward", FORWARD, T=T, n=n, m=m, x_ld=M, w_ld=M, res_ld=M, y_ld=M, z_ld=M)
        refused(lib, "ts2_op_linear_backward", BACKWARD, T=T, n=n, m=m, dy_ld=M, z_ld=M, x_ld=M, w_ld=M, dx_ld=M, dw_ld=M)
