"""How much scratch a dense layer's gradients take for K ranges: less than the library's pool keeps between calls."""
import pytest

from test_linear_gpu import ACT, KIND, capi, check, ptr, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_partial_sums_stay_inside_the_pool():
    T, n, m = 307_425, 19_456, 10_336
    lib = capi.load_library()
    x, dy, dw = torch.ones((T, n), device="cuda", dtype=torch.bfloat16), torch.ones((T, m), device="cuda", dtype=torch.bfloat16), torch.zeros((m, n), device="cuda")
    torch.cuda.synchronize()
    check(lib.ts2_dev_trim(0))
    before = torch.cuda.mem_get_info()[0]
    check(lib.ts2_op_linear_backward(0, stream(), KIND["bf16"], ACT["none"], T, n, m, ptr(dy), m, None, m, ptr(x), n, None, n, None, n, KIND["f32"], ptr(dw), n, None))
    taken = before - torch.cuda.mem_get_info()[0]  # scratch is given back when the device is waited for
    torch.cuda.synchronize()
    assert taken < 1.2e9, taken
    assert (dw == T).all()
