"""ts2_op_adamw: what decay does to parameters when it is as small as their rounding.

param, in [1, 2), is rounded to a step of 2^-23 each time, up or down at random because updates of about 1e-3 come on top.  So the mean over n parameters of (param - exact) is zero
up to 2^-23 / sqrt(12 n), six of which are allowed; the update's own errors, 2^-20 of it, have its random sign: 2^-20 of the mean update's deviation, 1e-3 / sqrt(n), six of
which are far less, and the sum that makes the update takes no more.  The product of rate and decay is an fp32 number, 2^-24 of itself for all alike."""
import ctypes as C

import pytest

from test_adamw_gpu import B1, B2, EPS, KIND, capi, check, np, stream

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("decay", [2e-5, 1e-4, 1e-3, 0.1])
def test_small_decays_keep_their_mean(bits, decay):
    n, rate = 1 << 20, float(np.float32(1e-3))
    decay = float(np.float32(decay))
    gen = torch.Generator(device="cuda").manual_seed(1)
    p = 1 + torch.rand(n, device="cuda", generator=gen)
    g = torch.randn(n, device="cuda", generator=gen)
    if bits == 32:
        m, v, ms, vs = torch.zeros(n, device="cuda"), torch.ones(n, device="cuda"), None, None
    else:  # v: 56 is one in e4m3, times 2^0
        m, v = torch.zeros(n, device="cuda", dtype=torch.uint8), torch.full((n,), 56, device="cuda", dtype=torch.uint8)
        ms, vs = torch.zeros(n // 32, device="cuda", dtype=torch.uint8), torch.full((n // 32,), 127, device="cuda", dtype=torch.uint8)
    p64, g64 = p.double(), g.double()
    up = rate * (1 - B1) * g64 / (1 - B1) / (((B2 + (1 - B2) * g64 * g64) / (1 - B2)).sqrt() + EPS)
    up *= 30  # the tensor's own rate, so that updates are about 1e-3
    want = p64 * (1 - 30 * rate * decay) - up
    table = (capi.AdamwTensor * 1)()
    t = table[0]
    t.param, t.grad, t.m, t.v, t.m_scale, t.v_scale, t.copy, t.n, t.rate, t.decay = *(None if x is None else x.data_ptr() for x in (p, g, m, v, ms, vs)), None, n, 30.0, decay
    check(capi.load_library().ts2_op_adamw(0, stream(), KIND["f32"], bits, KIND["none"], C.cast(table, C.c_void_p), 1, rate, B1, B2, EPS, 1, 1.0, None, 3))
    off = (p.double() - want).mean().item()
    assert abs(off) < 6 * (2.0 ** -23 / (12 * n) ** 0.5 + 2.0 ** -20 * 1e-3 / n ** 0.5) + 2.0 ** -24 * 30 * rate * decay * 1.5, (off, 30 * rate * decay * 1.5)
