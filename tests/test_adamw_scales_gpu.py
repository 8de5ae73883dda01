"""ts2_op_adamw: the order of the factors of a gradient, as the header has it.  Factors that are no powers of two, so that the order shows in moments of 8 bits, which are
defined to the bit; `verify` compares them."""
import pytest

from test_adamw_gpu import Tensor, np, verify

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("grad", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("scale,dev", [(0.3, 0.7), (-1.1, 3.3), (1.0 / 3, 1e-3)])
def test_two_factors(bits, grad, scale, dev):
    gen = torch.Generator(device="cuda").manual_seed(2)
    d = torch.tensor([dev], device="cuda")
    x = np.float32(1.0) + np.arange(1000, dtype=np.float32) * np.float32(1e-3)
    one = x * (np.float32(scale) * np.float32(dev))
    assert (one != x * np.float32(scale) * np.float32(dev)).any()  # the other order is another g
    verify([Tensor(n, gen, grad, bits) for n in (50_000, 33)], grad, bits, "none", 3, scale, d, seed=9)
