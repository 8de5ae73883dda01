"""ts2_op_moe_route_forward: groups ranked by the sum of two keys that are large and of opposite sign, or as large as fp32 gets.

ids are those of the definition in float64: ranks that differ by more than fp64 rounds.  A key near 10^4 is held to 2^-40 there, so ranks of different
groups, whose scores differ at random, are told apart."""
import pytest

from test_moe_route_gpu import case

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# neighbours in a group: a power of two from 8 on in rows that one warp's lanes hold at once, the same in longer rows, multiples of 8, others
GROUPS = [(64, 8, 4), (256, 8, 4), (256, 16, 8), (1024, 32, 16), (96, 4, 2), (240, 10, 5), (4, 2, 1), (64, 32, 16), (100, 10, 4)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,kept", GROUPS)
@pytest.mark.parametrize("size", [1e2, 1e3, 1e4])
def test_biases_that_cancel_in_a_group(score, E, groups, kept, size):
    """one expert of each group forced, the others pushed out: a group's rank is the sum of two scores, and its keys are `size`"""
    T = 3000 if E <= 128 else 600
    gen = torch.Generator(device="cuda").manual_seed(E + groups)
    b = torch.full((E,), -size, device="cuda")
    b[:: E // groups] = size
    case("f32", score, T, E, min(4, kept * E // groups), True, groups, kept, 2, b=b, seed=E)
    b = torch.where(torch.rand(E, device="cuda", generator=gen) < 0.5, -size, size)
    case("bf16", score, T, E, min(4, kept * E // groups), True, groups, kept, 2, b=b, seed=E)


def test_the_smallest_such_row():
    """exact ranks 1.147739 and 1.147875; the fp32 sums of the keys are 1.148438 and 1.147461"""
    logits = torch.tensor([[-0.35720438, 1.0258067, 2.0709758, -1.0468799]], device="cuda")
    b = torch.tensor([1e4, -1e4, 1e4, -1e4], device="cuda")
    case("f32", "sigmoid", 1, 4, 2, True, 2, 1, 2, logits=logits, b=b)
