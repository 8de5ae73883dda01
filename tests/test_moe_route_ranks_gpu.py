"""ts2_op_moe_route_forward: groups ranked by the sum of two keys that are large and of opposite sign, or as large as fp32 gets.

ids are those of the definition in float64: ranks that differ by more than fp64 rounds.  A key near 10^4 is held to 2^-40 there, so ranks of different
groups, whose scores differ at random, are told apart."""
import pytest

from test_moe_route_gpu import KIND, SCORE, capi, case, check, ptr, stream

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


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,kept", GROUPS)
def test_groups_of_one_key_without_a_bias_go_by_logits(score, E, groups, kept):
    """logits of some hundred, whose scores float64 takes for one, or for zero"""
    T, per, k = 200, E // groups, min(4, kept * E // groups)
    l = 300 * torch.randn((T, E), device="cuda", generator=torch.Generator(device="cuda").manual_seed(E))
    ids, w = torch.zeros((T, k), device="cuda", dtype=torch.int32), torch.zeros((T, k), device="cuda")
    check(capi.load_library().ts2_op_moe_route_forward(0, stream(), KIND["f32"], SCORE[score], ptr(l), E, T, E, k, None, groups, kept, 1, 1, 1.0, None, ptr(ids), ptr(w)))
    order = torch.sort(l.view(T, groups, per).amax(2), dim=1, descending=True, stable=True).indices[:, :kept]
    keep = torch.zeros((T, groups), device="cuda", dtype=torch.bool).scatter_(1, order, True)
    want = torch.sort(torch.where(keep.repeat_interleave(per, 1), l, float("-inf")), dim=1, descending=True, stable=True).indices[:, :k]
    assert torch.equal(ids, want.int())
