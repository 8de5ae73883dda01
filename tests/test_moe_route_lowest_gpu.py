"""ts2_op_moe_route_forward: biases of fp32's lowest and largest value, which take experts out or force them without being infinite.

Such an expert counts in its group and is chosen last (or first): in float64 a score beside a bias of 2^128 is rounded away, so among equal biases the lowest index
comes first."""
import pytest

from test_moe_route_gpu import case

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LOW, HIGH = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
# neighbours in a group: 8, 16, 32 in rows of 1024, 24, 10, 2
GROUPS = [(32, 4, 2), (256, 16, 8), (1024, 32, 4), (96, 4, 2), (60, 6, 3), (16, 8, 4)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("E,groups,kept", GROUPS)
def test_all_of_a_group_at_the_lowest_value(score, kind, E, groups, kept):
    """one group left, and the others fill up what is missing"""
    per = E // groups
    b = torch.full((E,), LOW, device="cuda")
    b[per:2 * per] = 0
    for top in (1, 2):
        case(kind, score, 50, E, min(32, per + 2, kept * per), True, groups, kept, top, b=b, seed=E)
    b[1] = 0.5 * LOW  # a group of one rank of its own
    case(kind, score, 50, E, min(32, per + 2, kept * per), True, groups, kept, 2, b=b, seed=E)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,groups,kept", GROUPS)
def test_groups_forced_by_the_largest_value(score, E, groups, kept):
    per = E // groups
    b = torch.zeros(E, device="cuda")
    b[:2], b[per:per + 2], b[2 * per - 1] = 0.75 * HIGH, HIGH, 0.875 * HIGH
    for keep in (1, kept):
        case("f32", score, 50, E, min(4, keep * per), True, groups, keep, 2, b=b, seed=E)
    b[:2] = torch.tensor([HIGH, LOW], device="cuda")  # keys that cancel
    case("f32", score, 50, E, min(4, kept * per), True, groups, kept, 2, b=b, seed=E)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_without_groups(score):
    b = torch.full((40,), LOW, device="cuda")
    b[[3, 9, 27]] = torch.tensor([0.1, HIGH, 0.0], device="cuda")
    case("f32", score, 50, 40, 8, True, b=b)
