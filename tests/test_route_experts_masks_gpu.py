"""DeviceRouteExperts where biases mask groups with the lowest value of a type: such experts are available, and their groups stay in the
order of their sums in 64 bits, which fp32 does not hold."""
import math

import pytest
import torch

import experts_plain as ep
from test_route_experts_gpu import check

pytestmark = pytest.mark.gpu

LOWEST = {"f32": torch.finfo(torch.float32).min, "bf16": torch.finfo(torch.bfloat16).min, "sum": -1.8e38}


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("lowest", sorted(LOWEST))
@pytest.mark.parametrize("E,groups,top,k", [(32, 8, 4, 8), (256, 8, 4, 8), (64, 16, 5, 16), (12, 3, 2, 6), (16, 16, 3, 2), (128, 2, 1, 4), (512, 8, 4, 8), (160, 8, 3, 6)])
def test_masked_groups(scoring, best, lowest, E, groups, top, k):
    size, low = E // groups, LOWEST[lowest]
    x = ep.normal(ep.gen(E + top), (37, E))
    last = torch.arange(E) >= E - size               # (all groups but the last are masked)
    check(x, torch.where(last, 0.0, low), k, scoring, True, groups, top, best)
    check(x.bfloat16(), torch.where(last, 0.0, low), k, scoring, True, groups, top, best)
    # every group; one expert of each left; one group's experts not available at all
    check(x, torch.full((E,), low), k, scoring, True, groups, top, best)
    check(x, torch.where(torch.arange(E) % size == size - 1, 0.1, low), k, scoring, True, groups, top, best)
    check(x, torch.where(torch.arange(E) < size, -math.inf, low), k, scoring, True, groups, top, best)


@pytest.mark.parametrize("E,groups,top,k", [(32, 8, 5, 12), (256, 8, 7, 16), (320, 8, 5, 12)])
def test_groups_of_different_lowest_values(E, groups, top, k):
    """Sums past fp32 are told apart by their values, and one that fp32 holds comes before them."""
    size = E // groups
    lows = [LOWEST["f32"], LOWEST["sum"], -1.7e38, LOWEST["bf16"], -1e38, LOWEST["f32"], -3.0, torch.finfo(torch.float32).max]
    bias = torch.tensor(lows).repeat_interleave(size)
    x = ep.normal(ep.gen(E), (21, E))
    x[4], x[5, ::3] = -math.inf, torch.finfo(torch.float32).min
    for scoring in ("softmax", "sigmoid"):
        check(x, bias, k, scoring, True, groups, top, 2)
        check(x, bias.flip(0), k, scoring, True, groups, top, 2)
