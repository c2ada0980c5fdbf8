"""DeviceRouteExperts where fp32 scores say nothing: tokens that the kernel of four tokens a wave leaves to 64 bits, alone in a wave, among
others, and all of a launch."""
import pytest
import torch

import experts_plain as ep
from test_route_experts_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("E,k,groups,top,best", [(8, 2, 1, 1, 1), (64, 8, 1, 1, 1), (256, 8, 1, 1, 1), (256, 8, 8, 4, 2), (128, 16, 4, 2, 1), (24, 6, 3, 2, 2)])
@pytest.mark.parametrize("T", [5, 130, 700])
def test_peaked_scores_and_biases_of_zero(scoring, kind, E, k, groups, top, best, T):
    """One expert has nearly all of the softmax (each of the others next to none of it), or every sigmoid is next to 0."""
    g = ep.gen(E + T)
    x = 8 * ep.normal(g, (T, E)) - 40
    check(x.to(ep.DT[kind]), torch.zeros(E), k, scoring, True, groups, top, best, live=T - 1)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("every", [1, 2, 3, 5, 64])
def test_some_tokens_in_doubt(scoring, every):
    """Tokens in doubt (scores that differ by less than fp32 has steps) beside others, in every place of a wave."""
    T, E, k = 333, 64, 6
    g = ep.gen(every)
    x = ep.normal(g, (T, E))
    x[::every] = 1 + ep.normal(g, (-(-T // every), E), scale=1e-6)
    x[7], x[9, 3] = float("inf"), float("inf")
    check(x, ep.normal(g, (E,), scale=0.1), k, scoring)
    check(x, torch.zeros(E), k, scoring, True, 8, 3, 2, scale=2.5)


@pytest.mark.parametrize("E,k,groups,top", [(256, 15, 1, 1), (256, 16, 1, 1), (256, 17, 1, 1), (160, 6, 8, 3), (32, 16, 2, 1), (16, 16, 1, 1)])
def test_as_many_picks_as_a_row_of_lanes(E, k, groups, top):
    g = ep.gen(E + k)
    x = ep.normal(g, (70, E))
    for scoring, bias in (("softmax", None), ("sigmoid", ep.normal(g, (E,), scale=0.1)), ("softmax", ep.normal(g, (E,), scale=1e-7))):
        check(x, bias, k, scoring, True, groups, top, 2)
