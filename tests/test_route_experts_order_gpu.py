"""DeviceRouteExperts where the order of the experts is hard to tell: scores that only 64 bits tell apart, ties, and more tokens than the
counts of a workgroup hold in a byte."""
import pytest
import torch

import experts_plain as ep
from test_route_experts_gpu import check, launch
import composable_kernel_amd as ck

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,k,groups,top", [(8, 2, 1, 1), (64, 8, 1, 1), (256, 8, 8, 4), (256, 16, 1, 1), (130, 31, 1, 1), (1024, 5, 1, 1), (600, 32, 4, 2)])
def test_sums_that_only_64_bits_tell_apart(scoring, E, k, groups, top):
    # beside a bias of 1000 a step of fp32 is 6e-5; the scores lie closer
    g = ep.gen(E + k)
    x = ep.normal(g, (40, E), scale=1e-3)
    check(x, torch.full((E,), 1000.0), k, scoring, True, groups, top, 1)
    check(x, 1000 + 2.0 ** -13 * torch.randint(0, 2, (E,), generator=g), k, scoring, False, groups, top, 2)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,k", [(8, 3), (64, 8), (256, 9), (256, 32), (512, 8), (1000, 32)])
def test_ties(scoring, biased, E, k):
    g = ep.gen(E + 7)
    x = torch.randint(0, 3, (70, E), generator=g).float()
    x[5], x[6] = 0.0, -0.0
    bias = torch.randint(0, 2, (E,), generator=g) * 0.25 if biased else None
    check(x, bias, k, scoring)
    check(x.bfloat16(), bias, k, scoring, False)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("E,k,T,live", [(8, 2, 65281, 65281), (8, 2, 70000, 65000), (128, 1, 66000, 66000), (1024, 2, 65600, 65555)])
def test_counts_that_no_byte_holds(kind, E, k, T, live):
    g = ep.gen(T)
    x = ep.normal(g, (T, E), ep.DT[kind])
    x[:, 1] += 2                                     # (an expert that most tokens take)
    op, arg, outs = launch(x, None, k, live=live)
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    ids, weights, offsets, rows, places = (t.cpu() for t in outs)
    want = x.float().sort(dim=1, descending=True, stable=True).indices[:, :k].int()
    want[live:] = -1
    assert torch.equal(ids, want)
    p = torch.gather(x.double(), 1, want.clamp(min=0).long()).softmax(dim=1)
    p[live:] = 0
    ep.near(weights, p, (2.0 ** -24 + 1e-13) * p.abs())
    flat = want.flatten().long()
    n = live * k
    order = torch.where(flat < 0, E, flat).sort(stable=True).indices
    assert torch.equal(rows[:n], order[:n].int()) and bool((rows[n:] == -1).all())
    assert torch.equal(offsets, torch.cat([torch.zeros(1, dtype=torch.long), torch.bincount(flat[:n], minlength=E).cumsum(0)]).int())
    back = torch.full((T * k,), -1, dtype=torch.int32)
    back[order[:n]] = torch.arange(n, dtype=torch.int32)
    assert torch.equal(places, back)


@pytest.mark.parametrize("E,k,bias", [(8, 2, False), (256, 8, True), (300, 32, True), (1024, 1, False)])
def test_no_tokens(E, k, bias):
    """The tables of no tokens: no logits are read, the offsets are 0."""
    offsets = torch.full((E + 2,), 7, dtype=torch.int32, device="cuda")
    op = ck.DeviceRouteExperts("f32")
    arg = op.MakeArgumentPointer(None, torch.zeros(E, device="cuda") if bias else None, None, None, None, offsets, None, None, 0, E, k, E)
    assert op.IsSupportedArgument(arg) and op.GetWorkSpaceSize(arg) == 0
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert offsets.tolist() == [0] * (E + 1) + [7]
