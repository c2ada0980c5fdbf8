"""DeviceRouteExperts against its formula in 64 bits: ids and tables as they are, weights to half a step of fp32."""
import math

import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def launch(x, bias, k, scoring="softmax", renormalise=True, groups=1, top_groups=1, best=1, scale=1.0, live=None, tables=True, pad=0):
    """Operator, argument and the outputs' tensors; x on the CPU, its rows `pad` elements further apart on the GPU."""
    T, E = x.shape
    xd = torch.full((T, E + pad), 50.0, dtype=x.dtype, device="cuda")
    xd[:, :E] = x.cuda()
    new = lambda *shape: torch.full(shape, 77, dtype=torch.int32, device="cuda")
    outs = [new(T, k), torch.full((T, k), 7.0, device="cuda")] + ([new(E + 1), new(T * k), new(T * k)] if tables else [None] * 3)
    kind = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}[x.dtype]
    op = ck.DeviceRouteExperts(kind, Scoring=scoring, Renormalise=renormalise)
    number = None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda")
    arg = op.MakeArgumentPointer(xd, None if bias is None else bias.cuda(), number, *outs, T, E, k, E + pad, groups, top_groups, best,
                                 ck.Scale(scale))
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    need = op.GetWorkSpaceSize(arg)
    if need:
        op.SetWorkSpacePointer(arg, torch.full((need,), 0x7B, dtype=torch.uint8, device="cuda"))
    return op, arg, outs


def check(x, bias, k, scoring="softmax", renormalise=True, groups=1, top_groups=1, best=1, scale=1.0, live=None, **kw):
    op, arg, outs = launch(x, bias, k, scoring, renormalise, groups, top_groups, best, scale, live, **kw)
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    want = ep.route(x, bias, k, scoring, renormalise, groups, top_groups, best, scale, live)
    ids, weights = outs[0].cpu(), outs[1].cpu()
    assert torch.equal(ids, want[0]), (ids != want[0]).nonzero()[:4].tolist()
    # (rounded once from 64 bits, in which a score takes some ten roundings)
    ep.near(weights, want[1], (2.0 ** -24 + 1e-13) * want[1].abs() + 2.0 ** -149, "weights")
    for name, got, w in zip(("offsets", "rows", "places"), outs[2:], want[2:]):
        assert got is None or torch.equal(got.cpu(), w), name


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (17, 64, 8), (64, 65, 3), (65, 256, 8), (5, 300, 32), (2, 1024, 7), (130, 129, 1)])
def test_sizes(kind, scoring, biased, T, E, k):
    g = ep.gen(T * 31 + E)
    x = ep.normal(g, (T, E), ep.DT[kind], 2.0)  # (16-bit logits of many experts hold ties)
    bias = ep.normal(g, (E,), scale=0.2) if biased else None
    check(x, bias, k, scoring)
    check(x, bias, k, scoring, renormalise=False, scale=2.5, pad=3)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("best", [1, 2])
@pytest.mark.parametrize("E,k,groups,top", [(64, 8, 8, 4), (60, 6, 4, 1), (12, 3, 12, 5), (256, 8, 8, 4), (192, 32, 64, 7), (1024, 4, 2, 1), (9, 9, 3, 2)])
def test_groups(scoring, biased, best, E, k, groups, top):
    g = ep.gen(E + groups)
    x = ep.normal(g, (70, E), torch.bfloat16, 1.0)
    x[3] = 0                                         # all alike: the lowest numbers
    x[5].masked_fill_(torch.rand(E, generator=g) < 0.8, -INF)
    x[6] = -INF
    bias = ep.normal(g, (E,), scale=0.5) if biased else None
    check(x, bias, k, scoring, True, groups, top, best)
    check(x, bias, k, scoring, False, groups, top, best)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_rows_that_masks_leave_little_of(scoring, biased):
    E, k = 12, 4
    x = ep.normal(ep.gen(1), (9, E))
    x[0] = -INF
    x[1] = NAN
    x[2, 1:] = -INF
    x[3, :10] = torch.finfo(torch.float32).min       # the type's lowest value is a value
    x[4, 3], x[4, 7] = INF, INF
    x[5, 2], x[5, 4], x[5, 9] = NAN, INF, -INF
    x[6] = torch.tensor([0.0, -0.0] * 6)             # one value
    x[7] = torch.linspace(-700, 700, E)
    x[8] = torch.linspace(-3e38, 3e38, E)
    bias = None
    if biased:
        bias = torch.zeros(E)
        bias[5], bias[6], bias[8] = -INF, NAN, 2.0
    check(x, bias, k, scoring)
    check(x, bias, k, scoring, renormalise=False)


def test_an_infinite_bias_comes_first():
    bias = torch.zeros(8)
    bias[6], bias[2] = INF, INF
    check(ep.normal(ep.gen(2), (4, 8)), bias, 3, "sigmoid")


@pytest.mark.parametrize("T", [20, 64, 65, 700, 5000])
@pytest.mark.parametrize("live", [0, 1, 19, -3, 100000])
def test_padded_batches(T, live):
    x = ep.normal(ep.gen(T), (T, 16), scale=2.0)
    x[T // 2] = -INF
    check(x, None, 2, live=live)


@pytest.mark.parametrize("T,E,k", [(257, 8, 2), (1000, 256, 8), (4097, 60, 6), (9000, 2, 1)])
def test_tables_of_many_tokens(T, E, k):
    g = ep.gen(T)
    x = ep.normal(g, (T, E), torch.bfloat16) + ep.normal(g, (1, E), torch.bfloat16, 2.0)
    check(x, None, k)
    check(x, None, k, tables=False)


def test_graph_and_another_stream():
    T, E, k = 300, 64, 4
    xs = [ep.normal(ep.gen(s), (T, E)) for s in range(3)]
    op, arg, outs = launch(xs[0], None, k, live=T)
    x, live = arg._keep[0][0], arg._keep[0][2]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    side = torch.cuda.Stream()
    for n, fresh in zip((300, 7, 150), xs):
        x.copy_(fresh)
        live.fill_(n)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.cpu().clone() for t in outs]
        with torch.cuda.stream(side):
            op.MakeInvokerPointer().Run(arg, ck.StreamConfig(side.cuda_stream))
        torch.cuda.synchronize()
        want = ep.route(fresh, None, k, "softmax", True, live=n)
        assert all(torch.equal(a, b.cpu()) for a, b in zip(got, outs))
        assert all(torch.equal(a, b) for a, b in zip([got[0]] + got[2:], (want[0],) + want[2:]))
