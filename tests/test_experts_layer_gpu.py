"""The int8 linear and mixture-of-experts operators in a row, as a layer runs them: route -> quantise -> experts up (gated, rows
gathered) -> quantise -> experts down -> a shared gated MLP on all tokens -> weighted sum on top of it. Every step is compared with its
plain form on the step's own inputs; the run again on another stream, and captured and replayed with other numbers of tokens, has to give
the same bits."""
import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep

pytestmark = pytest.mark.gpu


class Layer:
    """Weights and buffers of one layer for at most `tokens` tokens; `ranks`: the experts' products are launched in so many slices of the
    experts, as ranks that hold a part each would."""

    def __init__(self, tokens, hidden=256, inner=192, experts=12, k=3, groups=4, top_groups=2, scoring="sigmoid", seed=1, ranks=1):
        g = ep.gen(seed)
        self.T, self.H, self.I, self.E, self.k, self.groups, self.top, self.scoring = tokens, hidden, inner, experts, k, groups, top_groups, scoring
        new = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype, device="cuda")
        i32, f32, i8 = dict(dtype=torch.int32), dict(dtype=torch.float32), dict(dtype=torch.int8)
        weights = lambda e, n, m: (ep.codes(g, (e, n, m)).cuda(), ((0.5 + torch.rand(e, n, generator=g)) / (74 * m ** 0.5)).cuda())
        self.up, self.down = weights(experts, 2 * inner, hidden), weights(experts, hidden, inner)
        self.s_up, self.s_down = weights(1, 2 * inner, hidden), weights(1, hidden, inner)
        self.bias = ep.normal(g, (experts,), scale=0.2).cuda()
        self.x, self.logits, self.live = new(tokens, hidden), new(tokens, experts, **f32), new(1, **i32)
        pairs = tokens * k
        self.ids, self.w = new(tokens, k, **i32), new(tokens, k, **f32)
        self.offsets, self.rows, self.places = new(experts + 1, **i32), new(pairs, **i32), new(pairs, **i32)
        self.q, self.s = new(tokens, hidden, **i8), new(tokens, **f32)
        self.h, self.y = new(pairs, inner), new(pairs, hidden)
        self.qh, self.sh = new(pairs, inner, **i8), new(pairs, **f32)
        self.hs, self.qs, self.ss, self.out = new(tokens, inner), new(tokens, inner, **i8), new(tokens, **f32), new(tokens, hidden)
        self.ranks = ranks
        self.make()

    def make(self):
        T, H, I, E, k = self.T, self.H, self.I, self.E, self.k
        route, quant, combine = ck.DeviceRouteExperts("f32", self.scoring), ck.DeviceTokenQuantizeI8("bf16"), ck.DeviceExpertsCombine("bf16")
        up, down, mm_up, mm_down = (ck.DeviceExpertsGemmI8("bf16", True), ck.DeviceExpertsGemmI8("bf16"), ck.DeviceGemmTokenScaleI8("bf16", True),
                                    ck.DeviceGemmTokenScaleI8("bf16"))
        qz = lambda x, q, s: quant.MakeArgumentPointer(x, q, s, *x.shape, x.stride(0), q.stride(0))
        mm = lambda op, a, sa, w, c: op.MakeArgumentPointer(a, w[0], c, sa, w[1], None, a.shape[0], c.shape[1], a.shape[1], a.stride(0), w[0].stride(1),
                                                            c.stride(0))
        self.ops = [(route, route.MakeArgumentPointer(self.logits, self.bias, self.live, self.ids, self.w, self.offsets, self.rows, self.places, T, E, k,
                                                      E, self.groups, self.top, 2, ck.Scale(1.5))),
                    (quant, qz(self.x, self.q, self.s))]
        cuts = [E * r // self.ranks for r in range(self.ranks + 1)]
        products = lambda op, a, sa, w, c, rows, per: [
            (op, op.MakeArgumentPointer(a, w[0][i:j], c, sa, w[1][i:j], None, self.offsets[i:], rows, T * k, a.shape[0], j - i, c.shape[1], a.shape[1],
                                        a.stride(0), w[0].stride(1), c.stride(0), w[0].stride(0), per)) for i, j in zip(cuts, cuts[1:])]
        self.ops += products(up, self.q, self.s, self.up, self.h, self.rows, k) + [(quant, qz(self.h, self.qh, self.sh))]
        self.ops += products(down, self.qh, self.sh, self.down, self.y, None, 1)
        self.ops += [(mm_up, mm(mm_up, self.q, self.s, self.s_up, self.hs)), (quant, qz(self.hs, self.qs, self.ss)),
                     (mm_down, mm(mm_down, self.qs, self.ss, self.s_down, self.out)),
                     (combine, combine.MakeArgumentPointer(self.y, self.places, self.w, self.out, self.out, T, k, T * k, H, H, H, H))]
        for op, arg in self.ops:
            need = op.GetWorkSpaceSize(arg)
            if need:
                op.SetWorkSpacePointer(arg, torch.full((need,), 0x7F, dtype=torch.uint8, device="cuda"))

    def run(self, last=None):
        stream = torch.cuda.current_stream().cuda_stream
        for op, arg in self.ops[:last]:
            op.MakeInvokerPointer().Run(arg, ck.StreamConfig(stream))

    def begin(self, live, x, logits):
        self.live.fill_(live)
        self.x.copy_(x)
        self.logits.copy_(logits)

    def state(self):
        n = int(self.offsets[-1])   # (rows that belong to no expert are no result)
        return [t.clone() for t in (self.ids, self.w, self.offsets, self.rows, self.places, self.q, self.s, self.h[:n], self.y[:n], self.hs, self.out)]


def inputs(layer, seed):
    """(tokens that are there, activations, logits) of the steps; a token whose mask leaves no expert, one far from all others."""
    for i, live in enumerate((layer.T, 1, 0, layer.T // 2, layer.T)):
        g = ep.gen(seed + i)
        x, logits = ep.normal(g, (layer.T, layer.H), torch.bfloat16, 1.0 + i), ep.normal(g, (layer.T, layer.E), scale=2.0)
        logits[layer.T // 3] = -float("inf")
        x[layer.T // 2] *= 1000
        yield live, x.cuda(), logits.cuda()


def check(layer, live):
    L, cpu = layer, lambda t: t.cpu()
    ids, w, offsets, rows, places = ep.route(cpu(L.logits), cpu(L.bias), L.k, L.scoring, True, L.groups, L.top, 2, 1.5, live)
    for name, want in (("ids", ids), ("offsets", offsets), ("rows", rows), ("places", places)):
        assert torch.equal(cpu(getattr(L, name)), want), name
    ep.near(cpu(L.w), w, (2.0 ** -24 + 1e-13) * w.abs() + 2.0 ** -149, "weights")
    for x, q, s in ((L.x, L.q, L.s), (L.hs, L.qs, L.ss)):
        codes, scales = ep.quantize(cpu(x))
        assert torch.equal(cpu(q), codes) and torch.equal(cpu(s), scales)
    n = int(offsets[-1])
    codes, scales = ep.quantize(cpu(L.h[:n])) if n else (cpu(L.qh[:0]), cpu(L.sh[:0]))
    assert torch.equal(cpu(L.qh[:n]), codes) and torch.equal(cpu(L.sh[:n]), scales)
    for e in range(L.E):
        i, j = int(offsets[e]), int(offsets[e + 1])
        if i == j:
            continue
        token = (rows[i:j] // L.k).long()
        ep.near(cpu(L.h[i:j]), *ep.scaled(cpu(L.q)[token], cpu(L.up[0][e]), cpu(L.s)[token], cpu(L.up[1][e]), None, True, torch.bfloat16), f"up {e}")
        ep.near(cpu(L.y[i:j]), *ep.scaled(cpu(L.qh[i:j]), cpu(L.down[0][e]), cpu(L.sh[i:j]), cpu(L.down[1][e]), None, False, torch.bfloat16), f"down {e}")
    ep.near(cpu(L.hs), *ep.scaled(cpu(L.q), cpu(L.s_up[0][0]), cpu(L.s), cpu(L.s_up[1][0]), None, True, torch.bfloat16), "shared up")


@pytest.mark.parametrize("T,scoring", [(1, "softmax"), (40, "sigmoid"), (700, "softmax")])
def test_steps_of_a_layer(T, scoring):
    layer = Layer(T, scoring=scoring)
    for live, x, logits in inputs(layer, T):
        layer.begin(live, x, logits)
        layer.run(-1)
        shared = layer.out.cpu()
        ep.near(shared, *ep.scaled(layer.qs.cpu(), layer.s_down[0][0].cpu(), layer.ss.cpu(), layer.s_down[1][0].cpu(), None, False, torch.bfloat16),
                "shared down")
        op, arg = layer.ops[-1]
        op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        check(layer, live)
        ep.near(layer.out.cpu(), *ep.combine(layer.y.cpu(), layer.places.cpu().view(T, layer.k), layer.w.cpu(), shared, torch.bfloat16), "out")


def test_other_stream_graph_and_slices_give_the_same_bits():
    T, want = 90, []
    eager = Layer(T)
    for step in inputs(eager, 3):
        eager.begin(*step)
        eager.run()
        torch.cuda.synchronize()
        want.append(eager.state())

    aside, stream = Layer(T), torch.cuda.Stream()
    for i, step in enumerate(inputs(aside, 3)):
        aside.begin(*step)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            aside.run()
        torch.cuda.current_stream().wait_stream(stream)
        assert all(torch.equal(a, b) for a, b in zip(aside.state(), want[i])), i

    # three ranks' experts, one slice after the other
    sliced = Layer(T, ranks=3)
    for i, step in enumerate(inputs(sliced, 3)):
        sliced.begin(*step)
        sliced.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(sliced.state(), want[i])), i

    # one graph for all steps, the number of tokens read on the device; eager work of another layer between the replays
    captured, other = Layer(T), Layer(T, seed=9)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured.run()
    for i, step in enumerate(inputs(captured, 3)):
        captured.begin(*step)
        graph.replay()
        other.begin(*step)
        other.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured.state(), want[i])), i


def test_two_layers_at_once():
    """Two layers on two streams, each with its own buffers and workspaces, in turn without a wait between them."""
    layers, alone = [Layer(300, seed=s) for s in (1, 2)], [Layer(300, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for steps in zip(inputs(layers[0], 5), inputs(layers[1], 6)):
        for group in (layers, alone):
            for l, step in zip(group, steps):
                l.begin(*step)
        torch.cuda.synchronize()
        for l, s in zip(layers, streams):
            with torch.cuda.stream(s):
                l.run()
        torch.cuda.synchronize()
        for l, a in zip(layers, alone):
            a.run()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(l.state(), a.state()))
