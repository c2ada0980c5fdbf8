"""The 8-bit serving operators in a row, as a decoder's layer runs them: quantise -> project -> tables -> store -> attend ->
quantise -> project. Every step is compared with its plain form on the step's own inputs; the run again on another stream, and
captured and replayed, has to give the same bits."""
import pytest
import torch

import composable_kernel_amd as ck
import serving_plain as sp

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Layer:
    """Weights, cache and buffers of one layer for at most `tokens` new tokens of `batch` sequences."""

    def __init__(self, batch, tokens, hidden=256, heads=6, kv=2, D=64, size=16, blocks=40, width=8, code=E4M3, seed=1):
        g = sp.gen(seed)
        self.batch, self.tokens, self.hidden, self.heads, self.kv, self.D, self.size, self.width = batch, tokens, hidden, heads, kv, D, size, width
        self.qkv = (heads + 2 * kv) * D
        self.w = []
        for n, k in ((self.qkv, hidden), (hidden, heads * D)):
            self.w.append(((sp.normal(g, (n, k)) * 100).clamp(-448, 448).to(E4M3).cuda(),
                           ((1 + torch.rand(-(-n // 128), -(-k // 128), generator=g)) / 1600).cuda()))
        self.x = sp.normal(g, (tokens, hidden), torch.bfloat16).cuda()
        new = lambda *shape, dtype=torch.bfloat16: torch.zeros(*shape, dtype=dtype, device="cuda")
        self.qx, self.sx = new(tokens, hidden, dtype=E4M3), new(tokens, -(-hidden // 128), dtype=torch.float32)
        self.proj, self.att, self.out = new(tokens, self.qkv), new(tokens, heads * D), new(tokens, hidden)
        self.qo, self.so = new(tokens, heads * D, dtype=E4M3), new(tokens, -(-heads * D // 128), dtype=torch.float32)
        cache = [new(blocks, kv, size, D, dtype=code), new(blocks, kv, size, D, dtype=code), new(blocks, kv, dtype=torch.float32),
                 new(blocks, kv, dtype=torch.float32)]
        self.cache = cache
        self.free = _int(torch.randperm(blocks, generator=g).tolist())
        self.table = new(batch, width, dtype=torch.int32)
        self.ctx, self.news = _int([0] * batch), _int([0] * batch)
        self.cu, self.kvs = new(batch + 1, dtype=torch.int32), new(batch, dtype=torch.int32)
        self.slots, self.used = new(tokens, dtype=torch.int32), new(1, dtype=torch.int32)
        self.taken = 0
        self.make()

    def make(self):
        """The arguments, once: they hold the workspaces too."""
        T, hd, D = self.tokens, self.heads * self.D, self.D
        desc = ck.KvCache8(*self.cache)
        q = self.proj[:, :hd].view(T, self.heads, D)
        k = self.proj[:, hd:hd + self.kv * D].view(T, self.kv, D)
        v = self.proj[:, hd + self.kv * D:].view(T, self.kv, D)
        o = self.att.view(T, self.heads, D)
        quant, gemm, attn = ck.DeviceBlockQuantizeF8("bf16"), ck.DeviceGemmBlockScaleF8("bf16"), ck.DevicePagedAttention8("bf16")
        tables, store = ck.DeviceKvCacheTables(), ck.DeviceKvCacheStore8("bf16")
        mm = lambda a, sa, w, c: gemm.MakeArgumentPointer(a, w[0], c, sa, w[1], T, w[0].shape[0], w[0].shape[1], a.stride(0), w[0].stride(0),
                                                          c.stride(0), sa.stride(), w[1].stride())
        qz = lambda x, codes, s: quant.MakeArgumentPointer(x, codes, s, T, x.shape[1], x.stride(0), codes.stride(0), *s.stride())
        # MaxKvLen is what the tables can hold, so that one captured launch serves every later step
        self.ops = [(quant, qz(self.x, self.qx, self.sx)), (gemm, mm(self.qx, self.sx, self.w[0], self.proj)),
                    (tables, tables.MakeArgumentPointer(self.ctx, self.news, self.free, self.table, self.cu, self.kvs, self.slots, self.used,
                                                        self.batch, self.free.numel(), self.width, self.width, T, self.size)),
                    (store, store.MakeArgumentPointer(k, v, self.slots, desc, T, k.stride()[:2], v.stride()[:2])),
                    (attn, attn.MakeArgumentPointer(q, o, self.table, self.cu, self.kvs, desc, self.batch, T, self.heads,
                                                    self.width * self.size, self.width, self.width, q.stride()[:2], o.stride()[:2],
                                                    ck.Scale(D ** -0.5))),
                    (quant, qz(self.att, self.qo, self.so)), (gemm, mm(self.qo, self.so, self.w[1], self.out))]
        for op, arg in self.ops:
            need = op.GetWorkSpaceSize(arg)
            if need:
                op.SetWorkSpacePointer(arg, torch.full((need,), 0x7F, dtype=torch.uint8, device="cuda"))

    def run(self):
        stream = torch.cuda.current_stream().cuda_stream
        for op, arg in self.ops:
            op.MakeInvokerPointer().Run(arg, ck.StreamConfig(stream))

    def begin(self, ctx, news, x):
        """The inputs of a step, written into the buffers that the operators (or a captured graph of them) read. The free list is
        turned so that its next entries are at the front."""
        self.ctx.copy_(_int(ctx))
        self.news.copy_(_int(news))
        self.x.copy_(x)
        self.free.copy_(torch.roll(self.free, -self.taken))
        self.taken = 0

    def state(self):
        # rows of tokens that belong to no sequence are no result
        n = int(self.cu[-1])
        return [t.clone() for t in (self.table, self.cu, self.kvs, self.slots, self.used, self.out[:n], self.att[:n])] + [
            t.clone().view(torch.uint8) if t.dtype == E4M3 else t.clone() for t in self.cache]

    def end(self):
        self.taken = int(self.used[0])


def _near(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bool(bad.any()), (what, float((got.double() - want).abs().max()), bad.nonzero()[:4].tolist())


def _check(layer, before, news):
    """Every operator of the step against its plain form on that operator's own inputs."""
    L, n, hd, D = layer, sum(news), layer.heads * layer.D, layer.D
    half = sp.HALF_STEP[torch.bfloat16]
    for x, q, s, w, c in ((L.x, L.qx, L.sx, L.w[0], L.proj), (L.att[:n], L.qo[:n], L.so[:n], L.w[1], L.out[:n])):
        codes, scales = sp.quantize(x.cpu())
        assert sp.same_codes(q.cpu(), codes) and torch.equal(s.cpu(), scales)
        want, mag, cut = sp.gemm(q.cpu(), w[0].cpu(), s.cpu(), w[1].cpu())
        # half a step of the output, fp32 sums (128 products a group, its sum times the scales, the groups) and the instruction's cut
        sums = (128 + scales.shape[1] + 4) * 2.0 ** -23 * mag + cut
        _near(c.cpu(), want, half * (want.abs() + sums) + sums + 1e-30, "projection")
    cache = [t.cpu().clone() for t in before]
    slots = L.slots.cpu().tolist()
    proj = L.proj.cpu()
    sp.store(cache[0], cache[2], proj[:, hd:hd + L.kv * D].reshape(-1, L.kv, D), slots)
    sp.store(cache[1], cache[3], proj[:, hd + L.kv * D:].reshape(-1, L.kv, D), slots)
    for got, want in zip(L.cache, cache):
        assert sp.same_codes(got.cpu(), want) if got.dtype in (torch.int8, E4M3) else torch.equal(got.cpu(), want)
    q = proj[:n, :hd].reshape(n, L.heads, D)
    o, mag, big = sp.attention(q, L.table.cpu(), L.cu.cpu().tolist(), L.kvs.cpu().tolist(), *cache, D ** -0.5, True)
    bound = sp.attention_bound(o, mag, big, torch.bfloat16, D, L.width * L.size)
    _near(L.att[:n].cpu().view(n, L.heads, D), o, bound + sp.small_products(cache[3], cache[1].dtype, int(L.kvs.max())), "attention")


STEPS = [[20, 0, 3, 17], [1, 1, 1, 1], [1, 0, 1, 1], [0, 5, 30, 1], [1, 1, 1, 1]]


def _steps(layer, seed=5):
    """(context lengths, new lengths, activations) of the steps; the activations' rows behind the last new token are padding."""
    g, ctx = sp.gen(seed), [0] * layer.batch
    for i, news in enumerate(STEPS):
        yield list(ctx), news, sp.normal(g, (layer.tokens, layer.hidden), torch.bfloat16, 1.0 + i).cuda()
        ctx = [c + n for c, n in zip(ctx, news)]


@pytest.mark.parametrize("code", [E4M3, torch.int8])
def test_steps_of_a_layer(code):
    layer = Layer(4, 40, code=code)
    for ctx, news, x in _steps(layer):
        layer.begin(ctx, news, x)
        before = [t.clone() for t in layer.cache]
        layer.run()
        torch.cuda.synchronize()
        assert layer.kvs.cpu().tolist() == [c + n for c, n in zip(ctx, news)] and int(layer.cu[-1]) == sum(news)
        _check(layer, before, news)
        layer.end()


def test_other_stream_and_graph_give_the_same_bits():
    want = []
    eager = Layer(4, 40)
    for ctx, news, x in _steps(eager):
        eager.begin(ctx, news, x)
        eager.run()
        torch.cuda.synchronize()
        want.append(eager.state())
        eager.end()

    aside, stream = Layer(4, 40), torch.cuda.Stream()
    for i, (ctx, news, x) in enumerate(_steps(aside)):
        aside.begin(ctx, news, x)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            aside.run()
        torch.cuda.current_stream().wait_stream(stream)
        assert all(torch.equal(a, b) for a, b in zip(aside.state(), want[i])), i
        aside.end()

    # one graph for all steps, its lengths read on the device; eager work of another layer between the replays
    captured, other = Layer(4, 40), Layer(4, 40, seed=9)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured.run()
    for i, (ctx, news, x) in enumerate(_steps(captured)):
        captured.begin(ctx, news, x)
        graph.replay()
        other.begin([0] * 4, [3, 4, 5, 6], x)
        other.run()
        torch.cuda.synchronize()
        other.end()
        assert all(torch.equal(a, b) for a, b in zip(captured.state(), want[i])), i
        captured.end()


def test_two_layers_at_once():
    """Two layers on two streams, each with its own buffers and workspaces, in turn without a wait between them."""
    layers, alone = [Layer(4, 40, seed=s) for s in (1, 2)], [Layer(4, 40, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for steps in zip(_steps(layers[0], 5), _steps(layers[1], 6)):
        for group in (layers, alone):
            for l, (ctx, news, x) in zip(group, steps):
                l.begin(ctx, news, x)
        torch.cuda.synchronize()
        for l, s in zip(layers, streams):
            with torch.cuda.stream(s):
                l.run()
        torch.cuda.synchronize()
        for l, a in zip(layers, alone):
            a.run()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(l.state(), a.state()))
            l.end()
            a.end()
