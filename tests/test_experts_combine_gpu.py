"""DeviceExpertsCombine against its formula in 64 bits."""
import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep

pytestmark = pytest.mark.gpu


def check(T, k, N, kind, added, pads=(0, 0, 0), missing=0.0, in_place=False, seed=0):
    g, dt = ep.gen(seed + T + k + N), ep.DT[kind]
    P = T * k
    y = ep.normal(g, (P, N), dt)
    places = torch.randperm(P, generator=g).view(T, k).int()
    if missing:
        out = torch.rand(T, k, generator=g) < missing
        places[out] = torch.tensor([-1, P, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[torch.randint(0, 4, (int(out.sum()),), generator=g)]
        places[T // 2] = -1
    weights = torch.rand(T, k, generator=g)
    add = ep.normal(g, (T, N), dt) if added else None
    wide = lambda x, pad: torch.cat([x, torch.full((x.shape[0], pad), 9.0, dtype=dt)], dim=1).cuda()
    yd = wide(y, pads[0])
    ad = None if add is None else wide(add, pads[1])
    out = ad if in_place else torch.full((T, N + pads[2]), 55.0, dtype=dt, device="cuda")
    op = ck.DeviceExpertsCombine(kind)
    arg = op.MakeArgumentPointer(yd, places.cuda(), weights.cuda(), ad, out, T, k, P, N, N + pads[0], N + pads[1], N + (pads[1] if in_place else pads[2]))
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    out = out.cpu()
    assert bool((out[:, N:] == (9 if in_place else 55)).all())
    want, bound = ep.combine(y, places, weights, add, dt)
    ep.near(out[:, :N], want, bound, (T, k, N))


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (1, 8, 4096), (3, 2, 7), (5, 8, 2049), (9, 32, 100), (17, 3, 8), (300, 6, 513), (4, 9, 5000)])
def test_sizes(kind, added, T, k, N):
    check(T, k, N, kind, added)
    check(T, k, N, kind, added, pads=(3, 1, 5), missing=0.4)


def test_in_place_and_nothing_to_add():
    check(40, 4, 1000, "bf16", True, in_place=True)
    check(40, 4, 1000, "bf16", True, pads=(0, 8, 8), missing=0.9, in_place=True)
    check(6, 2, 300, "f32", False, missing=0.999)


def test_skipped_rows_are_not_read():
    """What no place names, and what weights of a place of -1 hold, does not affect the sum."""
    T, k, N = 4, 2, 64
    y = torch.full((T * k, N), float("nan"))
    y[0], y[3] = 1.0, 2.0
    places = torch.tensor([[0, -1], [-1, 3], [-1, -1], [3, 0]], dtype=torch.int32)
    w = torch.tensor([[2.0, float("nan")], [float("inf"), 1.0], [float("nan")] * 2, [1.0, 1.0]])
    out = torch.full((T, N), 9.0, device="cuda")
    op = ck.DeviceExpertsCombine("f32")
    op.MakeInvokerPointer().Run(op.MakeArgumentPointer(y.cuda(), places.cuda(), w.cuda(), None, out, T, k, T * k, N, N, N, N),
                                ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert out.cpu()[:, 0].tolist() == [2.0, 2.0, 0.0, 3.0]
