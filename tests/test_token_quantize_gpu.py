"""DeviceTokenQuantizeI8 against the formula's own steps on the CPU: codes and scales bit for bit."""
import pytest
import torch

import composable_kernel_amd as ck
import experts_plain as ep

pytestmark = pytest.mark.gpu


def check(x, kind, pad_x=0, pad_q=0, offset=0):
    M, K = x.shape
    xd = torch.zeros(M * (K + pad_x) + offset, dtype=x.dtype, device="cuda")[offset:].view(M, K + pad_x)
    xd[:, :K] = x.cuda()
    q = torch.full((M * (K + pad_q) + offset,), 99, dtype=torch.int8, device="cuda")[offset:].view(M, K + pad_q)
    s = torch.full((M + 1,), -1.0, device="cuda")
    op = ck.DeviceTokenQuantizeI8(kind)
    arg = op.MakeArgumentPointer(xd, q, s, M, K, K + pad_x, K + pad_q)
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    q, s = q.cpu(), s.cpu()
    assert bool((q[:, K:] == 99).all()) and s[M] == -1.0, "wrote behind the row"
    want_q, want_s = ep.quantize(x)
    assert torch.equal(s[:M].nan_to_num(-2.0), want_s.nan_to_num(-2.0))
    assert torch.equal(q[:, :K], want_q)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 7), (3, 8), (5, 511), (4, 513), (17, 1025), (9, 2049), (1, 4096), (3, 4104), (2, 8193), (2, 11008),
                                 (3, 12289), (2, 16384), (2, 16385), (1, 40001), (300, 130)])
def test_sizes(kind, M, K):
    check(ep.normal(ep.gen(M * 7919 + K), (M, K), ep.DT[kind], 3.0), kind)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("K", [264, 3001])
@pytest.mark.parametrize("pad_x,pad_q,offset", [(8, 16, 0), (1, 0, 0), (0, 3, 0), (0, 0, 1), (4, 4, 0)])
def test_strides_and_addresses(kind, K, pad_x, pad_q, offset):
    check(ep.normal(ep.gen(5), (19, K), ep.DT[kind]), kind, pad_x, pad_q, offset)


def test_the_ends_of_the_range_and_what_is_not_finite():
    inf, nan = float("inf"), float("nan")
    check(torch.tensor([[3.3e38, 1.0, -3.3e38], [1e-44, 0.0, 1e-40], [0.0, 0.0, -0.0], [2.0 ** -100, 2.0 ** -101, 0.0], [inf, 1.0, 2.0],
                        [1.0, nan, 2.0], [-inf, nan, 0.0], [127.0, 0.5, -1.5]]), "f32")
    x = ep.normal(ep.gen(9), (4, 3000), torch.bfloat16)
    x[0, 2999], x[1, 0], x[2, 1500] = nan, inf, -inf
    check(x, "bf16")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_values_half_way_between_codes(kind):
    """Rows of every mantissa of the largest value; x * 127 / amax half way between two codes where x has a bit pattern for it."""
    bits = 7 if kind == "bf16" else 10
    amax = (1 + torch.arange(2 ** bits) / 2 ** bits)[:, None].double()
    part = torch.arange(-127, 127).double().add(0.5)[None, :] / 127
    x = torch.cat([amax, (amax * part).to(ep.DT[kind]).double().clamp(-amax, amax)], dim=1).to(ep.DT[kind])
    ties = ((x.double() * 127 / amax) % 1 == 0.5).sum()
    assert int(ties) > 100
    check(x, kind)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_rows_of_nothing_have_the_smallest_scale(kind):
    s = torch.full((6,), 7.0, device="cuda")
    op = ck.DeviceTokenQuantizeI8(kind)
    arg = op.MakeArgumentPointer(None, None, s, 5, 0, 0, 0)
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert s.tolist() == [float(torch.tensor(2.0 ** -100) / 127)] * 5 + [7.0]
