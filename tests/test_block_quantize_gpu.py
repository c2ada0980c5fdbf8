"""DeviceBlockQuantizeF8 against the formula's own fp32 steps on the CPU: codes and scales bit for bit."""
import pytest
import torch

import composable_kernel_amd as ck
import serving_plain as sp

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def run(x, kind, m_fast=True, pad_x=0, pad_q=0, offset=0):
    """x on the CPU -> codes and scales [M, groups]; rows pad_* elements further apart, the operands `offset` elements in."""
    M, K = x.shape
    groups = -(-K // 128)
    xd = torch.zeros(M * (K + pad_x) + offset, dtype=x.dtype, device="cuda")[offset:].view(M, K + pad_x)
    xd[:, :K] = x.cuda()
    qd = torch.full((M * (K + pad_q) + offset,), 7.0, device="cuda").to(torch.float8_e4m3fn)
    q = qd[offset:].view(M, K + pad_q)
    s = torch.full((groups, M) if m_fast else (M, groups), -1.0, device="cuda")
    op = ck.DeviceBlockQuantizeF8(kind)
    strides = (1, M) if m_fast else (groups, 1)
    arg = op.MakeArgumentPointer(xd.data_ptr(), q.data_ptr(), s, M, K, K + pad_x, K + pad_q, *strides)
    assert op.IsSupportedArgument(arg), ck.capi.last_error()
    op.MakeInvokerPointer().Run(arg, ck.StreamConfig(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    q = q.cpu()
    assert bool((q[:, K:].float() == 7).all()), "wrote behind the row"
    return q[:, :K], (s.t() if m_fast else s).cpu()


def check(x, kind, **kw):
    q, s = run(x, kind, **kw)
    want_q, want_s = sp.quantize(x)
    assert torch.equal(s, want_s)
    assert sp.same_codes(q, want_q)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 127), (17, 129), (1, 4096), (33, 1000), (16, 520), (5, 640), (130, 2049)])
def test_sizes(kind, M, K):
    x = sp.normal(sp.gen(M * 7919 + K), (M, K), DT[kind], 3.0)
    check(x, kind)
    check(x, kind, m_fast=False)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("pad_x,pad_q,offset", [(8, 16, 0), (1, 0, 0), (0, 3, 0), (0, 0, 1), (4, 4, 0)])
def test_strides_and_addresses(kind, pad_x, pad_q, offset):
    check(sp.normal(sp.gen(5), (19, 264), DT[kind]), kind, pad_x=pad_x, pad_q=pad_q, offset=offset)


def test_every_code_and_the_ends_of_the_range():
    # one row holds every positive e4m3 value and the points half way between neighbours, its largest value 448: scale 1
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    between = (codes[1:] + codes[:-1]) / 2
    row = torch.zeros(1, 384)
    row[0, :127], row[0, 128:254] = codes, between
    row[0, 256:383] = -codes
    row[0, 127] = row[0, 255] = row[0, 383] = 448.0
    q, s = run(row, "f32")
    assert bool((s == 1.0).all())
    assert sp.same_codes(q, row.to(torch.float8_e4m3fn))
    check(torch.tensor([[3.3e38, 1.0, -3.3e38], [1e-44, 0.0, 1e-40], [0.0, 0.0, -0.0], [2.0 ** -100, 2.0 ** -101, 0.0]]), "f32")


def test_nan_and_infinity():
    x = sp.normal(sp.gen(9), (4, 256), torch.bfloat16)
    x[0, 5] = float("nan")
    x[1, 130] = float("inf")
    x[2, 7] = -float("inf")
    x[3, :128] = float("nan")
    q, s = run(x, "bf16")
    want_q, want_s = sp.quantize(x)
    assert torch.equal(s, want_s) and sp.same_codes(q, want_q)
    back = q.float() * s.repeat_interleave(128, dim=1)
    assert bool(back[0, 5].isnan()) and int(back[0].isnan().sum()) == 1
    assert bool(back[1, 128:].isnan().all()) and not bool(back[1, :128].isnan().any())
    assert bool(back[3, :128].isnan().all()) and not bool(back[3, 128:].isnan().any())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_values_half_way_between_codes(kind):
    """x * 448 / amax with 8 (11) bits in x and amax lies on the middle of two codes or 2^-16 and more away from it: every code is the
    one that 64 bits round to. Rows of every mantissa of amax; x = 0.75 amax, 0.65625 amax, ... where they have a bit pattern."""
    bits = 7 if kind == "bf16" else 10
    amax = (1 + torch.arange(2 ** bits) / 2 ** bits)[:, None].double()
    part = torch.tensor([(17 + 2 * i) * 2.0 ** -j / 28 * s for i in range(8) for j in range(1, 7) for s in (1, -1)]).double()
    x = torch.cat([amax, (amax * part).to(DT[kind]).double().clamp(-amax, amax), torch.zeros(2 ** bits, 31)], dim=1).to(DT[kind])
    assert x.shape[1] == 128
    q, s = run(x, kind)
    want = x.double() * 448 / amax
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -6))) - 3)
    ties = ((want / step) % 1 == 0.5).sum()
    assert int(ties) > 2 ** bits
    assert torch.equal(q.double(), torch.round(want / step) * step)
    check(x, kind)
