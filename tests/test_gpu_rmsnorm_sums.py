"""What the norm's forward promises of its roundings: squares in 64 bits, rstd rounded once, y
from three roundings of fp32; and its narrow rows in calls past the caches."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24  # half a step of fp32, relative


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("d", [1, 100, 128, 200, 256, 512, 1000, 1024, 1280, 4096, 8192, 16384])
def test_forward_roundings(d, stream):
    """rstd is off by its own rounding (2^-24) and what 64 bits lose; y in fp32 by that and those of
    two products, bf16's is half a step more; a scale by y's three in its block's largest value
    and that of the quotient by 448; a code is that of y in 64 bits (to half a step of its scale)."""
    T = 40000 // d + 3
    g = torch.Generator().manual_seed(d)
    x = torch.randn(T, d, generator=g).to(BF16)
    r = (3 * torch.randn(T, d, generator=g) * torch.exp2(torch.randint(-6, 7, (T, d), generator=g).float())).to(stream)
    gamma = 1 + 0.3 * torch.randn(d, generator=g)
    eps = float(torch.tensor(1e-5))
    s, rstd, y = ref.norm(x, r, gamma, eps, stream)
    ld = ref.up(d, 8)
    row = lambda t: torch.zeros(T, ld, dtype=t.dtype, device="cuda")[:, :d].copy_(t)  # noqa: E731
    S, Y = (torch.empty(T, ld, dtype=t, device="cuda")[:, :d] for t in (stream, BF16))
    C = torch.empty(T, ref.up(d, 16), dtype=torch.uint8, device="cuda")[:, :d]
    sc, rs = torch.empty(ref.blocks_of(d), T, device="cuda"), torch.empty(T, device="cuda")
    tmt_moe.rmsnorm_forward(row(x), row(r), gamma.cuda(), S=S, Y=Y, codes=C, scales=sc, rstd=rs)
    lost = 2.0 ** -48  # of 64 bits: fewer than 32 roundings of 2^-53
    assert torch.equal(S.cpu(), s)
    assert ((rs.cpu().double() - rstd).abs() <= rstd * (U + lost)).all()
    assert ((Y.cpu().double() - y).abs() <= y.abs() * (1 + 2.0 ** -8) * (3.01 * U) + y.abs() * 2.0 ** -8).all()
    most = torch.zeros(T, ref.up(d, 128), dtype=torch.float64)
    most[:, :d] = y.abs()
    want = most.view(T, -1, 128).amax(2).clamp(min=2.0 ** -100) / 448
    assert ((sc.cpu().double().t() - want).abs() <= want * 4.01 * U).all()
    q = y / want.repeat_interleave(128, 1)[:, :d]
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)  # at a power of 2 the finer one is below
    got = C.cpu().contiguous().view(ref.FP8).double()
    assert ((got - q).abs() <= step / 2 * (1 + 2.0 ** -40)).all()


@pytest.mark.parametrize("T,d,stream", [(60000, 128, BF16), (60000, 96, F32), (30000, 256, F32), (30000, 200, BF16),
                                        (260000, 128, BF16), (200000, 100, F32), (130000, 256, BF16), (90000, 252, F32)])
def test_narrow_rows_past_the_caches(T, d, stream):
    """Rows of 16 and 32 lanes: the same bits in a call whose outputs (whose inputs too, from 250 MB
    on) pass the caches as in calls of a few thousand rows."""
    g = torch.Generator(device="cuda").manual_seed(T)
    new = lambda rows, dtype, fill=0: torch.full((rows, ref.up(d, 16)), fill, dtype=dtype, device="cuda")[:, :d]  # noqa: E731
    X = new(T, BF16).copy_(torch.randn(T, d, device="cuda", generator=g))
    R = new(T, stream).copy_(torch.randn(T, d, device="cuda", generator=g))
    dY = new(T, BF16).copy_(torch.randn(T, d, device="cuda", generator=g))
    gamma = torch.randn(d, device="cuda", generator=g)

    def both(a, b):
        n = b - a
        S, C, Y, dS, rs, dg = new(n, stream), new(n, torch.uint8), new(n, BF16), new(n, stream), torch.empty(n, device="cuda"), torch.empty(d, device="cuda")
        sc = torch.empty(ref.blocks_of(d), n, device="cuda")
        tmt_moe.rmsnorm_forward(X[a:b], R[a:b], gamma, S=S, Y=Y, codes=C, scales=sc, rstd=rs)
        ws = torch.empty(tmt_moe.rmsnorm_workspace_size(n, d), dtype=torch.uint8, device="cuda")
        tmt_moe.rmsnorm_backward(dY[a:b], S, gamma, rs, dS, dg, ws, dR=R[a:b])
        return S, C, Y, rs, sc.t(), dS

    whole = both(0, T)
    for a in range(0, T, 5000):
        b = min(T, a + 5000)
        for name, big, small in zip(("S", "codes", "Y", "rstd", "scales", "dS"), whole, both(a, b)):
            assert torch.equal(big[a:b], small), (name, a)
