"""The norm's codes in e4m3's subnormals: those of 64 bits too, whatever the row's neighbours."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
EPS = float(torch.tensor(1e-5))


def _near_middles(d, stream, seed):
    """A row and gamma, whose values but for each block's first lie as near as fp32's gamma allows
    to the middle between two of e4m3's subnormals, and the codes of 64 bits."""
    g = torch.Generator().manual_seed(seed)
    r = (torch.randn(1, d, generator=g).abs() + 0.5).to(stream)
    v = r.double()[0]
    xh = v * (v.square().mean() + EPS) ** -0.5
    gamma = torch.ones(d, dtype=torch.float64)
    middle = (torch.randint(0, 8, (d,), generator=g).double() + 0.5) * 2.0 ** -9
    sign = torch.randint(0, 2, (d,), generator=g).double() * 2 - 1
    for c in range(0, d, 128):
        gamma[c + 1:c + 128] = (sign * middle / xh)[c + 1:c + 128] * xh[c] / 448
    gamma = gamma.float()
    y = xh * gamma.double()
    most = torch.stack([b.abs().max() for b in y.split(128)]).repeat_interleave(128)[:d]
    q = y * 448 / most
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    assert (q.abs() < 2.0 ** -6).sum() == d - ref.blocks_of(d)
    return r, gamma, q / step, step


def _right(got, q, step):
    """The codes of q steps, to nearest. In 64 bits q is off itself, by the two roundings of 448 / m
    and of the product, those of y's two products and half of the sum's, root's, quotient's and
    mean's, the same in m, and as many in the kernel: fewer than 32 of 2^-53 of at most 8
    steps for the subnormals, which decides between two codes where equal bf16 values make it the
    middle itself. There either is right."""
    tie = (q.abs() < 8) & ((q - torch.floor(q) - 0.5).abs() <= 32 * 8 * 2.0 ** -53)
    got = got / step
    return torch.where(tie, (got - q).abs() <= 0.5 + 2.0 ** -40, got == torch.round(q)).all().item()


def _codes(r, gamma):
    T, d = r.shape
    R = torch.zeros(T, ref.up(d, 8), dtype=r.dtype, device="cuda")[:, :d].copy_(r)
    C = torch.empty(T, ref.up(d, 16), dtype=torch.uint8, device="cuda")[:, :d]
    tmt_moe.rmsnorm_forward(None, R, gamma.cuda(), codes=C, scales=torch.empty(ref.blocks_of(d), T, device="cuda"))
    return C.contiguous()


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("d", [100, 128, 250, 256, 500, 1024, 1280, 4096, 8192, 16384])
def test_subnormal_codes_of_64_bits(d, stream):
    for seed in range(4):
        r, gamma, q, step = _near_middles(d, stream, seed)
        got = _codes(r, gamma).view(ref.FP8).double().cpu()[0]
        assert _right(got, q, step), (seed, (got / step != torch.round(q)).sum().item())


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("d", [128, 256])
def test_codes_do_not_depend_on_the_rows_beside(d, stream):
    """Rows that share a wave: one near the subnormals' middles, others of any value."""
    r, gamma, _, _ = _near_middles(d, stream, 1)
    alone = _codes(r, gamma)[0]
    g = torch.Generator().manual_seed(7)
    for k in range(200):
        rows = torch.cat([r, (3 * torch.randn(3, d, generator=g)).to(stream)])
        assert torch.equal(_codes(rows, gamma)[0], alone), k
