"""Products of code matrices that hold NaN codes."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ROWS, TILES = tmt_moe.FP8_ROWS, tmt_moe.FP8_TILES
NAN = 0x7f


def _codes(rows, K, seed):
    """Whole numbers, whose sums every kernel forms exactly, in rows padded with zeros."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    full = torch.zeros(rows, ref.up(K, 16), dtype=torch.uint8, device="cuda")
    full[:, :K] = torch.randint(-3, 4, (rows, K), generator=g, device="cuda").float().to(ref.FP8).view(torch.uint8)
    return full[:, :K]


def _scales(rows, K, tiles):
    return torch.ones((ref.blocks_of(rows), ref.blocks_of(K)) if tiles else (ref.blocks_of(K), rows), device="cuda")


def _product(a, b, tiles, y, beta=0.0):
    (M, K), N = a.shape, b.shape[0]
    blocks = TILES if tiles else ROWS
    size = tmt_moe.fp8_workspace_size(M, N, K, blocks)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    tmt_moe.fp8_matmul(a, _scales(M, K, False), b, _scales(N, K, tiles), y, beta=beta, blocks=blocks, workspace=ws)


# Sizes that give the workgroups of every kernel several units one after another, and the
# kernels that they reach: few rows; 64 x 64 (whole, split, paired); 128 x 128 (whole, split;
# fp32); 256 x 256 (K a multiple of 128 and not).
NAN_CODES = [
    (64, 2048, 140, True, BF16, "fp8_rows"), (777, 256, 4096, True, BF16, "fp8_rows"), (30, 64, 1000, False, F32, "fp8_rows"),
    (2560, 1640, 300, True, BF16, "fp8_quarter"), (2560, 1640, 300, False, BF16, "fp8_quarter"),
    (2560, 1640, 300, True, F32, "fp8_quarter"), (2560, 1640, 300, False, F32, "fp8_quarter"),
    (900, 264, 9000, True, BF16, "fp8_quarter"), (777, 1024, 2050, True, BF16, "fp8_quarter"),
    (2300, 1896, 500, True, BF16, "fp8_deep"), (2300, 1896, 500, False, BF16, "fp8_deep"),
    (2304, 1896, 6451, False, BF16, "fp8_deep"), (2048, 2048, 1000, False, F32, "fp8_quarter"),
    (4096, 4200, 1100, True, F32, "fp8_wide"), (4096, 4200, 1100, False, F32, "fp8_wide"),
    (8200, 4096, 768, True, BF16, "fp8_large"), (8190, 4088, 700, True, BF16, "fp8_large"),
]


@pytest.mark.parametrize("M,N,K,tiles,dtype,kernel", NAN_CODES)
def test_nan_codes_stay_in_their_row_and_column(M, N, K, tiles, dtype, kernel):
    """A NaN code makes its row of A's outputs, or its column of B's, NaN and no other: the rest has
    the bits of the product without them."""
    from launched_kernels import launched_kernels
    a, b = _codes(M, K, 1), _codes(N, K, 2)
    want, got = (torch.empty(M, N, dtype=dtype, device="cuda") for _ in range(2))
    assert any(kernel in k for k in launched_kernels(lambda: _product(a, b, tiles, want)))
    _product(a, b, tiles, want)
    g = torch.Generator(device="cuda").manual_seed(3)
    row = torch.rand(M, generator=g, device="cuda") < 0.05
    col = torch.rand(N, generator=g, device="cuda") < 0.05
    row[M - 1] = col[0] = True  # a tile's last rows and first columns among them
    for t, bad in ((a, row), (b, col)):
        at = bad.nonzero()[:, 0]
        t[at, torch.randint(0, K, at.shape, generator=g, device="cuda")] = NAN
    for beta in (0.0, 1.0):
        got.zero_()
        _product(a, b, tiles, got, beta)
        bad = row[:, None] | col[None, :]
        assert torch.equal(torch.isnan(got), bad), beta
        assert torch.equal(got.masked_fill(bad, 0), want.masked_fill(bad, 0)), beta
