"""The 8-bit layer's kernels where memory is far apart or much: row strides of 2^22 in every
product kernel, and calls whose outputs are stored past the caches."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ROWS, TILES = tmt_moe.FP8_ROWS, tmt_moe.FP8_TILES
WIDEST = 1 << 22


def _wide(rows, cols, dtype, fill):
    """(all of the memory, its rows' first `cols` elements) with rows 2^22 elements apart."""
    mem = torch.full(((rows - 1) * WIDEST + cols,), fill, dtype=dtype, device="cuda")
    return mem, mem.as_strided((rows, cols), (WIDEST, 1))


def _operand(rows, K, tiles, seed):
    """Dense codes, the same 2^22 bytes apart with NaN between, and their scales."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.zeros(rows, ref.up(K, 8), dtype=BF16, device="cuda")[:, :K].copy_(torch.randn(rows, K, device="cuda", generator=g))
    dense = torch.empty(rows, ref.up(K, 16), dtype=torch.uint8, device="cuda")
    scales = torch.empty((ref.blocks_of(rows), ref.blocks_of(K)) if tiles else (ref.blocks_of(K), rows), device="cuda")
    tmt_moe.fp8_quantize(x, dense[:, :K], scales, blocks=TILES if tiles else ROWS)
    wide = _wide(rows, ref.up(K, 16), torch.uint8, 0x7f)[1].copy_(dense)
    return dense[:, :K], wide[:, :K], scales


# Sizes that the plan gives to each tiled kernel, whole and split.
STRIDES = [
    (700, 1032, 2064, True, BF16, ["fp8_quarter_kernelILi64E"]), (1000, 2048, 1000, False, BF16, ["fp8_quarter_kernelILi64E"]),
    (900, 264, 9000, True, BF16, ["fp8_quarter_kernelILi64E", "linear_fixup_kernelILi64ELb0E"]),
    (1500, 2048, 400, True, BF16, ["fp8_deep_kernel"]), (500, 1000, 20000, True, BF16, ["fp8_deep_kernel", "linear_fixup_kernelILi128ELb0E"]),
    (4090, 4096, 640, True, BF16, ["fp8_large_kernelILb1E"]), (4090, 4096, 650, True, BF16, ["fp8_large_kernelILb0E"]),
    (1000, 2048, 1000, True, F32, ["fp8_quarter_kernelILi64E"]),
    (300, 264, 9000, True, F32, ["fp8_quarter_kernelILi64E", "linear_fixup_kernelILi64ELb1E"]),
    (2048, 2048, 1000, False, F32, ["fp8_quarter_kernelILi128E"]), (2048, 4096, 1100, False, F32, ["fp8_wide_kernel"]),
    (1100, 1304, 9000, True, F32, ["fp8_wide_kernel", "linear_fixup_kernelILi128ELb1E"]),
]


@pytest.mark.parametrize("M,N,K,tiles,dtype,names", STRIDES)
def test_the_widest_strides_of_every_tiled_kernel(M, N, K, tiles, dtype, names):
    """Operands and outputs in rows 2^22 elements apart give the bits of dense ones, stored and
    added to; what lies between the outputs' rows stays."""
    from launched_kernels import launched_kernels
    a, wide_a, sa = _operand(M, K, False, 1)
    b, wide_b, sb = _operand(N, K, tiles, 2)
    mem, z = _wide(M, N, dtype, 5.0)
    y = torch.empty(M, N, dtype=dtype, device="cuda")
    blocks = TILES if tiles else ROWS
    ws = torch.empty(max(tmt_moe.fp8_workspace_size(M, N, K, blocks), 1), dtype=torch.uint8, device="cuda")
    call = lambda a, b, y, beta: tmt_moe.fp8_matmul(a, sa, b, sb, y, beta=beta, blocks=blocks, workspace=ws)  # noqa: E731
    launched = launched_kernels(lambda: call(wide_a, wide_b, z, 0.0))
    assert len(launched) == len(names) and all(any(n in k for k in launched) for n in names), launched
    call(a, b, y, 0.0)
    call(wide_a, wide_b, z, 0.0)
    assert torch.isfinite(y).all() and torch.equal(y, z)
    call(a, b, y, 0.5)
    call(wide_a, wide_b, z, 0.5)
    assert torch.isfinite(y).all() and torch.equal(y, z)
    between = mem[N:N + (M - 1) * WIDEST].view(M - 1, WIDEST)
    assert (between[:, :64] == 5).all() and (between[:, WIDEST - N - 64:WIDEST - N] == 5).all()
    del mem, z, wide_a, wide_b, between
    torch.cuda.empty_cache()


@pytest.mark.parametrize("sides", ["", "_t", "both"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tiles", [False, True])
def test_quantize_past_the_caches(tiles, dtype, sides):
    """More than 16 MiB of codes, which are stored non-temporally: to the bit, in ragged rows and
    columns, nothing outside written."""
    rows, K = 9001, 2056
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float())).to(dtype)
    x[300, 700], x[5000, 2055] = float("nan"), -float("inf")
    args, checks = {}, []
    for side, v in (("", x), ("_t", x.t())):
        if sides not in ("both", side):
            continue
        r, c = v.shape
        codes, scales = ref.quantize(v, tiles)
        buf, view = ref.padded(torch.full((r, c), 99, dtype=torch.uint8, device="cuda"), ref.up(c, 16) + 16, 99)
        out = torch.full((scales.shape[0], scales.shape[1] + 3), 5.0, device="cuda")
        args["codes" + side], args["scales" + side] = view, out
        checks.append((codes, scales, buf, view, out, c))
    tmt_moe.fp8_quantize(x.cuda(), blocks=TILES if tiles else ROWS, **args)
    for codes, scales, buf, view, out, c in checks:
        assert torch.equal(view.cpu(), codes)
        assert torch.equal(out[:, :-3].cpu().nan_to_num(-1), scales.nan_to_num(-1)) and torch.isnan(scales).any()
        w = ref.up(c, 16)
        assert (buf[0] == 99).all() and (buf[-1] == 99).all() and (buf[1:-1, w:] == 99).all()
        assert (buf[1:-1, c:w] == 0).all() and (out[:, -3:] == 5).all()
