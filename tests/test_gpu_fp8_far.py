"""Matrices of more than 2^32 elements, in the quantiser, the norm, the products and the call that
turns codes: rows at both ends and around 2^31 and 2^32 elements have the bits of calls of those
rows alone."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ROWS, TILES = tmt_moe.FP8_ROWS, tmt_moe.FP8_TILES


def _spots(rows, K):
    """Whole tiles of rows, with those that hold element 2^31 and 2^32, and the last ones."""
    first = [0] + [(1 << b) // K // 128 * 128 for b in (31, 32)] + [rows // 128 * 128 - 128]
    assert rows * K > 1 << 32 and rows % 128
    return [(a, min(rows, a + 256)) for a in first]


@pytest.fixture(autouse=True)
def freed():
    yield
    torch.cuda.empty_cache()


def _random(rows, K, dtype, seed):
    return torch.empty(rows, K, dtype=dtype, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("tiles", [False, True])
def test_quantize(tiles):
    rows, K = (1 << 21) + 1003, 2056
    x = _random(rows, K, BF16, 1)
    codes = torch.empty(rows, ref.up(K, 16), dtype=torch.uint8, device="cuda")[:, :K]
    kb = ref.blocks_of(K)
    new = lambda n: torch.empty((ref.blocks_of(n), kb) if tiles else (kb, n), device="cuda")  # noqa: E731
    ct, st = torch.empty(K, ref.up(rows, 16), dtype=torch.uint8, device="cuda")[:, :rows], torch.empty((kb, ref.blocks_of(rows)) if tiles else (ref.blocks_of(rows), K), device="cuda")
    scales = new(rows)
    tmt_moe.fp8_quantize(x, codes, scales, ct, st, blocks=TILES if tiles else ROWS)
    for a, b in _spots(rows, K):
        n = b - a
        c, s = torch.empty(n, ref.up(K, 16), dtype=torch.uint8, device="cuda")[:, :K], new(n)
        t, ts = torch.empty(K, ref.up(n, 16), dtype=torch.uint8, device="cuda")[:, :n], torch.empty((kb, ref.blocks_of(n)) if tiles else (ref.blocks_of(n), K), device="cuda")
        tmt_moe.fp8_quantize(x[a:b], c, s, t, ts, blocks=TILES if tiles else ROWS)
        assert torch.equal(codes[a:b], c) and torch.equal(ct[:, a:b], t), a
        # a tile's rows past the spot's last are in the large call only where it ends inside a tile
        whole = slice(a // 128, a // 128 + ref.blocks_of(n))
        assert torch.equal(scales[whole] if tiles else scales[:, a:b], s), a
        assert torch.equal(st[:, whole] if tiles else st[whole], ts), a


def test_norm():
    """Wide rows, of which a launch takes more than a grid's first dimension holds."""
    T, d = (1 << 21) + 77, 2056
    R, X, dY, gamma = _random(T, d, BF16, 1), _random(T, d, BF16, 2), _random(T, d, BF16, 3), _random(1, d, F32, 4)[0]

    def both(a, b):
        n = b - a
        S, Y, dS = (torch.empty(n, d, dtype=BF16, device="cuda") for _ in range(3))
        C, sc = torch.empty(n, ref.up(d, 16), dtype=torch.uint8, device="cuda")[:, :d], torch.empty(ref.blocks_of(d), n, device="cuda")
        rs, dg = torch.empty(n, device="cuda"), torch.empty(d, device="cuda")
        tmt_moe.rmsnorm_forward(X[a:b], R[a:b], gamma, S=S, Y=Y, codes=C, scales=sc, rstd=rs)
        ws = torch.empty(tmt_moe.rmsnorm_workspace_size(n, d), dtype=torch.uint8, device="cuda")
        tmt_moe.rmsnorm_backward(dY[a:b], S, gamma, rs, dS, dg, ws, dR=R[a:b])
        return S, Y, C, sc.t(), rs, dS

    whole = both(0, T)
    for a, b in _spots(T, d):
        for name, big, small in zip(("S", "Y", "codes", "scales", "rstd", "dS"), whole, both(a, b)):
            assert torch.equal(big[a:b], small), (name, a)


@pytest.mark.parametrize("tiles,dtype", [(True, BF16), (False, F32)])
def test_product(tiles, dtype):
    """More than 2^32 codes of a, and as many outputs. Whole numbers, so that the kernel does not matter."""
    M, N, K = (1 << 22) + 1003, 1032, 1040
    g = torch.Generator(device="cuda").manual_seed(1)
    values = torch.arange(-3, 4, device="cuda").float().to(ref.FP8).view(torch.uint8)
    pick = lambda rows: values[torch.randint(0, 7, (rows, K), generator=g, device="cuda", dtype=torch.int32)]  # noqa: E731
    a, b = torch.empty(M, K, dtype=torch.uint8, device="cuda"), pick(N)
    for i in range(0, M, 1 << 19):
        a[i:i + (1 << 19)] = pick(min(M - i, 1 << 19))
    kb = ref.blocks_of(K)
    sa = torch.exp2(torch.randint(-1, 2, (kb, M), generator=g, device="cuda").float())
    sb = torch.ones((ref.blocks_of(N), kb) if tiles else (kb, N), device="cuda")
    y = torch.empty(M, N, dtype=dtype, device="cuda")
    blocks = TILES if tiles else ROWS
    ws = torch.empty(max(1, tmt_moe.fp8_workspace_size(M, N, K, blocks)), dtype=torch.uint8, device="cuda")
    tmt_moe.fp8_matmul(a, sa, b, sb, y, blocks=blocks, workspace=ws)
    for i, j in _spots(M, N):
        z = torch.empty(j - i, N, dtype=dtype, device="cuda")
        tmt_moe.fp8_matmul(a[i:j], sa[:, i:j].contiguous(), b, sb, z, blocks=blocks, workspace=ws)
        assert torch.equal(y[i:j], z) and z.abs().max() > 0, i


def test_transpose():
    rows, K = (1 << 21) + 1003, 2057
    x = torch.empty(rows, K, dtype=torch.uint8, device="cuda").random_(0, 256, generator=torch.Generator(device="cuda").manual_seed(1))
    y = torch.empty(K, ref.up(rows, 16), dtype=torch.uint8, device="cuda")[:, :rows]
    tmt_moe.fp8_transpose(x, y)
    for a, b in _spots(rows, K):
        assert torch.equal(y[:, a:b], x[a:b].t()), a
