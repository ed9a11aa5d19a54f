"""Code matrices that lie in columns: their products, and the call that lays them out in rows."""
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


def _in_columns(t, ld, offset=0):
    """The same values as a view whose columns are contiguous, `ld` apart, with NaN between them."""
    rows, K = t.shape
    buf = torch.full((offset + K * ld,), NAN, dtype=torch.uint8, device="cuda")
    view = buf[offset:].as_strided((rows, K), (1, ld))
    view.copy_(t)
    return view


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("M,N,K,spare,offset", [(1, 8, 1, 0, 0), (1, 64, 300, 0, 0), (2, 8, 130, 5, 1), (33, 136, 640, 7, 8), (100, 264, 1000, 0, 0),
                                                (129, 392, 143, 3, 5), (777, 512, 2048, 0, 0), (1280, 1280, 2048, 0, 16)])
def test_operands_in_columns(M, N, K, spare, offset, tiles, dtype):
    """A, B or both as the transposed view of rows: the bits of the product of rows."""
    a, b = _codes(M, K, M), _codes(N, K, N + 1)
    want, got = (torch.empty(M, N, dtype=dtype, device="cuda") for _ in range(2))
    _product(a, b, tiles, want)
    ca, cb = _in_columns(a, M + spare, offset), _in_columns(b, N + spare, offset)
    for x, y in ((ca, b), (a, cb), (ca, cb.view(ref.FP8))):
        got.fill_(float("nan"))
        _product(x, y, tiles, got)
        assert torch.equal(got, want)


def test_columns_on_another_stream_and_captured():
    """The rows that they are laid out in belong to the call's stream, or to the graph."""
    M, N, K = 500, 384, 2064
    b = _codes(N, K, 2)
    side, cols = torch.cuda.Stream(), torch.empty(K, M, dtype=torch.uint8, device="cuda")
    y = [torch.empty(M, N, device="cuda") for _ in range(3)]
    ws = torch.empty(max(1, tmt_moe.fp8_workspace_size(M, N, K, ROWS)), dtype=torch.uint8, device="cuda")
    sa, sb = _scales(M, K, False), _scales(N, K, False)
    call = lambda x, y, s=None: tmt_moe.fp8_matmul(x, sa, b, sb, y, blocks=ROWS, workspace=ws, stream=s)  # noqa: E731
    cols.copy_(_codes(M, K, 0).t())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(cols.t(), y[2])
    for k in range(3):
        a = _codes(M, K, 10 + k)
        cols.copy_(a.t())
        call(a, y[0])
        side.wait_stream(torch.cuda.current_stream())
        call(cols.t(), y[1], side)
        torch.cuda.current_stream().wait_stream(side)
        torch.full((M, ref.up(K, 16)), NAN, dtype=torch.uint8, device="cuda")  # what memory it can get is another's now
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])


@pytest.mark.parametrize("rows,K,ld,offset", [(1, 1, 1, 0), (1, 200, 200, 0), (200, 1, 1, 3), (16, 16, 16, 0), (127, 129, 129, 0), (128, 128, 136, 8),
                                              (130, 260, 264, 0), (1000, 77, 80, 0), (77, 1000, 1003, 2), (5000, 4104, 4104, 0)])
def test_transposed_codes(rows, K, ld, offset):
    """Every byte in its place, zeros up to the 16 bytes' end, nothing else written."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    buf = torch.randint(0, 256, (offset + rows * ld,), generator=g, device="cuda").to(torch.uint8)
    x = buf[offset:].as_strided((rows, K), (ld, 1))
    out, y = ref.padded(torch.full((K, rows), 99, dtype=torch.uint8, device="cuda"), ref.up(rows, 16) + 16, 99)
    tmt_moe.fp8_transpose(x, y)
    w = ref.up(rows, 16)
    assert torch.equal(y, x.t()) and (out[1:-1, rows:w] == 0).all()
    assert (out[0] == 99).all() and (out[-1] == 99).all() and (out[:, w:] == 99).all()
