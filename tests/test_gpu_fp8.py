"""Quantisation in blocks of 128 and the products of the 8-bit linear layer."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ROWS, TILES = tmt_moe.FP8_ROWS, tmt_moe.FP8_TILES


# ---- quantisation ----------------------------------------------------------------

def _quantize(x, tiles, sides="both", spare=0):
    """Codes and scales of both sides, with guards checked."""
    rows, K = x.shape
    ldx = ref.up(K, 8) + 8
    _, X = ref.padded(x.cuda(), ldx, float("nan"))
    rb, kb = ref.blocks_of(rows), ref.blocks_of(K)
    shape = ((rb, kb), (kb, rb)) if tiles else ((kb, rows), (rb, K))
    got, args, guards = [], {}, []
    for side, (r, c), (sr, sc) in (("", (rows, K), shape[0]), ("_t", (K, rows), shape[1])):
        if sides not in ("both", side):
            continue
        buf, codes = ref.padded(torch.full((r, c), 99, dtype=torch.uint8, device="cuda"), ref.up(c, 16) + 16, 99)
        scales = torch.full((sr, sc + spare), 5.0, device="cuda")
        args["codes" + side], args["scales" + side] = codes, scales
        guards.append((buf, c, scales, sc))
        got.append((codes, scales[:, :sc]))
    tmt_moe.fp8_quantize(X, blocks=TILES if tiles else ROWS, **args)
    for buf, c, scales, sc in guards:
        w = ref.up(c, 16)
        assert (buf[0] == 99).all() and (buf[-1] == 99).all() and (buf[1:-1, w:] == 99).all()
        assert (buf[1:-1, c:w] == 0).all() and (scales[:, sc:] == 5).all()
    return got


def _same(got, want):
    codes, scales = got
    assert torch.equal(codes.cpu(), want[0])
    assert torch.equal(scales.cpu().view(torch.int32), want[1].contiguous().view(torch.int32))


SHAPES = [(1, 1), (1, 128), (3, 16), (17, 40), (128, 128), (129, 127), (130, 257), (64, 1000), (1000, 64), (257, 384), (5, 4100)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("rows,K", SHAPES)
def test_quantize(rows, K, tiles, dtype):
    """To the bit, both sides, each side alone."""
    g = torch.Generator().manual_seed(rows * 7 + K)
    x = (torch.randn(rows, K, generator=g) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g).float())).to(dtype)
    want = ref.quantize(x, tiles), ref.quantize(x.t(), tiles)
    both = _quantize(x, tiles, spare=3)
    _same(both[0], want[0])
    _same(both[1], want[1])
    _same(_quantize(x, tiles, "")[0], want[0])
    _same(_quantize(x, tiles, "_t")[0], want[1])


@pytest.mark.parametrize("tiles", [False, True])
def test_quantize_large(tiles):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5003, 1288, generator=g).to(BF16)
    both = _quantize(x, tiles)
    _same(both[0], ref.quantize(x, tiles))
    _same(both[1], ref.quantize(x.t(), tiles))


@pytest.mark.parametrize("tiles", [False, True])
def test_quantize_special_values(tiles):
    """Zeros, subnormals, the largest values, infinities and NaN: a block that holds one of the
    last has a NaN for its scale and zeros for codes, the others are as ever."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(384, 640, generator=g)
    x[:128, :128] = 0
    x[:128, 128:256] *= 2.0 ** -140
    x[:128, 256:384] *= 2.0 ** -99
    x[128:256, :128] = 3.4028234663852886e38
    x[130, 200] = float("inf")
    x[131, 300] = float("nan")
    x[132, 400] = -float("inf")
    x[256:, 512:] = -0.0
    both = _quantize(x, tiles)
    _same((both[0][0], both[0][1].nan_to_num(-1)), (ref.quantize(x, tiles)[0], ref.quantize(x, tiles)[1].nan_to_num(-1)))
    t = ref.quantize(x.t(), tiles)
    _same((both[1][0], both[1][1].nan_to_num(-1)), (t[0], t[1].nan_to_num(-1)))
    for (_, s), w in zip(both, (ref.quantize(x, tiles), t)):
        assert torch.equal(torch.isnan(s.cpu()), torch.isnan(w[1]))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_every_step_of_the_codes(dtype):
    """All bf16 magnitudes below 1 next to a 448: every code, the midpoints between codes (ties
    to even) and e4m3's subnormals."""
    v = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(BF16).float()
    v = v[torch.isfinite(v) & (v.abs() <= 448)]
    v = v[:v.numel() // 127 * 127].view(-1, 127)
    x = torch.cat([v, torch.full((v.shape[0], 1), 448.0)], 1).to(dtype)
    _same(_quantize(x, False, "")[0], ref.quantize(x, False))


# ---- products ---------------------------------------------------------------------

def _operand(rows, K, tiles, seed, exact):
    """Codes in rows padded to 16 and scales on the device, and the values in 64 bits.
    exact: whole numbers times powers of two, whose sums fp32 holds."""
    g = torch.Generator().manual_seed(seed)
    rb, kb = ref.blocks_of(rows), ref.blocks_of(K)
    shape = (rb, kb) if tiles else (kb, rows)
    if exact:
        v = torch.randint(-3, 4, (rows, K), generator=g).float()
        s = torch.exp2(torch.randint(-1, 2, shape, generator=g).float())
    else:
        v = (torch.randn(rows, K, generator=g) * 100).clamp(-448, 448)  # e4m3 has no larger values
        s = torch.rand(shape, generator=g) * torch.exp2(torch.randint(-6, 6, shape, generator=g).float()) + 1e-3
    q = v.to(ref.FP8).view(torch.uint8)
    _, codes = ref.padded(q.cuda(), ref.up(K, 16) + 32, 0x7f)  # NaN outside
    codes.as_strided((rows, ref.up(K, 16)), codes.stride(), codes.storage_offset())[:, K:] = 0
    scales = torch.full((shape[0], shape[1] + 5), float("nan"), device="cuda")
    scales[:, :shape[1]] = s.cuda()
    return (codes, scales), ref.values(q, s, tiles)


def _product(M, N, K, tiles, dtype, exact=True, beta=0.0, seed=0, ldy=None):
    a, av = _operand(M, K, False, 2 * seed + 1, exact)
    b, bv = _operand(N, K, tiles, 2 * seed + 2, exact)
    y64 = av @ bv.t()
    g = torch.Generator().manual_seed(seed)
    old = torch.randint(-100, 100, (M, N), generator=g).to(dtype)
    buf, y = ref.padded((old if beta else torch.full((M, N), float("nan"), dtype=dtype)).cuda(), ldy or N + 16, 5.0)
    size = tmt_moe.fp8_workspace_size(M, N, K, TILES if tiles else ROWS)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if size else None
    tmt_moe.fp8_matmul(*a, *b, y, beta=beta, blocks=TILES if tiles else ROWS, workspace=ws)
    if beta:
        y64 = y64 + beta * old.double()
    got = y.cpu()
    if exact:  # one right result
        assert torch.equal(got, y64.float().to(dtype))
    else:
        # fp32 sums of a block's 128 products, the blocks' sums, two scales' product
        terms = av.abs() @ bv.abs().t() + abs(beta) * old.double().abs()
        tol = terms * (128 + ref.blocks_of(K) + 8) * 2.0 ** -24 + y64.abs() * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24)
        if dtype == BF16:
            # the 8-bit matrix instruction aligns 8 neighbouring products to the largest, whose
            # exponent's value is at most its own, and drops what lies 2^-13 below: up to 8 drops
            top = lambda v: torch.nn.functional.pad(v.abs(), (0, -K % 8)).view(v.shape[0], -1, 8).amax(2)  # noqa: E731
            tol = tol + top(av) @ top(bv).t() * 8 * 2.0 ** -13
        assert ((got.double() - y64).abs() <= tol).all()
    assert (buf[0] == 5).all() and (buf[-1] == 5).all() and (buf[1:-1, N:] == 5).all()


SIZES = [(1, 8, 16), (1, 8, 1), (2, 16, 130), (5, 24, 128), (16, 32, 256), (33, 136, 640), (64, 1024, 384), (100, 264, 1000),
         (128, 128, 128), (129, 392, 144), (256, 256, 2048), (300, 520, 1152), (777, 256, 4096), (130, 128, 16384)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product_to_the_bit(M, N, K, tiles, dtype):
    _product(M, N, K, tiles, dtype)


def _launched(M, N, K, tiles, dtype):
    """The kernels that a product of these sizes launches."""
    from launched_kernels import launched_kernels
    b = ref.blocks_of
    e = lambda r, c: torch.zeros(r, ref.up(c, 16), dtype=ref.FP8, device="cuda")[:, :c]  # noqa: E731
    size = tmt_moe.fp8_workspace_size(M, N, K, TILES if tiles else ROWS)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    args = (e(M, K), torch.ones(b(K), M, device="cuda"), e(N, K),
            torch.ones((b(N), b(K)) if tiles else (b(K), N), device="cuda"), torch.empty(M, N, dtype=dtype, device="cuda"))
    return launched_kernels(lambda: tmt_moe.fp8_matmul(*args, blocks=TILES if tiles else ROWS, workspace=ws))


# Sizes that reach every kernel, whole and split, a part of a round and several, with the
# (mangled) names that must be launched: template numbers are L<type><value>E.
ROW = "fp8_rows_kernelILb%dELb%dELi%dELi%dE"
KERNELS = [
    (5, 40, 300, True, BF16, [ROW % (1, 0, 1, 1)]), (64, 2048, 140, True, BF16, [ROW % (1, 0, 1, 2)]),
    (64, 4096, 130, False, BF16, [ROW % (0, 0, 2, 2)]), (63, 12288, 129, True, BF16, [ROW % (1, 0, 4, 4)]),
    (30, 64, 1000, False, F32, [ROW % (0, 1, 1, 1)]), (64, 4096, 200, True, F32, [ROW % (1, 1, 2, 2)]),
    (700, 1032, 2064, True, BF16, ["fp8_quarter_kernelILi64ELb1ELb0ELb0E"]), (1000, 2048, 1000, False, BF16, ["fp8_quarter_kernelILi64ELb0ELb0ELb0E"]),
    (777, 1024, 2050, True, BF16, ["fp8_quarter_kernelILi64ELb1ELb0ELb0ELb0ELi2E"]), (777, 1024, 700, True, BF16, ["fp8_quarter_kernelILi64ELb1ELb0ELb0ELb0ELi1E"]),
    (800, 1000, 1120, False, BF16, ["fp8_quarter_kernelILi64ELb0ELb0ELb0ELb0ELi2E"]), (1024, 1000, 1500, False, F32, ["fp8_quarter_kernelILi64ELb0ELb1ELb0ELb0ELi2E"]),
    (777, 256, 4096, True, BF16, [ROW % (1, 0, 2, 2) + "Lb0E"]), (64, 1024, 4096, True, BF16, [ROW % (1, 0, 1, 1) + "Lb0E"]),
    (100, 1024, 2050, False, F32, [ROW % (0, 1, 1, 2) + "Lb0E"]), (1000, 1000, 16000, False, F32, [ROW % (0, 1, 4, 4) + "Lb1E"]),
    (900, 264, 9000, True, BF16, ["fp8_quarter_kernelILi64ELb1ELb0ELb1E", "linear_fixup_kernelILi64ELb0E"]),
    (1500, 2048, 400, True, BF16, ["fp8_deep_kernelILb1ELb0E"]), (1100, 4000, 700, False, BF16, ["fp8_deep_kernelILb0ELb0E"]),
    (500, 1000, 20000, True, BF16, ["fp8_deep_kernelILb1ELb1E", "linear_fixup_kernelILi128ELb0E"]),
    (2304, 1896, 6451, False, BF16, ["fp8_deep_kernelILb0ELb0E", "fp8_deep_kernelILb0ELb1E", "linear_fixup_kernelILi128ELb0E"]),
    (4096, 4096, 640, True, BF16, ["fp8_large_kernelILb1E"]), (4090, 4096, 1100, True, BF16, ["fp8_large_kernelILb0E"]),
    (8190, 4088, 700, True, BF16, ["fp8_large_kernelILb0E"]), (8200, 4096, 768, True, BF16, ["fp8_large_kernelILb1E"]),
    (32700, 504, 1300, True, BF16, ["fp8_large_kernelILb0E"]),
    (1100, 4000, 700, False, F32, ["fp8_quarter_kernelILi64ELb0ELb1ELb0E"]),
    (300, 264, 9000, True, F32, ["fp8_quarter_kernelILi64ELb1ELb1ELb1E", "linear_fixup_kernelILi64ELb1E"]),
    (2304, 1896, 6451, False, F32, ["fp8_quarter_kernelILi64ELb0ELb1ELb0E", "fp8_quarter_kernelILi64ELb0ELb1ELb1E", "linear_fixup_kernelILi64ELb1E"]),
    (2048, 2048, 1000, False, F32, ["fp8_quarter_kernelILi128ELb0ELb1ELb0E"]),
    (600, 520, 16000, False, F32, ["fp8_quarter_kernelILi128ELb0ELb1ELb1E", "linear_fixup_kernelILi128ELb1E"]),
    (1100, 1304, 9000, True, F32, ["fp8_wide_kernelILb1ELb1E", "linear_fixup_kernelILi128ELb1E"]),
    (4096, 4200, 1100, False, F32, ["fp8_wide_kernelILb0ELb0E"]),
]


@pytest.mark.parametrize("M,N,K,tiles,dtype,names", KERNELS)
def test_every_kernel(M, N, K, tiles, dtype, names):
    """To the bit, stored and added to, with room behind the rows; then random values."""
    launched = _launched(M, N, K, tiles, dtype)
    assert len(launched) == len(names) and all(any(n in k for k in launched) for n in names), launched
    _product(M, N, K, tiles, dtype)
    _product(M, N, K, tiles, dtype, beta=0.5, ldy=N + 40)
    _product(M, N, K, tiles, dtype, exact=False)


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("M,N,K", [(7, 64, 200), (200, 264, 1024), (777, 512, 2048)])
def test_product_added(M, N, K, tiles):
    for dtype in (BF16, F32):
        _product(M, N, K, tiles, dtype, beta=0.5)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("M,N,K", [(3, 64, 512), (65, 128, 1000), (500, 640, 2048)])
def test_product_of_random_values(M, N, K, tiles, dtype):
    _product(M, N, K, tiles, dtype, exact=False)
    _product(M, N, K, tiles, dtype, exact=False, beta=-1.5)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_reduction_and_no_work(dtype):
    """K == 0 is beta * Y (and does not read Y with beta == 0); M == 0 and N == 0 are nothing."""
    e = lambda *s: torch.empty(s, dtype=ref.FP8, device="cuda")  # noqa: E731
    f = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    y = torch.full((5, 24), 3.0, dtype=dtype, device="cuda")
    tmt_moe.fp8_matmul(e(5, 0), f(0, 5), e(24, 0), f(1, 0), y, beta=2.0)
    assert (y == 6).all()
    y[0] = float("nan")
    tmt_moe.fp8_matmul(e(5, 0), f(0, 5), e(24, 0), f(0, 24), y, blocks=ROWS)
    assert (y == 0).all()
    tmt_moe.fp8_matmul(e(0, 128), f(1, 0), e(24, 128), f(1, 1), y[:0])
    tmt_moe.fp8_matmul(e(5, 128), f(1, 5), e(0, 128), f(0, 1), torch.empty(5, 0, dtype=dtype, device="cuda"))


@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("M", [3, 300])
def test_nan_scales_stay_in_their_block(M, tiles):
    N, K = 264, 384
    a, _ = _operand(M, K, False, 1, True)
    b, _ = _operand(N, K, tiles, 2, True)
    a[1][1, 2] = float("nan")
    if tiles:
        b[1][1, 0] = float("nan")
        bad = slice(128, 256)
    else:
        b[1][2, 77] = float("nan")
        bad = slice(77, 78)
    y = torch.empty(M, N, dtype=BF16, device="cuda")
    size = tmt_moe.fp8_workspace_size(M, N, K, TILES if tiles else ROWS)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    tmt_moe.fp8_matmul(*a, *b, y, blocks=TILES if tiles else ROWS, workspace=ws)
    want = torch.zeros(M, N, dtype=torch.bool)
    want[2] = True
    want[:, bad] = True
    assert torch.equal(torch.isnan(y).cpu(), want)


def test_training_step_together():
    """The layer as it is used: norm to codes, product, gradient to codes both ways, dX, dW, the
    norm's backward; against autograd in 64 bits through the values that the codes stand for."""
    T, d, n = 500, 384, 640
    g = torch.Generator().manual_seed(5)
    x, r = torch.randn(T, d, generator=g).to(BF16), torch.randn(T, d, generator=g).to(BF16)
    gamma, w = 1 + 0.2 * torch.randn(d, generator=g), torch.randn(n, d, generator=g) * d ** -0.5
    dy, dr = (torch.randn(T, n, generator=g) * 1e-2).to(BF16), (torch.randn(T, d, generator=g) * 1e-2).to(BF16)

    def held(rows, cols, tiles=False):
        rb, kb = ref.blocks_of(rows), ref.blocks_of(cols)
        return (torch.empty(rows, ref.up(cols, 16), dtype=ref.FP8, device="cuda")[:, :cols],
                torch.empty((rb, kb) if tiles else (kb, rows), device="cuda"))

    W, Wt = held(n, d, True), held(d, n, True)
    tmt_moe.fp8_quantize(w.cuda(), *W, *Wt, blocks=TILES)
    S, rstd, Y8, Ybf = torch.empty_like(x).cuda(), torch.empty(T, device="cuda"), held(T, d), torch.empty(T, d, dtype=BF16, device="cuda")
    tmt_moe.rmsnorm_forward(x.cuda(), r.cuda(), gamma.cuda(), S=S, Y=Ybf, codes=Y8[0], scales=Y8[1], rstd=rstd)
    out = torch.empty(T, n, dtype=BF16, device="cuda")

    def product(A, B, y, blocks, beta=0.0):
        size = tmt_moe.fp8_workspace_size(A[0].shape[0], B[0].shape[0], A[0].shape[1], blocks)
        tmt_moe.fp8_matmul(*A, *B, y, beta=beta, blocks=blocks,
                           workspace=torch.empty(size, dtype=torch.uint8, device="cuda") if size else None)

    product(Y8, W, out, TILES)
    Yt, G, Gt = held(d, T), held(T, n), held(n, T)
    tmt_moe.fp8_quantize(Ybf, codes_t=Yt[0], scales_t=Yt[1])
    tmt_moe.fp8_quantize(dy.cuda(), *G, *Gt)
    dh, dW = torch.empty(T, d, dtype=BF16, device="cuda"), torch.full((n, d), 1.0, device="cuda")
    product(G, Wt, dh, TILES)
    product(Gt, Yt, dW, ROWS, beta=1.0)
    dS, dgamma = torch.empty_like(S), torch.empty(d, device="cuda")
    tmt_moe.rmsnorm_backward(dh, S, gamma.cuda(), rstd, dS, dgamma,
                             torch.empty(tmt_moe.rmsnorm_workspace_size(T, d), dtype=torch.uint8, device="cuda"), dR=dr.cuda())

    val = lambda c, tiles=False: ref.values(c[0].cpu().view(torch.uint8), c[1].cpu(), tiles)  # noqa: E731
    far = lambda a, b: ((a.cpu().double() - b).norm() / b.norm()).item()  # noqa: E731
    # each product against the same product of the values that its codes stand for
    assert far(out, val(Y8) @ val(W, True).t()) < 2.0 ** -8
    assert far(dh, val(G) @ val(Wt, True).t()) < 2.0 ** -8
    assert far(dW - 1, val(Gt) @ val(Yt).t()) < 1e-5
    # and the whole against autograd: codes are off by at most 2^-4 of a value (in norm less)
    s64 = S.cpu().double().requires_grad_()
    g64, w64 = gamma.double().requires_grad_(), w.double().requires_grad_()
    h = s64 * (s64.square().mean(1, keepdim=True) + 1e-5).rsqrt() * g64
    y64 = h @ w64.t()
    y64.backward(dy.double())
    assert far(out, y64.detach()) < 2 * 2.0 ** -4
    assert far(dW - 1, w64.grad) < 2 * 2.0 ** -4
    assert far(dS.cpu().double() - dr.double(), s64.grad) < 2 * 2.0 ** -4
    assert far(dgamma, g64.grad) < 2 * 2.0 ** -4


@pytest.mark.parametrize("M,tiles,dtype", [(1, True, BF16), (64, True, BF16), (777, True, BF16), (700, False, F32), (3000, True, BF16)])
def test_repeats_and_captures(M, tiles, dtype):
    """The same bits on another stream and from a graph's replays with new inputs."""
    N, K = 1032, 2064
    blocks = TILES if tiles else ROWS
    a, _ = _operand(M, K, False, 1, False)
    b, _ = _operand(N, K, tiles, 2, False)
    size = tmt_moe.fp8_workspace_size(M, N, K, blocks)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    y = [torch.zeros(M, N, dtype=dtype, device="cuda") for _ in range(3)]
    tmt_moe.fp8_matmul(*a, *b, y[0], blocks=blocks, workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    tmt_moe.fp8_matmul(*a, *b, y[1], blocks=blocks, workspace=ws, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y[0], y[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tmt_moe.fp8_matmul(*a, *b, y[2], blocks=blocks, workspace=ws)
    for k in range(3):
        b[1].mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        tmt_moe.fp8_matmul(*a, *b, y[0], blocks=blocks, workspace=ws)
        assert torch.equal(y[0], y[2])


@pytest.mark.parametrize("M", [40, 300])
def test_the_widest_strides(M):
    """Code rows 2^22 bytes apart give the bits of dense ones; what lies between is NaN."""
    N, K, ld = 72, 1500, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(M)

    def operand(rows, blocks):
        x = torch.randn(rows, K, device="cuda", generator=g).to(BF16)
        X = torch.empty(rows, ref.up(K, 8), dtype=BF16, device="cuda")[:, :K].copy_(x)
        dense = torch.empty(rows, ref.up(K, 16), dtype=torch.uint8, device="cuda")
        shape = (ref.blocks_of(rows), ref.blocks_of(K)) if blocks == TILES else (ref.blocks_of(K), rows)
        scales = torch.empty(shape, device="cuda")
        tmt_moe.fp8_quantize(X, dense[:, :K], scales, blocks=blocks)
        wide = torch.full(((rows - 1) * ld + ref.up(K, 16),), 0x7f, dtype=torch.uint8, device="cuda")
        wide = wide.as_strided((rows, ref.up(K, 16)), (ld, 1)).copy_(dense)
        return dense[:, :K], wide[:, :K], scales

    a, wide_a, sa = operand(M, ROWS)
    for blocks in (TILES, ROWS):
        b, wide_b, sb = operand(N, blocks)
        for dtype in (BF16, F32):
            y, z = (torch.empty(M, N, dtype=dtype, device="cuda") for _ in range(2))
            ws = torch.empty(max(tmt_moe.fp8_workspace_size(M, N, K, blocks), 1), dtype=torch.uint8, device="cuda")
            tmt_moe.fp8_matmul(a, sa, b, sb, y, blocks=blocks, workspace=ws)
            tmt_moe.fp8_matmul(wide_a, sa, wide_b, sb, z, blocks=blocks, workspace=ws)
            assert torch.isfinite(y).all() and torch.equal(y, z)
