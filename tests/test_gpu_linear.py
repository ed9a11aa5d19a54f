"""The linear layer on microscaled numbers against plain products in 64 bits.

Tolerances: operands are exact, so an output is off by the fp32 sum's
rounding, at most (R + 2) 2^-23 of the sum of the terms' magnitudes for R
terms in any order, and by one rounding to its type, 2^-8 (bf16) or 2^-24
(fp32) of its value; beta adds one product and one sum in fp32.
"""
import numpy as np
import pytest
import torch

import mx_ref
import synthetic
import tmt_moe

pytestmark = pytest.mark.gpu

FP4, FP8 = tmt_moe.MX_FP4, tmt_moe.MX_FP8
BF16 = torch.bfloat16


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _rng(*key):
    return np.random.Generator(np.random.PCG64(list(key)))


def _bf16(x):
    """fp32 values that bf16 holds."""
    return synthetic.bf16_to_f32(synthetic.bf16_bits(np.asarray(x, np.float32)))


def _strided(a, ld, dtype, fill=float("nan")):
    """Device matrix with row stride ld, everything outside the rows `fill`,
    one row of it in front and one behind."""
    rows, cols = a.shape
    buf = torch.full(((rows + 2), ld), fill, dtype=dtype, device="cuda")
    view = buf[1:rows + 1, :cols]
    view.copy_(torch.from_numpy(np.ascontiguousarray(a)).to(dtype))
    return buf, view


def _scales(s, lds, fill=171):
    """[rows, K/32] scale bytes to block-major [K/32, lds] on the device."""
    out = torch.full((s.shape[1], lds), fill, dtype=torch.uint8, device="cuda")
    out[:, :s.shape[0]] = _dev(s.T)
    return out


def _up16(n):
    return max(16, (n + 15) // 16 * 16)


# ---- rows to codes and back -----------------------------------------------------

def _special(fmt):
    """Blocks where rounding, scales or the formats' ends can go wrong."""
    blocks = []
    rng = _rng(11)
    for e in (-126, -125, -120, -20, 0, 3, 60, 120, 125):
        for top in (1.0, 1.25, 1.5, 1.7421875, 1.75, 1.7578125, 1.9921875):
            b = np.zeros(32, np.float64)
            b[0] = top
            # every code, every border and its neighbours, in units of the block
            edge = np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.5]) / 4 * np.exp2(0)
            b[1:10] = edge
            b[10:19] = -edge * (1 + 2.0 ** -7)
            b[19:28] = edge * (1 - 2.0 ** -8)
            b[28:] = rng.standard_normal(4) * 2.0 ** -7
            blocks.append(np.ldexp(np.clip(b, -top, top), e))
    for v in (0.0, -0.0, 1e-45, -1e-40, 1.1754942e-38, 3.38e38, -3.38e38):
        blocks.append(np.full(32, v))
    for bad in (np.inf, -np.inf, np.nan):
        b = rng.standard_normal(32)
        b[rng.integers(32)] = bad
        blocks.append(b)
        blocks.append(np.full(32, bad))
    n = len(blocks)
    with np.errstate(over="ignore"):
        x = np.array(blocks, np.float32)
    return np.concatenate([x, x[rng.permutation(n)]], axis=1)


def _same_values(a, b):
    return np.array_equal(np.nan_to_num(a, nan=1234.5, posinf=1e300, neginf=-1e300),
                          np.nan_to_num(b, nan=1234.5, posinf=1e300, neginf=-1e300))


def _check_rows(x, fmt, f32, ldx=None, lds=None):
    rows, K = x.shape
    dtype = torch.float32 if f32 else BF16
    piece = 4 if f32 else 8
    ldx = ldx or (K + piece - 1) // piece * piece
    lds = lds or rows
    _, X = _strided(x, ldx, dtype)
    width = K // 2 if fmt == FP4 else K
    guard = 64
    codes_buf = torch.full((rows * width + guard,), 0xA5, dtype=torch.uint8, device="cuda")
    codes = codes_buf[:rows * width].view(rows, width)
    sc_buf = torch.full(((K // 32) * lds + guard,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = sc_buf[:(K // 32) * lds].view(K // 32, lds)
    tmt_moe.mx_quantize(X, codes, scales, fmt)
    ref_c, ref_s = mx_ref.quantize(x, fmt)
    got_s = scales.cpu().numpy()
    assert np.array_equal(got_s[:, :rows].T, ref_s)
    assert np.array_equal(codes.cpu().numpy(), ref_c)
    assert (got_s[:, rows:] == 0xA5).all() and (codes_buf[rows * width:] == 0xA5).all()
    assert (sc_buf[(K // 32) * lds:] == 0xA5).all()
    # back: exact in fp32, one rounding in bf16
    values = mx_ref.dequantize(ref_c, ref_s, fmt)
    for out in (torch.float32, BF16):
        pc = 4 if out == torch.float32 else 8
        buf, y = _strided(np.zeros((rows, K), np.float32), (K + pc - 1) // pc * pc + pc, out, fill=7.0)
        tmt_moe.mx_dequantize(codes, scales, y, fmt)
        want = torch.from_numpy(values.astype(np.float32)).to(out).double().numpy()
        assert _same_values(y.double().cpu().numpy(), want)
        assert (buf[0] == 7).all() and (buf[-1] == 7).all() and (buf[1:-1, K:] == 7).all()


@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("f32", [False, True])
def test_rows_special_values(fmt, f32):
    x = _special(fmt)
    _check_rows(x if f32 else _bf16_keep(x), fmt, f32)


def _bf16_keep(x):
    """bf16 values, infinities and NaN kept."""
    return torch.from_numpy(x).to(BF16).float().numpy()


@pytest.mark.parametrize("fmt", [FP4, FP8])
def test_every_bf16_value(fmt):
    """All finite bf16 values, 31 a block, each block topped by a value of
    the same magnitude or up to 2^6 larger."""
    bits = np.arange(65536, dtype=np.uint16)
    v = synthetic.bf16_to_f32(bits)
    v = v[np.isfinite(v)]
    order = np.argsort(np.abs(v), kind="stable")
    v = v[order]
    v = np.concatenate([v, np.zeros((-len(v)) % 31, np.float32)]).reshape(-1, 31)
    rows = []
    for up in (0, 1, 3, 6):
        with np.errstate(over="ignore"):
            top = np.minimum(np.abs(v).max(1).astype(np.float64) * 2.0 ** up, 3.3e38).astype(np.float32)
        rows.append(np.concatenate([_bf16(top)[:, None], v], axis=1))
    _check_rows(np.concatenate(rows), fmt, False)


@pytest.mark.parametrize("fmt", [FP4, FP8])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,K,ldx,lds", [
    (1, 32, None, None), (1, 4096, None, None), (3, 64, 72, 5), (63, 96, None, 64), (64, 128, 136, None),
    (65, 160, None, 67), (129, 224, 232, 256), (257, 256, None, None), (777, 288, None, 784), (130, 1056, 1064, 131),
    (5003, 64, None, None), (40, 4096, 4104, 48),
])
def test_rows_shapes(fmt, f32, rows, K, ldx, lds):
    rng = _rng(rows, K)
    x = rng.standard_normal((rows, K)) * np.exp(rng.uniform(-3, 3, (rows, 1)))
    _check_rows(x.astype(np.float32) if f32 else _bf16(x), fmt, f32, ldx, lds)


# ---- products ------------------------------------------------------------------

OPS = ("linear", "matmul", "dx", "dw")
_SIZE_OP = {"linear": tmt_moe.LINEAR_FORWARD, "matmul": tmt_moe.LINEAR_MATMUL, "dx": tmt_moe.LINEAR_DX,
            "dw": tmt_moe.LINEAR_DW}


class Problem:
    """One product's operands on the device and in 64 bits."""

    def __init__(self, op, T, N, K, seed=0, pad=0, spread=1.0):
        self.op, self.T, self.N, self.K = op, T, N, K
        rng = _rng(seed, T, N, K)
        self.lds = {"w": _up16(N) + 16 * (pad > 0), "x": _up16(T) + 16 * (pad > 0)}
        scale = lambda shape: rng.standard_normal(shape) * np.exp(rng.uniform(-spread, spread, (shape[0], 1)))  # noqa: E731
        if op == "dw":
            self.mx_c, self.mx_s = mx_ref.quantize(scale((T, K)).astype(np.float32), FP8)
            self.B = mx_ref.dequantize(self.mx_c, self.mx_s, FP8)  # [T, K]
        else:
            self.mx_c, self.mx_s = mx_ref.quantize((scale((N, K)) * K ** -0.5).astype(np.float32), FP4)
            self.B = mx_ref.dequantize(self.mx_c, self.mx_s, FP4)  # [N, K]
        if op == "matmul":
            self.xc, self.xs = mx_ref.quantize(scale((T, K)).astype(np.float32), FP4)
            self.A = mx_ref.dequantize(self.xc, self.xs, FP4)
        else:
            self.A = _bf16(scale((T, K if op == "linear" else N))).astype(np.float64)
        self.pad = pad
        self.upload()

    def upload(self):
        self.codes = _dev(self.mx_c)
        self.scales = _scales(self.mx_s, self.lds["x" if self.op == "dw" else "w"])
        if self.op == "matmul":
            self.x = (_dev(self.xc), _scales(self.xs, self.lds["x"]))
        else:
            _, self.x = _strided(self.A.astype(np.float32), self.A.shape[1] + self.pad, BF16)

    def out_shape(self):
        return {"linear": (self.T, self.N), "matmul": (self.T, self.N), "dx": (self.T, self.K), "dw": (self.N, self.K)}[self.op]

    def output(self, init=None):
        rows, cols = self.out_shape()
        a = np.full((rows, cols), np.nan, np.float32) if init is None else init
        return _strided(a, cols + self.pad, torch.float32 if self.op == "dw" else BF16, fill=5.0)

    def workspace(self, fill=0xFF):
        n = tmt_moe.linear_workspace_size(_SIZE_OP[self.op], self.T, self.N, self.K)
        return torch.full((n,), fill, dtype=torch.uint8, device="cuda") if n else None

    def call(self, y, ws, beta=0.0):
        if self.op == "matmul":
            tmt_moe.mxfp4_matmul(*self.x, self.codes, self.scales, y, beta=beta, workspace=ws)
        else:
            fn = {"linear": tmt_moe.mxfp4_linear, "dx": tmt_moe.mxfp4_linear_dx, "dw": tmt_moe.mxfp8_linear_dw}[self.op]
            fn(self.x, self.codes, self.scales, y, beta=beta, workspace=ws)

    def _product(self, A, B):
        A, B = _dev(A), _dev(B)
        r = A @ B.t() if self.op in ("linear", "matmul") else A @ B if self.op == "dx" else A.t() @ B
        return r.cpu().numpy()

    def reference(self):
        return self._product(self.A, self.B)

    def magnitude(self):
        return self._product(np.abs(self.A), np.abs(self.B))

    def check(self, y, init=None, beta=0.0, more=0.0):
        """more: a further absolute tolerance per output."""
        ref, mag = self.reference(), self.magnitude()
        R = {"linear": self.K, "matmul": self.K, "dx": self.N, "dw": self.T}[self.op]
        if init is not None:
            ref = ref + beta * init.astype(np.float64)
            mag = mag + abs(beta) * np.abs(init)
        got = y.double().cpu().numpy()
        tol = (R + 4) * 2.0 ** -23 * mag + np.abs(ref) * (2.0 ** -24 if self.op == "dw" else 2.0 ** -8) + more
        far = np.abs(got - ref) - tol
        worst = np.unravel_index(np.nanargmax(np.where(np.isnan(far), np.inf, far)), far.shape)
        assert (far <= 0).all(), (worst, got[worst], ref[worst], tol[worst])


def _run(op, T, N, K, pad=0, beta=0.0, seed=0):
    p = Problem(op, T, N, K, seed=seed, pad=pad)
    init = None
    if beta != 0.0:
        init = _rng(9, T).standard_normal(p.out_shape()).astype(np.float32)
        if op != "dw":
            init = _bf16(init)
    buf, y = p.output(init)
    p.call(y, p.workspace(), beta)
    p.check(y, init, beta)
    assert (buf[0] == 5).all() and (buf[-1] == 5).all() and (buf[1:-1, y.shape[1]:] == 5).all()
    return p


SHAPES = [
    (1, 16, 64), (1, 4096, 1024), (2, 48, 128), (3, 1040, 192), (8, 1024, 4096), (15, 272, 64), (16, 16, 4096),
    (17, 128, 320), (31, 80, 1024), (33, 4096, 64), (64, 1024, 4096), (65, 256, 256), (100, 144, 448), (127, 1280, 1280),
    (128, 128, 128), (129, 144, 192), (255, 272, 320), (256, 256, 64), (257, 528, 576), (300, 16, 4096), (513, 64, 1024),
    (777, 1024, 4096), (1024, 256, 256), (2048, 1280, 1280), (1500, 4112, 64), (5003, 1008, 960),
]


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("T,N,K", SHAPES)
def test_products(op, T, N, K):
    _run(op, T, N, K)


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("T,N,K,pad,beta", [
    (1, 64, 256, 8, 1.0), (5, 112, 192, 24, 0.0), (40, 1024, 1024, 8, -0.5), (130, 272, 320, 40, 1.0),
    (777, 336, 2048, 8, 0.25), (2100, 1296, 1344, 16, 1.0), (9000, 400, 448, 8, 1.0),
])
def test_strides_and_beta(op, T, N, K, pad, beta):
    """Rows wider than their width, NaN between them, an output that is read
    (beta != 0) or that starts as NaN (beta == 0)."""
    _run(op, T, N, K, pad, beta)


@pytest.mark.parametrize("op,T,N,K", [("linear", 16384, 4096, 1024), ("matmul", 16384, 4096, 1024),
                                      ("dx", 16384, 4096, 1024), ("dw", 16384, 4096, 1024), ("dw", 40001, 1024, 256),
                                      ("linear", 20011, 2736, 704), ("matmul", 20011, 2736, 704), ("dx", 20011, 2736, 704)])
def test_large_products(op, T, N, K):
    _run(op, T, N, K)


def test_no_tokens():
    """A weight gradient over no tokens is zero, or beta times what was there."""
    for beta in (0.0, 0.5):
        dW = torch.full((48, 128), 3.0, device="cuda")
        if beta == 0.0:
            dW.fill_(float("nan"))
        n = tmt_moe.linear_workspace_size(tmt_moe.LINEAR_DW, 0, 48, 128)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
        tmt_moe.mxfp8_linear_dw(torch.empty(0, 48, dtype=BF16, device="cuda"),
                                torch.empty(0, 128, dtype=torch.uint8, device="cuda"),
                                torch.empty(4, 16, dtype=torch.uint8, device="cuda"), dW, beta=beta, workspace=ws)
        assert (dW == (1.5 if beta else 0.0)).all()


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("T,N,K", [(7, 64, 256), (70, 272, 320), (600, 528, 576), (3000, 1280, 1280)])
def test_bad_values_stay_where_they_belong(op, T, N, K):
    """An infinity or a NaN in one row, and a block whose scale is NaN, reach
    the outputs that sum them and no others."""
    p = Problem(op, T, N, K, seed=3)
    rng = _rng(4, T)
    row, col = int(rng.integers(T)), int(rng.integers(N if op in ("dx", "dw") else K))
    mrow, mblk = int(rng.integers(len(p.mx_s))), int(rng.integers(K // 32))
    if op == "matmul":
        p.xs[row, col // 32] = 255
        p.A = mx_ref.dequantize(p.xc, p.xs, FP4)
    else:
        p.A[row, col] = np.inf if T % 2 else np.nan
    p.mx_s[mrow, mblk] = 255
    p.B = mx_ref.dequantize(p.mx_c, p.mx_s, FP8 if op == "dw" else FP4)
    p.upload()
    _, y = p.output()
    p.call(y, p.workspace())
    with np.errstate(all="ignore"):
        ok = np.isfinite(p._product(p.A, p.B))
    got = y.double().cpu().numpy()
    assert np.array_equal(np.isfinite(got), ok)
    assert ok.any() and not ok.all()
    p.A, p.B = np.where(np.isfinite(p.A), p.A, 0.0), np.where(np.isfinite(p.B), p.B, 0.0)
    ref, mag = p.reference(), p.magnitude()
    R = {"linear": K, "matmul": K, "dx": N, "dw": T}[op]
    tol = (R + 4) * 2.0 ** -23 * mag + np.abs(ref) * 2.0 ** -8
    assert (np.abs(got - ref)[ok] <= tol[ok]).all()


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("shift", [-100, 60])
def test_far_scales(op, shift):
    """Weights and checkpoints far from 1: scales are exponents, nothing is lost."""
    p = Problem(op, 70, 144, 192, seed=6)
    p.mx_s = (p.mx_s.astype(np.int32) + shift).astype(np.uint8)
    p.B = p.B * 2.0 ** shift
    p.upload()
    _, y = p.output()
    p.call(y, p.workspace())
    p.check(y)


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("T,N,K", [(1, 1024, 1024), (64, 1024, 4096), (300, 256, 2048), (2048, 1280, 1280)])
def test_captured_and_repeated(op, T, N, K):
    """Bit-identical from run to run, on another stream and in a replayed
    graph with other work in between; the workspace's content does not count."""
    p = Problem(op, T, N, K, seed=2)
    _, first = p.output()
    p.call(first, p.workspace(0xFF))
    _, again = p.output()
    ws = p.workspace(0x00)
    p.call(again, ws)
    assert torch.equal(first, again)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    _, third = p.output()
    with torch.cuda.stream(side):
        p.call(third, ws)
    side.synchronize()
    assert torch.equal(first, third)
    _, out = p.output()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        p.call(out, ws)
    for k in range(3):
        out.fill_(float(k))
        if ws is not None:
            ws.fill_(0xFF - k)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, out), k


def test_rows_past_4_gib():
    """Offsets beyond 32 bits: the last rows of a checkpoint of 2.2 GB and its
    products."""
    T, K, N = 2_200_003, 1024, 16
    lds = _up16(T)
    X = torch.empty(T, K, dtype=BF16, device="cuda")
    codes = torch.empty(T, K, dtype=torch.uint8, device="cuda")
    scales = torch.empty(K // 32, lds, dtype=torch.uint8, device="cuda")
    X.zero_()
    tail = _bf16(_rng(1).standard_normal((64, K)))
    X[-64:] = torch.from_numpy(tail).to(BF16)
    tmt_moe.mx_quantize(X, codes, scales, FP8)
    c, s = mx_ref.quantize(tail, FP8)
    assert np.array_equal(codes[-64:].cpu().numpy(), c)
    assert np.array_equal(scales[:, T - 64:T].cpu().numpy().T, s)
    assert (scales[:, :T - 64] == 127).all() and int(codes[:-64].max()) == 0
    dY = torch.zeros(T, N, dtype=BF16, device="cuda")
    g = _bf16(_rng(2).standard_normal((64, N)))
    dY[-64:] = torch.from_numpy(g).to(BF16)
    dW = torch.empty(N, K, device="cuda")
    n = tmt_moe.linear_workspace_size(tmt_moe.LINEAR_DW, T, N, K)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    tmt_moe.mxfp8_linear_dw(dY, codes, scales, dW, workspace=ws)
    V = mx_ref.dequantize(c, s, FP8)
    ref, mag = g.T.astype(np.float64) @ V, np.abs(g.T).astype(np.float64) @ np.abs(V)
    assert (np.abs(dW.double().cpu().numpy() - ref) <= 70 * 2.0 ** -23 * mag).all()
    wc, wsc = mx_ref.quantize((_rng(3).standard_normal((N, K)) / 32).astype(np.float32), FP4)
    Y = torch.empty(T, N, dtype=BF16, device="cuda")
    n = tmt_moe.linear_workspace_size(tmt_moe.LINEAR_FORWARD, T, N, K)
    ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
    tmt_moe.mxfp4_linear(X, _dev(wc), _scales(wsc, N), Y, workspace=ws)
    W = mx_ref.dequantize(wc, wsc, FP4)
    ref, mag = tail.astype(np.float64) @ W.T, np.abs(tail).astype(np.float64) @ np.abs(W.T)
    assert (np.abs(Y[-64:].double().cpu().numpy() - ref) <= (K + 4) * 2.0 ** -23 * mag + 2.0 ** -8 * np.abs(ref)).all()
    assert (Y[:-64] == 0).all()


def test_binding_refusals():
    X = torch.zeros(4, 64, dtype=BF16, device="cuda")
    Y = torch.zeros(4, 16, dtype=BF16, device="cuda")
    c = torch.zeros(16, 32, dtype=torch.uint8, device="cuda")
    s = torch.zeros(2, 16, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="must be a matrix"):
        tmt_moe.mxfp4_linear(X.float(), c, s, Y)
    with pytest.raises(ValueError, match="codes of W"):
        tmt_moe.mxfp4_linear(X, c[:8], s, Y)
    with pytest.raises(ValueError, match="scales of W"):
        tmt_moe.mxfp4_linear(X, c, s[:1], Y)
    with pytest.raises(ValueError, match="not on the current GPU"):
        tmt_moe.mxfp4_linear(X.cpu(), c, s, Y)
    with pytest.raises(ValueError, match="contiguous"):
        tmt_moe.mxfp4_linear(X.t().contiguous().t(), c, s, Y)
    with pytest.raises(ValueError, match="Y must be"):
        tmt_moe.mxfp4_linear(X, c, s, Y[:3])
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        tmt_moe.mx_quantize(X.half(), c, s)


# ---- together -------------------------------------------------------------------

def _train_step(T, N, K):
    """Quantise the masters, forward, keep the input in 8 bits, both gradients,
    AdamW, quantise again, and serve one token from the new weights."""
    rng = _rng(T, N)
    master = (rng.standard_normal((N, K)) * K ** -0.5).astype(np.float32)
    x, dy = _bf16(rng.standard_normal((T, K))), _bf16(rng.standard_normal((T, N)))
    M = _dev(master)
    state = {k: torch.zeros_like(M) for k in ("m", "v", "grad")}
    X, dY = _dev(x).to(BF16), _dev(dy).to(BF16)
    wc, wsc = torch.empty(N, K // 2, dtype=torch.uint8, device="cuda"), torch.empty(K // 32, N, dtype=torch.uint8, device="cuda")
    xc, xs = torch.empty(T, K, dtype=torch.uint8, device="cuda"), torch.empty(K // 32, _up16(T), dtype=torch.uint8, device="cuda")
    Y, dX = torch.empty(T, N, dtype=BF16, device="cuda"), torch.empty(T, K, dtype=BF16, device="cuda")
    size = max(tmt_moe.linear_workspace_size(op, T, N, K) for op in range(4))
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    opt = tmt_moe.AdamW([dict(master=M, **state)])
    tmt_moe.mx_quantize(M, wc, wsc)
    tmt_moe.mxfp4_linear(X, wc, wsc, Y, workspace=ws)
    tmt_moe.mx_quantize(X, xc, xs, FP8)
    tmt_moe.mxfp4_linear_dx(dY, wc, wsc, dX, workspace=ws)
    tmt_moe.mxfp8_linear_dw(dY, xc, xs, state["grad"], workspace=ws)
    opt.step(1, lr=1e-2, weight_decay=0.0)
    tmt_moe.mx_quantize(M, wc, wsc)
    y1 = torch.empty(1, N, dtype=BF16, device="cuda")
    tmt_moe.mxfp4_linear(X[:1], wc, wsc, y1, workspace=ws)
    torch.cuda.synchronize()
    W = mx_ref.dequantize(*mx_ref.quantize(master, FP4), FP4)
    X8 = mx_ref.dequantize(*mx_ref.quantize(x, FP8), FP8)
    new = M.cpu().numpy()
    W1 = mx_ref.dequantize(*mx_ref.quantize(new, FP4), FP4)
    x64, dy64 = x.astype(np.float64), dy.astype(np.float64)
    for got, a, b, half in ((Y, x64, W.T, 2.0 ** -8), (dX, dy64, W, 2.0 ** -8), (state["grad"], dy64.T, X8, 2.0 ** -24),
                            (y1, x64[:1], W1.T, 2.0 ** -8)):
        ref, mag = a @ b, np.abs(a) @ np.abs(b)
        assert (np.abs(got.double().cpu().numpy() - ref) <= (a.shape[1] + 4) * 2.0 ** -23 * mag + half * np.abs(ref)).all()
    # the update is AdamW's first step: lr times the gradient's sign, eps aside
    g = state["grad"].cpu().numpy()
    big = np.abs(g) > 1e-3
    assert np.abs((new - master)[big] + 1e-2 * np.sign(g)[big]).max() <= 1e-6
    # the checkpoint's gradient against the exact input's: each value of X8 is
    # within 2^-4 of X's
    exact = dy64.T @ x64
    assert (np.abs(g - exact) <= (2.0 ** -4 + 1e-5) * (np.abs(dy64).T @ np.abs(x64)) + 1e-30).all()
    opt.close()


@pytest.mark.parametrize("T,N,K", [(96, 256, 256), (777, 272, 320)])
def test_training_step_together(T, N, K):
    _train_step(T, N, K)


def test_gradients_by_differences():
    """L = <dY, X W^T> is linear in X and W: its differences are the gradients."""
    T, N, K = 33, 48, 64
    p, q = Problem("dx", T, N, K, seed=8), Problem("dw", T, N, K, seed=8)
    _, dX = p.output()
    p.call(dX, p.workspace())
    _, dW = q.output()
    q.call(dW, q.workspace())
    rng = _rng(12)
    loss = lambda X, W, dY: float((dY * (X @ W.T)).sum())  # noqa: E731
    h = 2.0 ** -6
    for _ in range(20):
        t, k, n = int(rng.integers(T)), int(rng.integers(K)), int(rng.integers(N))
        X = np.zeros((T, K))
        X[t, k] = h
        diff = (loss(X, p.B, p.A) - loss(-X, p.B, p.A)) / (2 * h)
        assert abs(float(dX[t, k]) - diff) <= abs(diff) * 2.0 ** -8 + 1e-5
        W = np.zeros((N, K))
        W[n, k] = h
        diff = (loss(q.B, W, q.A) - loss(q.B, -W, q.A)) / (2 * h)
        assert abs(float(dW[n, k]) - diff) <= abs(diff) * 2.0 ** -20 + 1e-5


def test_expert_weights_from_the_quantiser():
    """mx_quantize writes the block's own MXFP4 format: tmt_moe_forward_mxfp4 on
    its output equals the one on the host-made weights."""
    T, d, E, topk, h = 48, 256, 4, 2, 320
    case = synthetic.make_case(T, d, E, topk, h, seed=3, with_dy=False)
    as_bf16 = lambda a: _dev(a.view(np.int16)).view(BF16)  # noqa: E731
    outs = []
    for where in ("host", "gpu"):
        w = {}
        for name in ("W_up", "W_down"):
            if where == "host":
                q = synthetic.mxfp4_experts(case[name])
                w[name], w[name + "_s"] = _dev(q["codes"]), _dev(q["scales"])
            else:
                src = as_bf16(case[name])
                n, k = src.shape[1:]
                w[name] = torch.empty(E, n, k // 2, dtype=torch.uint8, device="cuda")
                w[name + "_s"] = torch.empty(E, k // 32, n, dtype=torch.uint8, device="cuda")
                for e in range(E):
                    tmt_moe.mx_quantize(src[e], w[name][e], w[name + "_s"][e])
        m = tmt_moe.MoE(T, d, E, topk, h, weight_format=tmt_moe.WEIGHTS_MXFP4)
        Y = torch.zeros(T, d, dtype=BF16, device="cuda")
        m.forward_mxfp4(as_bf16(case["X"]), as_bf16(case["Wr"]), w["W_up"], w["W_up_s"], w["W_down"], w["W_down_s"], Y, beta=0.0)
        outs.append(Y.cpu())
        m.close()
    assert torch.equal(*outs)


# ---- dispatch, ends of memory, streams ----------------------------------------------


@pytest.mark.parametrize("op,T,N,K,kernels", [
    ("linear", 1, 4096, 1024, ["linear_rows_kernelILi1ELi1ELi8ELi1E"]),
    ("linear", 16, 1024, 4096, ["linear_rows_kernelILi1ELi1ELi8ELi2E"]),
    ("linear", 64, 4096, 1024, ["linear_rows_kernelILi1ELi2ELi4ELi2E"]),
    ("linear", 64, 4096, 2048, ["linear_rows_kernelILi1ELi2ELi8ELi2E"]),
    ("linear", 128, 4096, 1024, ["linear_rows_kernelILi2ELi2ELi4ELi2E"]),
    ("linear", 256, 2048, 2048, ["linear_rows_kernelILi2ELi2ELi8ELi1E"]),
    ("linear", 600, 1280, 1024, ["linear_rows_kernelILi4ELi2ELi4ELi1E"]),
    ("linear", 777, 4096, 1024, ["linear_fwd_kernelILi128ELb0E"]),
    ("linear", 777, 1024, 4096, ["linear_fwd_kernelILi128ELb1E", "linear_fixup_kernelILi128ELb0E"]),
    ("linear", 16384, 4096, 1024, ["linear_fwd_kernelILi256ELb0E"]),
    ("matmul", 777, 4096, 1024, ["linear_mx_kernelILb0ELb1E"]),
    ("matmul", 777, 4096, 960, ["linear_mx_kernelILb0ELb0E"]),
    ("matmul", 128, 256, 8192, ["linear_mx_kernelILb1ELb1E", "linear_fixup_kernelILi128ELb0E"]),
    ("matmul", 128, 256, 8128, ["linear_mx_kernelILb1ELb0E", "linear_fixup_kernelILi128ELb0E"]),
    ("dx", 1024, 256, 256, ["linear_grad_kernelILi2ELi128ELb0E"]),
    ("dx", 64, 4096, 256, ["linear_grad_kernelILi2ELi128ELb1E", "linear_fixup_kernelILi128ELb0E"]),
    ("dx", 16384, 1024, 4096, ["linear_grad_kernelILi2ELi256ELb0E"]),
    ("dw", 128, 1024, 1024, ["linear_grad_kernelILi3ELi128ELb0E"]),
    ("dw", 2048, 256, 256, ["linear_grad_kernelILi3ELi128ELb1E", "linear_fixup_kernelILi128ELb1E"]),
    ("dw", 4096, 4096, 4096, ["linear_grad_kernelILi3ELi256ELb0E"]),
    ("dw", 16384, 4096, 1024, ["linear_grad_kernelILi3ELi256ELb1E", "linear_fixup_kernelILi256ELb1E"]),
])
def test_every_kernel_variant(op, T, N, K, kernels):
    """Each shape reaches the kernels that the plan should choose for it, and
    its result holds."""
    from launched_kernels import launched_kernels
    p = _run(op, T, N, K)
    _, y = p.output()
    ws = p.workspace()
    names = launched_kernels(lambda: p.call(y, ws))
    assert len(names) == len(kernels), names
    for want, name in zip(kernels, names):
        assert want in name, (want, name)


@pytest.mark.parametrize("op,T,N,K,kernel", [
    ("linear", 70 * 256, 1024, 4096, "linear_fwd_kernelILi256E"),
    ("dx", 70 * 256, 4096, 1024, "linear_grad_kernelILi2ELi256E"),
])
def test_whole_rounds_and_a_split_tail(op, T, N, K, kernel):
    """More tiles than fit at a time: whole ones, then the last round's parts
    and their sums."""
    from launched_kernels import launched_kernels
    p = _run(op, T, N, K)
    _, y = p.output()
    ws = p.workspace()
    names = launched_kernels(lambda: p.call(y, ws))
    assert [kernel + "Lb0E" in names[0], kernel + "Lb1E" in names[1], "linear_fixup_kernelILi256ELb0E" in names[2]] == [True] * 3, names


@pytest.mark.parametrize("op", OPS)
def test_operands_at_the_end_of_their_memory(op):
    """Operands that fill their allocations to the last byte (32 MiB, its own
    mapping), several units to a workgroup: nothing behind them is read."""
    torch.cuda.empty_cache()
    T = N = 4096
    K = 4096
    big = 16384 if op != "dw" else 4096
    T = big if op in ("linear", "matmul", "dx") else T
    N = 1024 if op in ("linear", "matmul", "dx") else N
    p = Problem(op, T, N, K if op != "dx" else 1024, seed=1)
    hold = []
    def own(t):  # t's values at the end of an allocation of whole 2 MiB pages
        n = t.numel() * t.element_size()
        page = 2 << 20
        whole = max((n + page - 1) // page * page, 12 << 20)
        buf = torch.empty(whole, dtype=torch.uint8, device="cuda")
        hold.append(buf)
        view = buf[whole - n:].view(t.dtype).view(t.shape)
        view.copy_(t)
        return view
    p.codes, p.scales = own(p.codes), own(p.scales)
    if op == "matmul":
        p.x = (own(p.x[0]), own(p.x[1]))
    else:
        p.x = own(p.x.contiguous())
    _, y = p.output()
    p.call(y, p.workspace())
    p.check(y)


def test_the_smallest_scales():
    """Scale byte 0 is 2^-127, in every product. MXFP4 values are multiples of
    2^-128 there, which bf16 holds (its subnormals are multiples of 2^-133);
    MXFP8 values are multiples of 2^-136 and each is rounded to a subnormal,
    off by at most 2^-134: the sum of |dY| times that comes on top."""
    for op in OPS:
        p = Problem(op, 20, 32, 128, seed=7, spread=0.1)
        p.mx_s[:] = 0
        p.B = mx_ref.dequantize(p.mx_c, p.mx_s, FP8 if op == "dw" else FP4)
        if op == "matmul":
            p.xs[:] = 250
            p.A = mx_ref.dequantize(p.xc, p.xs, FP4)
        else:
            p.A = _bf16(p.A * 2.0 ** 100).astype(np.float64)
        p.upload()
        _, y = p.output()
        p.call(y, p.workspace())
        p.check(y, more=np.abs(p.A).sum(0)[:, None] * 2.0 ** -134 if op == "dw" else 0.0)


def test_two_streams_at_once():
    """Calls that overlap on two streams, a workspace each."""
    ps = [Problem(op, 777, 1024, 2048, seed=s) for s, op in enumerate(("linear", "dw"))]
    outs, wss = [p.output()[1] for p in ps], [p.workspace() for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(10):
        for p, y, ws, st in zip(ps, outs, wss, streams):
            with torch.cuda.stream(st):
                p.call(y, ws)
    torch.cuda.synchronize()
    for p, y in zip(ps, outs):
        p.check(y)


def test_the_stream_argument():
    p = Problem("linear", 5, 64, 128)
    _, y = p.output()
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    tmt_moe.mxfp4_linear(p.x, p.codes, p.scales, y, workspace=p.workspace(), stream=st)
    st.synchronize()
    p.check(y)


def test_more_rows_than_a_grid_dimension_of_blocks():
    """4.3 million tokens of the narrowest layer: more than 65535 blocks of rows."""
    T, N, K = 4_300_001, 16, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    X = torch.empty(T, K, dtype=BF16, device="cuda").normal_(generator=g)
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device="cuda", generator=g)
    scales = torch.randint(120, 130, (K // 32, N), dtype=torch.uint8, device="cuda", generator=g)
    Y = torch.full((T + 1, N), 7.0, dtype=BF16, device="cuda")
    size = tmt_moe.linear_workspace_size(tmt_moe.LINEAR_FORWARD, T, N, K)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda") if size else None
    tmt_moe.mxfp4_linear(X, codes, scales, Y[:T], workspace=ws)
    W = torch.empty(N, K, dtype=torch.float32, device="cuda")
    tmt_moe.mx_dequantize(codes, scales, W, FP4)
    for at in (0, 2_097_100, 4_194_200, T - 1000):
        x, w = X[at:at + 1000].double().cpu(), W.double().cpu()
        want, most = x @ w.T, x.abs() @ w.abs().T
        assert ((Y[at:min(at + 1000, T)].double().cpu() - want).abs() <= (K + 2) * 2.0 ** -23 * most + 2.0 ** -8 * want.abs()).all()
    assert (Y[T] == 7.0).all()


@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_no_tokens_over_a_large_matrix(beta):
    """dW = beta dW past one pass of the launch's workgroups, rows padded."""
    N, K, ld = 4112, 4160, 4164
    buf = torch.full((N + 1, ld), 3.0, device="cuda")
    dW = buf[:N, :K]
    if beta == 0.0:
        dW.fill_(float("nan"))
    dY = torch.empty(0, N, dtype=BF16, device="cuda")
    codes = torch.empty(0, K, dtype=torch.uint8, device="cuda")
    scales = torch.empty(K // 32, 16, dtype=torch.uint8, device="cuda")
    tmt_moe.mxfp8_linear_dw(dY, codes, scales, dW, beta=beta)
    assert (dW == 3.0 * beta).all()
    assert (buf[:N, K:] == 3.0).all() and (buf[N] == 3.0).all()


def test_a_strided_workspace_is_refused():
    X = torch.zeros(16, 64, dtype=BF16, device="cuda")
    codes = torch.zeros(16, 32, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(2, 16, dtype=torch.uint8, device="cuda")
    Y = torch.zeros(16, 16, dtype=BF16, device="cuda")
    ws = torch.zeros(64, 64, dtype=torch.uint8, device="cuda")[:, :32]
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        tmt_moe.mxfp4_linear(X, codes, scales, Y, workspace=ws)


@pytest.mark.parametrize("T,N,K,pad,beta", [
    (8192, 2048, 4096, 0, 0.0), (8100, 2000, 4096, 16, 0.5), (16300, 2000, 2048, 8, 0.0), (4081, 4080, 8192, 0, 0.0),
    (16384, 2048, 2048, 0, -1.0),
])
def test_large_matmul_tiles(T, N, K, pad, beta):
    """MXFP4 x MXFP4 on 256 x 256 tiles: one round and two, whole and ragged."""
    from launched_kernels import launched_kernels
    p = _run("matmul", T, N, K, pad=pad, beta=beta)
    ws, outs = p.workspace(), [p.output()[1] for _ in range(3)]
    names = launched_kernels(lambda: p.call(outs[0], ws))
    assert len(names) == 1 and "linear_mx_large_kernel" in names[0], names
    for y in outs:
        p.call(y, ws)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("op", OPS)
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_the_widest_rows(op, beta):
    """Row strides of 2^22 elements: offsets inside a tile close to 2^31 bytes."""
    T, N, K = 300, 256, 320
    _run(op, T, N, K, pad=(1 << 22) - K, beta=beta)
