"""The products of the microscaled linear layer bit for bit.

Operands whose sums fp32 holds exactly (linear_exact.py) leave one right result
however long the reduction and however it is split, so there is no tolerance: a
lost step or tail, a sum or partial sum in fewer bits, a second rounding show.
Long reductions, outputs that are added to and wide rows reach every kernel,
the 256 x 256 tiles among them; each case names the kernels it must launch.
"""
import numpy as np
import pytest
import torch

import linear_exact
import mx_ref
import tmt_moe

pytestmark = pytest.mark.gpu

BF16, U8 = torch.bfloat16, torch.uint8
SIZE_OP = {"linear": tmt_moe.LINEAR_FORWARD, "matmul": tmt_moe.LINEAR_MATMUL, "dx": tmt_moe.LINEAR_DX,
           "dw": tmt_moe.LINEAR_DW}
ROWS_MAX = 1 << 22  # the widest row stride, in elements


def _up16(n):
    return max(16, (n + 15) // 16 * 16)


def _padded(t, ld, fill):
    """A view of t's values in rows of stride ld, one row in front and behind,
    `fill` outside."""
    buf = torch.full((t.shape[0] + 2, ld), fill, dtype=t.dtype, device="cuda")
    view = buf[1:t.shape[0] + 1, :t.shape[1]]
    view.copy_(t)
    return buf, view


def _scales(s, lds):
    """[K/32, rows] scales in rows of lds; past the last one NaN's byte."""
    out = torch.full((s.shape[0], lds), 255, dtype=U8, device="cuda")
    out[:, :s.shape[1]] = s
    return out


def _kernels(call):
    from launched_kernels import launched_kernels
    return launched_kernels(call)


class Call:
    """A product's operands on the device, its output with guards, the call."""

    def __init__(self, op, T, N, K, p, ldx=None, ldy=None, spare=0, beta=0.0, old=None):
        self.op = op
        mx_rows = T if op == "dw" else N
        self.w = (p["w"][0], _scales(p["w"][1], _up16(mx_rows) + spare))
        if op == "matmul":
            self.x = (p["x"][0], _scales(p["x"][1], _up16(T) + spare))
        else:
            _, self.x = _padded(p["x"], ldx or p["x"].shape[1], float("nan"))
        rows, cols = {"linear": (T, N), "matmul": (T, N), "dx": (T, K), "dw": (N, K)}[op]
        start = old if old is not None else torch.full((rows, cols), float("nan"), device="cuda")
        self.buf, self.y = _padded(start.to(torch.float32 if op == "dw" else BF16), ldy or cols, 5.0)
        size = tmt_moe.linear_workspace_size(SIZE_OP[op], T, N, K)
        self.ws = torch.full((size,), 255, dtype=U8, device="cuda") if size else None
        self.beta = beta

    def __call__(self):
        if self.op == "matmul":
            tmt_moe.mxfp4_matmul(*self.x, *self.w, self.y, beta=self.beta, workspace=self.ws)
        else:
            fn = {"linear": tmt_moe.mxfp4_linear, "dx": tmt_moe.mxfp4_linear_dx, "dw": tmt_moe.mxfp8_linear_dw}[self.op]
            fn(self.x, *self.w, self.y, beta=self.beta, workspace=self.ws)

    def guards(self):
        return bool((self.buf[0] == 5).all() and (self.buf[-1] == 5).all() and (self.buf[1:-1, self.y.shape[1]:] == 5).all())


def _check(op, T, N, K, kernels, pad=0, beta=0.0, ldx=None, ldy=None, signed=(False, True)):
    for sign in signed:
        p = linear_exact.operands(op, T, N, K, seed=5, signed=sign, device="cuda")
        exact = linear_exact.product(op, p["A"], p["B"])
        old = None
        if beta != 0.0:  # multiples of 4 that bf16 holds: beta times them is a whole number
            gen = torch.Generator(device="cuda").manual_seed(T + N)
            old = 4 * torch.randint(-63, 64, tuple(exact.shape), generator=gen, device="cuda").double()
            exact = exact + beta * old
        want = linear_exact.rounded(op, exact)
        del exact
        cols = want.shape[1]
        c = Call(op, T, N, K, p, ldx=ldx or (p["x"].shape[1] + pad if op != "matmul" else None), ldy=ldy or cols + pad,
                 spare=16 * (pad > 0), beta=beta, old=old)
        c()
        bad = (c.y != want).nonzero()
        assert bad.numel() == 0, (len(bad), bad[0].tolist(), float(c.y[tuple(bad[0])]), float(want[tuple(bad[0])]))
        assert c.guards()
    names = _kernels(c)
    assert len(names) == len(kernels) and all(k in n for k, n in zip(kernels, names)), names


def _fwd(tile, split, beta):
    return f"linear_fwd_kernelILi{tile}ELb{split}ELb{beta}E"


def _grad(op, tile, split, beta):
    return f"linear_grad_kernelILi{2 if op == 'dx' else 3}ELi{tile}ELb{split}ELb{beta}E"


def _mx(split, full, beta):
    return f"linear_mx_kernelILb{split}ELb{full}ELb{beta}E"


def _sums(tile, f32):
    return f"linear_fixup_kernelILi{tile}ELb{f32}E"


@pytest.mark.parametrize("op,T,N,K,pad,beta,kernels", [
    ("linear", 1, 4096, 1024, 8, 0.5, ["linear_rows_kernelILi1ELi1ELi8ELi1E"]),
    ("linear", 600, 1280, 1024, 0, -1.0, ["linear_rows_kernelILi4ELi2ELi4ELi1E"]),
    ("linear", 777, 4096, 1024, 8, 0.5, [_fwd(128, 0, 1)]),
    ("linear", 777, 1024, 4096, 8, 0.5, [_fwd(128, 1, 0), _sums(128, 0)]),
    ("linear", 16300, 4000, 1024, 0, 0.0, [_fwd(256, 0, 0)]),
    ("linear", 16300, 4000, 1024, 8, 0.5, [_fwd(256, 0, 1)]),
    ("linear", 17900, 1008, 4096, 8, -1.0, [_fwd(256, 0, 1), _fwd(256, 1, 0), _sums(256, 0)]),
    ("matmul", 777, 4096, 1024, 8, 0.5, [_mx(0, 1, 1)]),
    ("matmul", 777, 4096, 960, 8, -1.0, [_mx(0, 0, 1)]),
    ("matmul", 128, 256, 8128, 8, 0.5, [_mx(1, 0, 0), _sums(128, 0)]),
    ("matmul", 777, 1024, 4096, 0, 0.0, [_mx(1, 1, 0), _sums(128, 0)]),
    ("matmul", 8100, 2000, 4096, 16, 0.5, ["linear_mx_large_kernelILb1E"]),
    ("dx", 1024, 256, 256, 8, 0.5, [_grad("dx", 128, 0, 1)]),
    ("dx", 777, 4096, 1024, 8, -1.0, [_grad("dx", 128, 1, 0), _sums(128, 0)]),
    ("dx", 16300, 1040, 4032, 0, 0.0, [_grad("dx", 256, 0, 0)]),
    ("dx", 16300, 1040, 4032, 8, 0.5, [_grad("dx", 256, 0, 1)]),
    ("dx", 17900, 4080, 960, 8, 0.5, [_grad("dx", 256, 0, 1), _grad("dx", 256, 1, 0), _sums(256, 0)]),
    ("dw", 127, 1040, 1024, 8, 0.5, [_grad("dw", 128, 0, 1)]),
    ("dw", 2047, 1280, 1280, 8, -1.0, [_grad("dw", 128, 1, 0), _sums(128, 1)]),
    ("dw", 40001, 1024, 256, 0, 0.0, [_grad("dw", 128, 1, 0), _sums(128, 1)]),
    ("dw", 4001, 4080, 4032, 0, 0.0, [_grad("dw", 256, 0, 0)]),
    ("dw", 4001, 4080, 4032, 8, 0.5, [_grad("dw", 256, 0, 1)]),
    ("dw", 16383, 4080, 1024, 8, 0.5, [_grad("dw", 256, 1, 0), _sums(256, 1)]),
    ("dw", 40001, 1024, 1024, 8, -1.0, [_grad("dw", 256, 1, 0), _sums(256, 1)]),
])
def test_bit_for_bit(op, T, N, K, pad, beta, kernels):
    _check(op, T, N, K, kernels, pad, beta)


@pytest.mark.parametrize("op,T,N,K,kernels", [
    ("linear", 513, 4096, 1024, _fwd(128, 0, 0)),
    ("linear", 256, 65536, 1024, _fwd(256, 0, 0)),
    ("matmul", 256, 65536, 4096, "linear_mx_large_kernelILb0E"),
    ("dx", 256, 512, 65536, _grad("dx", 256, 0, 0)),
    ("dw", 512, 256, 65536, _grad("dw", 256, 0, 0)),
])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_the_widest_strides(op, T, N, K, kernels, beta):
    """Rows 2^22 elements apart in every matrix that has a stride: 256 rows of a
    tile are 2^31 bytes of bf16, 128 rows of a wave's fp32 outputs too."""
    kernels = [kernels] if beta == 0.0 else [kernels[:-2] + "1E"]
    _check(op, T, N, K, kernels, beta=beta, ldx=None if op == "matmul" else ROWS_MAX, ldy=ROWS_MAX, signed=(True,))


# ---- every code at every scale ---------------------------------------------------

_E2M1 = mx_ref.E2M1
_E4M3 = mx_ref.E4M3


def _value(table, codes, scales):
    """Codes and scale bytes as the products take them: in bf16, to nearest, which
    is exact but for e4m3's at scale bytes below 3; past bf16's range infinite."""
    v = table[codes] * mx_ref.e8m0(scales)
    with np.errstate(over="ignore"):
        return torch.from_numpy(v.astype(np.float32)).to(BF16).cuda()


def _same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0, posinf=3.0, neginf=-3.0),
                                                             b.nan_to_num(nan=0.0, posinf=3.0, neginf=-3.0))


@pytest.mark.parametrize("op,T,K,kernel", [
    ("linear", 1, 64, "linear_rows_kernel"), ("linear", 777, 1024, _fwd(128, 0, 0)), ("linear", 16384, 1024, _fwd(256, 0, 0)),
    ("matmul", 16, 64, _mx(0, 0, 0)), ("matmul", 777, 1024, _mx(0, 1, 0)), ("matmul", 8192, 4096, "linear_mx_large_kernelILb0E"),
])
def test_every_weight_at_every_scale(op, T, K, kernel):
    """A row of the weights for each code and scale byte, all its other codes
    zero, times ones: the outputs are the values."""
    N = 4096
    n = np.arange(N)
    s, c = n // 16, n % 16
    at = np.random.Generator(np.random.PCG64(K)).integers(K, size=N)
    codes = np.zeros((N, K), np.uint8)
    codes[n, at] = c
    scales = np.full((K // 32, N), 127, np.uint8)
    scales[at // 32, n] = s
    p = dict(w=(torch.from_numpy(codes[:, 0::2] | codes[:, 1::2] << 4).cuda(), torch.from_numpy(scales).cuda()))
    if op == "matmul":
        p["x"] = (torch.full((T, K // 2), 0x22, dtype=U8, device="cuda"), torch.full((K // 32, T), 127, dtype=U8, device="cuda"))
    else:
        p["x"] = torch.ones(T, K, dtype=BF16, device="cuda")
    call = Call(op, T, N, K, p)
    call()
    want = _value(_E2M1, c, s)
    assert torch.isfinite(want[16 * 120:16 * 130]).all() and want[16 * 255:].isnan().all()
    assert _same(call.y, want.expand(T, N))
    assert kernel in _kernels(call)[0]


@pytest.mark.parametrize("T,kernel", [(64, _grad("dx", 128, 0, 0)), (16384, _grad("dx", 256, 0, 0))])
def test_every_weight_at_every_scale_backward(T, kernel):
    """dX: row n of the weights is zero but for block n, which holds all codes at
    scale byte n."""
    N, K = 256, 8192
    c = np.arange(32) % 16
    codes = np.zeros((N, K), np.uint8)
    scales = np.full((K // 32, N), 127, np.uint8)
    for n in range(N):
        codes[n, 32 * n:32 * n + 32] = c
        scales[n, n] = n
    p = dict(w=(torch.from_numpy(codes[:, 0::2] | codes[:, 1::2] << 4).cuda(), torch.from_numpy(scales).cuda()),
             x=torch.ones(T, N, dtype=BF16, device="cuda"))
    call = Call("dx", T, N, K, p)
    call()
    want = _value(_E2M1, np.tile(c, N), np.repeat(np.arange(N), 32))
    assert _same(call.y, want.expand(T, K))
    assert kernel in _kernels(call)[0]


@pytest.mark.parametrize("N,kernel", [(16, _grad("dw", 128, 0, 0)), (2048, _grad("dw", 256, 0, 0))])
def test_every_checkpoint_value_at_every_scale(N, kernel):
    """dW: row t of the checkpoint is zero but for 256 columns, which hold all
    codes at scale byte t."""
    T, K = 256, 65536
    codes = np.zeros((T, K), np.uint8)
    scales = np.full((K // 32, T), 127, np.uint8)
    for t in range(T):
        codes[t, 256 * t:256 * t + 256] = np.arange(256)
        scales[8 * t:8 * t + 8, t] = t
    p = dict(w=(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()), x=torch.ones(T, N, dtype=BF16, device="cuda"))
    call = Call("dw", T, N, K, p)
    call()
    want = _value(_E4M3, np.tile(np.arange(256), T), np.repeat(np.arange(T), 256)).float()
    assert _same(call.y, want.expand(N, K))
    assert kernel in _kernels(call)[0]


# ---- rows ---------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", [mx_ref.FP4, mx_ref.FP8])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_the_widest_row(fmt, dtype):
    """One row of 2^31 - 32 columns, the most that 32 bits hold: to codes and back."""
    K = 2 ** 31 - 32
    gen = torch.Generator(device="cuda").manual_seed(fmt)
    X = torch.empty(1, K, dtype=dtype, device="cuda").normal_(generator=gen)
    codes = torch.full((1, K // 2 if fmt == mx_ref.FP4 else K), 0xA5, dtype=U8, device="cuda")
    scales = torch.full((K // 32, 1), 0xA5, dtype=U8, device="cuda")
    tmt_moe.mx_quantize(X, codes, scales, fmt)
    back = torch.full((1, K), float("nan"), dtype=dtype, device="cuda")
    tmt_moe.mx_dequantize(codes, scales, back, fmt)
    n = 1 << 16
    for at in (0, 2 ** 30 - 64, 2 ** 31 - 512 - n, K - n):
        c, s = mx_ref.quantize(X[:, at:at + n].float().cpu().numpy(), fmt)
        per = 2 if fmt == mx_ref.FP4 else 1
        assert np.array_equal(codes[:, at // per:(at + n) // per].cpu().numpy(), c)
        assert np.array_equal(scales[at // 32:(at + n) // 32].cpu().numpy().T, s)
        want = torch.from_numpy(mx_ref.dequantize(c, s, fmt).astype(np.float32)).to(dtype)
        assert torch.equal(back[:, at:at + n].cpu(), want)
    assert bool(back.isfinite().all())
