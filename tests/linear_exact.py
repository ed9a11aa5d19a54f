"""Operands of the microscaled linear layer whose products fp32 holds exactly.

Every value is a whole number of halves and the magnitudes of a sum's terms add
up to less than 2^24 of its smallest unit, so every partial sum in any order is
exact in fp32, and the result is known to the last bit however long the
reduction is. The terms are as large as that allows: sums of one sign fill the
24 bits, so one that is held in fewer, or that lacks a term, differs.
"""
import torch

OPS = ("linear", "matmul", "dx", "dw")
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# e4m3 codes of 0 .. 7
_E4M3_INTS = (0x00, 0x38, 0x40, 0x44, 0x48, 0x4A, 0x4C, 0x4E)


def _draw(gen, shape, n):
    return torch.randint(0, n, shape, generator=gen, device=gen.device)


def _fp4(gen, rows, K, spread, signed):
    """(packed codes, scale bytes [K/32, rows], values in 64 bits)."""
    codes = _draw(gen, (rows, K), 16 if signed else 8)
    scales = 127 + _draw(gen, (K // 32, rows), spread)
    values = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=gen.device)[codes]
    values = values * (2.0 ** (scales - 127).double()).t().repeat_interleave(32, dim=1)
    packed = (codes[:, 0::2] + 16 * codes[:, 1::2]).to(torch.uint8)
    return packed, scales.to(torch.uint8), values


def _fp8(gen, rows, K, spread, signed):
    ints = _draw(gen, (rows, K), 8)
    sign = _draw(gen, (rows, K), 2) if signed else torch.zeros_like(ints)
    scales = 127 + _draw(gen, (K // 32, rows), spread)
    codes = torch.tensor(_E4M3_INTS, device=gen.device)[ints] + 128 * sign
    values = (ints * (1 - 2 * sign)).double() * (2.0 ** (scales - 127).double()).t().repeat_interleave(32, dim=1)
    return codes.to(torch.uint8), scales.to(torch.uint8), values


def operands(op, T, N, K, seed=0, signed=False, device="cpu"):
    """dict: A, B (values in 64 bits, as `product` takes them), x (bf16 matrix,
    or (codes, scales) of MATMUL), w (codes, scales). Scales are [K/32, rows]."""
    gen = torch.Generator(device=device).manual_seed(seed + 131 * T + 7 * N + K)
    R = {"linear": K, "matmul": K, "dx": N, "dw": T}[op]
    if op == "matmul":
        # 12 2^(a - 1 + b - 1) 12 R of quarters, below 2^24
        a, b = next((a, b) for a, b in ((6, 6), (5, 5), (4, 4), (3, 3), (2, 2), (2, 1), (1, 1))
                    if R * 36 * 2 ** (a + b - 2) * 4 < 2 ** 24 - 2 ** 12)
        xc, xs, A = _fp4(gen, T, K, a, signed)
        wc, ws, B = _fp4(gen, N, K, b, signed)
        return dict(A=A, B=B, x=(xc, xs), w=(wc, ws))
    if op == "dw":
        wc, ws, B = _fp8(gen, T, K, 2, signed)
        most, unit = 14, 1.0
    else:
        wc, ws, B = _fp4(gen, N, K, 2, signed)
        most, unit = 12, 0.5
    top = min(255, int((2 ** 24 - 2 ** 12) * unit / (most * R)))
    assert top >= 1, "the reduction is too long for this test"
    A = _draw(gen, (T, K if op == "linear" else N), top + 1).double()
    if signed:
        A = A * (1 - 2 * _draw(gen, tuple(A.shape), 2)).double()
    return dict(A=A, B=B, x=A.to(torch.bfloat16), w=(wc, ws))


def product(op, A, B):
    """The operator's product in the operands' own type."""
    if op in ("linear", "matmul"):
        return A @ B.t()
    return A @ B if op == "dx" else A.t() @ B


def rounded(op, exact):
    """What the kernel returns for the exact sums: fp32 holds them, one rounding
    to the output's type."""
    once = exact.float()
    assert torch.equal(once.double(), exact), "a sum is not exact in fp32"
    return once if op == "dw" else once.to(torch.bfloat16)
