"""That comparing exact products bit for bit notices what it is meant to. The
mistakes are planted in the reference, on the CPU."""
import pytest
import torch

import linear_exact
import mx_ref

SHAPES = {"linear": (40, 64, 4096), "matmul": (40, 64, 4096), "dx": (40, 1024, 64), "dw": (40001, 64, 64)}


@pytest.mark.parametrize("signed", [False, True])
@pytest.mark.parametrize("op", linear_exact.OPS)
def test_the_codes_stand_for_the_values(op, signed):
    T, N, K = 40, 32, 128
    p = linear_exact.operands(op, T, N, K, seed=3, signed=signed)
    fmt = mx_ref.FP8 if op == "dw" else mx_ref.FP4
    assert (mx_ref.dequantize(p["w"][0].numpy(), p["w"][1].numpy().T, fmt) == p["B"].numpy()).all()
    if op == "matmul":
        assert (mx_ref.dequantize(p["x"][0].numpy(), p["x"][1].numpy().T, fmt) == p["A"].numpy()).all()
    else:
        assert (p["x"].double() == p["A"]).all()


@pytest.mark.parametrize("op", linear_exact.OPS)
def test_any_order_of_the_sum_is_exact(op):
    """fp32 in one chain, and in parts added afterwards."""
    T, N, K = SHAPES[op]
    for signed in (False, True):
        p = linear_exact.operands(op, T, N, K, seed=1, signed=signed)
        exact = linear_exact.product(op, p["A"], p["B"])
        once = linear_exact.rounded(op, exact)
        whole = linear_exact.product(op, p["A"].float(), p["B"].float())
        assert torch.equal(whole.double(), exact)
        parts = _parts(op, p, 8)
        total = parts[0]
        for q in parts[1:]:
            total = total + q
        assert torch.equal(total.double(), exact)
        assert once.dtype is (torch.float32 if op == "dw" else torch.bfloat16)


def _reduction(op, p):
    """Both operands with the reduction as dimension 0."""
    if op in ("linear", "matmul"):
        return p["A"].t().float(), p["B"].t().float()
    return (p["A"].t().float(), p["B"].float()) if op == "dx" else (p["A"].float(), p["B"].float())


def _parts(op, p, n):
    a, b = _reduction(op, p)
    step = -(-a.shape[0] // n)
    return [a[i:i + step].t() @ b[i:i + step] for i in range(0, a.shape[0], step)]


def _cut(x, bits):
    """x to `bits` significant bits, to nearest."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2 ** bits), e - bits)


@pytest.mark.parametrize("op", linear_exact.OPS)
def test_mistakes_are_noticed(op):
    T, N, K = SHAPES[op]
    p = linear_exact.operands(op, T, N, K, seed=2)
    want = linear_exact.rounded(op, linear_exact.product(op, p["A"], p["B"]))
    a, b = _reduction(op, p)
    R = a.shape[0]

    def differs(total):
        got = linear_exact.rounded(op, total.float().double())
        return (got != want).double().mean()

    # every comparison is of all outputs, so one that differs is enough; the
    # shares below say how plain the mistake is
    clear = 0.5 if op == "dw" else 0.01  # fp32 outputs, bf16 outputs
    assert differs(a.t() @ b) == 0
    for lost in (256, 64, R % 64 or 16):  # a split's last steps, one step, a ragged tail
        assert differs(a[:R - lost].t() @ b[:R - lost]) > 0.5, lost
    assert differs(a[:R - 1].t() @ b[:R - 1]) > clear  # one row
    parts = _parts(op, p, 8)  # partial sums in bf16; partial sums and the sum in fewer bits
    assert differs(sum(q.to(torch.bfloat16).float() for q in parts)) > clear
    if op == "dw":
        assert differs(sum(_cut(q, 16) for q in parts)) > clear
        assert differs(_cut(sum(parts), 20)) > clear
    swapped = a.clone()  # a row in its neighbour's place
    swapped[R // 2] = a[R // 2 - 1]
    assert differs(swapped.t() @ b) > clear
