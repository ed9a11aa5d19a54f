"""The root-mean-square norm with the residual's addition and 8-bit output, and its
backward, against 64 bits."""
import pytest
import torch

import fp8_ref as ref
import tmt_moe

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
# Additions that stand behind one another in a row's sum: 16 values of a lane, the
# butterfly's 6, 16 waves; each off by 2^-24 of the sum of magnitudes. The products,
# the mean, the root and the quotient add a few more.
ROW = (16 + 6 + 16 + 6) * 2.0 ** -24
OUT = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def _stream(t):
    return None if t is None else t.cuda()


def _inputs(T, d, stream, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, d, generator=g) * scale).to(BF16)
    r = (torch.randn(T, d, generator=g) * 3 * scale).to(stream)
    return x, r, 1 + 0.3 * torch.randn(d, generator=g)


def _check_codes(codes, scales, y, rstd_err):
    """codes and scales [d/128, T] against y in 64 bits."""
    T, d = y.shape
    pad = torch.zeros(T, ref.up(d, 128), dtype=torch.float64)
    pad[:, :d] = y.abs()
    m = pad.view(T, -1, 128).amax(2).clamp(min=2.0 ** -100)
    assert ((scales.double().t() - m / 448).abs() <= (m / 448) * (rstd_err + 2.0 ** -23)).all()
    s = ref.spread(scales, T, d, False)
    # half a step of a normal or a subnormal code, on a value off by the row's error
    tol = y.abs() * (2.0 ** -4 + 4 * (rstd_err + 2.0 ** -23)) + s * 2.0 ** -10
    assert ((codes.view(ref.FP8).double() * s - y).abs() <= tol).all()


WIDTHS = [1, 7, 8, 12, 17, 64, 127, 128, 129, 256, 500, 511, 512, 513, 1000, 1024, 1025, 1028, 1280, 2048, 2051, 4096, 4100,
          8192, 8200, 12345, 16384]


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("d", WIDTHS)
def test_forward(d, stream):
    """Every output at once, rows apart by more than their width, nothing outside written."""
    T = 5 if d > 2048 else 37
    x, r, gamma = _inputs(T, d, stream, d)
    s, rstd, y = ref.norm(x, r, gamma, 1e-5, stream)
    ld, ldc = ref.up(d, 8) + 8, ref.up(d, 16) + 16
    _, X = ref.padded(x.cuda(), ld, float("nan"))
    _, R = ref.padded(r.cuda(), ld, float("nan"))
    sb, S = ref.padded(torch.full((T, d), 7.0, dtype=stream, device="cuda"), ld, 5.0)
    yb, Y = ref.padded(torch.full((T, d), 7.0, dtype=BF16, device="cuda"), ld, 5.0)
    cb, C = ref.padded(torch.full((T, d), 99, dtype=torch.uint8, device="cuda"), ldc, 99)
    scales = torch.full((ref.blocks_of(d), T + 3), 5.0, device="cuda")
    rs = torch.full((T,), 5.0, device="cuda")
    tmt_moe.rmsnorm_forward(X, R, gamma.cuda(), S=S, Y=Y, codes=C, scales=scales, rstd=rs)
    assert torch.equal(S.cpu(), s)
    assert ((rs.cpu().double() - rstd).abs() <= rstd * ROW).all()
    assert ((Y.cpu().double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * ROW)).all()
    _check_codes(C.cpu(), scales[:, :T].cpu(), y, ROW + 2.0 ** -23)
    w16 = ref.up(d, 16)
    for buf in (sb, yb):
        assert (buf[0] == 5).all() and (buf[-1] == 5).all() and (buf[1:-1, d:] == 5).all()
    assert (cb[0] == 99).all() and (cb[-1] == 99).all() and (cb[1:-1, w16:] == 99).all()
    assert (cb[1:-1, d:w16] == 0).all()
    assert (scales[:, T:] == 5).all()


@pytest.mark.parametrize("T,d", [(1, 1024), (2, 1280), (777, 1280), (4099, 1024), (20001, 256), (1025, 4096)])
@pytest.mark.parametrize("stream", [BF16, F32])
def test_forward_many_rows(T, d, stream):
    x, r, gamma = _inputs(T, d, stream, T)
    s, rstd, y = ref.norm(x, r, gamma, 1e-6, stream)
    C = torch.empty(T, d, dtype=ref.FP8, device="cuda")
    scales, S = torch.empty(d // 128, T, device="cuda"), torch.empty(T, d, dtype=stream, device="cuda")
    Y, rs = torch.empty(T, d, dtype=BF16, device="cuda"), torch.empty(T, device="cuda")
    tmt_moe.rmsnorm_forward(x.cuda(), r.cuda(), gamma.cuda(), S=S, Y=Y, codes=C, scales=scales, rstd=rs, eps=1e-6)
    assert torch.equal(S.cpu(), s)
    assert ((Y.cpu().double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * ROW)).all()
    _check_codes(C.cpu().view(torch.uint8), scales.cpu(), y, ROW + 2.0 ** -23)


@pytest.mark.parametrize("which", ["X", "R bf16", "R fp32"])
def test_one_input(which):
    """The norm alone: the stream's first norm and its last."""
    x, r, gamma = _inputs(33, 384, F32 if which == "R fp32" else BF16)
    x, r = (x, None) if which == "X" else (None, r)
    s, rstd, y = ref.norm(x, r, gamma, 0.0, None)
    Y, rs = torch.empty(33, 384, dtype=BF16, device="cuda"), torch.empty(33, device="cuda")
    tmt_moe.rmsnorm_forward(_stream(x), _stream(r), gamma.cuda(), Y=Y, rstd=rs, eps=0.0)
    assert ((rs.cpu().double() - rstd).abs() <= rstd * ROW).all()
    assert ((Y.cpu().double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * ROW)).all()


@pytest.mark.parametrize("over", ["X", "R"])
@pytest.mark.parametrize("d", [1000, 2056])
def test_sum_in_place(over, d):
    """S takes the place of the sublayer's output or of the stream."""
    x, r, gamma = _inputs(29, d, BF16)
    s, _, y = ref.norm(x, r, gamma, 1e-5, BF16)
    X, R, Y = x.cuda(), r.cuda(), torch.empty(29, d, dtype=BF16, device="cuda")
    tmt_moe.rmsnorm_forward(X, R, gamma.cuda(), S=X if over == "X" else R, Y=Y)
    assert torch.equal((X if over == "X" else R).cpu(), s)
    assert ((Y.cpu().double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * ROW)).all()


def test_special_rows():
    """A row of zeros, of the smallest and of large values, with an infinity, with a NaN; its
    neighbours do not notice."""
    d = 256
    x, r, gamma = _inputs(7, d, BF16)
    x[1], r[1] = 0, 0
    x[2], r[2] = 2.0 ** -120, 0
    x[3], r[3] = 2.0 ** 59, 0
    x[4, 200] = float("inf")
    x[5, 3] = float("nan")
    C, sc = torch.empty(7, d, dtype=torch.uint8, device="cuda"), torch.empty(2, 7, device="cuda")
    Y, rs = torch.empty(7, d, dtype=BF16, device="cuda"), torch.empty(7, device="cuda")
    tmt_moe.rmsnorm_forward(x.cuda(), r.cuda(), gamma.cuda(), Y=Y, codes=C, scales=sc, rstd=rs)
    _, _, y = ref.norm(x, r, gamma, 1e-5, BF16)
    fine = [0, 1, 2, 3, 6]
    assert ((Y.cpu().double()[fine] - y[fine]).abs() <= y[fine].abs() * (2.0 ** -8 + 2 * ROW)).all()
    _check_codes(C.cpu()[fine], sc.cpu()[:, fine], y[fine], ROW + 2.0 ** -23)
    # an infinity: rstd is 0, so the row is 0 but for NaN at the infinity and in its block of codes
    assert rs[4] == 0 and torch.isnan(Y[4, 200]) and (Y[4, :200] == 0).all()
    assert torch.isnan(sc[1, 4]) and (C[4, 128:] == 0).all() and sc[0, 4].item() == (torch.tensor(2.0 ** -100) / 448).item()
    assert torch.isnan(Y[5]).all() and torch.isnan(sc[:, 5]).all() and (C[5] == 0).all()


def _backward(T, d, stream, with_dr, seed=0, in_place=False):
    g = torch.Generator().manual_seed(seed)
    s = (torch.randn(T, d, generator=g) * 3).to(stream)
    dy = (torch.randn(T, d, generator=g) * 1e-2).to(BF16)
    dr = (torch.randn(T, d, generator=g) * 1e-2).to(stream) if with_dr else None
    gamma = 1 + 0.3 * torch.randn(d, generator=g)
    rstd = (s.double().square().mean(1) + 1e-5).rsqrt().float()
    ds, dgamma, size, gsize = ref.norm_grad(dy, s, gamma, rstd, dr)
    ld = ref.up(d, 8) + 8
    _, DY = ref.padded(dy.cuda(), ld, float("nan"))
    _, S = ref.padded(s.cuda(), ld, float("nan"))
    ob, DS = ref.padded((dr if in_place else torch.zeros(T, d, dtype=stream)).cuda(), ld, 5.0)
    DR = DS if in_place else ref.padded(dr.cuda(), ld, float("nan"))[1] if with_dr else None
    gb = torch.full((d + 8,), 5.0, device="cuda")
    ws = torch.full((tmt_moe.rmsnorm_workspace_size(T, d),), 255, dtype=torch.uint8, device="cuda")
    tmt_moe.rmsnorm_backward(DY, S, gamma.cuda(), rstd.cuda(), DS, gb[:d], ws, dR=DR)
    tol = size * ROW + (ds.abs() + (0 if dr is None else dr.double().abs())) * 2.0 ** -23 + ds.abs() * OUT[stream]
    assert ((DS.cpu().double() - ds).abs() <= tol).all()
    # rows that a wave adds up one after another (1024 and more waves), the waves, the sums of workgroups
    seq = (T + 1023) // 1024 + 4 + 16 + 40
    assert ((gb[:d].cpu().double() - dgamma).abs() <= gsize * seq * 2.0 ** -24).all()
    assert (gb[d:] == 5).all() and (ob[0] == 5).all() and (ob[-1] == 5).all() and (ob[1:-1, d:] == 5).all()


@pytest.mark.parametrize("stream", [BF16, F32])
@pytest.mark.parametrize("with_dr", [False, True])
@pytest.mark.parametrize("d", WIDTHS)
def test_backward(d, with_dr, stream):
    _backward(5 if d > 2048 else 37, d, stream, with_dr, d)


@pytest.mark.parametrize("T,d,stream", [(1, 1024, BF16), (5003, 1000, BF16), (9001, 512, F32), (3000, 2048, F32), (700, 8192, BF16)])
def test_backward_many_rows(T, d, stream):
    _backward(T, d, stream, True, T)


@pytest.mark.parametrize("stream", [BF16, F32])
def test_backward_in_place(stream):
    _backward(300, 1032, stream, True, 3, in_place=True)


def test_backward_against_differences():
    """dS and dgamma against central differences of the formula, in 64 bits."""
    g = torch.Generator().manual_seed(1)
    T, d, h = 3, 24, 1e-4
    s, gamma = torch.randn(T, d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)
    dy = torch.randn(T, d, generator=g).to(BF16)
    rstd = (s.double().square().mean(1) + 1e-5).rsqrt()

    def loss(s, gamma):
        return (dy.double() * s * (s.square().mean(1) + 1e-5).rsqrt()[:, None] * gamma).sum()

    dS, dG = torch.empty(T, d, device="cuda"), torch.empty(d, device="cuda")
    ws = torch.empty(tmt_moe.rmsnorm_workspace_size(T, d), dtype=torch.uint8, device="cuda")
    tmt_moe.rmsnorm_backward(dy.cuda(), s.cuda(), gamma.cuda(), rstd.float().cuda(), dS, dG, ws)
    s64, g64 = s.double(), gamma.double()
    for i in range(T * d):
        e = torch.zeros(T * d, dtype=torch.float64)
        e[i] = h
        e = e.view(T, d)
        # third derivatives of s rstd are of the order of 10: h^2 * 10; the sums in fp32
        assert abs((loss(s64 + e, g64) - loss(s64 - e, g64)) / (2 * h) - dS.view(-1)[i].item()) < 1e-5
    for i in range(d):
        e = torch.zeros(d, dtype=torch.float64)
        e[i] = h
        assert abs((loss(s64, g64 + e) - loss(s64, g64 - e)) / (2 * h) - dG[i].item()) < 1e-5


def test_no_rows():
    x = torch.empty(0, 64, dtype=BF16, device="cuda")
    gamma, dgamma = torch.ones(64, device="cuda"), torch.full((64,), 5.0, device="cuda")
    tmt_moe.rmsnorm_forward(x, x, gamma, S=x, Y=x, codes=x.to(ref.FP8), scales=torch.empty(1, 0, device="cuda"))
    tmt_moe.rmsnorm_backward(x, x, gamma, torch.empty(0, device="cuda"), x, dgamma, None)
    assert (dgamma == 0).all()


@pytest.mark.parametrize("d", [1, 100, 1001])
def test_one_dense_row(d):
    """One row of any length needs no room behind it, but for the codes."""
    x, r, gamma = _inputs(1, d, F32, d)
    s, rstd, y = ref.norm(x, r, gamma, 1e-5, F32)
    S, Y, dS = torch.empty(1, d, device="cuda"), torch.empty(1, d, dtype=BF16, device="cuda"), torch.empty(1, d, device="cuda")
    C, sc = torch.empty(1, ref.up(d, 16), dtype=torch.uint8, device="cuda"), torch.empty(ref.blocks_of(d), 1, device="cuda")
    rs, dg = torch.empty(1, device="cuda"), torch.empty(d, device="cuda")
    ws = torch.empty(tmt_moe.rmsnorm_workspace_size(1, d), dtype=torch.uint8, device="cuda")
    tmt_moe.rmsnorm_forward(x.cuda(), r.cuda(), gamma.cuda(), S=S, Y=Y, codes=C[:, :d], scales=sc, rstd=rs)
    assert torch.equal(S.cpu(), s) and (C[:, d:] == 0).all()
    assert ((Y.cpu().double() - y).abs() <= y.abs() * (2.0 ** -8 + 2 * ROW)).all()
    _check_codes(C[:, :d].cpu(), sc.cpu(), y, ROW + 2.0 ** -23)
    tmt_moe.rmsnorm_backward(Y, S, gamma.cuda(), rs, dS, dg, ws)
    want = Y.cpu().double()[0] * S.cpu().double()[0] * rs.cpu().double()
    assert ((dg.cpu().double() - want).abs() <= want.abs() * 2.0 ** -22).all()  # two products, a sum of one term


@pytest.mark.parametrize("fn", ["forward", "backward"])
def test_repeats_and_captures(fn):
    """The same bits on another stream and from a graph's replays with new inputs."""
    T, d = 1500, 1160
    x, r, gamma = (t.cuda() for t in _inputs(T, d, BF16))
    ws = torch.empty(tmt_moe.rmsnorm_workspace_size(T, d), dtype=torch.uint8, device="cuda")
    rs = torch.rand(T, device="cuda") + 0.5

    def call(x, o, stream=None):
        if fn == "forward":
            tmt_moe.rmsnorm_forward(x, r, gamma, S=o[0], Y=o[1], codes=o[2], scales=o[3], rstd=o[4], stream=stream)
        else:
            tmt_moe.rmsnorm_backward(x, r, gamma, rs, o[0], o[5], ws, dR=r, stream=stream)

    def outs():
        return (torch.zeros_like(x), torch.zeros_like(x), torch.zeros(T, ref.up(d, 16), dtype=ref.FP8, device="cuda")[:, :d],
                torch.zeros(ref.blocks_of(d), T, device="cuda"), torch.zeros(T, device="cuda"), torch.zeros(d, device="cuda"))

    bits = lambda o: [t.contiguous().view(torch.uint8).clone() for t in o]  # noqa: E731
    side, a, b, c = torch.cuda.Stream(), outs(), outs(), outs()
    call(x, a)
    side.wait_stream(torch.cuda.current_stream())
    call(x, b, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(i, j) for i, j in zip(bits(a), bits(b)))
    graph, held = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        call(held, c)
    for k in range(3):
        held.copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        call(held, a)
        assert all(torch.equal(i, j) for i, j in zip(bits(a), bits(c)))


@pytest.mark.parametrize("T,d,stream", [(40000, 1024, F32), (40000, 1024, BF16), (9000, 512, BF16), (20000, 4096, BF16), (5000, 16000, F32)])
def test_large_calls_as_small_ones(T, d, stream):
    """A row's results do not depend on how many rows a call has, nor on how it passes memory:
    the same bits as in calls of 500 rows."""
    g = torch.Generator(device="cuda").manual_seed(T)
    X = torch.randn(T, d, device="cuda", generator=g).to(BF16)
    R = torch.randn(T, d, device="cuda", generator=g).to(stream)
    dY, gamma = torch.randn(T, d, device="cuda", generator=g).to(BF16), torch.randn(d, device="cuda", generator=g)

    def both(a, b):
        n = b - a
        S, C = torch.empty(n, d, dtype=stream, device="cuda"), torch.empty(n, d, dtype=torch.uint8, device="cuda")
        Y, rs = torch.empty(n, d, dtype=BF16, device="cuda"), torch.empty(n, device="cuda")
        sc = torch.empty(d // 128, n, device="cuda")
        tmt_moe.rmsnorm_forward(X[a:b], R[a:b], gamma, S=S, Y=Y, codes=C, scales=sc, rstd=rs)
        dS, dg = torch.empty(n, d, dtype=stream, device="cuda"), torch.empty(d, device="cuda")
        ws = torch.empty(tmt_moe.rmsnorm_workspace_size(n, d), dtype=torch.uint8, device="cuda")
        tmt_moe.rmsnorm_backward(dY[a:b], S, gamma, rs, dS, dg, ws, dR=R[a:b])
        return S, C, Y, rs, sc.t(), dS, dg

    whole = both(0, T)
    for a in range(0, T, 500):
        b = min(T, a + 500)
        for name, big, small in zip(("S", "codes", "Y", "rstd", "scales", "dS"), whole, both(a, b)):
            assert torch.equal(big[a:b], small), (name, a)
    # dgamma: no addition is off by more than 2^-24 of the sum of magnitudes, and no value
    # stands behind more than the rows of its lane (160 here), 16 rows of a workgroup and 1024
    # workgroups; the product adds 3 roundings
    dg, most = torch.zeros(d, dtype=torch.float64, device="cuda"), torch.zeros(d, dtype=torch.float64, device="cuda")
    for a in range(0, T, 500):
        t = dY[a:a + 500].double() * whole[0][a:a + 500].double() * whole[3][a:a + 500].double()[:, None]
        dg, most = dg + t.sum(0), most + t.abs().sum(0)
    assert ((whole[6].double() - dg).abs() <= most * (160 + 16 + 1024 + 3) * 2.0 ** -24).all()


@pytest.mark.parametrize("d", [1024, 1280, 100])
@pytest.mark.parametrize("stream", [BF16, F32])
def test_codes_of_64_bits(d, stream):
    """No code above e4m3's subnormals goes another way than that of the norm in 64 bits."""
    T = (1 << 24) // d
    g = torch.Generator(device="cuda").manual_seed(d)
    ld = ref.up(d, 8)
    X = torch.randn(T, ld, device="cuda", generator=g).to(BF16)[:, :d]
    R = (3 * torch.randn(T, ld, device="cuda", generator=g)).to(stream)[:, :d]
    gamma = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    C = torch.empty(T, ref.up(d, 16), dtype=torch.uint8, device="cuda")[:, :d]
    scales, S = torch.empty(ref.blocks_of(d), T, device="cuda"), torch.empty(T, ld, dtype=stream, device="cuda")[:, :d]
    tmt_moe.rmsnorm_forward(X, R, gamma, S=S, codes=C, scales=scales)
    s = S.double()
    y = s * (s.square().mean(1, keepdim=True) + float(torch.tensor(1e-5))) ** -0.5 * gamma.double()
    for c in range(0, d, 128):
        q = y[:, c:c + 128]
        q = q * 448 / q.abs().amax(1, keepdim=True)
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)  # no |q| is a power of 2 but by chance
        want = torch.round(q / step) * step
        got = C[:, c:c + 128].contiguous().view(ref.FP8).double()
        assert torch.equal(got[q.abs() >= 2.0 ** -6], want[q.abs() >= 2.0 ** -6])
