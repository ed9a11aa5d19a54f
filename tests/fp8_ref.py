"""Blocks of e4m3 codes with fp32 scales, and the norm in front of them, restated
for the tests: quantisation operation by operation in fp32 (it is exact to the bit),
everything else in 64 bits."""
import torch

BLOCK = 128
FP8 = torch.float8_e4m3fn


def up(n, of):
    return (n + of - 1) // of * of


def blocks_of(n):
    return (n + BLOCK - 1) // BLOCK


def padded(t, ld, fill=0):
    """A view of t's values in rows of `ld`, a row in front and behind; `fill` outside."""
    buf = torch.full((t.shape[0] + 2, ld), fill, dtype=t.dtype, device=t.device)
    view = buf[1:t.shape[0] + 1, :t.shape[1]]
    view.copy_(t)
    return buf, view


def quantize(x, tiles):
    """(codes, uint8 [rows, K], scales) of x (CPU, bf16 or fp32)."""
    x = x.float()
    rows, K = x.shape
    h = BLOCK if tiles else 1
    b = torch.zeros(up(rows, h), up(K, BLOCK))
    b[:rows, :K] = x
    b = b.view(up(rows, h) // h, h, -1, BLOCK)
    m = b.abs().amax((1, 3), keepdim=True)
    bad = ~torch.isfinite(m) | torch.isnan(b).any(3, keepdim=True).any(1, keepdim=True)
    m = m.clamp(min=2.0 ** -100)
    q = torch.where(bad, torch.zeros_like(b), b * (torch.tensor(448.0) / m)).to(FP8).view(torch.uint8)
    s = torch.where(bad, torch.full_like(m, float("nan")), m / torch.tensor(448.0)).view(b.shape[0], b.shape[2])
    q = q.view(-1, b.shape[2] * BLOCK)[:rows, :K].contiguous()
    return q, s if tiles else s.t().contiguous()


def spread(scales, rows, K, tiles):
    """A scale for every value, 64 bits."""
    s = scales.double()
    if tiles:
        return s.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :K]
    return s.t()[:rows].repeat_interleave(BLOCK, 1)[:, :K]


def values(codes, scales, tiles):
    return codes.view(FP8).double() * spread(scales, *codes.shape, tiles)


def norm(x, r, gamma, eps, stream):
    """(S in its type, rstd, y), the latter two in 64 bits."""
    if r is None:
        s = x
    elif x is None:
        s = r
    else:
        s = (x.float() + r.float()).to(stream)
    w = s.double()
    rstd = (w.square().mean(1) + eps).rsqrt()
    return s, rstd, w * rstd[:, None] * gamma.double()


def norm_grad(dy, s, gamma, rstd, dr):
    """dS and dgamma, and the magnitudes that their roundings are relative to."""
    dy, w, g, r = dy.double(), s.double(), gamma.double(), rstd.double()[:, None]
    gg, xh = dy * g, w * r
    c = (gg * xh).mean(1, keepdim=True)
    ds = r * (gg - xh * c)
    size = r * (gg.abs() + xh.abs() * (gg * xh).abs().mean(1, keepdim=True))
    if dr is not None:
        ds = ds + dr.double()
    return ds, (dy * xh).sum(0), size, (dy * xh).abs().sum(0)
