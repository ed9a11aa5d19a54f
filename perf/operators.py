"""Performance cases of the linear layer on microscaled (MX) numbers.

Blocks of 32 values along a row share one power-of-two scale (an e8m0 byte s,
2^(s - 127)). MXFP4 holds e2m1 codes, two a byte, the low nibble first; MXFP8
holds e4m3 codes. Scales lie block-major, [K/32][rows rounded up to 16].

Kinds of work, one operator each:

  quantize  rows to codes and scales and back to the values they stand for:
            expert weights after an optimizer step, activation checkpoints;
  linear    Y = X W^T with bf16 activations and MXFP4 weights: serving;
  matmul    the same with the activations rounded to MXFP4 in the pass too;
  dx        dX = dY W, the gradient at the layer's input;
  dw        dW = dY^T X from X kept as an MXFP8 checkpoint, in fp32.

Sizes are those of ``synthetic.CONFIGS``, of TMT's default width and of the
reference's profile shape. Activations are N(0, 1) with rows of different
scale, weights N(0, 1/sqrt(fan_in)), made on the GPU from the seed alone.
"""
import math
import os
import sys

import torch

own = False

MXFP4, MXFP8 = "mxfp4", "mxfp8"


def listed():
    return [
        # One expert's fp32 masters to MXFP4 after an optimizer step.
        {"name": "quantize_expert", "kind": "quantize", "format": MXFP4, "dtype": "fp32", "rows": 4096, "K": 1024},
        # The input of a large training step kept in 8 bits for the backward.
        {"name": "checkpoint_batch", "kind": "quantize", "format": MXFP8, "dtype": "bf16", "rows": 32768, "K": 1024},
        # Sampling one stream: the smallest call there is.
        {"name": "linear_decode_1", "kind": "linear", "T": 1, "N": 4096, "K": 1024},
        # A serving step over 64 streams, down-projection.
        {"name": "linear_decode_64", "kind": "linear", "T": 64, "N": 1024, "K": 4096},
        # A prompt of ragged length.
        {"name": "linear_prompt_777", "kind": "linear", "T": 777, "N": 4096, "K": 1024},
        # A large evaluation batch.
        {"name": "linear_batch", "kind": "linear", "T": 16384, "N": 4096, "K": 1024},
        # A ragged prompt with the activations in 4 bits as well.
        {"name": "matmul_prompt_777", "kind": "matmul", "T": 777, "N": 1024, "K": 4096},
        # The largest evaluation batch, activations in 4 bits.
        {"name": "matmul_batch", "kind": "matmul", "T": 65536, "N": 4096, "K": 1024},
        # A training step's layer at TMT's default width (batch 8 x 128 tokens).
        {"name": "dx_default_width", "kind": "dx", "T": 1024, "N": 256, "K": 256},
        # The input gradient of the large model's up-projection.
        {"name": "dx_batch", "kind": "dx", "T": 32768, "N": 4096, "K": 1024},
        # The weight gradient at the reference's profile shape.
        {"name": "dw_profile_shape", "kind": "dw", "T": 2048, "N": 1280, "K": 1280},
        # The weight gradient of the large model's up-projection.
        {"name": "dw_batch", "kind": "dw", "T": 32768, "N": 4096, "K": 1024},
    ]


_LARGEST = 65536 * 4096 * 1024  # T N K of the largest listed case


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _multiple(rng, lo, hi, of):
    return max(of, (_log(rng, lo, hi) + of // 2) // of * of)


def draw(rng):
    pick = rng.random()
    if pick < 0.2:
        K = _multiple(rng, 64, 4096, 32)
        fmt = rng.choice((MXFP4, MXFP8))
        return {"kind": "quantize", "format": fmt, "dtype": rng.choice(("fp32", "bf16")),
                "rows": _log(rng, 1, min(65536, (1 << 26) // K)), "K": K}
    kind = "linear" if pick < 0.5 else "matmul" if pick < 0.65 else "dx" if pick < 0.82 else "dw"
    N, K = _multiple(rng, 64, 4096, rng.choice((16, 64))), _multiple(rng, 64, 4096, 64)
    low = {"linear": 1, "matmul": 16, "dx": 64, "dw": 64}[kind]
    if kind == "linear" and rng.random() < 0.4:  # serving steps
        return {"kind": kind, "T": _log(rng, 1, 128), "N": N, "K": K}
    return {"kind": kind, "T": _log(rng, low, min(65536, _LARGEST // (4 * N * K))), "N": N, "K": K}


# ---- the numbers -------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exponent(amax, fmt):
    """The blocks' exponents. MXFP4: floor(log2 amax) - 2. MXFP8: the smallest e with amax <= 448 * 2^e."""
    frac, ex = torch.frexp(amax)  # amax = frac * 2^ex, frac in [0.5, 1)
    e = ex.int() - 3 if fmt == MXFP4 else ex.int() - 9 + (frac > 0.875).int()
    return torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e))


def _round4(a):
    """Index of the e2m1 magnitude nearest to a >= 0, ties to the even index, saturating."""
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=a.device)
    low, high = torch.bucketize(a, bounds), torch.bucketize(a, bounds, right=True)
    return torch.where(low % 2 == 0, low, high)


def _round8(a):
    """The e4m3 magnitude nearest to a in [0, 448], ties to even."""
    step = torch.ldexp(torch.ones_like(a), (torch.frexp(a)[1] - 1).clamp(min=-6) - 3)
    return torch.round(a / step) * step


def _rounded(x, fmt):
    """x [rows, K] rounded to the format: (magnitude [rows, K/32, 32], sign, exponent [rows, K/32]) in 32 bits."""
    rows, K = x.shape
    b = x.float().view(rows, K // 32, 32)
    e = _exponent(b.abs().amax(2), fmt)
    a = torch.ldexp(b.abs(), -e[:, :, None])
    return _round4(a) if fmt == MXFP4 else _round8(a), torch.signbit(b), e


def _values(x, fmt):
    """The values that x stands for in the format, 32 bits [rows, K]."""
    q, neg, e = _rounded(x, fmt)
    if fmt == MXFP4:
        q = torch.tensor(_E2M1, device=x.device)[q]
    v = torch.ldexp(q, e[:, :, None])
    return torch.where(neg, -v, v).view(x.shape)


def _scale_rows(e):
    """Exponents [rows, K/32] to scale bytes [K/32, rows rounded up to 16]."""
    s = torch.zeros(e.shape[1], (e.shape[0] + 15) // 16 * 16, dtype=torch.uint8, device=e.device)
    s[:, :e.shape[0]] = (e + 127).to(torch.uint8).t()
    return s


def _encode(x, fmt):
    """Codes and scale bytes of x [rows, K], as a program keeps them."""
    q, neg, e = _rounded(x, fmt)
    if fmt == MXFP8:
        codes = torch.where(neg, -q, q).to(torch.float8_e4m3fn).view(torch.uint8).view(x.shape)
    else:
        code = (q.to(torch.uint8) | (neg.to(torch.uint8) << 3)).view(x.shape)
        codes = code[:, 0::2] | (code[:, 1::2] << 4)
    return codes, _scale_rows(e)


def _decode(codes, scales, fmt):
    """The values that codes and scale bytes stand for, 32 bits [rows, K]."""
    rows = codes.shape[0]
    if fmt == MXFP4:
        grid = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=codes.device)
        v = grid[torch.stack((codes & 15, codes >> 4), dim=2).int()].view(rows, -1, 32)
    else:
        v = codes.view(torch.float8_e4m3fn).float().view(rows, -1, 32)
    return torch.ldexp(v, scales[:, :rows].t().int()[:, :, None] - 127).view(rows, -1)


# ---- inputs --------------------------------------------------------------------

def _activations(gen, T, K):
    """Rows of different scale, as a residual stream has them."""
    x = torch.randn((T, K), generator=gen, device="cuda")
    return (x * (0.5 + 1.5 * torch.rand((T, 1), generator=gen, device="cuda"))).to(torch.bfloat16)


def _inputs(case, seed):
    """The tensors that exist before the call."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "quantize":
        rows, K = case["rows"], case["K"]
        if case["dtype"] == "fp32":
            return {"x": torch.randn((rows, K), generator=gen, device="cuda") * K ** -0.5}
        return {"x": _activations(gen, rows, K)}
    T, N, K = case["T"], case["N"], case["K"]
    s = {}
    if case["kind"] != "dw":
        s["codes"], s["scales"] = _encode(torch.randn((N, K), generator=gen, device="cuda") * K ** -0.5, MXFP4)
    if case["kind"] in ("linear", "matmul"):
        s["X"] = _activations(gen, T, K)
    else:
        s["dY"] = torch.randn((T, N), generator=gen, device="cuda").to(torch.bfloat16)
    if case["kind"] == "dw":
        s["codes"], s["scales"] = _encode(_activations(gen, T, K), MXFP8)
    return s


def prepare(case, seed):
    """Inputs and output buffers of a running program."""
    s = _inputs(case, seed)
    kind, u8 = case["kind"], dict(dtype=torch.uint8, device="cuda")
    if kind == "quantize":
        rows, K = case["rows"], case["K"]
        s["y"] = torch.empty_like(s["x"])
    elif kind in ("linear", "matmul"):
        s["Y"] = torch.empty((case["T"], case["N"]), dtype=torch.bfloat16, device="cuda")
        rows, K = case["T"], case["K"]
    elif kind == "dx":
        s["dX"] = torch.empty((case["T"], case["K"]), dtype=torch.bfloat16, device="cuda")
    else:
        s["dW"] = torch.empty((case["N"], case["K"]), device="cuda")
    if kind in ("quantize", "matmul"):  # codes and scales that the pass makes
        half = 1 if case.get("format") == MXFP8 else 2
        s["q"] = torch.empty((rows, K // half), **u8)
        s["q_scales"] = torch.empty((K // 32, (rows + 15) // 16 * 16), **u8)
    return dict(s, case=case)


# ---- one pass --------------------------------------------------------------------

def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        return {"y": _values(s["x"], case["format"]).to(s["x"].dtype)}
    if kind == "linear":
        return {"Y": (s["X"].float() @ _decode(s["codes"], s["scales"], MXFP4).t()).to(torch.bfloat16)}
    if kind == "matmul":
        return {"Y": (_values(s["X"], MXFP4) @ _decode(s["codes"], s["scales"], MXFP4).t()).to(torch.bfloat16)}
    if kind == "dx":
        return {"dX": (s["dY"].float() @ _decode(s["codes"], s["scales"], MXFP4)).to(torch.bfloat16)}
    return {"dW": s["dY"].float().t() @ _decode(s["codes"], s["scales"], MXFP8)}


def _library():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "test-model-thing-cuda_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tmt_moe
    return tmt_moe


_OPS = {"linear": "LINEAR_FORWARD", "matmul": "LINEAR_MATMUL", "dx": "LINEAR_DX", "dw": "LINEAR_DW"}


def _kernels(s):
    lib, case = _library(), s["case"]
    kind = case["kind"]
    if kind == "quantize":
        fmt = lib.MX_FP4 if case["format"] == MXFP4 else lib.MX_FP8
        lib.mx_quantize(s["x"], s["q"], s["q_scales"], fmt)
        lib.mx_dequantize(s["q"], s["q_scales"], s["y"], fmt)
        return {"y": s["y"]}
    if "workspace" not in s:  # kept by the program from its first step on
        size = lib.linear_workspace_size(getattr(lib, _OPS[kind]), case["T"], case["N"], case["K"])
        s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    if kind == "linear":
        lib.mxfp4_linear(s["X"], s["codes"], s["scales"], s["Y"], workspace=s["workspace"])
        return {"Y": s["Y"]}
    if kind == "matmul":
        lib.mx_quantize(s["X"], s["q"], s["q_scales"], lib.MX_FP4)
        lib.mxfp4_matmul(s["q"], s["q_scales"], s["codes"], s["scales"], s["Y"], workspace=s["workspace"])
        return {"Y": s["Y"]}
    if kind == "dx":
        lib.mxfp4_linear_dx(s["dY"], s["codes"], s["scales"], s["dX"], workspace=s["workspace"])
        return {"dX": s["dX"]}
    lib.mxfp8_linear_dw(s["dY"], s["codes"], s["scales"], s["dW"], workspace=s["workspace"])
    return {"dW": s["dW"]}


def run(s):
    return _kernels(s) if own else _plain(s)


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    kind, K = case["kind"], case["K"]
    if kind == "quantize":
        n = case["rows"] * K
        size = 4 if case["dtype"] == "fp32" else 2
        held = (0.5 if case["format"] == MXFP4 else 1.0) + 1.0 / 32
        return {"bytes": n * (2 * size + 2 * held), "flops": 4 * n}  # codes and scales written, then read
    T, N = case["T"], case["N"]
    w4 = 0.5 + 1.0 / 32
    flops = 2 * T * N * K
    if kind == "linear":
        return {"bytes": 2 * T * K + w4 * N * K + 2 * T * N, "flops": flops}
    if kind == "matmul":
        return {"bytes": 2 * T * K + 2 * w4 * T * K + w4 * N * K + 2 * T * N, "flops": flops}
    if kind == "dx":
        return {"bytes": 2 * T * N + w4 * N * K + 2 * T * K, "flops": flops}
    return {"bytes": 2 * T * N + (1 + 1.0 / 32) * T * K + 4 * N * K, "flops": flops}


# ---- the same in 64 bits --------------------------------------------------------------

def _held64(x, fmt):
    """x [rows, K] rounded to the format, by multiples of each binade's step."""
    b = x.double().view(x.shape[0], -1, 32)
    amax = b.abs().amax(2, keepdim=True)
    safe = torch.where(amax > 0, amax, torch.ones_like(amax))
    top = torch.floor(torch.log2(safe))
    # log2 may round across a power of two
    top = top + (torch.exp2(top + 1) <= safe).double() - (torch.exp2(top) > safe).double()
    if fmt == MXFP4:
        e, least, digits, most = top - 2, 0, 1, 6.0
    else:
        e, least, digits, most = top - 8 + (safe > 448 * torch.exp2(top - 8)).double(), -6, 3, 448.0
    unit = torch.exp2(torch.where(amax > 0, e.clamp(-127, 127), torch.zeros_like(e)))
    v = b / unit
    binade = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40)))
    binade = binade + (torch.exp2(binade + 1) <= v.abs()).double() - (torch.exp2(binade) > v.abs()).double()
    step = torch.exp2(binade.clamp(min=least) - digits)
    return (torch.round(v / step) * step).clamp(-most, most).mul(unit).view(x.shape)


def _decode64(codes, scales, fmt):
    """Codes by their sign, exponent and mantissa bits."""
    rows = codes.shape[0]
    if fmt == MXFP4:
        c = torch.empty((rows, codes.shape[1] * 2), dtype=torch.int32, device=codes.device)
        c[:, 0::2], c[:, 1::2] = codes.int() & 15, codes.int() >> 4
        neg, ex, man, digits, bias = c >> 3, (c >> 1) & 3, c & 1, 1, 1
    else:
        c = codes.int()
        neg, ex, man, digits, bias = c >> 7, (c >> 3) & 15, c & 7, 3, 7
    frac = man.double() / (1 << digits) + (ex > 0).double()
    v = frac * torch.exp2((ex.clamp(min=1) - bias).double()) * (1 - 2 * neg)
    unit = torch.exp2(scales[:, :rows].double() - 127).t()
    return (v.view(rows, -1, 32) * unit[:, :, None]).view(rows, -1)


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return {"y": _held64(s["x"], case["format"])}
    if kind == "linear":
        return {"Y": s["X"].double() @ _decode64(s["codes"], s["scales"], MXFP4).t()}
    if kind == "matmul":
        return {"Y": _held64(s["X"], MXFP4) @ _decode64(s["codes"], s["scales"], MXFP4).t()}
    if kind == "dx":
        return {"dX": s["dY"].double() @ _decode64(s["codes"], s["scales"], MXFP4)}
    return {"dW": s["dY"].double().t() @ _decode64(s["codes"], s["scales"], MXFP8)}
