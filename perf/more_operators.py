"""Performance cases of the linear layer in 8-bit floating point and of the norm in front of it.

Codes are e4m3, with one fp32 scale for each block of 128 values: 1 x 128 of a
row (activations and gradients) or tiles of 128 x 128 (weights). With m the
block's largest magnitude, and at least 2^-100, a code is the e4m3 value
nearest to x * (448 / m) and the scale is m / 448. Scales of rows lie
block-major, [K/128][rows]; those of tiles as [rows/128][K/128].

Kinds of work, one operator each:

  norm           S = X + R, the residual stream; root-mean-square norm of S,
                 out as bf16, as codes with scales, or both;
  norm_backward  dS (with the stream's own gradient added) and dgamma;
  quantize       a matrix to codes in its own order and transposed, in one
                 pass: weights in tiles, a layer's output gradient in rows;
  product        Y = A B^T with B in tiles: the layer's forward, and its input
                 gradient with the transposed codes;
  gradient       dW = dY^T X in fp32 from the transposed codes of both.

Sizes are those of ``synthetic.CONFIGS``, of the reference's profile shape and
of ragged prompts and batches. Inputs are made on the GPU from the seed alone.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
BLOCK = 128
FP8 = torch.float8_e4m3fn
_STREAM = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # Sampling one stream: the norm ahead of an 8-bit layer.
        {"name": "norm_decode", "kind": "norm", "T": 1, "d": 1024, "stream": "bf16", "residual": True, "out": "fp8"},
        # A prompt of ragged length at the profile shape's width; a router reads the bf16 rows, the layer the codes.
        {"name": "norm_prompt", "kind": "norm", "T": 777, "d": 1280, "stream": "bf16", "residual": True, "out": "both"},
        # A large training step with the residual stream in fp32.
        {"name": "norm_batch", "kind": "norm", "T": 32768, "d": 1024, "stream": "fp32", "residual": True, "out": "fp8"},
        # A ragged batch of an uneven width, backward.
        {"name": "norm_backward_ragged", "kind": "norm_backward", "T": 5003, "d": 1000, "stream": "bf16", "residual": True},
        # The backward of the large training step.
        {"name": "norm_backward_batch", "kind": "norm_backward", "T": 32768, "d": 1024, "stream": "fp32", "residual": True},
        # A layer's fp32 masters after an optimizer step: codes for the forward and for the input gradient.
        {"name": "quantize_weights", "kind": "quantize", "blocks": "tiles", "dtype": "fp32", "rows": 4096, "K": 1024},
        # A layer's output gradient: codes for the input gradient and, transposed, for the weight gradient.
        {"name": "quantize_gradient", "kind": "quantize", "blocks": "rows", "dtype": "bf16", "rows": 32768, "K": 4096},
        # Sampling one stream through the layer: the smallest call there is.
        {"name": "product_decode_1", "kind": "product", "M": 1, "N": 4096, "K": 1024},
        # A prompt of ragged length, down-projection.
        {"name": "product_prompt_777", "kind": "product", "M": 777, "N": 1024, "K": 4096},
        # The up-projection of the large training step.
        {"name": "product_batch", "kind": "product", "M": 32768, "N": 4096, "K": 1024},
        # The weight gradient at the reference's profile shape.
        {"name": "gradient_profile_shape", "kind": "gradient", "T": 2048, "N": 1280, "K": 1280},
        # The weight gradient of the large training step's up-projection.
        {"name": "gradient_batch", "kind": "gradient", "T": 32768, "N": 4096, "K": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, of):
    return max(of, (_log(rng, lo, hi) + of // 2) // of * of)


def draw(rng):
    pick = rng.random()
    if pick < 0.4:
        d = _width(rng, 64, 8192, rng.choice((1, 8, 128)))
        case = {"kind": "norm" if pick < 0.25 else "norm_backward", "T": _log(rng, 1, min(32768, (1 << 25) // d)), "d": d,
                "stream": rng.choice(("bf16", "fp32")), "residual": rng.random() < 0.75}
        return dict(case, out=rng.choice(("fp8", "bf16", "both"))) if pick < 0.25 else case
    if pick < 0.55:
        K = _width(rng, 64, 8192, rng.choice((1, 128)))
        return {"kind": "quantize", "blocks": rng.choice(("rows", "tiles")), "dtype": rng.choice(("fp32", "bf16")),
                "rows": _log(rng, 1, min(32768, (1 << 26) // K)), "K": K}
    N, K = _width(rng, 64, 8192, rng.choice((8, 128))), _width(rng, 64, 8192, rng.choice((16, 128)))
    most = min(32768, (1 << 37) // (N * K))
    if pick < 0.85:
        return {"kind": "product", "M": _log(rng, 1, 128 if rng.random() < 0.4 else most), "N": N, "K": K}
    return {"kind": "gradient", "T": _log(rng, 64, most), "N": N, "K": K}


def _up(n, of):
    return (n + of - 1) // of * of


# ---- inputs --------------------------------------------------------------------

def _padded(x, of):
    """x as a view of rows whose stride is a multiple of `of` elements."""
    if x.shape[1] % of == 0:
        return x
    full = torch.zeros((x.shape[0], _up(x.shape[1], of)), dtype=x.dtype, device=x.device)
    full[:, :x.shape[1]] = x
    return full[:, :x.shape[1]]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rows(gen, T, d):
    """Rows of different scale, as a layer puts out."""
    return _randn(gen, T, d) * (0.5 + 1.5 * torch.rand((T, 1), generator=gen, device="cuda"))


def _held(x, blocks):
    """Codes and scales as a program has them from earlier calls; the codes' rows start at multiples of 16 bytes."""
    q, s = _encode(x, blocks)
    return _padded(q.to(FP8).view(torch.uint8), 16).view(FP8), s


def _inputs(case, seed):
    """The tensors that exist before the call."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind in ("norm", "norm_backward"):
        T, d, stream = case["T"], case["d"], _STREAM[case["stream"]]
        outliers = 1 + 15 * (torch.rand(d, generator=gen, device="cuda") < 0.01).float()  # a few wide channels
        s = {"gamma": 1 + 0.2 * _randn(gen, d)}
        if kind == "norm":
            if case["residual"] or stream is torch.bfloat16:
                s["X"] = _padded(_rows(gen, T, d).to(torch.bfloat16), 8)
            if case["residual"] or "X" not in s:
                s["R"] = _padded((4 * _randn(gen, T, d) * outliers).to(stream), 8)
        else:
            s["dY"] = _padded((1e-3 * _rows(gen, T, d)).to(torch.bfloat16), 8)
            s["S"] = _padded((4 * _randn(gen, T, d) * outliers).to(stream), 8)
            s["rstd"] = (s["S"].double().square().mean(1) + EPS).rsqrt().float()
            if case["residual"]:
                s["dR"] = _padded((1e-3 * _randn(gen, T, d)).to(stream), 8)
        return s
    if kind == "quantize":
        x = _rows(gen, case["rows"], case["K"]) * case["K"] ** -0.5
        return {"x": _padded(x.to(_STREAM[case["dtype"]]), 8)}
    N, K = case["N"], case["K"]
    if kind == "product":
        A, B, blocks = _rows(gen, case["M"], K).to(torch.bfloat16), _randn(gen, N, K) * K ** -0.5, "tiles"
    else:
        A, B, blocks = _rows(gen, case["T"], N).t(), _rows(gen, case["T"], K).t(), "rows"
    s = {}
    s["A"], s["A_scales"] = _held(A, "rows")
    s["B"], s["B_scales"] = _held(B, blocks)
    return s


def prepare(case, seed):
    """Inputs and output buffers of a running program."""
    s = _inputs(case, seed)
    kind = case["kind"]

    def empty(rows, cols, dtype, of=8):
        return torch.empty((rows, _up(cols, of)), dtype=dtype, device="cuda")[:, :cols]

    if kind in ("norm", "norm_backward"):
        T, d, stream = case["T"], case["d"], _STREAM[case["stream"]]
        if kind == "norm_backward":
            s["dS"], s["dgamma"] = empty(T, d, stream), torch.empty(d, device="cuda")
        else:
            s["rstd"] = torch.empty(T, device="cuda")
            if case["residual"]:
                s["S"] = empty(T, d, stream)
            if case["out"] != "fp8":
                s["Y"] = empty(T, d, torch.bfloat16)
            if case["out"] != "bf16":
                s["codes"], s["scales"] = empty(T, d, FP8, 16), torch.empty((_up(d, BLOCK) // BLOCK, T), device="cuda")
    elif kind == "quantize":
        rows, K = case["rows"], case["K"]
        rb, kb = _up(rows, BLOCK) // BLOCK, _up(K, BLOCK) // BLOCK
        tiles = case["blocks"] == "tiles"
        s["codes"], s["codes_t"] = empty(rows, K, FP8, 16), empty(K, rows, FP8, 16)
        s["scales"] = torch.empty((rb, kb) if tiles else (kb, rows), device="cuda")
        s["scales_t"] = torch.empty((kb, rb) if tiles else (rb, K), device="cuda")
    elif kind == "product":
        s["Y"] = empty(case["M"], case["N"], torch.bfloat16)
    else:
        s["dW"] = empty(case["N"], case["K"], torch.float32)
    return dict(s, case=case)


# ---- one pass: the plain forms -----------------------------------------------------

def _blocked(x, rows_of):
    """x, zeros added to whole blocks, as [row blocks, rows_of, column blocks, 128]."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[1] % BLOCK, 0, -x.shape[0] % rows_of))
    return x.view(x.shape[0] // rows_of, rows_of, x.shape[1] // BLOCK, BLOCK)


def _encode(x, blocks):
    """(values that the codes hold, in 32 bits, scales) of x."""
    b = _blocked(x, BLOCK if blocks == "tiles" else 1)
    m = b.abs().amax((1, 3), keepdim=True).clamp(min=2.0 ** -100)
    a = (b * (448.0 / m)).abs().clamp(max=448.0)
    step = torch.ldexp(torch.ones_like(a), (torch.frexp(a)[1] - 1).clamp(min=-6) - 3)
    q = torch.copysign(torch.round(a / step) * step, b).view(b.shape[0] * b.shape[1], -1)[:x.shape[0], :x.shape[1]]
    s = (m / 448.0).view(b.shape[0], b.shape[2])
    return q, s if blocks == "tiles" else s.t().contiguous()


def _values(codes, scales, blocks):
    """What codes and scales stand for, in 32 bits."""
    rows, K = codes.shape
    if blocks == "tiles":
        s = scales.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :K]
    else:
        s = scales.t().repeat_interleave(BLOCK, 1)[:, :K]
    return codes.float() * s


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "norm":
        x = s["X"].float() + s["R"].float() if case["residual"] else s.get("X", s.get("R")).float()
        x = x.to(_STREAM[case["stream"]])
        out = {"S": x} if case["residual"] else {}
        x = x.float()
        out["rstd"] = 1.0 / torch.sqrt(x.square().mean(1) + EPS)
        y = x * out["rstd"][:, None] * s["gamma"]
        if case["out"] != "fp8":
            out["Y"] = y.to(torch.bfloat16)
        if case["out"] != "bf16":
            q, out["scales"] = _encode(y, "rows")
            out["codes"] = q.to(FP8)
        return out
    if kind == "norm_backward":
        dy, xh = s["dY"].float(), s["S"].float() * s["rstd"][:, None]
        g = dy * s["gamma"]
        ds = s["rstd"][:, None] * (g - xh * (g * xh).mean(1, keepdim=True))
        if case["residual"]:
            ds = ds + s["dR"].float()
        return {"dS": ds.to(_STREAM[case["stream"]]), "dgamma": (dy * xh).sum(0)}
    if kind == "quantize":
        x, blocks = s["x"], case["blocks"]
        q, scales = _encode(x, blocks)
        qt, scales_t = _encode(x.t(), blocks)
        return {"codes": q.to(FP8), "scales": scales, "codes_t": qt.to(FP8), "scales_t": scales_t}
    tiles = kind == "product"
    y = _values(s["A"], s["A_scales"], "rows") @ _values(s["B"], s["B_scales"], "tiles" if tiles else "rows").t()
    return {"Y": y.to(torch.bfloat16)} if tiles else {"dW": y}


# ---- one pass: the framework's calls -------------------------------------------------

def _library():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "test-model-thing-cuda_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tmt_moe
    return tmt_moe


def _workspace(s, size):
    """Kept by the program from its first step on."""
    if "workspace" not in s:
        s["workspace"] = torch.empty(max(size(), 1), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _kernels(s):
    lib, case = _library(), s["case"]
    kind = case["kind"]
    if kind == "norm":
        lib.rmsnorm_forward(s.get("X"), s.get("R"), s["gamma"], S=s.get("S"), Y=s.get("Y"), codes=s.get("codes"),
                            scales=s.get("scales"), rstd=s["rstd"], eps=EPS)
        return {k: s[k] for k in ("S", "Y", "codes", "scales", "rstd") if k in s}
    if kind == "norm_backward":
        ws = _workspace(s, lambda: lib.rmsnorm_workspace_size(case["T"], case["d"]))
        lib.rmsnorm_backward(s["dY"], s["S"], s["gamma"], s["rstd"], s["dS"], s["dgamma"], ws, dR=s.get("dR"))
        return {"dS": s["dS"], "dgamma": s["dgamma"]}
    if kind == "quantize":
        lib.fp8_quantize(s["x"], s["codes"], s["scales"], s["codes_t"], s["scales_t"],
                         blocks=lib.FP8_TILES if case["blocks"] == "tiles" else lib.FP8_ROWS)
        return {k: s[k] for k in ("codes", "scales", "codes_t", "scales_t")}
    y, blocks = ("Y", lib.FP8_TILES) if kind == "product" else ("dW", lib.FP8_ROWS)
    ws = _workspace(s, lambda: lib.fp8_workspace_size(s["A"].shape[0], s["B"].shape[0], s["A"].shape[1], blocks))
    lib.fp8_matmul(s["A"], s["A_scales"], s["B"], s["B_scales"], s[y], blocks=blocks, workspace=ws)
    return {y: s[y]}


def run(s):
    return _kernels(s) if own else _plain(s)


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_backward"):
        n, stream = case["T"] * case["d"], 2 if case["stream"] == "bf16" else 4
        if kind == "norm":
            size = 2 + 2 * stream if case["residual"] else stream  # X, R in, S out; or the one input
            size += {"fp8": 1 + 4 / BLOCK, "bf16": 2, "both": 3 + 4 / BLOCK}[case["out"]]
            return {"bytes": n * size + 4 * case["T"] + 4 * case["d"], "flops": 6 * n}
        size = 2 + 2 * stream + (stream if case["residual"] else 0)
        return {"bytes": n * size + 4 * case["T"] + 8 * case["d"], "flops": 10 * n}
    if kind == "quantize":
        n = case["rows"] * case["K"]
        scales = 8 / BLOCK ** 2 if case["blocks"] == "tiles" else 8 / BLOCK
        return {"bytes": n * ((4 if case["dtype"] == "fp32" else 2) + 2 + scales), "flops": 6 * n}
    if kind == "product":
        M, N, K, out = case["M"], case["N"], case["K"], 2
        scales = 4 * M * K / BLOCK + 4 * N * K / BLOCK ** 2
    else:
        M, N, K, out = case["N"], case["K"], case["T"], 4
        scales = 4 * (M + N) * K / BLOCK
    return {"bytes": M * K + N * K + scales + out * M * N, "flops": 2 * M * N * K}


# ---- the same in 64 bits --------------------------------------------------------------

def _amax64(x, blocks):
    """The largest magnitude of each value's block, spread over the block, and once a block."""
    rows, K = x.shape
    most = torch.stack([c.abs().amax(1) for c in x.split(BLOCK, 1)], 1)
    if blocks == "tiles":
        most = torch.stack([c.amax(0) for c in most.split(BLOCK, 0)], 0)
    most = most.clamp(min=2.0 ** -100)
    column = torch.arange(K, device=x.device) // BLOCK
    row = torch.arange(rows, device=x.device) // (BLOCK if blocks == "tiles" else 1)
    return most[row][:, column], most


def _encode64(x, blocks):
    spread, most = _amax64(x, blocks)
    v = x * 448.0 / spread
    binade = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -40)))
    binade = binade + (torch.exp2(binade + 1) <= v.abs()).double() - (torch.exp2(binade) > v.abs()).double()
    step = torch.exp2(binade.clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448), most / 448.0 if blocks == "tiles" else (most / 448.0).t()


def _values64(codes, scales, blocks):
    rows, K = codes.shape
    c = codes.contiguous().view(torch.uint8).int()
    v = torch.where((c >> 3) & 15 == 0, (c & 7).double() / 512, (8 + (c & 7)).double() * torch.exp2(((c >> 3) & 15).double() - 10))
    column = torch.arange(K, device=c.device) // BLOCK
    row = torch.arange(rows, device=c.device)
    s = scales[row // BLOCK][:, column] if blocks == "tiles" else scales[column][:, row].t()
    return v * (1 - 2 * (c >> 7)) * s.double()


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        terms = [s[k].double() for k in ("X", "R") if k in s]
        x = sum(terms[1:], terms[0])
        if case["residual"]:
            x = x.to(_STREAM[case["stream"]]).double()
        rstd = (torch.linalg.vector_norm(x, dim=1) ** 2 / x.shape[1] + EPS) ** -0.5
        y = s["gamma"].double() * (x * rstd[:, None])
        out = {"rstd": rstd}
        if case["residual"]:
            out["S"] = x
        if case["out"] != "fp8":
            out["Y"] = y
        if case["out"] != "bf16":
            out["codes"], out["scales"] = _encode64(y, "rows")
        return out
    if kind == "norm_backward":
        # y_i = gamma_i x_i r with r = (mean(x^2) + eps)^(-1/2), dr/dx_j = -r^3 x_j / d
        x, dy, r = s["S"].double(), s["dY"].double(), s["rstd"].double()[:, None]
        dr = (dy * s["gamma"].double() * x).sum(1, keepdim=True)
        ds = dy * s["gamma"].double() * r - r ** 3 * x * dr / x.shape[1]
        return {"dS": ds + s["dR"].double() if "dR" in s else ds, "dgamma": (dy * x * r).sum(0)}
    if kind == "quantize":
        x = s["x"].double()
        codes, scales = _encode64(x, case["blocks"])
        codes_t, scales_t = _encode64(x.t(), case["blocks"])
        return {"codes": codes, "scales": scales, "codes_t": codes_t, "scales_t": scales_t}
    tiles = kind == "product"
    y = _values64(s["A"], s["A_scales"], "rows") @ _values64(s["B"], s["B_scales"], "tiles" if tiles else "rows").t()
    return {"Y" if tiles else "dW": y}
