"""Refusals of the 8-bit linear layer and its norm: every check comes before any launch, so
these run without a GPU (pointers are never followed). Then what the binding refuses itself."""
import ctypes

import pytest
import torch

import tmt_moe

A, U, V = 0x10000, 0x10008, 0x10002  # 16-byte aligned, 8 bytes, 2 bytes
i64, f32, size = ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


def refused(rc, text):
    assert rc == -1, (rc, tmt_moe.last_error())
    assert text in tmt_moe.last_error(), tmt_moe.last_error()


FORWARD = dict(T=4, d=256, dtype=0, X=A, ldx=256, R=A, ldr=256, gamma=A, eps=1e-5, S=A, lds=256, Y=A, ldy=256, codes=A,
               ldc=256, scales=A, ldsc=4, rstd=A)


def _forward(q):
    return tmt_moe.load_library().tmt_moe_rmsnorm_forward(
        None, q["T"], q["d"], q["dtype"], q["X"], q["ldx"], q["R"], q["ldr"], q["gamma"], q["eps"], q["S"], q["lds"],
        q["Y"], q["ldy"], q["codes"], q["ldc"], q["scales"], q["ldsc"], q["rstd"])


@pytest.mark.parametrize("change,text", [
    (dict(T=-1), "T=-1"), (dict(T=(1 << 30) + 1), "T="), (dict(d=0), "d=0"), (dict(d=16385), "d=16385"), (dict(dtype=2), "dtype"),
    (dict(X=0, R=0), "both NULL"), (dict(R=0, dtype=1), "without R"), (dict(S=0, Y=0, codes=0, rstd=0), "all NULL"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(X=U), "X must be 16-byte"), (dict(ldx=255), "X"), (dict(ldx=260), "X"), (dict(R=U), "R must be"), (dict(ldr=252), "R"),
    (dict(dtype=1, ldr=258), "R"), (dict(gamma=0), "gamma"), (dict(gamma=U), "gamma"), (dict(S=U), "S must be"), (dict(lds=260), "S"),
    (dict(Y=U), "Y must be"), (dict(ldy=8), "Y"), (dict(codes=U), "codes"), (dict(ldc=264), "codes"), (dict(ldc=240), "codes"),
    (dict(scales=0), "scales"), (dict(scales=V), "scales"), (dict(ldsc=3), "scales"), (dict(rstd=V), "rstd"),
    (dict(ldx=(1 << 22) + 8), "over"), (dict(ldsc=(1 << 31) + 1), "scales"),
])
def test_norm_forward_refusals(change, text):
    refused(_forward(dict(FORWARD, **change)), text)


BACKWARD = dict(T=4, d=256, dtype=0, dY=A, lddy=256, S=A, lds=256, gamma=A, rstd=A, dR=A, lddr=256, dS=A, ldds=256, dgamma=A,
                ws=A, bytes=1 << 40)


def _backward(q):
    return tmt_moe.load_library().tmt_moe_rmsnorm_backward(
        None, q["T"], q["d"], q["dtype"], q["dY"], q["lddy"], q["S"], q["lds"], q["gamma"], q["rstd"], q["dR"], q["lddr"],
        q["dS"], q["ldds"], q["dgamma"], q["ws"], q["bytes"])


@pytest.mark.parametrize("change,text", [
    (dict(T=-1), "T=-1"), (dict(d=0), "d=0"), (dict(d=16385), "d=16385"), (dict(dtype=-1), "dtype"),
    (dict(dY=0), "dY"), (dict(dY=U), "dY"), (dict(lddy=128), "dY"), (dict(S=0), "S must"), (dict(S=U), "S must"), (dict(lds=0), "S"),
    (dict(gamma=0), "gamma"), (dict(rstd=0), "rstd"), (dict(rstd=V), "rstd"), (dict(dR=U), "dR"), (dict(lddr=260), "dR"),
    (dict(dS=0), "dS"), (dict(dS=U), "dS"), (dict(ldds=255), "dS"), (dict(dgamma=0), "dgamma"), (dict(dgamma=U), "dgamma"),
    (dict(ws=0), "workspace"), (dict(ws=A + 16), "workspace"), (dict(bytes=16), "workspace of 16"),
])
def test_norm_backward_refusals(change, text):
    refused(_backward(dict(BACKWARD, **change)), text)


QUANT = dict(blocks=0, dtype=0, X=A, ldx=256, rows=32, K=256, codes=A, ldc=256, scales=A, lds=256, codes_t=A, ldct=32, scales_t=A,
             ldst=256)


def _quantize(q):
    return tmt_moe.load_library().tmt_moe_fp8_quantize(
        None, q["blocks"], q["dtype"], q["X"], q["ldx"], q["rows"], q["K"], q["codes"], q["ldc"], q["scales"], q["lds"],
        q["codes_t"], q["ldct"], q["scales_t"], q["ldst"])


@pytest.mark.parametrize("change,text", [
    (dict(blocks=2), "blocks"), (dict(blocks=-1), "blocks"), (dict(dtype=3), "dtype"), (dict(rows=-1), "rows=-1"), (dict(K=-5), "K=-5"),
    (dict(codes=0, codes_t=0), "both NULL"), (dict(X=0), "X"), (dict(X=U), "X"), (dict(ldx=252), "X"), (dict(dtype=1, ldx=258), "X"),
    (dict(codes=U), "codes"), (dict(ldc=240), "codes"), (dict(ldc=264), "codes"), (dict(scales=0), "scales"), (dict(lds=31), "scales"),
    (dict(codes_t=U), "codes_t"), (dict(ldct=16), "codes_t"), (dict(ldct=40), "codes_t"), (dict(scales_t=0), "scales_t"),
    (dict(ldst=255), "scales_t"), (dict(blocks=1, lds=1), "scales"), (dict(blocks=1, ldst=0), "scales_t"), (dict(scales=V), "scales"),
    (dict(rows=1 << 30, K=1 << 9, ldx=1 << 9), "2^23"), (dict(rows=1 << 23, lds=1 << 23, ldct=1 << 23), "over"),
])
def test_quantize_refusals(change, text):
    refused(_quantize(dict(QUANT, **change)), text)


PRODUCT = dict(blocks=1, dtype=0, M=4, N=256, K=256, A=A, lda=256, As=A, ldas=4, B=A, ldb=256, Bs=A, ldbs=2, Y=A, ldy=256, beta=0.0,
               ws=A, bytes=1 << 40)


def _product(q):
    return tmt_moe.load_library().tmt_moe_fp8_matmul(
        None, q["blocks"], q["dtype"], q["M"], q["N"], q["K"], q["A"], q["lda"], q["As"], q["ldas"], q["B"], q["ldb"], q["Bs"],
        q["ldbs"], q["Y"], q["ldy"], q["beta"], q["ws"], q["bytes"])


@pytest.mark.parametrize("change,text", [
    (dict(blocks=2), "blocks"), (dict(dtype=2), "dtype"), (dict(M=-1), "M=-1"), (dict(N=-8), "N=-8"), (dict(N=12), "N=12"),
    (dict(K=-1), "K=-1"), (dict(K=(1 << 22) + 1), "K="), (dict(N=(1 << 22) + 8), "N="), (dict(M=(1 << 30) + 1), "M="),
    (dict(M=1 << 30, N=1 << 11), "2^40"), (dict(A=0), "A must"), (dict(A=U), "A must"), (dict(lda=248), "A"), (dict(lda=264), "A"),
    (dict(As=0), "A_scale"), (dict(As=V), "A_scale"), (dict(ldas=3), "A_scale"), (dict(B=0), "B must"), (dict(B=U), "B must"),
    (dict(ldb=128), "B"), (dict(Bs=0), "B_scale"), (dict(ldbs=1), "B_scale"), (dict(blocks=0, ldbs=255), "B_scale"),
    (dict(Y=0), "Y must"), (dict(Y=U), "Y must"), (dict(ldy=248), "Y"), (dict(ldy=260), "Y"), (dict(dtype=1, ldy=258), "Y"),
])
def test_product_refusals(change, text):
    refused(_product(dict(PRODUCT, **change)), text)


def test_no_work_is_no_work():
    assert _forward(dict(FORWARD, T=0, ldx=0, gamma=0, scales=0)) == 0
    assert _quantize(dict(QUANT, rows=0, X=0)) == 0 and _quantize(dict(QUANT, K=0, X=0)) == 0
    assert _product(dict(PRODUCT, M=0, A=0)) == 0 and _product(dict(PRODUCT, N=0, Y=0)) == 0


def test_workspaces():
    """They serve fewer rows too, and bad sizes are refused."""
    for blocks in (tmt_moe.FP8_TILES, tmt_moe.FP8_ROWS):
        for N, K in ((64, 4096), (1024, 4096), (4096, 1024), (4096, 16384), (1280, 1280)):
            last = 0
            for M in (0, 1, 64, 65, 128, 777, 1000, 2048, 5000, 16384, 65536, 100000):
                now = tmt_moe.fp8_workspace_size(M, N, K, blocks)
                assert now >= last and now <= 256 << 20
                last = now
    last = 0
    for T in (0, 1, 5, 100, 1000, 4096, 5000, 100000, 1 << 30):
        now = tmt_moe.rmsnorm_workspace_size(T, 1000)
        assert now >= last and now <= 64 << 20
        last = now
    for call in (lambda: tmt_moe.fp8_workspace_size(1, 12, 64), lambda: tmt_moe.fp8_workspace_size(-1, 8, 64),
                 lambda: tmt_moe.fp8_workspace_size(1, 8, 64, 2), lambda: tmt_moe.rmsnorm_workspace_size(4, 16385)):
        with pytest.raises(tmt_moe.MoeError):
            call()
    for call in (lambda: tmt_moe.fp8_workspace_size(1 << 32, 8, 64), lambda: tmt_moe.rmsnorm_workspace_size(1, (1 << 32) + 5)):
        with pytest.raises(ValueError, match="32 bits"):
            call()


# ---- the binding --------------------------------------------------------------------

BF16, F32, U8, FP8 = torch.bfloat16, torch.float32, torch.uint8, torch.float8_e4m3fn


class Stand:
    """What the binding asks a tensor for."""

    def __init__(self, shape, dtype, device=0, strides=None):
        self.shape, self.dtype, self.device, self._dev = tuple(shape), dtype, f"cuda:{device}", device
        self._strides = strides or ((shape[1], 1) if len(shape) == 2 else (1,))
        self.nbytes = 1 << 40

    def get_device(self):
        return self._dev

    def stride(self, i=None):
        return self._strides if i is None else self._strides[i]

    def is_contiguous(self):
        return self._strides[-1] == 1

    def dim(self):
        return len(self.shape)

    def data_ptr(self):
        return 0x10000

    def storage_offset(self):
        return 0

    def untyped_storage(self):
        class Storage:
            nbytes = staticmethod(lambda: self.shape[0] * self._strides[0])
        return Storage()


class Library:
    """Takes every call and keeps its arguments."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args)) or 0


@pytest.fixture
def lib(monkeypatch):
    fake = Library()
    monkeypatch.setattr(tmt_moe, "load_library", lambda *a: fake)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0, raising=False)
    return fake


def _calls(T=48, d=256, N=128, device=0, stream=None, **other):
    b = lambda n: (n + 127) // 128  # noqa: E731
    t = dict(X=Stand((T, d), BF16, device), gamma=Stand((d,), F32), codes=Stand((T, d), U8), scales=Stand((b(d), T), F32),
             rstd=Stand((T,), F32), W=Stand((N, d), FP8), W_scales=Stand((b(N), b(d)), F32), Y=Stand((T, N), BF16),
             codes_t=Stand((d, T), U8), scales_t=Stand((b(T), d), F32), ws=Stand((1, 1 << 20), U8))
    t.update(other)
    return {
        "forward": lambda: tmt_moe.rmsnorm_forward(t["X"], None, t["gamma"], codes=t["codes"], scales=t["scales"], rstd=t["rstd"], stream=stream),
        "backward": lambda: tmt_moe.rmsnorm_backward(t["X"], t["X"], t["gamma"], t["rstd"], t["X"], t["gamma"], t["ws"], stream=stream),
        "quantize": lambda: tmt_moe.fp8_quantize(t["X"], t["codes"], t["scales"], t["codes_t"], t["scales_t"], stream=stream),
        "matmul": lambda: tmt_moe.fp8_matmul(t["codes"], t["scales"], t["W"], t["W_scales"], t["Y"], stream=stream),
    }


ENTRIES = ["forward", "backward", "quantize", "matmul"]


@pytest.mark.parametrize("entry", ENTRIES)
def test_the_stand_ins_reach_the_library(lib, entry):
    _calls()[entry]()
    assert len(lib.calls) == 1


@pytest.mark.parametrize("entry", ENTRIES)
def test_sizes_past_32_bits_are_refused(lib, entry):
    with pytest.raises(ValueError, match="32 bits"):
        _calls(T=(1 << 32) + 5)[entry]()
    assert not lib.calls


class Queue:
    def __init__(self, device):
        self.cuda_stream, self.device_index, self.device = 0x7000, device, torch.device("cuda", device)


@pytest.mark.parametrize("entry", ENTRIES)
def test_another_gpu_is_refused(lib, entry):
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        _calls(stream=Queue(1))[entry]()
    bad = dict(codes=Stand((48, 256), U8, 1)) if entry == "matmul" else dict(X=Stand((48, 256), BF16, 1))
    with pytest.raises(ValueError, match="not on the current GPU"):
        _calls(**bad)[entry]()
    assert not lib.calls


@pytest.mark.parametrize("entry,bad,text", [
    ("forward", dict(X=Stand((48, 256), F32)), "X must be|stream"), ("forward", dict(gamma=Stand((255,), F32)), "gamma"),
    ("forward", dict(gamma=Stand((256,), BF16)), "gamma"), ("forward", dict(codes=Stand((48, 256), BF16)), "uint8"),
    ("forward", dict(codes=Stand((47, 256), U8)), "codes"), ("forward", dict(scales=None), "scales"),
    ("forward", dict(scales=Stand((2, 47), F32)), "scales"), ("forward", dict(scales=Stand((1, 48), F32)), "scales"),
    ("forward", dict(rstd=Stand((47,), F32)), "rstd"), ("backward", dict(rstd=Stand((48,), BF16)), "rstd"),
    ("quantize", dict(codes_t=Stand((48, 256), U8)), "codes_t"), ("quantize", dict(scales_t=Stand((1, 255), F32)), "scales_t"),
    ("quantize", dict(scales=None), "go together"), ("quantize", dict(codes_t=Stand((256, 48), U8, 0, (1, 256))), "contiguous"),
    ("matmul", dict(W=Stand((128, 255), FP8)), "B must be"), ("matmul", dict(W_scales=Stand((2, 2), F32)), "B_scales"),
    ("matmul", dict(Y=Stand((48, 127), BF16)), "Y must be"), ("matmul", dict(Y=Stand((48, 128), torch.float16)), "bfloat16 or float32"),
])
def test_binding_refusals(lib, entry, bad, text):
    with pytest.raises(ValueError, match=text):
        _calls(**bad)[entry]()
    assert not lib.calls


def test_codes_whose_last_row_ends_early_are_refused(lib):
    """A row of 250 codes ends at byte 256, the last one too."""
    with pytest.raises(ValueError, match="last row"):
        _calls(d=250, codes=Stand((48, 250), U8, 0, (250, 1)))["forward"]()
    assert not lib.calls


def test_a_single_row_has_any_stride(lib):
    """Its stride is not used, whatever a view left there."""
    _calls(T=1, X=Stand((1, 256), BF16, 0, (1, 1)), codes=Stand((1, 256), U8, 0, (7, 1)))["forward"]()
    args = lib.calls[0][1]
    assert args[5] == 256 and args[15] == 256
