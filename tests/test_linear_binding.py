"""The Python binding of the microscaled linear layer: what it has to refuse
itself, before the C ABI sees 32-bit sizes and bare addresses. Tensors are
stand-ins that know a shape, a type, strides and a device, so that this runs
without a GPU and nothing is launched."""
import pytest
import torch

import tmt_moe

BF16, U8 = torch.bfloat16, torch.uint8


class Stand:
    """What the binding asks a tensor for."""

    def __init__(self, rows, cols, dtype, device=0):
        self.shape, self.dtype, self.device, self._dev = (rows, cols), dtype, f"cuda:{device}", device

    def get_device(self):
        return self._dev

    def stride(self):
        return self.shape[1], 1

    def is_contiguous(self):
        return True

    def dim(self):
        return 2

    def data_ptr(self):
        return 0x10000


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


def _calls(T, N, K, stream=None):
    """Each entry point on a layer of these sizes."""
    lds = (max(T, N) + 15) // 16 * 16
    w = Stand(N, K // 2, U8), Stand(K // 32, N, U8)
    x4, x8, xs = Stand(T, K // 2, U8), Stand(T, K, U8), Stand(K // 32, lds, U8)
    X, Y, W = Stand(T, K, BF16), Stand(T, N, BF16), Stand(N, K, torch.float32)
    return {
        "quantize": lambda: tmt_moe.mx_quantize(X, x8, xs, tmt_moe.MX_FP8, stream=stream),
        "dequantize": lambda: tmt_moe.mx_dequantize(x4, xs, X, tmt_moe.MX_FP4, stream=stream),
        "linear": lambda: tmt_moe.mxfp4_linear(X, *w, Y, stream=stream),
        "matmul": lambda: tmt_moe.mxfp4_matmul(x4, xs, *w, Y, stream=stream),
        "dx": lambda: tmt_moe.mxfp4_linear_dx(Y, *w, X, stream=stream),
        "dw": lambda: tmt_moe.mxfp8_linear_dw(Y, x8, xs, W, stream=stream),
    }


ENTRIES = ["quantize", "dequantize", "linear", "matmul", "dx", "dw"]


@pytest.mark.parametrize("entry", ENTRIES)
def test_the_stand_ins_reach_the_library(lib, entry):
    _calls(48, 32, 128)[entry]()
    assert len(lib.calls) == 1


@pytest.mark.parametrize("entry", ENTRIES)
@pytest.mark.parametrize("T", [1 << 31, (1 << 32) + 5])
def test_sizes_past_32_bits_are_refused(lib, entry, T):
    """2^32 + 5 rows must not become 5."""
    with pytest.raises(ValueError, match="32 bits"):
        _calls(T, 16, 64)[entry]()
    assert not lib.calls


@pytest.mark.parametrize("sizes", [((1 << 32) + 1, 16, 64), (1, (1 << 32) + 16, 64), (1, 16, (1 << 32) + 64), (1 << 31, 16, 64)])
def test_workspace_sizes_past_32_bits_are_refused(sizes):
    for op in range(4):
        with pytest.raises(ValueError, match="32 bits"):
            tmt_moe.linear_workspace_size(op, *sizes)


class Queue:
    """A torch.cuda.Stream as the binding sees it."""

    def __init__(self, device):
        self.cuda_stream, self.device_index, self.device = 0x7000, device, torch.device("cuda", device)


@pytest.mark.parametrize("entry", ENTRIES)
def test_a_stream_of_another_gpu_is_refused(lib, entry):
    """Work goes to the current GPU, whose memory the operands are in."""
    _calls(48, 32, 128, stream=Queue(0))[entry]()
    assert len(lib.calls) == 1 and lib.calls[0][1][0] == 0x7000
    with pytest.raises(ValueError, match="stream is on cuda:1"):
        _calls(48, 32, 128, stream=Queue(1))[entry]()
    assert len(lib.calls) == 1
