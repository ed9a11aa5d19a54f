"""Code matrices in columns, without a GPU: what the transposing call refuses, and what the binding
hands on to it."""
import contextlib

import pytest
import torch

import tmt_moe
from test_fp8_args import BF16, F32, FP8, U8, Library, Queue, Stand, lib, refused  # noqa: F401

A = 0x10000
CALL = dict(codes=A + 3, ldc=301, rows=200, K=300, codes_t=A, ldct=208)


def _transpose(q):
    return tmt_moe.load_library().tmt_moe_fp8_transpose(None, q["codes"], q["ldc"], q["rows"], q["K"], q["codes_t"], q["ldct"])


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows=-1"), (dict(K=-1), "K=-1"), (dict(codes=0), "codes must"), (dict(ldc=299), "row stride 299"),
    (dict(ldc=(1 << 22) + 1), "row stride"), (dict(codes_t=0), "codes_t must"), (dict(codes_t=A + 8), "codes_t must be 16-byte"),
    (dict(ldct=192), "codes_t"), (dict(ldct=200), "codes_t"), (dict(rows=1 << 30, K=1 << 9, ldc=1 << 9), "2^23"),
    (dict(rows=1 << 23, ldct=1 << 23), "over"),
])
def test_transpose_refusals(change, text):
    refused(_transpose(dict(CALL, **change)), text)


def test_nothing_to_transpose():
    assert _transpose(dict(CALL, rows=0, codes=0)) == 0 and _transpose(dict(CALL, K=0, codes_t=0)) == 0


@pytest.fixture
def laid_out(lib, monkeypatch):  # noqa: F811
    """Rows that the binding asks torch for, on which stream."""
    made, on = [], []
    monkeypatch.setattr(torch.cuda, "stream", lambda s: on.append(s) or contextlib.nullcontext())

    class Rows(Stand):
        def __getitem__(self, at):
            return Stand((self.shape[0], at[1].stop), self.dtype, 0, self._strides)

    monkeypatch.setattr(torch, "empty", lambda shape, dtype, device: made.append(shape) or Rows(shape, dtype))
    monkeypatch.setattr(Stand, "t", lambda self: Stand(self.shape[::-1], self.dtype, self._dev, self._strides[::-1]), raising=False)
    return made, on


def _matmul(A=None, B=None, **other):
    q = dict(A=A or Stand((48, 250), U8, 0, (256, 1)), A_scales=Stand((2, 48), F32), B=B or Stand((128, 250), FP8, 0, (256, 1)),
             B_scales=Stand((1, 2), F32), Y=Stand((48, 128), BF16), stream=None)
    q.update(other)
    tmt_moe.fp8_matmul(q["A"], q["A_scales"], q["B"], q["B_scales"], q["Y"], stream=q["stream"])


def test_columns_are_laid_out_in_rows(lib, laid_out):  # noqa: F811
    queue = Queue(0)
    _matmul(Stand((48, 250), U8, 0, (1, 50)), Stand((128, 250), FP8, 0, (1, 128)), stream=queue)
    assert laid_out == ([(48, 256), (128, 256)], [queue, queue])
    names = [c[0] for c in lib.calls]
    assert names == ["tmt_moe_fp8_transpose", "tmt_moe_fp8_transpose", "tmt_moe_fp8_matmul"]
    # rows K, columns M, the columns' stride; then the product of rows of 256
    assert lib.calls[0][1][2:5] == (50, 250, 48) and lib.calls[0][1][6] == 256
    assert lib.calls[2][1][7] == 256 and lib.calls[2][1][11] == 256


def test_rows_are_not(lib, laid_out):  # noqa: F811
    _matmul()
    _matmul(Stand((48, 1), U8, 0, (16, 7)), Stand((128, 1), FP8, 0, (16, 7)), A_scales=Stand((1, 48), F32), B_scales=Stand((1, 1), F32))
    assert not laid_out[0] and [c[0] for c in lib.calls] == ["tmt_moe_fp8_matmul"] * 2


@pytest.mark.parametrize("bad,text", [
    (dict(A=Stand((48, 250), BF16, 0, (1, 48))), "A must be uint8"), (dict(A=Stand((48, 250), U8, 1, (1, 48))), "not on the current GPU"),
    (dict(B=Stand((128, 249), U8, 0, (1, 128))), "B must be"), (dict(A=Stand((48, 250), U8, 0, (512, 2))), "rows of A must be contiguous"),
    (dict(A=Stand((48, 250), U8, 0, (1, 48)), Y=Stand((47, 128), BF16)), "Y must be"),
    (dict(A=Stand((48, 250), U8, 0, (1, 48)), A_scales=Stand((2, 47), F32)), "A_scales"),
])
def test_nothing_is_laid_out_for_a_call_that_is_refused(lib, laid_out, bad, text):  # noqa: F811
    with pytest.raises(ValueError, match=text):
        _matmul(**bad)
    assert not lib.calls and not laid_out[0]
