"""Refusals of the microscaled linear layer: every check comes before any
launch, so these run without a GPU (pointers are never followed)."""
import ctypes

import numpy as np
import pytest

import mx_ref
import synthetic
import tmt_moe

A, U = 0x10000, 0x10008  # a 16-byte aligned address and one that is not
i64, f32, size = ctypes.c_int64, ctypes.c_float, ctypes.c_size_t


def refused(rc, text):
    assert rc == -1, (rc, tmt_moe.last_error())
    assert text in tmt_moe.last_error()


QUANT = dict(format=0, dtype=0, X=A, ldx=64, rows=4, K=64, codes=A, scales=A, lds=16)


@pytest.mark.parametrize("change,text", [
    (dict(format=2), "format"), (dict(format=-1), "format"), (dict(dtype=2), "dtype"),
    (dict(rows=-1), "rows"), (dict(K=0), "K=0"), (dict(K=48), "K=48"), (dict(K=-32), "K=-32"),
    (dict(ldx=32), "ldx"), (dict(ldx=68), "ldx"), (dict(dtype=1, ldx=66), "ldx"), (dict(lds=3), "lds"),
    (dict(X=0), "non-NULL"), (dict(codes=0), "non-NULL"), (dict(scales=0), "non-NULL"),
    (dict(X=U), "aligned"), (dict(codes=U), "aligned"),
])
def test_rows_refusals(change, text):
    lib = tmt_moe.load_library()
    q = dict(QUANT, **change)
    refused(lib.tmt_moe_mx_quantize(None, q["format"], q["dtype"], q["X"], i64(q["ldx"]), q["rows"], q["K"],
                                    q["codes"], q["scales"], i64(q["lds"])), text)
    refused(lib.tmt_moe_mx_dequantize(None, q["format"], q["codes"], q["scales"], i64(q["lds"]), q["rows"], q["K"],
                                      q["dtype"], q["X"], i64(q["ldx"])), text)


def test_no_rows_is_no_work():
    lib = tmt_moe.load_library()
    assert lib.tmt_moe_mx_quantize(None, 0, 0, None, i64(0), 0, 64, None, None, i64(0)) == 0
    assert lib.tmt_moe_mx_dequantize(None, 1, None, None, i64(0), 0, 64, 1, None, i64(0)) == 0
    assert lib.tmt_moe_mxfp4_linear(None, 0, 16, 64, None, i64(0), None, None, i64(0), None, i64(0), f32(0), None, size(0)) == 0


PRODUCT = dict(T=4, N=32, K=64, x=A, ldx=64, w=A, ws=A, wlds=32, y=A, ldy=64, workspace=0x10000, bytes=1 << 40)


def _product(op, q):
    lib = tmt_moe.load_library()
    fn = {"linear": lib.tmt_moe_mxfp4_linear, "dx": lib.tmt_moe_mxfp4_linear_dx, "dw": lib.tmt_moe_mxfp8_linear_dw}[op]
    return fn(None, q["T"], q["N"], q["K"], q["x"], i64(q["ldx"]), q["w"], q["ws"], i64(q["wlds"]), q["y"],
              i64(q["ldy"]), f32(0), q["workspace"], size(q["bytes"]))


@pytest.mark.parametrize("op", ["linear", "dx", "dw"])
@pytest.mark.parametrize("change,text", [
    (dict(T=-1), "T=-1"), (dict(N=0), "N=0"), (dict(N=24), "N=24"), (dict(K=32), "K=32"), (dict(K=0), "K=0"),
    (dict(x=0), "non-NULL"), (dict(x=U), "aligned"), (dict(ldx=16), "stride"), (dict(ldx=68), "stride"),
    (dict(w=0), "non-NULL"), (dict(ws=0), "non-NULL"), (dict(w=U), "aligned"), (dict(ws=U), "aligned"),
    (dict(wlds=40), "scale stride"), (dict(wlds=0), "scale stride"),
    (dict(y=0), "non-NULL"), (dict(y=U), "aligned"), (dict(ldy=16), "stride"), (dict(ldy=66), "stride"),
])
def test_product_refusals(op, change, text):
    refused(_product(op, dict(PRODUCT, **change)), text)


@pytest.mark.parametrize("change,text", [
    (dict(xs=0), "non-NULL"), (dict(xq=U), "aligned"), (dict(xlds=0), "scale stride"), (dict(xlds=24), "scale stride"),
])
def test_matmul_refusals(change, text):
    q = dict(xq=A, xs=A, xlds=16, **{k: v for k, v in PRODUCT.items() if k not in ("x", "ldx")})
    q.update(change)
    lib = tmt_moe.load_library()
    refused(lib.tmt_moe_mxfp4_matmul(None, q["T"], q["N"], q["K"], q["xq"], q["xs"], i64(q["xlds"]), q["w"], q["ws"],
                                     i64(q["wlds"]), q["y"], i64(q["ldy"]), f32(0), q["workspace"], size(q["bytes"])), text)


@pytest.mark.parametrize("args,text", [
    ((4, 16, 64, 64), "op"), ((-1, 16, 64, 64), "op"), ((0, -1, 64, 64), "T=-1"), ((1, 16, 8, 64), "N=8"),
    ((2, 16, 64, 96), "K=96"),
])
def test_workspace_size_refusals(args, text):
    with pytest.raises(tmt_moe.MoeError) as e:
        tmt_moe.linear_workspace_size(*args)
    assert e.value.code == -1 and text in str(e.value)


@pytest.mark.parametrize("op", range(4))
def test_a_workspace_serves_fewer_tokens(op):
    for N, K in ((16, 64), (256, 256), (1024, 4096), (4096, 1024), (1280, 1280)):
        last = 0
        for T in (0, 1, 16, 17, 64, 65, 127, 128, 129, 300, 777, 1024, 2048, 5003, 16384, 65536):
            now = tmt_moe.linear_workspace_size(op, T, N, K)
            assert now >= last, (N, K, T)
            last = now


def test_a_missing_or_small_workspace_is_refused():
    for op, name in enumerate(("linear", None, "dx", "dw")):
        if name is None:
            continue
        for T, N, K in ((300, 256, 4096), (777, 1024, 4096), (2048, 256, 256)):
            need = tmt_moe.linear_workspace_size(op, T, N, K)
            if need == 0:
                continue
            q = dict(PRODUCT, T=T, N=N, K=K, ldx=max(N, K), ldy=max(N, K), wlds=max(T + 15, N) // 16 * 16)
            refused(_product(name, dict(q, workspace=0, bytes=need)), "workspace")
            refused(_product(name, dict(q, workspace=0x10010, bytes=need)), "workspace")
            refused(_product(name, dict(q, bytes=need - 1)), "smaller")


def test_the_reference_rounds_to_the_nearest_code():
    """mx_ref's MXFP8 against a search over all codes, and both formats' error
    bounds: half a step of the value, 2^-4 (e4m3), saturation aside."""
    rng = np.random.Generator(np.random.PCG64(5))
    x = (rng.standard_normal((64, 96)) * np.exp(rng.uniform(-20, 20, (64, 1)))).astype(np.float32)
    codes, scales = mx_ref.quantize(x, mx_ref.FP8)
    back = mx_ref.dequantize(codes, scales, mx_ref.FP8)
    unit = np.repeat(mx_ref.e8m0(scales), 32, axis=1)
    assert np.all(np.abs(back - x) <= np.maximum(np.abs(x) * 2.0 ** -4, unit * 2.0 ** -10))
    a = np.abs(x / unit)
    near = np.abs(a[:, :, None] - mx_ref.E4M3[:127]).min(axis=2)
    assert np.array_equal(near, np.abs(np.abs(back / unit) - a))
    assert a.max() <= 448 and np.all(np.abs(x).reshape(64, 3, 32).max(2) * 2 > 448 * mx_ref.e8m0(scales))
    codes, scales = mx_ref.quantize(x, mx_ref.FP4)
    assert np.array_equal(mx_ref.dequantize(codes, scales, mx_ref.FP4), synthetic.mxfp4_dequantize(codes, scales))


@pytest.mark.parametrize("rows,K", [(1 << 28, 32), (1 << 28, 256), (1 << 24, 4096), (2 ** 31 - 1, 4096)])
def test_rows_past_one_launch_are_refused(rows, K):
    lib = tmt_moe.load_library()
    refused(lib.tmt_moe_mx_quantize(None, 0, 0, A, i64(K), rows, K, A, A, i64(rows)), "2^36")
    refused(lib.tmt_moe_mx_dequantize(None, 1, A, A, i64(rows), rows, K, 1, A, i64(K)), "2^36")


@pytest.mark.parametrize("op", ["linear", "dx", "dw"])
@pytest.mark.parametrize("T,N,K,ld", [
    (2 ** 31 - 1, 1024, 64, 1024), (2 ** 31 - 1, 16, 1024, 1024), (1, 1 << 22, 1 << 20, 1 << 22),
])
def test_outputs_past_32_bit_tile_counts_are_refused(op, T, N, K, ld):
    q = dict(PRODUCT, T=T, N=N, K=K, ldx=ld, ldy=ld, wlds=1 << 22)
    refused(_product(op, q), "2^40")


@pytest.mark.parametrize("change", [dict(ldx=(1 << 22) + 64), dict(ldy=(1 << 22) + 64), dict(wlds=(1 << 27) + 16)])
@pytest.mark.parametrize("op", ["linear", "dx", "dw"])
def test_strides_past_the_limits_are_refused(op, change):
    refused(_product(op, dict(PRODUCT, **change)), "is over")


def test_tokens_past_the_limit_are_refused():
    refused(_product("linear", dict(PRODUCT, T=(1 << 30) + 1)), "T=1073741825 is over")
