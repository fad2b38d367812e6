"""8-bit linear: what the entry points refuse, without a GPU."""
import re
from pathlib import Path

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lithe_b200 import _lib
from lithe_b200.kernels import QuantizedRows, _launch, int8_linear, quantize_rows, quantize_weight


def _linear(q=0x10000, q_stride=128, xs=0x20000, w=0x30000, w_stride=128, ws=0x40000, bias=None, out=0x50000,
            dtype=_lib.DTYPE_BF16, rows=4, n=8, k=100, h=None, b_dec=None, rps=0, rank=0):
    return _lib.lib().lithe_int8_linear(q, q_stride, xs, w, w_stride, ws, bias, out, dtype, rows, n, k, h, b_dec, rps,
                                        rank, None, None)


@pytest.mark.parametrize("over,code", [
    ({"dtype": _lib.DTYPE_F32}, _lib.ERR_ARG),
    ({"rows": -1}, _lib.ERR_ARG),
    ({"n": 0}, _lib.ERR_ARG),
    ({"k": 0}, _lib.ERR_ARG),
    ({"k": 131073, "q_stride": 131088, "w_stride": 131088}, _lib.ERR_UNSUPPORTED),
    ({"rows": 2 ** 31 - 1}, _lib.ERR_UNSUPPORTED),
    ({"n": 2 ** 31 - 1}, _lib.ERR_UNSUPPORTED),
    ({"q": 0x10008}, _lib.ERR_ARG),
    ({"q": None}, _lib.ERR_ARG),
    ({"q_stride": 100}, _lib.ERR_ARG),
    ({"w_stride": 96}, _lib.ERR_ARG),
    ({"w": 0x30001}, _lib.ERR_ARG),
    ({"xs": None}, _lib.ERR_ARG),
    ({"ws": 0x40002}, _lib.ERR_ARG),
    ({"out": None}, _lib.ERR_ARG),
    ({"out": 0x50001}, _lib.ERR_ARG),
    ({"bias": 0x60001}, _lib.ERR_ARG),
    ({"h": 0x70000}, _lib.ERR_ARG),
    ({"h": 0x70000, "b_dec": 0x80000, "rps": 2, "rank": 8}, _lib.ERR_UNSUPPORTED),
    ({"h": 0x70000, "b_dec": 0x80000, "rps": 3, "rank": 16}, _lib.ERR_ARG),
    ({"h": 0x70000, "b_dec": 0x80000, "rps": 0, "rank": 16}, _lib.ERR_ARG),
    ({"h": 0x70002, "b_dec": 0x80000, "rps": 2, "rank": 16}, _lib.ERR_ARG),
    ({"h": 0x70000, "b_dec": 0x80000, "rps": 2, "rank": 16, "dtype": _lib.DTYPE_F16}, _lib.ERR_UNSUPPORTED),
])
def test_c_linear_refuses(over, code):
    assert _linear(**over) == code
    assert _lib.lib().lithe_last_error()


def test_c_linear_without_rows_is_a_no_op():
    assert _linear(rows=0, q=None, out=None) == _lib.OK


def _quant(x=0x10000, dtype=_lib.DTYPE_BF16, rows=4, k=100, x_stride=100, q=0x20000, q_stride=112, scale=0x30000):
    return _lib.lib().lithe_quantize_rows(x, dtype, rows, k, x_stride, q, q_stride, scale, None)


@pytest.mark.parametrize("over,code", [
    ({"dtype": _lib.DTYPE_F32}, _lib.ERR_ARG),
    ({"rows": -1}, _lib.ERR_ARG),
    ({"k": 0}, _lib.ERR_ARG),
    ({"k": 200000, "q_stride": 200000}, _lib.ERR_UNSUPPORTED),
    ({"x": None}, _lib.ERR_ARG),
    ({"x": 0x10001}, _lib.ERR_ARG),
    ({"x_stride": -1}, _lib.ERR_ARG),
    ({"q": 0x20004}, _lib.ERR_ARG),
    ({"q_stride": 104}, _lib.ERR_ARG),
    ({"q_stride": 96}, _lib.ERR_ARG),
    ({"scale": None}, _lib.ERR_ARG),
])
def test_c_quantize_refuses(over, code):
    assert _quant(**over) == code


def _dynamic(x=0x10000, x_stride=100, w=0x30000, w_stride=128, rows=4, n=8, k=100, dtype=_lib.DTYPE_BF16, h=None,
             b_dec=None, space=0x20000, size=4 * (112 + 4)):
    return _lib.lib().lithe_int8_linear_dynamic(x, x_stride, w, w_stride, 0x40000, None, 0x50000, dtype, rows, n, k, h,
                                                b_dec, 2, 16, None, space, size, None)


@pytest.mark.parametrize("over,code", [
    ({"x": None}, _lib.ERR_ARG),
    ({"x": 0x10001}, _lib.ERR_ARG),
    ({"x_stride": -100}, _lib.ERR_ARG),
    ({"w": 0x30004}, _lib.ERR_ARG),
    ({"dtype": _lib.DTYPE_F32}, _lib.ERR_ARG),
    ({"space": None}, _lib.ERR_ARG),
    ({"space": 0x20008}, _lib.ERR_ARG),
    ({"size": 4 * (112 + 4) - 1}, _lib.ERR_ARG),
    ({"h": 0x70000}, _lib.ERR_ARG),
    ({"k": 200000, "w_stride": 200000}, _lib.ERR_UNSUPPORTED),
])
def test_c_dynamic_refuses(over, code):
    assert _dynamic(**over) == code
    assert _lib.lib().lithe_last_error()


def test_workspace_bytes():
    lib = _lib.lib()
    assert lib.lithe_int8_workspace_bytes(4, 100) == 4 * (112 + 4)
    assert lib.lithe_int8_workspace_bytes(0, 100) == 0
    assert lib.lithe_int8_workspace_bytes(2 ** 31 - 1, 131072) == (2 ** 31 - 1) * (131072 + 4)
    assert _dynamic(rows=0, x=None, space=None, size=0) == _lib.OK


def test_python_checks():
    with pytest.raises(ValueError, match="CUDA"):
        int8_linear(torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(ValueError, match="CUDA"):
        quantize_rows(torch.zeros(2, 8, dtype=torch.bfloat16))
    with FakeTensorMode():
        x = torch.empty(2, 8, device="cuda")
        with pytest.raises(TypeError):
            quantize_rows(x)
        with pytest.raises(ValueError, match=r"k >= 1"):
            quantize_rows(torch.empty(2, 0, dtype=torch.bfloat16, device="cuda"))
        with pytest.raises(ValueError, match=r"\(n, k\)"):
            quantize_weight(torch.empty(2, 3, 8, dtype=torch.bfloat16, device="cuda"))
        with pytest.raises(RuntimeError, match="inference-only"):
            quantize_rows(torch.empty(2, 8, dtype=torch.bfloat16, device="cuda", requires_grad=True))
        with pytest.raises(RuntimeError, match="inference-only"):
            int8_linear(torch.empty(2, 8, dtype=torch.bfloat16, device="cuda"), None, None,
                        torch.empty(4, dtype=torch.bfloat16, device="cuda", requires_grad=True))


def test_launch_checks(monkeypatch):
    """Every disagreement of shapes, types and strides is refused before the kernel is called."""
    monkeypatch.setattr(_launch, "_require_cuda", lambda t, what: None)
    bf = torch.bfloat16
    ok = dict(q=torch.zeros(6, 32, dtype=torch.int8), x_scale=torch.zeros(6), weight=torch.zeros(4, 32, dtype=torch.int8),
              weight_scale=torch.zeros(4), bias=torch.zeros(4, dtype=bf), out=torch.zeros(6, 4, dtype=bf),
              h=torch.zeros(6, 16, dtype=bf), b_dec=torch.zeros(2, 4, 16, dtype=bf))
    for key, bad in [("q", torch.zeros(6, 31, dtype=torch.int8)), ("q", torch.zeros(6, 32, dtype=torch.uint8)),
                     ("q", torch.zeros(6, 40, dtype=torch.int8)[:, :32]), ("x_scale", torch.zeros(5)),
                     ("x_scale", torch.zeros(6, dtype=torch.float64)), ("weight", torch.zeros(4, 32)),
                     ("weight", torch.zeros(32, 4, dtype=torch.int8).t()), ("weight_scale", torch.zeros(8)[::2]),
                     ("bias", torch.zeros(4)), ("bias", torch.zeros(5, dtype=bf)), ("out", torch.zeros(6, 5, dtype=bf)),
                     ("out", torch.zeros(6, 4)), ("h", None), ("h", torch.zeros(5, 16, dtype=bf)),
                     ("h", torch.zeros(6, 16)), ("b_dec", torch.zeros(4, 4, 16, dtype=bf)),
                     ("b_dec", torch.zeros(0, 4, 16, dtype=bf)), ("b_dec", torch.zeros(2, 5, 16, dtype=bf)),
                     ("b_dec", None)]:
        with pytest.raises((ValueError, TypeError)):
            _launch.int8_linear_(**{**ok, key: bad})


def test_sizes_beyond_32_bits_are_refused(monkeypatch):
    monkeypatch.setattr(_launch, "_require_cuda", lambda t, what: None)
    x = torch.zeros(1, 1, dtype=torch.bfloat16).expand(2 ** 32 + 5, 1)
    w, ws = torch.zeros(4, 16, dtype=torch.int8)[:, :1], torch.zeros(4)
    with pytest.raises(NotImplementedError):
        int8_linear(x, w, ws)
    with pytest.raises(NotImplementedError):
        quantize_rows(x)
    with pytest.raises(NotImplementedError):
        int8_linear(x[:1], w[:1].expand(2 ** 31, 1), ws[:1].expand(2 ** 31))


def test_ops_know_their_shapes():
    import lithe_b200.kernels.ops  # noqa: F401
    with FakeTensorMode():
        x = torch.empty(6, 40, dtype=torch.float16, device="cuda")
        q, scale = torch.ops.lithe_b200.quantize_rows(x)
        assert tuple(q.shape) == (6, 40) and q.stride(0) == 48 and q.dtype == torch.int8 and tuple(scale.shape) == (6,)
        y = torch.ops.lithe_b200.int8_linear_dynamic(x.view(2, 3, 40), q[:3], scale[:3], None, None, None)
        assert tuple(y.shape) == (2, 3, 3) and y.dtype == torch.float16
        y = torch.ops.lithe_b200.int8_linear(q, scale, q[:3], scale[:3], None, None, None, True)
        assert tuple(y.shape) == (6, 3) and y.dtype == torch.float16


def test_what_the_quantisation_writes_is_read_by_ordinary_loads():
    """The linear may start while q and the scales are being written, so it must not read them as memory
    that is constant for its lifetime (__ldg)."""
    source = (Path(_lib.__file__).parent / "csrc" / "int8_linear.cu").read_text()
    body = source[source.index("struct Params {"):source.index("extern \"C\"")]         # the linear's kernels
    constant = re.findall(r"__ldg\(((?:[^()]|\((?:[^()]|\([^()]*\))*\))*)\)", body)
    assert constant and not [c for c in constant if re.search(r"\bx_scale\b|\bp\.q\b|\brow\b", c)], constant
    load = body[body.index("uint4 load16("):]
    assert "return *reinterpret_cast<const uint4*>(row + k0)" in load[:load.index("\n}\n")]


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("which", ["x", "bias", "weight_scale", "h", "b_dec"])
def test_every_operand_is_inference_only(which, quantized):
    """No operand's gradient is lost silently: with grad mode on, one that requires a gradient is refused."""
    bf = torch.bfloat16
    with FakeTensorMode():
        ops = dict(x=torch.empty(6, 32, dtype=bf, device="cuda"), weight=torch.empty(4, 32, dtype=torch.int8, device="cuda"),
                   weight_scale=torch.empty(4, device="cuda"), bias=torch.empty(4, dtype=bf, device="cuda"),
                   h=torch.empty(6, 16, dtype=bf, device="cuda"), b_dec=torch.empty(2, 4, 16, dtype=bf, device="cuda"))
        if quantized:
            ops["x"] = QuantizedRows(torch.empty(6, 32, dtype=torch.int8, device="cuda"), torch.empty(6, device="cuda"), (6,), bf)
        (ops["x"].scale if which == "x" and quantized else ops[which]).requires_grad_()
        with pytest.raises(RuntimeError, match="inference-only"):
            int8_linear(**ops)
