"""Calls from several threads: a thread whose first CUDA call is one of ours."""
import threading

import pytest
import torch

from lithe_b200 import device_errors
from lithe_b200.kernels import (PackedBank, PackedLayout, PackedLoRALinear, int8_linear, qk_norm_rotate, quantize_rows,
                                quantize_weight, rotate_axes)
from tests.test_gpu_int8 import make

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def run(fn):
    got = []

    def body():
        try:
            got.append(fn())
        except Exception as e:
            got.append(e)

    t = threading.Thread(target=body)
    t.start()
    return t, got


def first_calls():
    bank = PackedBank(PackedLayout.from_modules([{"name": "m", "shape_a": [16, 256], "shape_b": [512, 16]}]), 4, "cuda")
    bank.fill_random(seed=1)
    lin = torch.nn.Linear(256, 512, device="cuda", dtype=BF).requires_grad_(False)
    x = make((2, 256, 256), BF, 1)
    w, ws = quantize_weight(lin.weight)
    q = make((2, 5, 4, 64), BF, 3)
    pos = torch.arange(5, device="cuda").view(5, 1)
    calls = {"int8_linear": lambda: int8_linear(x, w, ws), "rotate_axes": lambda: rotate_axes(q, pos, (64,)),
             "qk_norm_rotate": lambda: qk_norm_rotate(q, q, None, None, pos, (64,))[0],
             "quantize_rows": lambda: quantize_rows(x).q}
    for rows in (9, 40, 512):
        rq = quantize_rows(make((rows, 256), BF, rows))
        calls[f"int8_linear of {rows} quantised rows"] = lambda rq=rq: int8_linear(rq, w, ws)
    for name, kw in (("adapters", {}), ("adapters in the product", {"fused_gemm": True}), ("8-bit base", {"int8_base": True})):
        layer = PackedLoRALinear(lin, bank, "m", 16, 1.0, **kw)
        layer.assign = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
        calls[name] = lambda layer=layer: (setattr(layer, "_bdec_cache", None), layer(x))[1]
    return calls


def test_the_first_call_of_a_thread():
    with torch.no_grad():
        for name, call in first_calls().items():
            want = call()
            torch.cuda.synchronize()

            def fn():
                with torch.no_grad():
                    return call()

            t, got = run(fn)
            t.join(60)
            assert got and torch.is_tensor(got[0]), (name, got)
            torch.cuda.synchronize()
            assert torch.equal(got[0], want), name
    assert device_errors() == 0
