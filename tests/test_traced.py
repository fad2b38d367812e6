"""The operators where a call is recorded rather than run (make_fx, FakeTensorMode): they reach the record as
torch ops, and results have their shapes.  No GPU."""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from lithe_b200.kernels import int8_linear, qk_norm_rotate, quantize_rows, rotate_axes

BF = torch.bfloat16


def test_recorded_as_ops():
    def f(q, k, pos, x, w, ws):
        q, k = qk_norm_rotate(q, k, None, None, pos, (32, 32))
        rotate_axes(q, pos, (32, 32), out=q)
        return q, k, rotate_axes(k, pos, (32, 32)), int8_linear(quantize_rows(x), w, ws), int8_linear(x, w, ws)

    with FakeTensorMode():
        args = (torch.empty(2, 4, 3, 64, dtype=BF, device="cuda"), torch.empty(2, 4, 1, 64, dtype=BF, device="cuda"),
                torch.empty(4, 2, device="cuda"), torch.empty(2, 3, 40, dtype=BF, device="cuda"),
                torch.empty(5, 48, dtype=torch.int8, device="cuda")[:, :40], torch.empty(5, device="cuda"))
        shapes = [tuple(t.shape) for t in f(*args)]
        graph = make_fx(f)(*args).graph
    assert shapes == [(2, 4, 3, 64), (2, 4, 1, 64), (2, 4, 1, 64), (2, 3, 5), (2, 3, 5)]
    ops = [n.target._schema.name for n in graph.nodes if n.op == "call_function" and hasattr(n.target, "_schema")]
    mine = [n.split("::")[1] for n in ops if n.startswith("lithe_b200::")]
    assert mine == ["qk_norm_rotate_", "rotate_axes_", "rotate_axes_", "quantize_rows", "int8_linear",
                    "int8_linear_dynamic"]
