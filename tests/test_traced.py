"""The operators where a call is recorded rather than run (make_fx, FakeTensorMode): they reach the record as
torch ops, and results have their shapes; and forward-mode derivatives.  No GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from lithe_b200.kernels import int8_linear, qk_norm_rotate, quantize_rows, rotate_axes
from lithe_b200.kernels.layers import _inference_only

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


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """A dual tensor's tangent would be lost: refused in every operand, in no_grad too (forward mode is on there)."""
    with FakeTensorMode(), torch.set_grad_enabled(grad), fwAD.dual_level():
        x = torch.empty(2, 4, 3, 64, device="cuda")
        pos = torch.empty(4, 1, device="cuda")
        dual, dpos = fwAD.make_dual(x, x.clone()), fwAD.make_dual(pos, pos.clone())
        rows = torch.empty(3, 64, dtype=BF, device="cuda")
        w, ws = torch.empty(5, 64, dtype=torch.int8, device="cuda"), torch.empty(5, device="cuda")
        for call in (lambda: rotate_axes(dual, pos, (64,)), lambda: rotate_axes(x, dpos, (64,)),
                     lambda: qk_norm_rotate(x, dual, None, None, pos, (64,)),
                     lambda: qk_norm_rotate(x, x, fwAD.make_dual(x[0, 0, 0], x[0, 0, 1]), None, pos, (64,)),
                     lambda: quantize_rows(fwAD.make_dual(rows, rows.clone())),
                     lambda: int8_linear(fwAD.make_dual(rows, rows.clone()), w, ws),
                     lambda: int8_linear(rows, w, fwAD.make_dual(ws, ws.clone())),
                     lambda: _inference_only(fwAD.make_dual(rows, rows.clone()))):
            with pytest.raises(RuntimeError, match="inference-only"):
                call()
        assert rotate_axes(x, pos, (64,)).shape == x.shape              # an open level alone is none
