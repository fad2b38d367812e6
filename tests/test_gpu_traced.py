"""Traced calls (torch.jit.trace, make_fx): the trace holds the kernels and computes on new inputs what an
eager call does, bit for bit."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from lithe_b200 import device_errors
from lithe_b200.kernels import (Int8Linear, PackedBank, PackedLayout, int8_linear, qk_norm_rotate, quantize_rows,
                                quantize_weight, rotate_axes, wrap_packed)
from tests.test_gpu_int8 import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def traced(how, fn, args):
    return torch.jit.trace(fn, args, check_trace=False) if how == "jit" else make_fx(fn)(*args)


@pytest.mark.parametrize("how", ["jit", "fx"])
def test_operators(how):
    w, ws = quantize_weight(make((40, 96), BF, 2))
    wq = 1 + make((64,), BF, 3, 0.1)

    def f(q, k, pos, x):
        a, b = qk_norm_rotate(q, k, wq, None, pos, (32, 32))
        return a, b, rotate_axes(q, pos, (32, 32)), int8_linear(x, w, ws), int8_linear(quantize_rows(x), w, ws)

    def inputs(seed):
        return (make((2, 5, 4, 64), BF, seed), make((2, 5, 2, 64), BF, seed + 1),
                torch.arange(10, device=DEV).view(5, 2) * seed, make((2, 7, 96), BF, seed + 2))

    with torch.no_grad():
        g = traced(how, f, inputs(1))
        for seed in (1, 9):
            assert all(torch.equal(a, b) for a, b in zip(g(*inputs(seed)), f(*inputs(seed))))
    assert device_errors() == 0


@pytest.mark.parametrize("how", ["jit", "fx"])
def test_given_outputs(how):
    def f(q, k, pos, joint):
        qk_norm_rotate(q, k, None, None, pos, (64,), out_q=joint[:, 2:, 0], out_k=joint[:, 2:, 1])
        return rotate_axes(q, pos, (64,), out=q)

    def inputs(seed):
        return (make((2, 5, 4, 64), BF, seed), make((2, 5, 4, 64), BF, seed + 1),
                torch.arange(5, device=DEV).view(5, 1) * seed, torch.zeros(2, 7, 2, 4, 64, dtype=BF, device=DEV))

    with torch.no_grad():
        g = traced(how, f, inputs(1))
        a, b = inputs(9), inputs(9)
        assert torch.equal(g(*a), f(*b))
        assert torch.equal(a[0], b[0]) and torch.equal(a[3], b[3]) and bool(b[3][:, 2:].abs().amax() > 0)


@pytest.mark.parametrize("how", ["jit", "fx"])
def test_layer(how):
    with torch.no_grad():
        layer = Int8Linear.from_linear(torch.nn.Linear(96, 40, device=DEV, dtype=BF))
        g = traced(how, layer, (make((3, 5, 96), BF, 1),))
        x = make((3, 5, 96), BF, 2)
        assert torch.equal(g(x), layer(x))


@pytest.mark.parametrize("how", ["jit", "fx"])
@pytest.mark.parametrize("int8", [False, True])
def test_layers_keep_nothing_in_a_trace(how, int8):
    """q, k and v of a block traced after eager calls have left a B factor and a shared preparation behind: the
    trace has its own, so that it follows the routing tensor and the bank."""
    names = ["b.attn.to_q", "b.attn.to_k", "b.attn.to_v"]
    bank = PackedBank(PackedLayout.from_modules([{"name": n, "shape_a": [16, 256], "shape_b": [256, 16]} for n in names]),
                      8, DEV)
    bank.fill_random(seed=1)
    block = torch.nn.Module()
    block.b = torch.nn.Module()
    block.b.attn = torch.nn.Module()
    for n in names:
        setattr(block.b.attn, n.split(".")[-1], torch.nn.Linear(256, 256, device=DEV, dtype=BF).requires_grad_(False))
    layers = list(wrap_packed(block, bank, scaling=2.0, int8_base=int8, fused_gemm=not int8).values())
    ids = torch.tensor([1, 4], dtype=torch.int32, device=DEV)
    for m in layers:
        m.assign = ids

    def f(x):
        return tuple(m(x) for m in layers)

    with torch.no_grad():
        x = make((2, 128, 256), BF, 1)
        f(x)
        layers[0](x)                                 # leaves the other two's results pending
        g = traced(how, f, (x,))
        ids.copy_(torch.tensor([3, 0], dtype=torch.int32))
        y = make((2, 128, 256), BF, 2)
        assert all(torch.equal(a, b) for a, b in zip(g(y), f(y)))
        bank.fill_random(seed=7)
        assert all(torch.equal(a, b) for a, b in zip(g(x), f(x)))
    assert device_errors() == 0
