"""Calls from several threads: a thread whose first CUDA call is one of ours; and two threads calling one set
of layers, of which neither gets what the other's input or routing prepared, wherever one is interrupted."""
import threading

import pytest
import torch

from lithe_b200 import device_errors, serve
from lithe_b200.flux_model import FluxConfig, FluxShapedTransformer, lora_targets
from lithe_b200.kernels import (PackedBank, PackedLayout, PackedLoRALinear, int8_linear, layers, qk_norm_rotate,
                                quantize_rows, quantize_weight, rotate_axes, wrap_packed)
from tests.helpers import random_adapter
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


def qkv(how):
    """(q, k, v of one block, a function that forgets what they keep)."""
    torch.manual_seed(31)
    cfg = FluxConfig.tiny()
    model = FluxShapedTransformer(cfg).cuda().bfloat16().eval()
    if how == "attached":
        ads = [random_adapter([(n, m.in_features, m.out_features) for n, m in lora_targets(model)], rank=16, seed=50 + s)
               for s in range(2)]
        router, named = serve.attach_adapters(model, ads, fused_gemm=True)
        router.set([[(1, 1.0)], [(0, 0.5)]])
        got = [next(m for n, m in named.items() if n.endswith(f"transformer_blocks.0.attn.to_{c}") and "single" not in n)
               for c in "qkv"]
    else:
        bank = PackedBank(PackedLayout.from_modules([{"name": n, "shape_a": [16, m.in_features],
                                                      "shape_b": [m.out_features, 16]} for n, m in lora_targets(model)]), 4, "cuda")
        bank.fill_random(seed=3)
        named = wrap_packed(model, bank, scaling=20.0, fused_gemm=how == "fused", int8_base=how == "int8")
        ids = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
        for m in named.values():
            m.assign = ids
        got = [named[f"transformer_blocks.0.attn.to_{c}"] for c in "qkv"]
    group = got[0].prep_group
    assert group is not None and all(m.prep_group is group for m in got)

    def forget():
        for m in got:
            m._bdec_cache = None
        group._key, group._ready = None, {}
        if hasattr(group, "_bdec_key"):
            group._bdec_key = None
    return got, forget


@pytest.mark.parametrize("how", ["fused", "int8", "attached"])
def test_interrupted_while_it_leaves_results(how, monkeypatch):
    """A thread is stopped between making its siblings' results and naming the input they are for; the other
    thread calls q on its own input meanwhile (or as soon as it may)."""
    (q, k, v), forget = qkv(how)
    x, y = (torch.randn(2, 256, 256, device="cuda").bfloat16() for _ in range(2))
    with torch.no_grad():
        want = [(m(x), m(y)) for m in (q, k, v) if forget() is None]
        forget()
    init = layers._InputKey.__init__
    inside, other_done, first_done = (threading.Event() for _ in range(3))

    def slow(self, x3, *rest):
        if x3 is x:
            inside.set()
            other_done.wait(2.0)
        init(self, x3, *rest)

    monkeypatch.setattr(layers._InputKey, "__init__", slow)

    def first():
        try:
            with torch.no_grad():
                return q(x), k(x), v(x)
        finally:
            first_done.set()

    def second():
        inside.wait(10.0)
        with torch.no_grad():
            a = q(y)
            other_done.set()
            first_done.wait(10.0)
            return a, k(y), v(y)

    threads = [run(first), run(second)]
    for t, _ in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert inside.is_set()
    for i, (_, got) in enumerate(threads):
        assert got and isinstance(got[0], tuple), got
        assert all(torch.equal(g, w[i]) for g, w in zip(got[0], want))
    assert device_errors() == 0


def test_interrupted_while_it_reads_a_kept_factor(monkeypatch):
    """A thread has found its routing's kept B factor, and another thread's call under another routing replaces
    it before it is taken."""
    (q, _, _), _ = qkv("fused")
    q.prep_group = None
    x = torch.randn(2, 256, 256, device="cuda").bfloat16()
    ids = q.assign
    other = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        q.assign = other
        want_other = q(x)
        q.assign = ids
        want = q(x)                                      # leaves its B factor kept
    matches = layers._RouteKey.matches
    main = threading.get_ident()

    def slow(self, i, extra):
        hit = matches(self, i, extra)
        if hit and threading.get_ident() == main and i is ids:
            q.assign = other
            t, got = run(lambda: call())
            t.join(60)
            q.assign = ids
            assert got and torch.is_tensor(got[0]), got
            assert torch.equal(got[0], want_other)
        return hit

    def call():
        with torch.no_grad():
            return q(x)

    monkeypatch.setattr(layers._RouteKey, "matches", slow)
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
