"""The layers under torch.inference_mode, whose tensors count no versions: nothing that depends on one is
kept, nothing raises, and the results are those of no_grad, bit for bit."""
import pytest
import torch

from lithe_b200 import device_errors, kohya, serve
from lithe_b200.flux_model import FluxConfig, FluxShapedTransformer, lora_targets
from lithe_b200.kernels import PackedBank, PackedLayout, wrap_packed
from tests.helpers import random_adapter

pytestmark = pytest.mark.gpu


def served(seed, attach):
    """(model, its inputs, what `attach(model, targets)` gives), seeded."""
    torch.manual_seed(seed)
    cfg = FluxConfig.tiny()
    model = FluxShapedTransformer(cfg).cuda().bfloat16().eval()
    got = attach(model, lora_targets(model))
    lat = torch.randn(2, 256, cfg.in_channels, device="cuda").bfloat16()
    txt = torch.randn(2, 256, cfg.text_dim, device="cuda").bfloat16()
    pooled = torch.randn(2, cfg.pooled_dim, device="cuda").bfloat16()
    return model, (lat, txt, pooled, torch.full((2,), 0.5, device="cuda")), got


@pytest.mark.parametrize("fused_gemm", [False, True])
@pytest.mark.parametrize("attached_inside", [False, True])
def test_attached_adapters(fused_gemm, attached_inside):
    def attach(model, targets):
        ads = [random_adapter([(n, m.in_features, m.out_features) for n, m in targets], rank=16, seed=30 + s)
               for s in range(3)]
        with torch.inference_mode(attached_inside):
            return serve.attach_adapters(model, ads, fused_gemm=fused_gemm)

    model, args, (router, _) = served(9, attach)
    routes = [[[(2, 1.0)], [(0, 0.5)]], [[(1, 1.0)], [(0, 0.5)]], [[(1, 0.25)], []]]
    want = []
    with torch.no_grad():
        for route in routes:
            router.set(route)
            want.append(model(*args))
    with torch.inference_mode():
        for _ in range(2):
            for route, w in zip(routes, want):
                router.set(route)
                assert torch.equal(model(*args), w) and torch.equal(model(*args), w)
        router.set(routes[0])
        model(*args)
        router.ids[0, 0] = 1                         # an in-place change of the routing is seen
        assert torch.equal(model(*args), want[1])
    with torch.no_grad():
        router.set(routes[2])
        assert torch.equal(model(*args), want[2])
    assert device_errors() == 0


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("key_format", ["diffusers", "kohya"])
def test_a_bank_made_under_inference_mode(key_format, int8):
    def attach(model, targets):
        if key_format == "kohya":
            cfg = model.cfg
            mods = kohya.kohya_flux_modules(rank=16, double_blocks=cfg.double_blocks, single_blocks=cfg.single_blocks,
                                            hidden=cfg.hidden, mlp_ratio=cfg.mlp_ratio)
        else:
            mods = [{"name": n, "shape_a": [16, m.in_features], "shape_b": [m.out_features, 16]} for n, m in targets]
        lay = PackedLayout.from_modules(mods)
        with torch.inference_mode():
            bank = PackedBank(lay, 4, "cuda")
            bank.fill_random(seed=5)
            wrapped = wrap_packed(model, bank, key_format, scaling=20.0, fused_gemm=not int8, int8_base=int8)
        return bank, wrapped

    model, args, (bank, wrapped) = served(11, attach)
    for m in wrapped.values():
        m.assign = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    other = PackedBank(bank.layout, 4, "cuda")
    other.words.copy_(bank.words)
    with torch.inference_mode():
        got = model(*args)
        bank.fill_random(seed=6)                     # new adapters in the same slots
        moved = model(*args)
        bank.words.copy_(other.words)
        assert torch.equal(model(*args), got) and not torch.equal(moved, got)
    with torch.no_grad():
        assert torch.equal(model(*args), got)
        for m in wrapped.values():                   # a bank that counts versions gives the same
            m.bank = other
        assert torch.equal(model(*args), got) and torch.equal(model(*args), got)
    assert device_errors() == 0


def in_a_new_process(code):
    """What a first call leaves behind needs a process without earlier ones."""
    import subprocess
    import sys
    from pathlib import Path
    got = subprocess.run([sys.executable, "-c", "import torch\n" + code], cwd=Path(__file__).resolve().parents[1],
                         capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip().endswith("ok"), got.stderr[-2000:]


def test_errors_of_a_first_call_under_inference_mode_can_be_cleared():
    in_a_new_process("""
from lithe_b200 import device_errors
from lithe_b200.kernels import PackedBank, PackedLayout, wrap_packed, PackedLoRALinear
lay = PackedLayout.from_modules([{"name": "m", "shape_a": [16, 128], "shape_b": [128, 16]}])
with torch.inference_mode():
    bank = PackedBank(lay, 2, "cuda")
    layer = PackedLoRALinear(torch.nn.Linear(128, 128, device="cuda", dtype=torch.bfloat16), bank, "m", 16, 1.0)
    layer.assign = torch.tensor([7], dtype=torch.int32, device="cuda")       # out of range: reported, not followed
    layer(torch.zeros(1, 4, 128, device="cuda", dtype=torch.bfloat16))
assert device_errors() != 0
assert device_errors() == 0
print("ok")
""")


@pytest.mark.parametrize("setup", ["int8", "int8 layer", "bank", "index"])
def test_a_first_call_inside_a_capture_leaves_the_error_word_alone(setup):
    """The error word is there before a graph is captured: replays do not clear the errors in it."""
    in_a_new_process(f"""
from lithe_b200 import device_errors
from lithe_b200.kernels import (IndexLoRALinear, Int8Linear, PackedBank, PackedLayout, PackedLoRALinear, _launch, int8_linear,
                                quantize_weight)
from lithe_b200 import codebook as cb
bf = torch.bfloat16
x = torch.ones(1, 40, 128, device="cuda", dtype=bf)
lin = torch.nn.Linear(128, 128, device="cuda", dtype=bf).requires_grad_(False)
if {setup!r} == "int8":
    w, ws = quantize_weight(lin.weight)
    call = lambda: int8_linear(x, w, ws)
elif {setup!r} == "int8 layer":         # as from a checkpoint: filled on the CPU, then moved
    call = lambda: layer(x)
    layer = Int8Linear(128, 128, torch.ones(128, 128, dtype=torch.int8), torch.ones(128)).cuda()
elif {setup!r} == "bank":
    lay = PackedLayout.from_modules([{{"name": "m", "shape_a": [16, 128], "shape_b": [128, 16]}}])
    layer = PackedLoRALinear(lin, PackedBank(lay, 2, "cuda"), "m", 16, 1.0)
    layer.assign = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = lambda: layer(x)
else:
    idx = torch.zeros(2, 3, 32, dtype=torch.int32, device="cuda")
    layer = IndexLoRALinear(lin, idx, idx, *cb.twin_pools(), 16, 1.0)
    layer.assign = torch.zeros(1, dtype=torch.int32, device="cuda")
    call = lambda: layer(x)
lin(x)                                  # (cuBLAS lays out its own before a capture)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(graph):
    out = call()
assert device_errors() == 0             # before any replay
_launch.error_word(torch.device("cuda", 0)).fill_(4)
graph.replay()
assert device_errors() == 4
print("ok")
""")
