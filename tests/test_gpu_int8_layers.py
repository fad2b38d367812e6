"""The 8-bit linears, the norm and the rotation as the layers and the model use them.

Tolerances: the layer tests compare with the formulas in 64 bits on the layer's own operands (as in
test_gpu_int8.py: half a rounding step of the result and 40 half steps of fp32 of what is added); two
bf16 roundings apart (the adapters added in a second pass) is another half step of the base's
result.  The model tests compare two ways of computing the same model in bf16, whose roundings
differ at every linear: relative Frobenius 3e-2, as the model's other paths are compared.
"""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

from lithe_b200 import device_errors
from lithe_b200.flux_model import FluxConfig, FluxShapedTransformer, lora_targets, rope_axes, rope_positions
from lithe_b200.kernels import (Int8Linear, PackedBank, PackedLayout, PackedLoRALinear, int8_linear, qk_norm_rotate,
                                quantize_rows, wrap_int8, wrap_linears, wrap_packed)
from tests.helpers import rel_fro
from tests.test_gpu_int8 import check, exact_linear, make
from tests.test_gpu_rotary import check as check_turn
from tests.test_gpu_rotary import exact_norm, exact_turn

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def linear(k, n, dtype=BF, bias=True, seed=0):
    lin = nn.Linear(k, n, bias=bias, device=DEV, dtype=dtype)
    with torch.no_grad():
        lin.weight.copy_(make((n, k), dtype, seed + 1, 0.03))
        if bias:
            lin.bias.copy_(make((n,), dtype, seed + 2, 0.1))
    return lin


@pytest.mark.parametrize("k,n,dtype,bias", [(64, 40, BF, True), (100, 24, torch.float16, True), (1001, 33, BF, False)])
def test_int8_linear_layer(k, n, dtype, bias):
    lin = linear(k, n, dtype, bias)
    layer = Int8Linear.from_linear(lin)
    x = make((3, 50, k), dtype, 7)
    with torch.no_grad():
        got = layer(x)
        check(got, *exact_linear(x, layer.weight, layer.weight_scale, layer.bias))
        assert layer.weight.shape == (n, k) and rel_fro(got.float(), lin(x).float()) < 3e-2      # 8-bit steps of both
        again = Int8Linear(k, n, torch.zeros_like(layer.weight_q), torch.zeros_like(layer.weight_scale), layer.bias)
        again.load_state_dict(layer.state_dict())
        assert torch.equal(again(x), got)
        scale = layer.weight_scale.clone()
        other = layer.to(torch.float16 if dtype == BF else BF)
        assert other.weight_scale.dtype == torch.float32 and torch.equal(other.weight_scale, scale)
        other(x.to(torch.float16 if dtype == BF else BF))
    with pytest.raises(ValueError):
        Int8Linear(k, n, torch.zeros(n, k + 16, dtype=torch.int8), torch.zeros(n))
    with pytest.raises(RuntimeError, match="inference-only"):
        layer.to(dtype)(x.requires_grad_())


def bank_of(shapes, slots=8, seed=1):
    lay = PackedLayout.from_modules([{"name": n, "shape_a": [16, k], "shape_b": [o, 16]} for n, k, o in shapes])
    bank = PackedBank(lay, slots, DEV)
    bank.fill_random(seed=seed)
    return bank


@pytest.mark.parametrize("tokens", [1, 8, 9, 37, 128, 300, 512])
@pytest.mark.parametrize("k,n", [(128, 200), (320, 256), (640, 1032)])
def test_adapters_on_an_8_bit_base(k, n, tokens):
    bank = bank_of([("m", k, n)])
    layer = PackedLoRALinear(linear(k, n), bank, "m", 16, 2.0, int8_base=True)
    assert isinstance(layer.base, Int8Linear)
    layer.assign = torch.tensor([3, -1, 6, 3], dtype=torch.int32, device=DEV)
    layer.weights = torch.tensor([1.0, 1.0, 0.5, -2.0], device=DEV)
    x = make((4, tokens, k), BF, 5)
    with torch.no_grad():
        got = layer(x)
        base = layer.base(x)
        assert torch.equal(got[1], base[1])                              # unrouted: the base linear's bits
        h, b_dec = torch.ops.lithe_b200.lora_prep(x, bank.words, bank.words, layer._va, layer._vb, bank.n_slots,
                                                  layer.assign, layer.weights, n, layer._lut, 2.0, True)
        want, mag = exact_linear(x, layer.base.weight, layer.base.weight_scale, layer.base.bias, h, b_dec)
        if layer._int8_expand_ok(x):
            check(got, want, mag)
        else:
            tol = 2.0 ** -8 * (want.abs() + 2 * base.double().abs()) + 40 * 2.0 ** -24 * mag
            assert ((got.double() - want).abs() <= tol).all()
        # a new routing is seen, and the old one again
        layer.assign = torch.tensor([0, 0, 0, 0], dtype=torch.int32, device=DEV)
        moved = layer(x)
        layer.assign = torch.tensor([3, -1, 6, 3], dtype=torch.int32, device=DEV)
        assert torch.equal(layer(x), got) and not torch.equal(moved[0], got[0])
    assert device_errors() == 0


def test_no_samples_and_two_dimensions():
    bank = bank_of([("m", 128, 256)])
    layer = PackedLoRALinear(linear(128, 256), bank, "m", 16, 1.0, int8_base=True)
    with torch.no_grad():
        assert layer(torch.empty(0, 20, 128, dtype=BF, device=DEV)).shape == (0, 20, 256)
        x = make((5, 128), BF, 1)
        layer.assign = torch.arange(5, dtype=torch.int32, device=DEV)
        assert torch.equal(layer(x), layer(x[:, None])[:, 0])


def test_attention_block_chain():
    """The block as a served model runs it, step by step against the formulas on each step's own inputs:
    activations quantised once for q, k and v, 8-bit products with the adapters' expand, norm and rotation
    into the joint sequence of two streams, attention, 8-bit output projection."""
    b, heads, hd, n_txt, n_img = 2, 4, 64, 24, 100
    d = heads * hd
    names = [f"{s}.{p}" for s in ("txt", "img") for p in "qkv"]
    bank = bank_of([(n, d, d) for n in names])
    ids = torch.tensor([2, 5], dtype=torch.int32, device=DEV)
    pos = rope_positions(n_txt, n_img, DEV)
    axes = rope_axes(hd)
    joint = [torch.full((b, n_txt + n_img, heads, hd), float("nan"), dtype=BF, device=DEV) for _ in range(3)]
    norms = [1 + make((hd,), BF, 30 + i, 0.1) for i in range(4)]
    with torch.no_grad():
        for s, (stream, tokens, at) in enumerate((("txt", n_txt, 0), ("img", n_img, n_txt))):
            x = make((b, tokens, d), BF, 10 + s)
            rows = quantize_rows(x)
            outs = []
            for i, p in enumerate("qkv"):
                layer = PackedLoRALinear(linear(d, d, seed=100 * s + 10 * i), bank, f"{stream}.{p}", 16, 1.5, int8_base=True)
                layer.assign = ids
                h, b_dec = layer._expand_operands(x)
                y = int8_linear(rows, layer.base.weight, layer.base.weight_scale, layer.base.bias, h=h, b_dec=b_dec)
                assert torch.equal(y, layer(x))
                check(y, *exact_linear(x, layer.base.weight, layer.base.weight_scale, layer.base.bias, h, b_dec))
                outs.append(y.view(b, tokens, heads, hd))
            here = slice(at, at + tokens)
            qk_norm_rotate(outs[0], outs[1], norms[2 * s], norms[2 * s + 1], pos[here], axes, out_q=joint[0][:, here],
                           out_k=joint[1][:, here])
            joint[2][:, here] = outs[2]
            for y, w, j in ((outs[0], norms[2 * s], joint[0]), (outs[1], norms[2 * s + 1], joint[1])):
                check_turn(j[:, here], *exact_turn(exact_norm(y, w, 1e-6), pos[here], axes, 1e4, "interleaved"), 24)
        assert not any(j.isnan().any() for j in joint)
        q, k, v = (j.transpose(1, 2) for j in joint)
        o = F.scaled_dot_product_attention(q, k, v).transpose(1, 2).reshape(b, n_txt + n_img, d)
        proj = Int8Linear.from_linear(linear(d, d, seed=900))
        check(proj(o), *exact_linear(o, proj.weight, proj.weight_scale, proj.bias))
    assert device_errors() == 0


class PlainInt8(nn.Module):
    """The 8-bit base with decoded adapters, by its formula in 64 bits, rounded once."""

    def __init__(self, layer, a, b):
        super().__init__()
        self.layer, self.a, self.b = layer, a, b

    def forward(self, x):
        lin = self.layer.base
        y, _ = exact_linear(x, lin.weight, lin.weight_scale, lin.bias)
        for i in range(x.shape[0]):
            h = (self.layer.scaling * (x[i].double() @ self.a[i].double().t())).to(x.dtype).double()
            y[i] += h @ self.b[i].double().t()
        return y.to(x.dtype)


def tiny(seed, fused_qk, state=None):
    torch.manual_seed(seed)
    cfg = FluxConfig.tiny()
    cfg.fused_qk = fused_qk
    model = FluxShapedTransformer(cfg).cuda().bfloat16().eval()
    if state is not None:
        model.load_state_dict(state)
    lat = torch.randn(2, 81, cfg.in_channels, device=DEV).bfloat16()
    txt = torch.randn(2, 23, cfg.text_dim, device=DEV).bfloat16()
    pooled = torch.randn(2, cfg.pooled_dim, device=DEV).bfloat16()
    return model, (lat, txt, pooled, torch.full((2,), 0.5, device=DEV))


def test_model_with_the_fused_norm_and_rotation():
    model, args = tiny(3, False)
    fused, _ = tiny(3, True, model.state_dict())
    with torch.no_grad():
        want, got = model(*args), fused(*args)
    assert rel_fro(got.float(), want.float()) < 2e-2


def test_model_on_8_bit_bases():
    model, args = tiny(4, True)
    state = {k: v.clone() for k, v in model.state_dict().items()}
    targets = lora_targets(model)
    bank = bank_of([(n, m.in_features, m.out_features) for n, m in targets], seed=5)
    wrapped = wrap_packed(model, bank, scaling=20.0, int8_base=True)
    ids = torch.tensor([2, 7], dtype=torch.int32, device=DEV)
    for m in wrapped.values():
        m.assign = ids
    others = [n for n, m in model.named_modules() if isinstance(m, nn.Linear)]
    assert set(wrap_int8(model, others)) == set(others)
    assert not any(isinstance(m, nn.Linear) for m in model.modules())
    plain, _ = tiny(4, False, state)
    from lithe_b200.kernels import split_decoded
    dec = bank.decode([2, 7], dtype=BF)
    per = [split_decoded(dec[i], bank.layout) for i in range(2)]
    wrap_linears(plain, [n for n, _ in targets], lambda n, lin: PlainInt8(wrapped[n], [p[n][0] for p in per], [p[n][1] for p in per]))
    wrap_int8(plain, others)
    with torch.no_grad():
        got, want = model(*args).float(), plain(*args).float()
        groups = {id(m.prep_group): m.prep_group for m in wrapped.values() if m.prep_group is not None}
        assert len(groups) == 6 and all(g._key is None and not g._ready for g in groups.values())
        for m in wrapped.values():
            m.prep_group = None
        assert torch.equal(model(*args).float(), got)                    # grouped or alone: the same bits
        for m in wrapped.values():
            m.assign = torch.full((2,), -1, dtype=torch.int32, device=DEV)
        unrouted = model(*args).float()
    # the two agree, and far better than either does with the model without its adapters
    assert rel_fro(got, want) < min(3e-2, 0.5 * rel_fro(got, unrouted))
    assert device_errors() == 0


def test_compiled_model_on_8_bit_bases():
    torch._dynamo.reset()
    model, args = tiny(6, True)
    targets = lora_targets(model)
    bank = bank_of([(n, m.in_features, m.out_features) for n, m in targets], seed=7)
    wrapped = wrap_packed(model, bank, scaling=20.0, int8_base=True)
    for m in wrapped.values():
        m.assign = torch.tensor([2, 7], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        eager = model(*args)
        assert torch.equal(torch.compile(model, fullgraph=True, backend="aot_eager")(*args), eager)


@pytest.mark.parametrize("int8", [True, False])
def test_inference_mode(int8):
    """Under inference_mode torch counts no versions: nothing is shared, and the results are the same."""
    model, args = tiny(8, int8)
    if not int8:
        args = (make((2, 256, 16), BF, 1), make((2, 256, 64), BF, 2), *args[2:])
    targets = lora_targets(model)
    bank = bank_of([(n, m.in_features, m.out_features) for n, m in targets], seed=9)
    wrapped = wrap_packed(model, bank, scaling=20.0, int8_base=int8, fused_gemm=not int8)
    with torch.no_grad():
        for m in wrapped.values():
            m.assign = torch.tensor([1, 3], dtype=torch.int32, device=DEV)
        want = model(*args)
    with torch.inference_mode():
        ids = torch.tensor([1, 3], dtype=torch.int32, device=DEV)
        for m in wrapped.values():
            m.assign = ids
        assert torch.equal(model(*args), want)
        ids.copy_(torch.tensor([4, 4], dtype=torch.int32, device=DEV))
        moved = model(*args)
        x = make((1, 3, 2, 64), BF, 1)
        qk_norm_rotate(x, x.clone(), None, None, torch.zeros(3, 1, device=DEV), (64,), out_q=x)
    assert not torch.equal(moved, want)


def test_captured_layer():
    bank = bank_of([("m", 256, 512)])
    layer = PackedLoRALinear(linear(256, 512), bank, "m", 16, 2.0, int8_base=True)
    layer.assign = torch.tensor([1, 4], dtype=torch.int32, device=DEV)
    x = make((2, 40, 256), BF, 1)
    with torch.no_grad():
        layer(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        x.copy_(make((2, 40, 256), BF, 2))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(x))


@pytest.mark.parametrize("int8", [True, False])
def test_captured_block_computes_its_own(int8):
    """q, k and v of one block, called on an input before and while a graph is captured: replays follow the
    input's and the routing's new values, also once the layers have gone on to another routing."""
    names = ["b.attn.to_q", "b.attn.to_k", "b.attn.to_v"]
    bank = bank_of([(n, 256, 256) for n in names])
    block = nn.Module()
    block.b = nn.Module()
    block.b.attn = nn.Module()
    for i, n in enumerate(names):
        setattr(block.b.attn, n.split(".")[-1], linear(256, 256, seed=20 * i))
    layers = list(wrap_packed(block, bank, scaling=2.0, int8_base=int8, fused_gemm=not int8).values())
    ids = torch.tensor([1, 4], dtype=torch.int32, device=DEV)
    for m in layers:
        m.assign = ids
    assert layers[0].prep_group is not None
    x = make((2, 128, 256), BF, 1)
    with torch.no_grad():
        layers[0](x)                                 # leaves the other two's results pending
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs = [m(x) for m in layers]
            pending = len(layers[0].prep_group._ready)
        assert pending == 0                          # one preparation, shared among the three
        x.copy_(make((2, 128, 256), BF, 2))
        ids.copy_(torch.tensor([3, 0], dtype=torch.int32, device=DEV))
        other = torch.tensor([5, 5], dtype=torch.int32, device=DEV)
        for m in layers:
            m.assign = other
            m(make((2, 128, 256), BF, 3))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for m, g in zip(layers, got):
            m.assign = ids
            assert torch.equal(m(x), g)


def test_results_shared_on_one_stream_alone():
    """A kept B factor is used on the stream that made it; another stream's call makes its own."""
    bank = bank_of([("m", 256, 512)])
    layer = PackedLoRALinear(linear(256, 512), bank, "m", 16, 2.0, int8_base=True)
    layer.assign = torch.tensor([1, 4], dtype=torch.int32, device=DEV)
    x = make((2, 40, 256), BF, 1)
    with torch.no_grad():
        want = layer(x)
        kept = layer._bdec_cache[1]
        assert torch.equal(layer(x), want) and layer._bdec_cache[1] is kept
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = layer(x)
            assert layer._bdec_cache[1] is not kept
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("batch,n_img,n_txt", [(0, 9, 5), (2, 9, 0), (2, 0, 5), (1, 1, 1)])
def test_model_on_empty_batches_and_streams(batch, n_img, n_txt):
    model, (lat, txt, pooled, t) = tiny(5, False)
    fused, _ = tiny(5, True, model.state_dict())
    args = (lat[:batch, :n_img], txt[:batch, :n_txt], pooled[:batch], t[:batch])
    with torch.no_grad():
        want, got = model(*args), fused(*args)
    assert got.shape == want.shape == (batch, n_img, 16)
    assert got.numel() == 0 or rel_fro(got.float(), want.float()) < 2e-2
