"""The FLUX-shaped model's host side without a GPU: recorded on fake CUDA tensors, or plain on the CPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

from lithe_b200.flux_model import FluxConfig, FluxShapedTransformer


def inputs(cfg, batch=2, n_img=9, n_txt=5, device="cuda", dtype=torch.bfloat16):
    return (torch.zeros(batch, n_img, cfg.in_channels, device=device, dtype=dtype),
            torch.zeros(batch, n_txt, cfg.text_dim, device=device, dtype=dtype),
            torch.zeros(batch, cfg.pooled_dim, device=device, dtype=dtype), torch.zeros(batch, device=device))


def fake_model(cfg):
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device("cuda"):
            return FluxShapedTransformer(cfg)
    finally:
        torch.set_default_dtype(torch.float32)


@pytest.mark.parametrize("built", [False, True])
def test_fused_qk_is_one_switch(built):
    """cfg.fused_qk alone decides the form, whatever it was when the model was built: a fused call for each
    stream of each block, or none."""
    with FakeTensorMode(), torch.no_grad():
        cfg = FluxConfig.tiny()
        cfg.fused_qk = built
        model, args = fake_model(cfg), inputs(cfg)
        for fused in (not built, built):
            model.cfg.fused_qk = fused
            graph = make_fx(model)(*args).graph
            calls = [n for n in graph.nodes if "qk_norm_rotate_" in str(n.target)]
            assert len(calls) == (2 * cfg.double_blocks + cfg.single_blocks if fused else 0)
            assert model(*args).shape == (2, 9, cfg.in_channels)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("batch,n_img,n_txt", [(0, 9, 5), (2, 9, 0), (2, 0, 5), (1, 1, 1)])
def test_empty_batches_and_streams(batch, n_img, n_txt, fused):
    with FakeTensorMode(), torch.no_grad():
        cfg = FluxConfig.tiny()
        cfg.fused_qk = fused
        got = fake_model(cfg)(*inputs(cfg, batch, n_img, n_txt))
    assert got.shape == (batch, n_img, cfg.in_channels)


@pytest.mark.parametrize("weights,latents", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                             (torch.bfloat16, torch.bfloat16)])
def test_the_time_embedding_has_the_weights_type(weights, latents):
    """Under autocast the latents may have another type than the weights; the embedding goes by the weights."""
    cfg = FluxConfig.tiny()
    model = FluxShapedTransformer(cfg).to(weights)
    seen = []
    model.time_in.register_forward_pre_hook(lambda mod, args: seen.append(args[0].dtype))
    with torch.no_grad(), torch.autocast("cpu", torch.bfloat16):
        model(*inputs(cfg, device="cpu", dtype=latents))
    assert seen == [weights]


def test_the_time_embedding_of_an_8_bit_embedder():
    class Wrapped(torch.nn.Module):                  # an embedder without a weight of its own
        def __init__(self, base):
            super().__init__()
            self.base = base

        def forward(self, x):
            return self.base(x)

    cfg = FluxConfig.tiny()
    model = FluxShapedTransformer(cfg).to(torch.bfloat16)
    model.x_embedder = Wrapped(model.x_embedder)
    with torch.no_grad():
        assert model(*inputs(cfg, device="cpu")).dtype == torch.bfloat16
