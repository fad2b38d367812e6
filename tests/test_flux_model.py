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
