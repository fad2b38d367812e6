"""Linear layers on 8-bit integers: activations quantised per token, weights per output channel.

    q[r, k] = x[r, k] * 127 / max |x[r]|  to the nearest whole number, ties to even
    y[r, n] = (q[r] . w[n]) * (max |x[r]| / 127) * scale[n] + bias[n] + h[r] . b_dec[sample(r), n]

The products are summed exactly (int32), the rest in fp32, and y is rounded once.  The last term
is the adapters' rank-16 expand of ``lora_gemm`` (h and b_dec from ``lora_prep``): the base
linear of a served model in half the weight bytes and on the faster tensor-core type, with the
routed adapters still added before the rounding.  No counterpart in the reference.

Inference only, like the layers.  The calls run on the current stream of their inputs' device and
take their results and workspace (a byte per activation and a scale per row) from torch's caching
allocator, so they can be captured into a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _launch


class QuantizedRows(NamedTuple):
    """Activations as 8-bit rows: ``q`` (rows, k) int8, ``scale`` (rows,) fp32, and the leading
    shape and dtype of the tensor they stand for (the shape and dtype of a linear's result)."""
    q: torch.Tensor
    scale: torch.Tensor
    shape: Tuple[int, ...]
    dtype: torch.dtype


def quantize_rows(x: torch.Tensor) -> QuantizedRows:
    """x (..., k) bfloat16 or float16 as 8-bit rows, each with its own scale.

    Linears that read the same x can share the result (``int8_linear`` takes it in x's place).
    A row with an infinity or a NaN gets scale NaN, so every result of it is NaN.
    """
    _launch._require_cuda(x, "x")
    if x.dtype not in _launch.ACTIVATION_DTYPES:
        raise TypeError(f"x must be one of {_launch.ACTIVATION_DTYPES}, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., k) with k >= 1, got {tuple(x.shape)}")
    _launch.inference_only(x)
    k = x.shape[-1]
    if x.numel() // k > _launch._MOST:
        raise NotImplementedError(f"x: {x.numel() // k} rows are above {_launch._MOST}")
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    if k > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    if _launch.recorded(x):
        q, scale = torch.ops.lithe_b200.quantize_rows(x2)
    else:
        q = torch.empty(x2.shape[0], _launch.padded(k), dtype=torch.int8, device=x.device)[:, :k]
        scale = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
        _launch.quantize_rows_(x2, q, scale)
    return QuantizedRows(q, scale, tuple(x.shape[:-1]), x.dtype)


def quantize_weight(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """A linear's weight (n, k), bfloat16 or float16, as (int8 weight (n, k), scale (n,) fp32) for
    ``int8_linear``.  The int8 rows start on 16-byte boundaries (their stride is k rounded up)."""
    if weight.dim() != 2:
        raise ValueError(f"weight must be (n, k), got {tuple(weight.shape)}")
    got = quantize_rows(weight.detach())
    _launch.laid_out(got.q)
    return got.q, got.scale


def int8_linear(x: Union[torch.Tensor, QuantizedRows], weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, *, h: Optional[torch.Tensor] = None,
                b_dec: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (..., k) times the int8 ``weight`` (n, k), plus bias, plus the adapters' expand: (..., n).

    x is bfloat16 or float16 (quantised here, per row) or what ``quantize_rows`` returned; the
    result has its dtype.  ``weight`` and ``weight_scale`` from ``quantize_weight`` (or any int8
    rows that start on 16-byte boundaries, with one fp32 scale each); ``bias`` (n,) of x's dtype.
    ``h`` (rows, 16) and ``b_dec`` (samples, n, 16), both bfloat16 as ``lora_prep`` gives them,
    add h . b_dec[sample]^T; every sample has rows / samples consecutive rows (bfloat16 x only).
    Any number of rows, n >= 1, k up to 131072.
    """
    if isinstance(x, QuantizedRows):
        _launch.inference_only(x.scale, bias, weight_scale, h, b_dec)
        n = weight.shape[0]
        if _launch.recorded(x.q):
            out = torch.ops.lithe_b200.int8_linear(x.q, x.scale, weight, weight_scale, bias, h, b_dec,
                                                   x.dtype == torch.float16)
        else:
            out = torch.empty(x.q.shape[0], n, dtype=x.dtype, device=x.q.device)
            _launch.int8_linear_(x.q, x.scale, weight, weight_scale, bias, out, h, b_dec)
        return out.view(*x.shape, n)
    _launch.inference_only(x, bias, weight_scale, h, b_dec)
    if _launch.recorded(x):
        return torch.ops.lithe_b200.int8_linear_dynamic(x, weight, weight_scale, bias, h, b_dec)
    return _launch.int8_linear_dynamic(x, weight, weight_scale, bias, h, b_dec)
