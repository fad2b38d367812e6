"""Rotary positions with several axes, and the per-head RMS norm of q and k in the same pass.

The step between the q / k projections of an attention block and its attention: images and
video give every token one position per axis (time, row, column), each axis turns its own slice
of a head's value pairs, and models of this kind normalise each head of q and k first.

    angle(token, pair) = positions[token, axis] * theta ** (-2 i / axes[axis])

with i the pair's index inside its axis's slice of axes[axis] / 2 pairs (slices in order).
``pairing`` "interleaved" turns neighbours (2p, 2p + 1), "halves" turns p with p + sum(axes) / 2;
values from sum(axes) on are left as they are.  Everything is computed in fp32 (the angle's
revolutions in fp64) and rounded once.

The reference's pipelines take both steps from diffusers; they have no counterpart in it.
Inference only, like the layers.  Both calls run on the current stream of their inputs' device,
allocate nothing but their results, and can be captured into a CUDA graph.
"""
from __future__ import annotations

import functools
import math
import operator
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from . import _launch


def _written(*tensors: torch.Tensor) -> None:
    """Move the version counters of tensors written behind torch's back, as an in-place op does (tensors
    of inference_mode have none and are passed over)."""
    torch.autograd.graph.increment_version(tensors)


@functools.lru_cache(maxsize=256)
def _checked_rotation(dim: int, axes: Tuple[int, ...], theta: float, pairing: str) -> int:
    if pairing not in _launch.PAIRINGS:
        raise ValueError(f"pairing must be one of {tuple(_launch.PAIRINGS)}, got {pairing!r}")
    if not 1 <= len(axes) <= _lib.MAX_AXES:
        raise ValueError(f"1 to {_lib.MAX_AXES} axes, got {len(axes)}")
    if any(a < 0 or a % 2 for a in axes) or sum(axes) > dim:
        raise ValueError(f"the axes' dims {axes} must be even, not negative and sum to at most the head dim {dim}")
    if not (theta > 0.0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive and finite, got {theta}")
    return _launch.PAIRINGS[pairing]


def _rotation(dim: int, axes: Sequence[int], theta: float, pairing: str,
              recorded: bool) -> Tuple[Tuple[int, ...], float, int]:
    """(axes, theta, the pairing's code), plain numbers, checked.  (They are made plain before the lookup: an
    object that can change, a tensor say, is one key with its old value.)"""
    axes, theta = tuple(map(operator.index, axes)), float(theta)
    check = _checked_rotation.__wrapped__ if recorded else _checked_rotation
    return axes, theta, check(dim, axes, theta, pairing)


def rotate_axes(x: torch.Tensor, positions: torch.Tensor, axes: Sequence[int], *, theta: float = 10000.0,
                pairing: str = "interleaved", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (batch, tokens, heads, dim) with every head turned by its token's positions.

    ``positions`` (tokens, len(axes)), or (batch, tokens, len(axes)) for positions of each
    sample's own; int32, int64 or float32, on x's device.  ``axes``: the head's values each axis
    turns (even, summing to at most dim); dim even, at most 256.  x is bfloat16, float16 or
    float32, with any strides over samples, tokens and heads (a slice of a fused q / k / v
    projection).  The result is a new tensor, or ``out``: x itself to rotate in place, or memory
    apart from x and the positions.
    """
    _launch._check_heads(x, "x")
    _launch.inference_only(x, positions, out)
    as_op = _launch.recorded(x)
    axes, theta, code = _rotation(x.shape[3], axes, theta, pairing, as_op)
    fresh = out is None
    if fresh:
        out = x.new_empty(x.shape)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if as_op:
        if out is x:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            torch.ops.lithe_b200.rotate_axes_(out, x, positions, list(axes), theta, code)
            return x.copy_(out)
        torch.ops.lithe_b200.rotate_axes_(out, x, positions, list(axes), theta, code)
        return out
    _launch.rotate_axes_(x, out, positions, axes, theta, code, True, fresh)
    if not fresh:
        _written(out)
    return out


def qk_norm_rotate(q: torch.Tensor, k: torch.Tensor, weight_q: Optional[torch.Tensor],
                   weight_k: Optional[torch.Tensor], positions: torch.Tensor, axes: Sequence[int], *,
                   theta: float = 10000.0, eps: float = 1e-6, pairing: str = "interleaved",
                   out_q: Optional[torch.Tensor] = None,
                   out_k: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, k) with every head RMS-normalised, weighted and turned by its token's positions.

    q (batch, tokens, heads, dim) and k (batch, tokens, kv_heads, dim), any strides over the
    first three dimensions.  ``weight_q`` / ``weight_k`` (dim,) of q's type or float32, or None
    for a norm without weights.  ``positions``, ``axes``, ``theta`` and ``pairing`` as in
    ``rotate_axes``.  The results are new tensors, or ``out_q`` / ``out_k``: slices of a joint
    [text; image] buffer, or q and k themselves (apart from all else that the call reads).
    """
    _launch._check_heads(q, "q")
    _launch._check_heads(k, "k", q)
    _launch.inference_only(q, k, weight_q, weight_k, positions, out_q, out_k)
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative, got {eps}")
    as_op = _launch.recorded(q)
    axes, theta, code = _rotation(q.shape[3], axes, theta, pairing, as_op)
    fresh = out_q is None and out_k is None
    if out_q is None:
        out_q = q.new_empty(q.shape)
    if out_k is None:
        out_k = k.new_empty(k.shape)
    if not positions.is_contiguous():
        positions = positions.contiguous()
    if as_op:
        oq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out_q is q else out_q
        ok = torch.empty(k.shape, dtype=k.dtype, device=k.device) if out_k is k else out_k
        torch.ops.lithe_b200.qk_norm_rotate_(oq, ok, q, k, weight_q, weight_k, positions, list(axes), theta, eps, code)
        return (q.copy_(oq) if out_q is q else oq), (k.copy_(ok) if out_k is k else ok)
    _launch.qk_norm_rotate_(q, k, out_q, out_k, weight_q, weight_k, positions, axes, theta, eps, code, True, fresh)
    if not fresh:
        _written(out_q, out_k)
    return out_q, out_k
