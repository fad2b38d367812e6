"""Tensor-level wrappers over the C ABI (one function per entry point of include/lithe_b200.h).

They check devices, dtypes and layouts, pass raw device pointers and the current torch
stream to liblithe_b200, and raise on a non-zero return.  No host synchronisation: the
kernels' device-side error word is read only by ``device_errors``.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import struct
import threading
from typing import Optional, Sequence, Tuple

import numpy as np
import torch
from torch.autograd import forward_ad

from .. import _lib

# Activation dtypes the sgmv kernels compute in, and their C-ABI codes.
ACTIVATION_DTYPES = (torch.bfloat16, torch.float16)
_DTYPE_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}

_err_words: dict = {}
_err_lock = threading.Lock()


def error_word(device: torch.device) -> torch.Tensor:
    """The int32 device error word the kernels of ``device`` OR their LITHE_DEVERR_* bits into."""
    t = _err_words.get(getattr(device, "index", None))
    if t is not None:
        return t
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    with _err_lock, torch.inference_mode(False):         # (device_errors clears it in any mode)
        t = _err_words.get(device.index)
        if t is None:
            t = torch.zeros(1, dtype=torch.int32, device=device)
            _err_words[device.index] = t
    return t


def device_errors(device=None, clear: bool = True) -> int:
    """Synchronise with ``device``'s error word and return its LITHE_DEVERR_* bits."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    w = error_word(device)
    val = int(w.item())
    if clear and val:
        w.zero_()
    return val


def raise_device_errors(device=None) -> None:
    bits = device_errors(device)
    if bits:
        names = [n for b, n in ((_lib.DEVERR_SLOT, "adapter slot out of range"),
                                (_lib.DEVERR_INDEX, "index outside [0, 512) in an integer bank"),
                                (_lib.DEVERR_TIMEOUT, "pipeline wait timed out")) if bits & b]
        raise ValueError("lithe_b200 kernel reported: " + "; ".join(names))


def _require_cuda(t: torch.Tensor, what: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor (lithe_b200 has no CPU path), got {t.device}")


_SMS: dict = {}


def _sm_count(device: torch.device) -> int:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    if idx not in _SMS:
        _SMS[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _SMS[idx]


# The current stream's handle without the Python object around it (which costs more than a launch).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_handle(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def ordered_after(device: torch.device) -> Optional[Tuple[int, int]]:
    """What a later call must share with this one to find its results made: the current stream and the
    CUDA-graph capture in progress there (0 for none).  None when the stream cannot be queried."""
    stream = stream_handle(device)
    capture = _lib.lib().lithe_capture_id(stream)
    return None if capture < 0 else (stream, capture)


_tracing_state = getattr(torch._C, "_get_tracing_state", lambda: None)
_dispatch_modes = getattr(torch._C, "_len_torch_dispatch_stack", lambda: 0)
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def recorded(t: torch.Tensor) -> bool:
    """Whether a call on ``t`` is recorded or interpreted instead of only run -- torch.compile, jit.trace, a
    dispatch mode (make_fx, FakeTensorMode), a tensor subclass -- so that it must reach its kernel as a torch op."""
    return (torch.compiler.is_compiling() or _tracing_state() is not None or _dispatch_modes() > 0
            or type(t) not in _PLAIN)


def laid_out(t: torch.Tensor) -> None:
    """Called where weights or banks are laid out: ``t``'s device gets its error word, so that no graph capture is
    the first to need it.  A word made inside one is zeroed, with the errors in it, by every replay."""
    if t.is_cuda and not recorded(t):
        error_word(t.device)


def differentiated(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether a derivative through one of the tensors is being recorded: it requires a gradient while grad mode
    is on, or carries a forward-mode tangent.  The kernels have none to give."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if getattr(forward_ad, "_current_level", -1) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def inference_only(*tensors: Optional[torch.Tensor]) -> None:
    if (torch.is_grad_enabled() or getattr(forward_ad, "_current_level", -1) >= 0) and differentiated(*tensors):
        raise RuntimeError("lithe_b200 operators are inference-only: run them under torch.no_grad()")


_lut_cache: dict = {}


def lut_array(lut) -> ctypes.Array:
    """The level LUT as a ctypes float array (cached per LUT array object; LUTs are immutable)."""
    if isinstance(lut, ctypes.Array):
        return lut
    key = id(lut)
    hit = _lut_cache.get(key)
    if hit is not None and hit[0] is lut:
        return hit[1]
    arr = _lib.float_array(np.asarray(lut, dtype=np.float32).reshape(-1))
    if len(_lut_cache) > 256:
        _lut_cache.clear()
    _lut_cache[key] = (lut, arr)
    return arr


_lut_list_cache: dict = {}


def lut_from_list(lut) -> ctypes.Array:
    """A flat list of LUT floats (the form the custom ops take) as a ctypes array, cached by
    the list's values."""
    key = tuple(float(v) for v in lut)
    arr = _lut_list_cache.get(key)
    if arr is None:
        if len(_lut_list_cache) > 256:
            _lut_list_cache.clear()
        arr = _lib.float_array(key)
        _lut_list_cache[key] = arr
    return arr


_NO_CONTEXT = contextlib.nullcontext()
# The current device without torch.cuda's look at whether CUDA is up (a tensor of the device is at hand).
_raw_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def device_ctx(device: torch.device):
    """torch.cuda.device(device), or a no-op when it is already the current device."""
    if device.index is None or device.index == _raw_device():
        return _NO_CONTEXT
    return torch.cuda.device(device)


def index_view(base: torch.Tensor, fmt: int, levels: int, slot_stride: int, offset: int,
               level_stride: int = 0) -> _lib.IndexView:
    return _lib.IndexView(base.data_ptr(), fmt, levels, slot_stride, offset, level_stride)


def level_major_view(idx: torch.Tensor) -> _lib.IndexView:
    """View of an (n_slots, L, n_blocks) int16/int32 contiguous bank."""
    fmt = {torch.int16: _lib.IDX_I16, torch.int32: _lib.IDX_I32}.get(idx.dtype)
    if fmt is None or idx.dim() != 3 or not idx.is_contiguous():
        raise ValueError("integer index banks must be contiguous (n_slots, L, n_blocks) int16/int32")
    return index_view(idx, fmt, idx.shape[1], idx.shape[1] * idx.shape[2], 0, idx.shape[2])


# Which form of the fused op the layers use: "fused" decodes the factor chunks inside the SGMV
# kernel for every 64-token tile (lithe_sgmv_index); "staged" decodes each routed adapter's
# chunks once per call into a workspace (lithe_sgmv_index_ws) and streams them with the tiles.
# Results are bit-identical; on B200 the fused form is faster on every FLUX shape measured
# (the staged main loop pays a second bulk copy per stage), so it is the default.
DEFAULT_MODE = "fused"


def workspace_bytes(batch: int, d_in: int, d_out: int) -> int:
    return int(_lib.lib().lithe_sgmv_workspace_bytes(batch, d_in, d_out))


def sgmv_index_(x: torch.Tensor, out: torch.Tensor, *, accumulate: bool, view_a: _lib.IndexView,
                view_b: _lib.IndexView, n_slots: int, ids: torch.Tensor, weights: Optional[torch.Tensor],
                rank: int, lut: np.ndarray, scaling: float, err: Optional[torch.Tensor] = None,
                mode: Optional[str] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lithe_sgmv_index(_typed, _ws) on torch tensors; ``out`` (B, M, d_out) is written in place.

    x is bfloat16 or float16; out has x's dtype, or float32 when ``accumulate`` is False (the
    delta alone, lithe_sgmv_index_typed).  ``mode`` "fused" or "staged" (None: DEFAULT_MODE);
    a staged call (bf16 only) takes ``workspace`` (uint8 CUDA tensor) or allocates one from
    torch's caching allocator.
    """
    _require_cuda(x, "x")
    if x.dtype not in ACTIVATION_DTYPES:
        raise TypeError(f"x must be one of {ACTIVATION_DTYPES}, got {x.dtype}")
    if out.dtype != x.dtype and not (out.dtype == torch.float32 and not accumulate):
        raise TypeError(f"out must have x's dtype ({x.dtype}), or float32 when not accumulating; got {out.dtype}")
    if x.dim() != 3 or out.dim() != 3 or x.shape[:2] != out.shape[:2]:
        raise ValueError(f"x (B, M, d_in) and out (B, M, d_out) disagree: {tuple(x.shape)} vs {tuple(out.shape)}")
    if not (x.is_contiguous() and out.is_contiguous()):
        raise ValueError("x and out must be contiguous")
    if out.device != x.device or ids.device != x.device:
        raise ValueError("x, out and ids must be on the same device")
    if ids.dtype != torch.int32 or ids.dim() != 1 or ids.numel() != x.shape[0] or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous (B,) int32 tensor")
    if weights is not None and (weights.dtype != torch.float32 or weights.device != x.device
                                or weights.numel() != x.shape[0] or not weights.is_contiguous()):
        raise ValueError("weights must be a contiguous (B,) float32 tensor on x's device")
    if err is None:
        err = error_word(x.device)
    bsz, m, d_in = x.shape
    mode = mode or DEFAULT_MODE
    if mode not in ("staged", "fused"):
        raise ValueError(f"mode must be 'staged' or 'fused', got {mode!r}")
    common = (x.data_ptr(), out.data_ptr(), 1 if accumulate else 0, ctypes.byref(view_a), ctypes.byref(view_b),
              int(n_slots), ids.data_ptr(), weights.data_ptr() if weights is not None else None,
              bsz, m, d_in, out.shape[2], int(rank), lut_array(lut), float(scaling), err.data_ptr())
    typed = x.dtype != torch.bfloat16 or out.dtype != torch.bfloat16
    if typed and mode == "staged":
        raise NotImplementedError("the staged form takes bfloat16 x and out")
    with torch.cuda.device(x.device):
        if typed:
            rc = _lib.lib().lithe_sgmv_index_typed(*common[:-1], _DTYPE_CODE[x.dtype], _DTYPE_CODE[out.dtype],
                                                   common[-1], stream_handle(x.device))
        elif mode == "fused":
            rc = _lib.lib().lithe_sgmv_index(*common, stream_handle(x.device))
        else:
            need = workspace_bytes(bsz, d_in, out.shape[2])
            if workspace is None or workspace.numel() < need:
                workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)
            _require_cuda(workspace, "workspace")
            rc = _lib.lib().lithe_sgmv_index_ws(*common, workspace.data_ptr(), workspace.numel(),
                                                stream_handle(x.device))
    _lib.check(rc, "lithe_sgmv_index_typed" if typed else "lithe_sgmv_index" if mode == "fused"
               else "lithe_sgmv_index_ws")
    return out


def decode_packed_(words: torch.Tensor, n_blocks: int, levels: int, sides: Optional[torch.Tensor],
                   lut: np.ndarray, out: torch.Tensor) -> torch.Tensor:
    _require_cuda(words, "words")
    if words.dtype not in (torch.int64, torch.uint64) or not words.is_contiguous():
        raise ValueError("words must be a contiguous 64-bit tensor")
    if out.dtype not in (torch.bfloat16, torch.float32) or not out.is_contiguous():
        raise ValueError("out must be a contiguous bfloat16/float32 tensor")
    if out.numel() != n_blocks * 64:
        raise ValueError("out must hold n_blocks * 64 values")
    if words.numel() * 7 < n_blocks * levels:
        raise ValueError(f"words ({words.numel()}) too short for {n_blocks} blocks x {levels} levels")
    if sides is not None and (sides.dtype != torch.int8 or sides.numel() != n_blocks or sides.device != words.device):
        raise ValueError("sides must be an int8 tensor with one entry per block on the words' device")
    with torch.cuda.device(words.device):
        rc = _lib.lib().lithe_decode_packed(
            words.data_ptr(), int(n_blocks), int(levels), sides.data_ptr() if sides is not None else None,
            lut_array(lut), out.data_ptr(), _lib.DTYPE_F32 if out.dtype == torch.float32 else _lib.DTYPE_BF16,
            stream_handle(words.device))
    _lib.check(rc, "lithe_decode_packed")
    return out


def decode_packed_batch_(bank: torch.Tensor, slot_ids: torch.Tensor, n_blocks: int, levels: int,
                         sides: Optional[torch.Tensor], lut: np.ndarray, out: torch.Tensor,
                         err: Optional[torch.Tensor] = None) -> torch.Tensor:
    _require_cuda(bank, "bank")
    if bank.dim() != 2 or bank.dtype not in (torch.int64, torch.uint64) or not bank.is_contiguous():
        raise ValueError("bank must be a contiguous (n_slots, slot_stride) 64-bit tensor")
    if slot_ids.dtype != torch.int32 or slot_ids.device != bank.device or not slot_ids.is_contiguous():
        raise ValueError("slot_ids must be a contiguous int32 tensor on the bank's device")
    if out.dtype not in (torch.bfloat16, torch.float32) or not out.is_contiguous() \
            or out.numel() != slot_ids.numel() * n_blocks * 64:
        raise ValueError("out must be a contiguous (n_sel, n_blocks, 64) bfloat16/float32 tensor")
    if err is None:
        err = error_word(bank.device)
    with torch.cuda.device(bank.device):
        rc = _lib.lib().lithe_decode_packed_batch(
            bank.data_ptr(), bank.shape[1], bank.shape[0], slot_ids.data_ptr(), slot_ids.numel(), int(n_blocks),
            int(levels), sides.data_ptr() if sides is not None else None, lut_array(lut), out.data_ptr(),
            _lib.DTYPE_F32 if out.dtype == torch.float32 else _lib.DTYPE_BF16, err.data_ptr(),
            stream_handle(bank.device))
    _lib.check(rc, "lithe_decode_packed_batch")
    return out


def pack_raw_(raw: torch.Tensor, segments: torch.Tensor, levels: int, words: torch.Tensor,
              err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lithe_pack_raw: raw (n,) uint16/int16 payload on the device -> packed ``words`` in place.

    ``segments`` is the (n_segments, 3) int64 device table of (raw_offset, first_block, n_blocks).
    """
    _require_cuda(raw, "raw")
    if raw.dtype not in (torch.int16, torch.uint16) or raw.dim() != 1 or not raw.is_contiguous():
        raise ValueError("raw must be a contiguous 1-D 16-bit tensor")
    if segments.dtype != torch.int64 or segments.dim() != 2 or segments.shape[1] != 3 \
            or not segments.is_contiguous() or segments.device != raw.device:
        raise ValueError("segments must be a contiguous (n, 3) int64 tensor on raw's device")
    if words.dtype not in (torch.int64, torch.uint64) or not words.is_contiguous() or words.device != raw.device:
        raise ValueError("words must be a contiguous 64-bit tensor on raw's device")
    if err is None:
        err = error_word(raw.device)
    with torch.cuda.device(raw.device):
        rc = _lib.lib().lithe_pack_raw(raw.data_ptr(), raw.numel(), segments.data_ptr(), segments.shape[0],
                                       int(levels), words.data_ptr(), words.numel(), err.data_ptr(),
                                       stream_handle(raw.device))
    _lib.check(rc, "lithe_pack_raw")
    return words


def lora_gemm_(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], out: torch.Tensor,
               h: Optional[torch.Tensor] = None, b_dec: Optional[torch.Tensor] = None, rows_per_sample: int = 0,
               err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lithe_lora_gemm: out (rows, n) = x (rows, k) . weight^T + bias [+ h . b_dec[sample]^T], bf16."""
    _require_cuda(x, "x")
    for t, name in ((x, "x"), (weight, "weight"), (out, "out")):
        if t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != x.device:
            raise ValueError(f"{name} must be a contiguous bfloat16 tensor on x's device")
    if x.dim() != 2 or weight.dim() != 2 or out.dim() != 2:
        raise ValueError("x (rows, k), weight (n, k) and out (rows, n) must be 2-D")
    rows, k = x.shape
    n = weight.shape[0]
    if weight.shape[1] != k or tuple(out.shape) != (rows, n):
        raise ValueError(f"shapes disagree: x {tuple(x.shape)}, weight {tuple(weight.shape)}, out {tuple(out.shape)}")
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.numel() != n or not bias.is_contiguous()):
        raise ValueError("bias must be a contiguous (n,) bfloat16 tensor")
    rank = 0
    if h is not None:
        if b_dec is None or h.dtype != torch.bfloat16 or b_dec.dtype != torch.bfloat16 \
                or not h.is_contiguous() or not b_dec.is_contiguous():
            raise ValueError("h and b_dec must be contiguous bfloat16 tensors")
        rank = h.shape[-1]
        if h.numel() != rows * rank or b_dec.shape[-2:] != (n, rank):
            raise ValueError("h must be (rows, rank) and b_dec (samples, n, rank)")
    if err is None:
        err = error_word(x.device)
    with device_ctx(x.device):
        rc = _lib.lib().lithe_lora_gemm(
            x.data_ptr(), weight.data_ptr(), bias.data_ptr() if bias is not None else None, out.data_ptr(), rows, n,
            k, h.data_ptr() if h is not None else None, b_dec.data_ptr() if b_dec is not None else None,
            int(rows_per_sample), int(rank), err.data_ptr(), stream_handle(x.device))
    _lib.check(rc, "lithe_lora_gemm")
    return out


def prep_workspace_bytes(batch: int, m: int, d_in: int) -> int:
    """Bytes of workspace the split shrink of lithe_lora_prep_ws needs on the current device."""
    n = int(_lib.lib().lithe_lora_prep_workspace_bytes(batch, m, d_in))
    if n < 0:
        _lib.check(n, "lithe_lora_prep_workspace_bytes")
    return n


# The split shrink's cross-CTA combine costs about as much as 20-30 stages of x streaming
# (measured on B200: at 14 x 4096 x 3072 the split and whole-tile forms time the same, with the
# busiest whole-tile CTA 23 stages above the average; at 14 x 4096 x 12288, 91 stages above,
# the split is 7% faster).  It is taken when the busiest whole-tile CTA would run at least this
# many stages more than the average.
PREP_SPLIT_MIN_GAIN_STAGES = 48


def prep_split_pays(batch: int, m: int, d_in: int, sms: int) -> bool:
    units = -(-m // 64) * batch
    stages = -(-d_in // 128)
    if units <= 0 or sms <= 0:
        return False
    busiest = -(-units // min(units, sms)) * stages
    return busiest - units * stages / min(units * stages, sms) >= PREP_SPLIT_MIN_GAIN_STAGES


def lora_prep_(x: torch.Tensor, *, view_a: _lib.IndexView, view_b: _lib.IndexView, n_slots: int, ids: torch.Tensor,
               weights: Optional[torch.Tensor], d_out: int, lut: np.ndarray, scaling: float,
               h: Optional[torch.Tensor], b_dec: Optional[torch.Tensor], err: Optional[torch.Tensor] = None,
               split: Optional[bool] = None, workspace: Optional[torch.Tensor] = None) -> None:
    """lithe_lora_prep: h (B*M, 16) and b_dec (B, d_out, 16), bf16, for lithe_lora_gemm's fused expand.
    Either may be None to skip its half (not both).  With ``split`` h comes from
    lithe_lora_prep_ws, whose CTAs take equal runs of the x stages rather than of 64-token
    tiles; ``workspace`` (uint8 CUDA tensor of at least prep_workspace_bytes) is then used,
    or one is allocated from torch's caching allocator.  ``split=None`` takes the split where
    prep_split_pays says so."""
    _require_cuda(x, "x")
    if x.dtype != torch.bfloat16 or x.dim() != 3 or not x.is_contiguous():
        raise ValueError("x must be a contiguous (B, M, d_in) bfloat16 tensor")
    bsz, m, d_in = x.shape
    if h is None and b_dec is None:
        raise ValueError("h and b_dec are both None")
    if h is not None and (h.dtype != torch.bfloat16 or h.numel() != bsz * m * 16 or not h.is_contiguous()
                          or h.device != x.device):
        raise ValueError("h must be a contiguous (B*M, 16) bfloat16 tensor on x's device")
    if b_dec is not None and (b_dec.dtype != torch.bfloat16 or b_dec.numel() != bsz * d_out * 16
                              or not b_dec.is_contiguous() or b_dec.device != x.device):
        raise ValueError("b_dec must be a contiguous (B, d_out, 16) bfloat16 tensor on x's device")
    if ids.dtype != torch.int32 or ids.numel() != bsz or ids.device != x.device or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous (B,) int32 tensor on x's device")
    if err is None:
        err = error_word(x.device)
    with device_ctx(x.device):
        common = (x.data_ptr(), ctypes.byref(view_a), ctypes.byref(view_b), int(n_slots), ids.data_ptr(),
                  weights.data_ptr() if weights is not None else None, bsz, m, d_in, int(d_out), 16, lut_array(lut),
                  float(scaling), h.data_ptr() if h is not None else None,
                  b_dec.data_ptr() if b_dec is not None else None, err.data_ptr())
        if split is None:
            split = prep_split_pays(bsz, m, d_in, _sm_count(x.device))
        if split and h is not None and bsz * m > 0:
            if workspace is None:
                workspace = torch.empty(max(prep_workspace_bytes(bsz, m, d_in), 16), dtype=torch.uint8,
                                        device=x.device)
            _require_cuda(workspace, "workspace")
            rc = _lib.lib().lithe_lora_prep_ws(*common, workspace.data_ptr(), workspace.numel(),
                                                stream_handle(x.device))
            _lib.check(rc, "lithe_lora_prep_ws")
        else:
            rc = _lib.lib().lithe_lora_prep(*common, stream_handle(x.device))
            _lib.check(rc, "lithe_lora_prep")


def prep_multi_workspace_bytes(batch: int, d_in: int, n_targets: int) -> int:
    return int(_lib.lib().lithe_lora_prep_multi_workspace_bytes(batch, d_in, n_targets))


def lora_prep_multi_(x: torch.Tensor, *, views_a: Sequence[_lib.IndexView], views_b: Sequence[_lib.IndexView],
                     d_outs: Sequence[int], n_slots: int, ids: torch.Tensor, weights: Optional[torch.Tensor],
                     lut: np.ndarray, scalings: Sequence[float], hs: Sequence[torch.Tensor],
                     b_decs: Sequence[Optional[torch.Tensor]], err: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None) -> None:
    """lithe_lora_prep_multi: h and b_dec of up to 4 rank-16 linears that read the same x, with
    x streamed once.  hs[t] (B*M, 16) and b_decs[t] (B, d_outs[t], 16) are bf16; a b_dec entry
    may be None."""
    _require_cuda(x, "x")
    if x.dtype != torch.bfloat16 or x.dim() != 3 or not x.is_contiguous():
        raise ValueError("x must be a contiguous (B, M, d_in) bfloat16 tensor")
    n = len(views_a)
    if not (1 <= n <= 4) or not (len(views_b) == len(d_outs) == len(scalings) == len(hs) == len(b_decs) == n):
        raise ValueError("1 to 4 targets, with one view pair, d_out, scaling, h and b_dec each")
    bsz, m, d_in = x.shape
    for h, bd, d_out in zip(hs, b_decs, d_outs):
        if h.dtype != torch.bfloat16 or h.numel() != bsz * m * 16 or not h.is_contiguous() or h.device != x.device:
            raise ValueError("every h must be a contiguous (B*M, 16) bfloat16 tensor on x's device")
        if bd is not None and (bd.dtype != torch.bfloat16 or bd.numel() != bsz * d_out * 16
                               or not bd.is_contiguous() or bd.device != x.device):
            raise ValueError("every b_dec must be a contiguous (B, d_out, 16) bfloat16 tensor on x's device")
    if ids.dtype != torch.int32 or ids.numel() != bsz or ids.device != x.device or not ids.is_contiguous():
        raise ValueError("ids must be a contiguous (B,) int32 tensor on x's device")
    if err is None:
        err = error_word(x.device)
    if workspace is None:
        workspace = torch.empty(max(prep_multi_workspace_bytes(bsz, d_in, n), 16), dtype=torch.uint8,
                                device=x.device)
    _require_cuda(workspace, "workspace")
    va = (_lib.IndexView * n)(*views_a)
    vb = (_lib.IndexView * n)(*views_b)
    with device_ctx(x.device):
        rc = _lib.lib().lithe_lora_prep_multi(
            x.data_ptr(), n, va, vb, (ctypes.c_int32 * n)(*[int(d) for d in d_outs]), int(n_slots), ids.data_ptr(),
            weights.data_ptr() if weights is not None else None, bsz, m, d_in, 16, lut_array(lut),
            (ctypes.c_float * n)(*[float(v) for v in scalings]), (ctypes.c_void_p * n)(*[h.data_ptr() for h in hs]),
            (ctypes.c_void_p * n)(*[bd.data_ptr() if bd is not None else None for bd in b_decs]), err.data_ptr(),
            workspace.data_ptr(), workspace.numel(), stream_handle(x.device))
    _lib.check(rc, "lithe_lora_prep_multi")


def pack_raw_batch_(raw: torch.Tensor, segments: torch.Tensor, levels: int, bank: torch.Tensor,
                    slot_ids: Optional[torch.Tensor], n_words: int, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lithe_pack_raw_batch: raw (n, payload) 16-bit rows -> bank rows slot_ids[i] (words [0, n_words))."""
    _require_cuda(raw, "raw")
    if raw.dtype not in (torch.int16, torch.uint16) or raw.dim() != 2 or raw.stride(1) != 1 or raw.stride(0) % 8:
        raise ValueError("raw must be a (n, payload) 16-bit tensor with unit inner stride and an 8-aligned row stride")
    if segments.dtype != torch.int64 or segments.dim() != 2 or segments.shape[1] != 3 \
            or not segments.is_contiguous() or segments.device != raw.device:
        raise ValueError("segments must be a contiguous (n, 3) int64 tensor on raw's device")
    if bank.dim() != 2 or bank.dtype not in (torch.int64, torch.uint64) or not bank.is_contiguous() \
            or bank.device != raw.device:
        raise ValueError("bank must be a contiguous (n_slots, slot_stride) 64-bit tensor on raw's device")
    if slot_ids is not None and (slot_ids.dtype != torch.int32 or slot_ids.numel() != raw.shape[0]
                                 or not slot_ids.is_contiguous() or slot_ids.device != raw.device):
        raise ValueError("slot_ids must be a contiguous (n,) int32 tensor on raw's device")
    if err is None:
        err = error_word(raw.device)
    with device_ctx(raw.device):
        rc = _lib.lib().lithe_pack_raw_batch(
            raw.data_ptr(), raw.stride(0), raw.shape[0], raw.shape[1], segments.data_ptr(), segments.shape[0],
            int(levels), bank.data_ptr(), bank.shape[1], bank.shape[0],
            slot_ids.data_ptr() if slot_ids is not None else None, int(n_words), err.data_ptr(),
            stream_handle(raw.device))
    _lib.check(rc, "lithe_pack_raw_batch")
    return bank


# ------------------------------------------------------------------------------------------
# Rotation and per-head norm
# ------------------------------------------------------------------------------------------
_POS_CODE = {torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64, torch.float32: _lib.POS_F32}
PAIRINGS = {"interleaved": _lib.PAIR_INTERLEAVED, "halves": _lib.PAIR_HALVES}


@functools.lru_cache(maxsize=256)
def _axis_arrays(axes: tuple, theta: float) -> tuple:
    """The axes' dims and the pairs' frequencies theta^(-2 i / dim), as the C entries take them."""
    freqs = [theta ** (-2.0 * i / d) for d in axes for i in range(d // 2)]
    return (ctypes.c_int32 * max(1, len(axes)))(*axes), (ctypes.c_double * max(1, len(freqs)))(*freqs)


_MOST = 2 ** 31 - 1025       # a dimension the C entries take (ctypes would cut a larger one to 32 bits)


def _check_sizes(t: torch.Tensor, name: str) -> None:
    if t.numel() > _MOST and max(t.shape) > _MOST:
        raise NotImplementedError(f"{name}: a dimension of {tuple(t.shape)} is above {_MOST}")


def _heads_strides(t: torch.Tensor) -> tuple:
    """(sample, token, head) strides; a dimension of one element has none that matters."""
    b, s, h, _ = t.shape
    sb, ss, sh, _ = t.stride()
    return (sb if b != 1 else 0, ss if s != 1 else 0, sh if h != 1 else 0)


_pack_view = struct.Struct("PqqqiI").pack


def _heads_layout(t: torch.Tensor, shape: Optional[Sequence[int]] = None,
                  strides: Optional[Sequence[int]] = None) -> tuple:
    """(lithe_heads_view of ``t``, the address of its first byte, the one behind its last, whether its heads,
    tokens and samples follow one another without meeting).  ``shape``, ``strides``: t's, where they are at hand."""
    b, s, h, d = t.shape if shape is None else shape
    sb, ss, sh, _ = t.stride() if strides is None else strides
    apart = True
    inner = d
    if h == 1:
        sh = 0
    else:
        apart = sh >= inner
        inner += (h - 1) * sh
    if s == 1:
        ss = 0
    else:
        apart = apart and ss >= inner
        inner += (s - 1) * ss
    if b == 1:
        sb = 0
    else:
        apart = apart and sb >= inner
        inner += (b - 1) * sb
    first = t.data_ptr()
    return _pack_view(first, sb, ss, sh, h, 0), first, first + inner * t.element_size(), apart


def _output_layout(t: torch.Tensor, name: str, like: torch.Tensor) -> tuple:
    """_heads_layout of an output that the caller gave, checked against the input it belongs to."""
    shape, strides = t.shape, t.stride()
    if not t.is_cuda or t.dtype != like.dtype or t.device != like.device or len(shape) != 4 or strides[3] != 1:
        _check_heads(t, name, like)
    if shape != like.shape:
        raise ValueError(f"{name} must be {tuple(like.shape)}, got {tuple(shape)}")
    return _heads_layout(t, shape, strides)


def _check_heads(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> None:
    if not t.is_cuda:
        _require_cuda(t, name)
    if t.dtype not in _DTYPE_CODE:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    shape = t.shape
    if len(shape) != 4:
        raise ValueError(f"{name} must be (batch, tokens, heads, dim), got {tuple(shape)}")
    if t.numel() > _MOST:
        _check_sizes(t, name)
    if t.stride()[3] != 1 and shape[3] > 1:
        raise ValueError(f"{name}: the values of a head must be contiguous (stride 1), got stride {t.stride(3)}")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have the inputs' type and device ({like.dtype}, {like.device}), got "
                         f"{t.dtype}, {t.device}")


def _has_own_elements(t: torch.Tensor) -> bool:
    """Whether no two of ``t``'s elements share an address (an expanded tensor's do)."""
    reach = 0
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s <= reach:
            return False
        reach += (n - 1) * s
    return True


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two (batch, tokens, heads, dim) tensors certainly share no element: their bytes do
    not meet, or they are slices of one buffer that leave each other's part of every token alone."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    _, a0, a1, _ = _heads_layout(a)
    _, b0, b1, _ = _heads_layout(b)
    if a1 <= b0 or b1 <= a0:
        return True
    sa, sb = _heads_strides(a), _heads_strides(b)
    if a.shape[:2] != b.shape[:2] or sa[:2] != sb[:2]:
        return False
    size = a.element_size()
    if (b0 - a0) % size:
        return False
    inner_a = (a.shape[2] - 1) * sa[2] + a.shape[3]
    inner_b = (b.shape[2] - 1) * sb[2] + b.shape[3]
    spans = []                      # (period both repeat with, what each covers of one period)
    if a.shape[1] > 1:
        if a.shape[0] == 1 or sa[0] % sa[1] == 0:
            spans.append((sa[1], inner_a, inner_b))
        inner_a, inner_b = inner_a + (a.shape[1] - 1) * sa[1], inner_b + (b.shape[1] - 1) * sb[1]
    if a.shape[0] > 1:
        spans.append((sa[0], inner_a, inner_b))
    for period, in_a, in_b in spans:
        d = ((b0 - a0) // size) % period if period > 0 else 0
        if d >= in_a and d + in_b <= period:
            return True
    return False


def _same_view(a: torch.Tensor, b: torch.Tensor) -> bool:
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and _heads_strides(a) == _heads_strides(b)


def _check_outputs(ins: Sequence[torch.Tensor], outs: Sequence[torch.Tensor], names: Sequence[str],
                   layouts: Optional[Sequence[tuple]] = None) -> None:
    """Every output is its own input (in place) or shares no element with an input or another output.
    ``layouts``: _heads_layout of the inputs and the outputs, where they are at hand."""
    n = len(ins)
    if layouts is None:
        layouts = [_heads_layout(t) for t in (*ins, *outs)]
    for i, o in enumerate(outs):
        _, o0, o1, apart = layouts[n + i]
        if not apart and not _has_own_elements(o):
            raise ValueError(f"{names[i]} has elements that share an address")
        for j in range(n + i):
            x = layouts[j]
            if x[2] <= o0 or o1 <= x[1]:
                continue
            if j >= n:
                if not _apart(o, outs[j - n]):
                    raise ValueError(f"{names[i]} overlaps {names[j - n]}")
            elif not (i == j and _same_view(o, ins[j])) and not _apart(o, ins[j]):
                raise ValueError(f"{names[i]} overlaps an input (it may be its own input's very view)")


def _rotation_args(x: torch.Tensor, positions: torch.Tensor, axes: tuple, theta: float, pairing: int) -> tuple:
    code = _POS_CODE.get(positions.dtype)
    if code is None:
        raise TypeError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    if positions.device != x.device:
        raise ValueError("positions must be on the inputs' device")
    b, s = x.shape[:2]
    shape, n = positions.shape, len(axes)
    if shape != (s, n) and shape != (b, s, n):
        raise ValueError(f"positions must be ({s}, {n}) or ({b}, {s}, {n}), got {tuple(shape)}")
    if not positions.is_contiguous():
        raise ValueError("positions must be contiguous")
    dims, freqs = _axis_arrays(axes, theta)
    return positions.data_ptr(), code, len(shape) - 2, dims, n, freqs, pairing, stream_handle(x.device)


def _check_read(first: int, size: int, what: str, out: tuple, name: str) -> None:
    """The output (its _heads_layout) does not reach over ``size`` bytes from ``first`` on, which every token reads."""
    if first < out[2] and out[1] < first + size:
        raise ValueError(f"{name} overlaps {what}")


def rotate_axes_(x: torch.Tensor, out: torch.Tensor, positions: torch.Tensor, axes: Sequence[int], theta: float,
                 pairing: int, checked: bool = False, fresh: bool = False) -> torch.Tensor:
    """lithe_rotate_axes on torch tensors: ``out`` (batch, tokens, heads, dim) is written.  ``checked``: the
    caller has checked x; ``fresh``: and made ``out`` for this call."""
    if not checked:
        _check_heads(x, "x")
    of_x = _heads_layout(x)
    of_out = _heads_layout(out) if fresh else of_x if out is x else _output_layout(out, "out", x)
    if not fresh:
        _check_outputs((x,), (out,), ("out",), (of_x, of_out))
        _check_read(positions.data_ptr(), positions.nbytes, "positions", of_out, "out")
    b, s, _, d = x.shape
    args = (of_x[0], of_out[0], _DTYPE_CODE[x.dtype], b, s, d,
            *_rotation_args(x, positions, tuple(axes), theta, pairing))
    with device_ctx(x.device):
        rc = _lib.lib().lithe_rotate_axes(*args)
    if rc:
        _lib.check(rc, "lithe_rotate_axes")
    return out


def qk_norm_rotate_(q: torch.Tensor, k: torch.Tensor, out_q: torch.Tensor, out_k: torch.Tensor,
                    weight_q: Optional[torch.Tensor], weight_k: Optional[torch.Tensor], positions: torch.Tensor,
                    axes: Sequence[int], theta: float, eps: float, pairing: int, checked: bool = False,
                    fresh: bool = False) -> None:
    """lithe_qk_norm_rotate on torch tensors: ``out_q`` and ``out_k`` are written.  ``checked``: the caller
    has checked q and k; ``fresh``: and made both outputs for this call."""
    if not checked:
        _check_heads(q, "q")
        _check_heads(k, "k", q)
    if fresh:
        layouts = [_heads_layout(t) for t in (q, k, out_q, out_k)]
    else:
        layouts = [_heads_layout(q), _heads_layout(k), _output_layout(out_q, "out_q", q), _output_layout(out_k, "out_k", k)]
        _check_outputs((q, k), (out_q, out_k), ("out_q", "out_k"), layouts)
    b, s, _, d = q.shape
    kb, ks, _, kd = k.shape
    if kb != b or ks != s or kd != d:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in batch, tokens and dim")
    dtype = weight_dtype = q.dtype
    for w, name in ((weight_q, "weight_q"), (weight_k, "weight_k")):
        if w is None:
            continue
        if w.dtype != dtype and w.dtype != torch.float32:
            raise TypeError(f"{name} must be {dtype} or float32, got {w.dtype}")
        if w.shape != (d,) or w.device != q.device or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous ({d},) tensor on q's device")
        weight_dtype = w.dtype
    if weight_q is not None and weight_k is not None and weight_q.dtype != weight_k.dtype:
        raise TypeError(f"weight_q and weight_k must have one type, got {weight_q.dtype} and {weight_k.dtype}")
    of_q, of_k, of_out_q, of_out_k = layouts
    at_q = weight_q.data_ptr() if weight_q is not None else None
    at_k = weight_k.data_ptr() if weight_k is not None else None
    if not fresh:
        lo, hi = min(of_out_q[1], of_out_k[1]), max(of_out_q[2], of_out_k[2])
        for t, first, what in ((positions, positions.data_ptr(), "positions"), (weight_q, at_q, "weight_q"), (weight_k, at_k, "weight_k")):
            if first is None or first >= hi or first + t.nbytes <= lo:
                continue
            _check_read(first, t.nbytes, what, of_out_q, "out_q")
            _check_read(first, t.nbytes, what, of_out_k, "out_k")
    args = (of_q[0], of_k[0], of_out_q[0], of_out_k[0], at_q, at_k, _DTYPE_CODE[weight_dtype], eps,
            _DTYPE_CODE[dtype], b, s, d, *_rotation_args(q, positions, tuple(axes), theta, pairing))
    with device_ctx(q.device):
        rc = _lib.lib().lithe_qk_norm_rotate(*args)
    if rc:
        _lib.check(rc, "lithe_qk_norm_rotate")


# ------------------------------------------------------------------------------------------
# 8-bit integer linear
# ------------------------------------------------------------------------------------------
def quantize_rows_(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """lithe_quantize_rows: x (rows, k) bf16 / fp16 -> q (rows, k) int8 and scale (rows,) fp32."""
    _require_cuda(x, "x")
    if x.dtype not in ACTIVATION_DTYPES:
        raise TypeError(f"x must be one of {ACTIVATION_DTYPES}, got {x.dtype}")
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"x must be (rows, k) with contiguous rows, got {tuple(x.shape)}, strides {x.stride()}")
    if q.shape != x.shape or q.dtype != torch.int8 or q.device != x.device or (q.shape[1] > 1 and q.stride(1) != 1):
        raise ValueError("q must be an int8 tensor of x's shape with contiguous rows, on x's device")
    if scale.dtype != torch.float32 or scale.numel() != x.shape[0] or not scale.is_contiguous() \
            or scale.device != x.device:
        raise ValueError("scale must be a contiguous (rows,) float32 tensor on x's device")
    _check_sizes(x, "x")
    rows, k = x.shape
    with device_ctx(x.device):
        rc = _lib.lib().lithe_quantize_rows(x.data_ptr(), _DTYPE_CODE[x.dtype], rows, k,
                                            x.stride(0) if rows > 1 else 0, q.data_ptr(),
                                            q.stride(0) if rows > 1 else padded(k), scale.data_ptr(),
                                            stream_handle(x.device))
    _lib.check(rc, "lithe_quantize_rows")


def padded(k: int) -> int:
    """Bytes between the starts of 8-bit rows of k values: rows start on 16-byte boundaries."""
    return -(-k // 16) * 16


def _int8_weight(weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor], dtype: torch.dtype,
                 dev: torch.device, k: int) -> tuple:
    """The checks of a linear's int8 weight, scale and bias; (n, bytes between the weight's rows)."""
    if weight.dtype != torch.int8 or weight.device != dev:
        raise TypeError(f"weight must be int8 on {dev}, got {weight.dtype} on {weight.device}")
    if weight.dim() != 2 or weight.shape[1] != k:
        raise ValueError(f"weight must be (n, {k}), got {tuple(weight.shape)}")
    if weight.numel() > _MOST:
        _check_sizes(weight, "weight")
    n = weight.shape[0]
    stride, inner = weight.stride()
    if n == 1:
        stride = padded(k)
    if (k > 1 and inner != 1) or stride % 16 or weight.data_ptr() % 16:
        raise ValueError("weight: int8 rows must be contiguous and start on 16-byte boundaries "
                         f"(strides {weight.stride()})")
    if weight_scale.dtype != torch.float32 or weight_scale.numel() != n or not weight_scale.is_contiguous() \
            or weight_scale.device != dev:
        raise ValueError(f"weight_scale must be a contiguous ({n},) float32 tensor on x's device")
    if bias is not None and (bias.dtype != dtype or bias.numel() != n or not bias.is_contiguous()
                             or bias.device != dev):
        raise ValueError(f"bias must be a contiguous ({n},) {dtype} tensor on x's device")
    return n, stride


_NO_EXPAND = (None, None, 0, 0)


def _int8_expand(h: Optional[torch.Tensor], b_dec: Optional[torch.Tensor], rows: int, n: int,
                 dev: torch.device) -> tuple:
    """The checks of the expand's operands; their (h, b_dec, rows per sample, rank) arguments."""
    if h is None and b_dec is None:
        return _NO_EXPAND
    if h is None or b_dec is None:
        raise ValueError("h and b_dec come together")
    for t, name in ((h, "h"), (b_dec, "b_dec")):
        if t.dtype != torch.bfloat16 or not t.is_contiguous() or t.device != dev:
            raise ValueError(f"{name} must be a contiguous bfloat16 tensor on x's device")
    if h.dim() != 2 or h.shape[0] != rows or b_dec.dim() != 3 or b_dec.shape[1] != n \
            or b_dec.shape[2] != h.shape[1]:
        raise ValueError(f"h must be ({rows}, rank) and b_dec (samples, {n}, rank), got {tuple(h.shape)} and "
                         f"{tuple(b_dec.shape)}")
    samples = b_dec.shape[0]
    if rows and (samples == 0 or rows % samples):
        raise ValueError(f"b_dec's {samples} samples do not divide {rows} rows")
    return h.data_ptr(), b_dec.data_ptr(), rows // samples if samples else 0, h.shape[1]


def int8_linear_(q: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                 bias: Optional[torch.Tensor], out: torch.Tensor, h: Optional[torch.Tensor] = None,
                 b_dec: Optional[torch.Tensor] = None, err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lithe_int8_linear: out (rows, n) from q (rows, k), x_scale (rows,), weight (n, k), weight_scale (n,)."""
    _require_cuda(q, "q")
    dev = q.device
    if q.dim() != 2 or q.dtype != torch.int8:
        raise ValueError(f"q must be (rows, k) int8, got {tuple(q.shape)} {q.dtype}")
    _check_sizes(q, "q")
    rows, k = q.shape
    q_stride = q.stride(0) if rows > 1 else padded(k)
    if (k > 1 and q.stride(1) != 1) or q_stride % 16 or q.data_ptr() % 16:
        raise ValueError(f"q: int8 rows must be contiguous and start on 16-byte boundaries (strides {q.stride()})")
    n, w_stride = _int8_weight(weight, weight_scale, bias, out.dtype, dev, k)
    if out.dtype not in ACTIVATION_DTYPES or out.shape != (rows, n) or not out.is_contiguous() or out.device != dev:
        raise ValueError(f"out must be a contiguous ({rows}, {n}) bfloat16 or float16 tensor on q's device")
    if x_scale.dtype != torch.float32 or x_scale.numel() != rows or not x_scale.is_contiguous() \
            or x_scale.device != dev:
        raise ValueError(f"x_scale must be a contiguous ({rows},) float32 tensor on q's device")
    expand = _int8_expand(h, b_dec, rows, n, dev)
    if rows == 0:
        return out
    if err is None:
        err = error_word(dev)
    with device_ctx(dev):
        rc = _lib.lib().lithe_int8_linear(
            q.data_ptr(), q_stride, x_scale.data_ptr(), weight.data_ptr(), w_stride, weight_scale.data_ptr(),
            bias.data_ptr() if bias is not None else None, out.data_ptr(), _DTYPE_CODE[out.dtype], rows, n, k,
            *expand, err.data_ptr(), stream_handle(dev))
    if rc:
        _lib.check(rc, "lithe_int8_linear")
    return out


def int8_linear_dynamic(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                        bias: Optional[torch.Tensor], h: Optional[torch.Tensor] = None,
                        b_dec: Optional[torch.Tensor] = None) -> torch.Tensor:
    """lithe_int8_linear_dynamic: (..., n) from x (..., k) bf16 / fp16, quantised within the call."""
    _require_cuda(x, "x")
    dev, dtype, shape = x.device, x.dtype, x.shape
    if dtype not in ACTIVATION_DTYPES:
        raise TypeError(f"x must be one of {ACTIVATION_DTYPES}, got {dtype}")
    if not shape or shape[-1] < 1:
        raise ValueError(f"x must be (..., k) with k >= 1, got {tuple(shape)}")
    k = shape[-1]
    if x.is_contiguous():
        rows, x_stride = x.numel() // k, k
    else:
        x = x.reshape(-1, k)
        if k > 1 and x.stride(1) != 1:
            x = x.contiguous()
        rows = x.shape[0]
        x_stride = x.stride(0) if rows > 1 else k
    if rows > _MOST:
        raise NotImplementedError(f"x: {rows} rows are above {_MOST}")
    n, w_stride = _int8_weight(weight, weight_scale, bias, dtype, dev, k)
    expand = _NO_EXPAND if h is None and b_dec is None else _int8_expand(h, b_dec, rows, n, dev)
    out = x.new_empty((*shape[:-1], n))
    if rows == 0:
        return out
    x_ptr = x.data_ptr()
    if rows == 1 and k <= 16384 and not (k % 8 or x_ptr % 16):
        space, size = None, 0           # the kernel quantises such a row itself
    else:
        size = rows * (padded(k) + 4)
        space = torch.empty(size, dtype=torch.uint8, device=dev)
    with device_ctx(dev):
        rc = _lib.lib().lithe_int8_linear_dynamic(
            x_ptr, x_stride, weight.data_ptr(), w_stride, weight_scale.data_ptr(),
            bias.data_ptr() if bias is not None else None, out.data_ptr(), _DTYPE_CODE[dtype], rows, n, k, *expand,
            error_word(dev).data_ptr(), space.data_ptr() if space is not None else None, size, stream_handle(dev))
    if rc:
        _lib.check(rc, "lithe_int8_linear_dynamic")
    return out
