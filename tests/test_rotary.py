"""Multi-axis rotation and per-head norm: what the entry points refuse, without a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lithe_b200 import _lib
from lithe_b200.kernels import _launch, qk_norm_rotate, rotary, rotate_axes


def _view(**over):
    a = dict(base=0x10000, sample_stride=1024, token_stride=256, head_stride=64, heads=4)
    a.update(over)
    return _lib.HeadsView(*a.values())


def _rotate(x=None, out=None, dtype=_lib.DTYPE_BF16, batch=1, tokens=4, dim=64, positions=0x30000, pos_type=_lib.POS_F32,
            axes=(16, 24, 24), n_axes=None, freqs=(1.0,) * 128, pairing=0):
    x, out = x or _view(), out or _view(base=0x20000)
    arr = (ctypes.c_int32 * max(1, len(axes)))(*axes)
    return _lib.lib().lithe_rotate_axes(ctypes.byref(x), ctypes.byref(out), dtype, batch, tokens, dim, positions,
                                        pos_type, 0, arr, len(axes) if n_axes is None else n_axes,
                                        None if freqs is None else (ctypes.c_double * len(freqs))(*freqs), pairing, None)


@pytest.mark.parametrize("over,code", [
    ({"dtype": 7}, _lib.ERR_ARG),
    ({"batch": -1}, _lib.ERR_ARG),
    ({"dim": 63}, _lib.ERR_ARG),
    ({"dim": 0}, _lib.ERR_ARG),
    ({"dim": 258}, _lib.ERR_UNSUPPORTED),
    ({"axes": (16, 24, 26)}, _lib.ERR_ARG),           # more than the head's dim
    ({"axes": (15, 24)}, _lib.ERR_ARG),
    ({"axes": (-2, 24)}, _lib.ERR_ARG),
    ({"axes": (2147483646, 4)}, _lib.ERR_ARG),
    ({"n_axes": 0}, _lib.ERR_ARG),
    ({"axes": (2,) * 9}, _lib.ERR_ARG),
    ({"freqs": None}, _lib.ERR_ARG),
    ({"freqs": (1.0,) * 31 + (float("nan"),)}, _lib.ERR_ARG),
    ({"freqs": (float("inf"),) + (1.0,) * 127}, _lib.ERR_ARG),
    ({"pairing": 2}, _lib.ERR_ARG),
    ({"pos_type": 3}, _lib.ERR_ARG),
    ({"positions": None}, _lib.ERR_ARG),
    ({"x": _view(base=None)}, _lib.ERR_ARG),
    ({"x": _view(base=0x10001)}, _lib.ERR_ARG),
    ({"x": _view(heads=0)}, _lib.ERR_ARG),
    ({"x": _view(heads=2 ** 30 + 1)}, _lib.ERR_UNSUPPORTED),
    ({"x": _view(token_stride=-256)}, _lib.ERR_ARG),
    ({"out": _view(heads=3)}, _lib.ERR_ARG),
])
def test_c_entry_refuses(over, code):
    assert _rotate(**over) == code
    assert _lib.lib().lithe_last_error()


def test_c_entry_without_tokens_is_a_no_op():
    assert _rotate(tokens=0) == _lib.OK
    assert _rotate(batch=0, positions=None) == _lib.OK


def test_c_norm_entry_refuses():
    v, arr = _view(), (ctypes.c_int32 * 1)(16)

    def call(eps=1e-6, wtype=_lib.DTYPE_BF16, k=v):
        return _lib.lib().lithe_qk_norm_rotate(ctypes.byref(v), None if k is None else ctypes.byref(k), ctypes.byref(v),
                                               ctypes.byref(v), None, None, wtype, eps, _lib.DTYPE_BF16, 1, 0, 64,
                                               0x30000, 0, 0, arr, 1, (ctypes.c_double * 8)(), 0, None)
    assert call() == _lib.OK
    assert call(eps=-1.0) == _lib.ERR_ARG
    assert call(wtype=_lib.DTYPE_F16) == _lib.ERR_ARG
    assert call(k=None) == _lib.ERR_ARG


def test_python_checks():
    cpu = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        rotate_axes(cpu, torch.zeros(4, 1), (64,))
    with FakeTensorMode():
        x = torch.empty(2, 4, 3, 64, dtype=torch.bfloat16, device="cuda")
        pos = torch.empty(4, 2, device="cuda")
        with pytest.raises(ValueError, match="axes"):
            rotate_axes(x, pos, (64, 2))
        with pytest.raises(ValueError, match="axes"):
            rotate_axes(x, pos, (3, 2))
        with pytest.raises(ValueError, match="axes"):
            rotate_axes(x, pos, ())
        with pytest.raises(ValueError, match="pairing"):
            rotate_axes(x, pos, (32, 32), pairing="pairs")
        with pytest.raises(ValueError, match="theta"):
            rotate_axes(x, pos, (32, 32), theta=-1.0)
        with pytest.raises(TypeError):
            rotate_axes(x.double(), pos, (32, 32))
        with pytest.raises(ValueError, match="batch, tokens"):
            rotate_axes(x[0], pos, (32, 32))
        with pytest.raises(ValueError, match="contiguous"):
            rotate_axes(x.transpose(2, 3), pos, (2,))
        with pytest.raises(RuntimeError, match="inference-only"):
            rotate_axes(x.float().requires_grad_(), pos, (32, 32))
        with pytest.raises(TypeError):
            rotate_axes(x, pos, (32.5, 2))
        with pytest.raises(RuntimeError, match="inference-only"):
            rotate_axes(x, pos, (32, 32), out=torch.empty(2, 4, 3, 64, dtype=x.dtype, device="cuda", requires_grad=True))
        with pytest.raises(NotImplementedError):
            rotate_axes(x[:1].expand(2 ** 31, 4, 3, 64), pos, (32, 32))
        with pytest.raises(ValueError, match="eps"):
            qk_norm_rotate(x, x, None, None, pos, (32, 32), eps=-1.0)
        with pytest.raises(ValueError, match="type and device"):
            qk_norm_rotate(x, x.float(), None, None, pos, (32, 32))


def test_rotation_arguments():
    x = torch.zeros(2, 4, 3, 64)
    for pos in (torch.zeros(4, 3), torch.zeros(3, 2), torch.zeros(1, 4, 2), torch.zeros(2, 4)):
        with pytest.raises(ValueError, match="positions"):
            _launch._rotation_args(x, pos, (32, 32), 1e4, 0)
    with pytest.raises(TypeError, match="positions"):
        _launch._rotation_args(x, torch.zeros(4, 2, dtype=torch.float16), (32, 32), 1e4, 0)
    with pytest.raises(ValueError, match="contiguous"):
        _launch._rotation_args(x, torch.zeros(2, 4).t(), (32, 32), 1e4, 0)


def test_overlap_checks():
    buf = torch.zeros(2, 5, 3, 4, 8)
    q, k, v = buf.unbind(2)
    _launch._check_outputs((q, k), (q, k), ("q", "k"))                  # in place in a fused projection
    assert _launch._apart(q, k) and _launch._apart(v, q)
    one = torch.zeros(1, 5, 3, 4, 8)
    assert _launch._apart(one[:, :, 0], one[:, :, 2])
    token = torch.zeros(2, 1, 3, 4, 8)
    assert _launch._apart(token[:, :, 0], token[:, :, 1])
    joint = torch.zeros(2, 9, 4, 8)
    assert not _launch._apart(joint[:, :5], joint[:, 4:])
    assert _launch._apart(joint[:1, :4], joint[:1, 4:8])
    assert _launch._apart(torch.zeros(3, 2, 2, 8), torch.zeros(3, 2, 2, 8))
    assert not _launch._apart(q, q)
    with pytest.raises(ValueError, match="overlaps an input"):
        _launch._check_outputs((joint[:, :8],), (joint[:, 1:],), ("out",))
    with pytest.raises(ValueError, match="overlaps an input"):
        _launch._check_outputs((q, k), (k, q), ("out_q", "out_k"))      # swapped: one would read the other's result
    with pytest.raises(ValueError, match="overlaps out_q"):
        _launch._check_outputs((torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 4, 8)), (q, q), ("out_q", "out_k"))
    with pytest.raises(ValueError, match="share an address"):
        _launch._check_outputs((), (torch.zeros(1, 1, 1, 8).expand(2, 3, 1, 8),), ("out",))


def test_ops_are_registered():
    import lithe_b200.kernels.ops  # noqa: F401
    with FakeTensorMode():
        x = torch.empty(2, 4, 3, 64, dtype=torch.bfloat16, device="cuda")
        pos = torch.empty(4, 2, device="cuda")
        assert torch.ops.lithe_b200.rotate_axes_(torch.empty_like(x), x, pos, [32, 32], 1e4, 0) is None
        assert torch.ops.lithe_b200.qk_norm_rotate_(torch.empty_like(x), torch.empty_like(x), x, x, None, None, pos,
                                                    [32, 32], 1e4, 1e-6, 0) is None


@pytest.mark.parametrize("which", ["positions", "weight_q", "weight_k", "q", "k"])
def test_every_operand_is_inference_only(which):
    with FakeTensorMode():
        ops = dict(q=torch.empty(2, 4, 3, 64, device="cuda"), k=torch.empty(2, 4, 3, 64, device="cuda"),
                   weight_q=torch.empty(64, device="cuda"), weight_k=torch.empty(64, device="cuda"),
                   positions=torch.empty(4, 2, device="cuda"))
        ops[which].requires_grad_()
        with pytest.raises(RuntimeError, match="inference-only"):
            qk_norm_rotate(*ops.values(), (32, 32))
        if which == "positions":
            with pytest.raises(RuntimeError, match="inference-only"):
                rotate_axes(ops["k"], ops["positions"], (32, 32))


def test_no_answer_is_kept_for_an_object_that_can_change():
    """axes and theta may come as tensors or arrays: each call takes the numbers that they hold then."""
    rotation = rotary._rotation
    theta, axis = torch.tensor(1e4), torch.tensor(16)
    assert rotation(64, (axis, 24), theta, "interleaved", False) == ((16, 24), 1e4, 0)
    theta.fill_(256.0)
    axis.fill_(8)
    assert rotation(64, (axis, 24), theta, "interleaved", False) == ((8, 24), 256.0, 0)
    assert rotation(64, [8, 24], 256, "halves", False) == ((8, 24), 256.0, 1)
    assert all(type(a) is int for a in rotation(64, (True + 7, axis), 1, "halves", False)[0])
    with pytest.raises(TypeError):
        rotation(64, (8.0, 24), 256, "halves", False)       # though (8, 24) is known
    axis.fill_(7)
    with pytest.raises(ValueError, match="even"):
        rotation(64, (axis, 24), theta, "interleaved", False)


def test_outputs_apart_from_what_every_token_reads(monkeypatch):
    """An output that reaches over the positions or the norms' weights is refused: tokens would read each
    other's results there."""
    monkeypatch.setattr(_launch, "_require_cuda", lambda t, what: None)
    buf = torch.zeros(2 * 3 * 2 * 8 + 64)
    out = buf[:96].view(2, 3, 2, 8)
    x, k = torch.ones(2, 3, 2, 8), torch.ones(2, 3, 2, 8)
    for pos in (buf[80:86].view(3, 2), buf[95:101].view(3, 2), buf[:12].view(2, 3, 2)):
        with pytest.raises(ValueError, match="out overlaps positions"):
            _launch.rotate_axes_(x, out, pos, (4, 4), 1e4, 0)
        with pytest.raises(ValueError, match="out_k overlaps positions"):
            _launch.qk_norm_rotate_(x, k, x, out, None, None, pos, (4, 4), 1e4, 1e-6, 0)
    pos = torch.zeros(3, 2)
    with pytest.raises(ValueError, match="out_q overlaps weight_k"):
        _launch.qk_norm_rotate_(x, k, out, k, None, buf[89:97], pos, (4, 4), 1e4, 1e-6, 0)
    behind, none = _launch._heads_layout(out), _launch._heads_layout(buf[:0].view(0, 3, 2, 8))
    for view in (behind, none):                             # next to an output, and an output without elements
        _launch._check_read(buf[96:].data_ptr(), 24, "positions", view, "out")
