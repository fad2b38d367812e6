"""Offsets beyond 32 bits: rows, tokens and results behind the first 2^31 elements have the bits that they have
in a call of their own (a row or token does not depend on the others)."""
import pytest
import torch

from lithe_b200.kernels import int8_linear, qk_norm_rotate, quantize_rows, quantize_weight, rotate_axes
from tests.test_gpu_int8 import make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


@pytest.mark.parametrize("expand", [False, True])
def test_results(expand):
    samples, rps, n, k = 700, 256, 12288, 64
    rows = samples * rps
    assert rows * n > 2 ** 31
    x = make((rows, k), BF, 1)
    w, ws = quantize_weight(make((n, k), BF, 2, 0.02))
    h, b_dec = (make((rows, 16), BF, 4), make((samples, n, 16), BF, 5, 0.1)) if expand else (None, None)
    got = int8_linear(x, w, ws, h=h, b_dec=b_dec)
    for s in (0, samples // 2, samples - 1):
        at = slice(s * rps, (s + 1) * rps)
        want = int8_linear(x[at], w, ws, h=None if h is None else h[at], b_dec=None if h is None else b_dec[s:s + 1])
        if expand:          # one sample alone takes another path, whose expand adds in another order: 16 terms in fp32
            mag = want.double().abs() + h[at].double().abs() @ b_dec[s].double().abs().t()
            assert ((got[at].double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs() + 80 * 2.0 ** -24 * mag).all()
        else:
            assert torch.equal(got[at], want)


def test_activations():
    rows, k, n = 16400, 131072, 24
    assert rows * k > 2 ** 31
    x = torch.empty(rows, k, dtype=BF, device=DEV)
    for i in range(0, rows, 1024):
        x[i:i + 1024].copy_(make((min(1024, rows - i), k), BF, i))
    w, ws = quantize_weight(make((n, k), BF, 2, 0.02))
    got, q = int8_linear(x, w, ws), quantize_rows(x)
    for at in (slice(0, 40), slice(rows // 2, rows // 2 + 3), slice(rows - 40, rows)):
        assert torch.equal(got[at], int8_linear(x[at], w, ws))
        alone = quantize_rows(x[at])
        assert torch.equal(q.q[at], alone.q) and torch.equal(q.scale[at], alone.scale)


def test_tokens():
    tokens, heads, dim, axes = 360000, 24, 256, (64, 96, 96)
    assert tokens * heads * dim > 2 ** 31
    x = torch.empty(1, tokens, heads, dim, dtype=BF, device=DEV)
    for i in range(0, tokens, 30000):
        x[:, i:i + 30000].copy_(make((1, min(30000, tokens - i), heads, dim), BF, i))
    pos = torch.randint(0, 10 ** 6, (tokens, 3), device=DEV)
    got = rotate_axes(x, pos, axes)
    normed, _ = qk_norm_rotate(x, x[:, :, :1], None, None, pos, axes, out_q=torch.empty_like(x))
    for at in (slice(0, 5), slice(tokens // 2, tokens // 2 + 5), slice(tokens - 5, tokens)):
        assert torch.equal(got[:, at], rotate_axes(x[:, at], pos[at], axes))
        assert torch.equal(normed[:, at], qk_norm_rotate(x[:, at], x[:, at, :1], None, None, pos[at], axes)[0])
